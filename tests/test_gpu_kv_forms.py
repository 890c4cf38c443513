"""GPU tests of the paged cache's calls that its documentation allows beside the
usual ones, against the same oracle, within the same bound (test_gpu_kv.py)."""
import numpy as np
import pytest

from oracle import cbx_kv_oracle as KV
from oracle import cbx_t3_oracle as T3
from test_gpu_kv import D, Dev, bound, caches, cbx, run, say, store  # noqa: F401
from test_gpu_kv import test_prompts_match_oracle as prompts_match
from test_gpu_kv import test_shared_prefix_matches_oracle as shared_matches
from test_gpu_kv import test_step_matches_oracle as step_matches
from test_gpu_kv_t3 import H, L_, N, TOL, V, Server, small  # noqa: F401

pytestmark = pytest.mark.gpu


def pool_of(rng, lens, page, n_prefix=0, parent=None, prefix_len=None, extra=2):
    """Room for lens positions and one more of each stream."""
    n_pages = sum(-(-(x + 1) // page) for x in lens) + extra
    return KV.Pool(len(lens), max(-(-(max(lens) + 1) // page), 1), page, n_pages, n_prefix=n_prefix,
                   parent=parent, prefix_len=prefix_len, free=rng.permutation(n_pages))


# ------------------------------------------------------------------ prompts without a list of tiles

UNLISTED = [  # (already cached, new) of each stream, key heads, heads a key head, prefix or 0
    ([(0, 1)], 2, 1, 0), ([(0, 251)], 4, 1, 0),
    ([(5, 64), (16, 65), (40, 3), (0, 0), (9, 129)], 2, 1, 45),
    ([(0, 0), (0, 0), (3, 7), (0, 0)], 1, 5, 20),
    ([(3, i % 3) for i in range(70)], 1, 3, 0),
    ([(0, 9)] * 3 + [(0, 0)] * 61 + [(1, 30)], 1, 64, 0),
    ([(0, (1, 0, 0, 2)[i % 4]) for i in range(4200)], 1, 1, 0),  # three rounds of 64 streams
    ([(100, 130)] * 24, 8, 1, 0),  # whole tiles a workgroup
]


@pytest.mark.parametrize("short", [False, True], ids=["none", "too-few"])
@pytest.mark.parametrize("streams,n_kv,group,prefix", UNLISTED,
                         ids=[f"{len(x[0])}x{x[0][0][1]}-{x[2]}" for x in UNLISTED])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_prompts_without_a_list_of_tiles(cbx, streams, n_kv, group, prefix, dtype, short):  # noqa: F811
    """Rows planned without tiles, or given to the attention with fewer than they
    need: the outputs are those with the plan's list, bit for bit, and the oracle's."""
    torch, mod, s = cbx
    rng = np.random.default_rng(len(streams) + group)
    n0 = 1 if prefix else 0
    had = [prefix] * n0 + [x[0] for x in streams]
    new = [0] * n0 + [x[1] for x in streams]
    n = len(had)
    say("no list", len(streams), streams[0], n_kv, group, dtype, short)
    pool = pool_of(rng, [a + b for a, b in zip(had, new)], 16, n0, [-1] * n0 + [n0 - 1] * len(streams),
                   [0] * n0 + [prefix] * len(streams))
    d = Dev(torch, mod, pool)
    if sum(had):
        d.plan(s, d.rows(False, sum(had)), n_new=had)
    c = caches(torch, rng, pool, n_kv, getattr(torch, dtype))
    store(torch, rng, pool, c, 0, had)
    T = mod.Sampler.kv_tile_rows(n_kv * group, n_kv)
    listed = d.rows(False, sum(new) + 5, tile_rows=T)
    plan = d.plan(s, listed, n_new=new)
    want, x = run(cbx, d, listed, plan, c, n_kv, group, rng, sd=2.0)
    b = {k: t for k, t in listed.b.items() if k != "tiles"}
    if short:
        b["tiles"] = listed.b["tiles"][:-1].fill_(-1)
    r = mod.Sampler.kv_rows(**b, tile_rows=T if short else 0)
    got, _ = run(cbx, d, r, plan, c, n_kv, group, rng, q=x["q"], kn=x["kn"], vn=x["vn"])
    assert np.array_equal(got, want)


def test_t3_prompts_without_a_list_of_tiles(small):  # noqa: F811
    """The transformer's prompt rows, with the plan's tiles, none, and too few."""
    torch, mod, s, dm, _ = small
    x = torch.randn((70, N), device="cuda", generator=torch.Generator("cuda").manual_seed(2)) * 0.7
    out = []
    for tiles in ("listed", "none", "few"):
        torch.manual_seed(1)
        srv = Server(torch, mod, s, dm, 5, 0, torch.float32)
        r = srv.rows(70, step=False, tiles=tiles == "listed")
        srv.plan(r, n_new=[9, 0, 33, 27, 1])
        if tiles == "few":
            f = torch.zeros((1, 4), dtype=torch.int32, device="cuda")
            r.tiles, r.n_tiles, r._tensors = f.data_ptr(), 1, r._tensors + (f,)
        say("t3", tiles)
        hid = torch.full((70, N), 7.0, device="cuda")
        s.t3_kv(dm, srv.cache, srv.streams, r, hid, inputs=x)
        torch.cuda.synchronize()
        out.append(hid.cpu().numpy())
    assert np.array_equal(out[0], out[1]) and np.array_equal(out[0], out[2])
    assert np.isfinite(out[0]).all() and (out[0] != 7.0).all()


# ------------------------------------------------------------------ streams


def test_a_workspace_outlives_its_call_on_another_stream(cbx):  # noqa: F811
    """A call put on a busy stream and its KvAttn dropped: torch does not hand the
    workspace to the stream that it was made on until the call has ended."""
    torch, mod, s = cbx
    rng = np.random.default_rng(3)
    pool = pool_of(rng, [1500, 900], 16)
    d = Dev(torch, mod, pool)
    d.plan(s, d.rows(False, 2400), n_new=[1500, 900])
    c = caches(torch, rng, pool, 2, torch.float32)
    store(torch, rng, pool, c, 0, [1500, 900])
    r = d.rows(True, tiles=False)
    plan = d.plan(s, r)
    want, x = run(cbx, d, r, plan, c, 2, 1, rng)
    side = torch.cuda.Stream()
    out = torch.empty((2, 2 * D), device="cuda")
    a = mod.Sampler.kv_attn(mod.Sampler.kv_cache(*c), d.streams, r, x["q"], out, k=x["kn"], v=x["vn"])
    at, size = a.workspace, a.workspace_bytes
    assert size
    torch.cuda.synchronize()
    say("another stream")
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    s.kv_attend(a, stream=side.cuda_stream)
    del a
    other = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]
    assert at not in [t.data_ptr() for t in other]
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)


# ------------------------------------------------------------------ heads, pages, rows already stored


@pytest.mark.parametrize("group", [16, 17, 40, 64])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_steps_of_many_heads_a_key_head(cbx, dtype, group):  # noqa: F811
    """More pairs of a row than a wave holds: several workgroups a row, each with
    the row's new key; prefixes' tiles of one to four rows."""
    step_matches(cbx, [31, 0, 130, 64], dtype, 2, group, 16)
    shared_matches(cbx, [40, 70], [(0, 40, 0), (0, 33, 100), (-1, 0, 20), (1, 70, 16), (1, 1, 7), (0, 2, 3)],
                   dtype, 1, group, 16)


@pytest.mark.parametrize("page", [128, 256])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_large_pages(cbx, dtype, page):  # noqa: F811
    step_matches(cbx, [127, 0, 128, 700, 255, 256], dtype, 2, 1, page)
    step_matches(cbx, [300, 1], dtype, 2, 4, page)
    shared_matches(cbx, [300], [(0, 300, 0), (0, 255, 130), (0, 257, 255), (-1, 0, 256)], dtype, 2, 1, page)
    prompts_match(cbx, [200], [(0, 200, 100, 200), (0, 129, 0, 127), (-1, 0, 256, 3)], dtype, 2, 1, page)


@pytest.mark.parametrize("n_kv,group", [(2, 1), (1, 4)])
@pytest.mark.parametrize("n", [3, 90], ids=["few", "many"])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_rows_already_stored(cbx, dtype, n, n_kv, group):  # noqa: F811
    """Calls without new keys and values: the cache holds them."""
    torch, mod, s = cbx
    rng = np.random.default_rng(n)
    had = [50] + [(5 * i) % 61 for i in range(n)]
    say("stored", dtype, n, n_kv, group)
    new = [0] + [1 + (7 * i) % 50 for i in range(n)]
    pool = pool_of(rng, [a + b for a, b in zip(had, new)], 16, 1, [-1] + [0] * n,
                   [0] + [(50, 33, 0)[i % 3] for i in range(n)])
    d = Dev(torch, mod, pool)
    d.plan(s, d.rows(False, sum(had)), n_new=had)
    c = caches(torch, rng, pool, n_kv, getattr(torch, dtype))
    store(torch, rng, pool, c, 0, had)
    T = mod.Sampler.kv_tile_rows(n_kv * group, n_kv)
    for step in (False, True):
        r = d.rows(step, sum(new), tile_rows=T)
        plan = d.plan(s, r, n_new=[0] + [1] * n if step else new)
        run(cbx, d, r, plan, c, n_kv, group, rng, sd=2.0)
        run(cbx, d, r, plan, c, n_kv, group, rng, sd=2.0, new=False)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_t3_steps_of_whole_rows(small, dtype):  # noqa: F811
    """As many streams as rows are not cut for: each row goes from its one
    workgroup straight into the next product's parts.  The tolerance is
    test_gpu_kv_t3.py's."""
    torch, mod, s, dm, rm = small
    n, half = 256, dtype == "float16"
    say("t3 whole rows", dtype)
    rng = np.random.default_rng(12)
    srv = Server(torch, mod, s, dm, n, 0, getattr(torch, dtype), n_pages=3 * n)
    oracles = [T3.new_cache(n, L_, H, 64)]
    if half:
        oracles.append(tuple(c.astype(np.float16) for c in T3.new_cache(n, L_, H, 64)))
    own = np.array([1 + (7 * i) % 30 for i in range(n)])
    x = (rng.standard_normal((own.sum(), N)) * 0.7).astype(np.float32)
    srv.prompt(x, own.tolist())
    for i, f in enumerate(np.cumsum(own) - own):
        for c in oracles:
            T3.prefill(rm, x[f:f + own[i]], *c, i, 0)
    moved = 0.0
    for turn in range(3):
        tokens, state = rng.integers(0, V, n), [1 if i % 9 == turn else 0 for i in range(n)]
        active = np.array(state) == 0
        got = srv.step(tokens, state, False)
        want = [T3.step(rm, tokens, own.copy(), *c, active=active) for c in oracles]
        if half:
            moved = max(moved, np.abs(want[1] - want[0])[active].max())
        err = np.abs(got - want[-1]) - TOL * np.abs(want[-1])
        assert err[active].max() <= TOL + 2 * moved, (turn, err[active].max(), moved)
        assert np.all(got[~active] == 0.0)
        own[active] += 1


# ------------------------------------------------------------------ large scores


@pytest.mark.parametrize("form", ["step", "shared", "prompt"])
@pytest.mark.parametrize("size", [1e6, 1e10, 1e20, -1e10, -1e30])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("group", [1, 2, 4])
def test_large_scores(cbx, dtype, group, size, form):  # noqa: F811
    """Finite scores of any size: the j-th key from the end has size (1 + j / 64),
    so one key of each row is larger than all others by size / 64 at least and the
    output is its value: a weight of 1, or a power of two, and the division, each
    rounded once or twice (8 u; fp16 parts of a weight that is no power of two cut
    off at 2^-20 in the sum and the product alike, 32 u)."""
    torch, mod, s = cbx
    rng = np.random.default_rng(4)
    say("large", dtype, group, size, form)
    n_kv, n, plen = 2, 5, 20
    own = [0, 3, 17, 40, 63]
    n0 = 1 if form == "shared" else 0
    had = [plen] * n0 + [x - (x > plen) * plen if n0 else x for x in own]
    pool = pool_of(rng, had, 16, n0, [-1] * n0 + [n0 - 1] * n, [0] * n0 + [plen] * n)
    d = Dev(torch, mod, pool)
    d.plan(s, d.rows(False, sum(had) + 1), n_new=had)
    c = caches(torch, rng, pool, n_kv, getattr(torch, dtype))
    store(torch, rng, pool, c, 0, had)
    T = mod.Sampler.kv_tile_rows(n_kv * group, n_kv)
    new = [0] * n0 + [1] * n
    r = d.rows(form != "prompt", sum(new), tiles=form != "step", tile_rows=T)
    plan = d.plan(s, r, n_new=new)
    rows = [i for i in range(r.n_rows) if plan["position"][i] >= 0]
    # keys: 1 + j / 64 (exact in either type) in dimension 0 alone, j shuffled over
    # the positions that a row sees
    kc, vc = (t[0].float().cpu().numpy() for t in c)
    kc[:] = 0.0
    kn = np.zeros((r.n_rows, n_kv, D), np.float32)
    vn = rng.standard_normal((r.n_rows, n_kv, D)).astype(np.float32)
    if dtype == "float16":
        vn = vn.astype(np.float16).astype(np.float32)
    want = np.zeros((r.n_rows, n_kv, D))
    shared = rng.permutation(plen) if n0 else []
    for x in range(plen if n0 else 0):
        kc[pool.tables[0, x // 16], :, x % 16, 0] = 1 + shared[x] / 64
    for i in rows:
        st, pos = (i if form != "prompt" else plan["stream"][i]), int(plan["position"][i])
        mine = pos + 1 - (plen if n0 else 0)
        j = list(shared) + list(rng.permutation(mine) + len(shared))
        at = KV.keys_of(pool, st, pos)
        for x in range(len(shared), pos):
            kc[at[x][0], :, at[x][1], 0] = 1 + j[x] / 64
        kn[i, :, 0] = 1 + j[pos] / 64
        best = int(np.argmax(j) if size > 0 else np.argmin(j))
        want[i] = vn[i] if best == pos else vc[at[best][0], :, at[best][1]]
    for t, x in zip(c, (kc, vc)):
        t[0].copy_(torch.from_numpy(x))
    q = np.zeros((r.n_rows, n_kv * group, D), np.float32)
    q[..., 0] = size * 8
    out = torch.empty((r.n_rows, n_kv * group * D), device="cuda")
    t = lambda a: torch.from_numpy(a.reshape(r.n_rows, -1)).cuda()  # noqa: E731
    s.kv_attend(mod.Sampler.kv_attn(mod.Sampler.kv_cache(*c), d.streams, r, t(q), out, k=t(kn), v=t(vn)))
    got = out.cpu().numpy().reshape(r.n_rows, n_kv, group, D)[rows]
    want = want[rows][:, :, None]
    assert np.abs(got - want).max() <= 40 * 2.0 ** -24 * np.abs(want).max(), np.abs(got - want).max((1, 2, 3))


@pytest.mark.parametrize("form", ["step", "few", "many"])
@pytest.mark.parametrize("size", [1.0, 1e6, 3e7, 1e9, 1e10, 1e20, -3e7, -1e10, -1e30])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("group", [1, 4])
def test_large_equal_scores(cbx, dtype, group, size, form):  # noqa: F811
    """Keys of two kinds, all scores of a kind the same to the bit, wherever they
    are met: the output is the mean of the larger kind's values (at size 1 the
    softmax of both), within the bound of n equal scores; the larger kind first,
    last, or in turn."""
    torch, mod, s = cbx
    rng = np.random.default_rng(6)
    say("equal", dtype, group, size, form)
    n_kv, lens = 2, [0, 5, 40, 100, 333] + [70] * (60 if form == "many" else 0)
    pool = pool_of(rng, lens, 16)
    d = Dev(torch, mod, pool)
    d.plan(s, d.rows(False, sum(lens)), n_new=lens)
    c = caches(torch, rng, pool, n_kv, getattr(torch, dtype))
    store(torch, rng, pool, c, 0, lens)
    T = mod.Sampler.kv_tile_rows(n_kv * group, n_kv)
    r = d.rows(form == "step", len(lens), tiles=form != "step", tile_rows=T)
    plan = d.plan(s, r, n_new=[1] * len(lens))
    vn = rng.standard_normal((len(lens), n_kv, D)).astype(getattr(np, dtype)).astype(np.float32)
    t = lambda a: torch.from_numpy(a.reshape(len(lens), -1)).cuda()  # noqa: E731
    q = np.zeros((len(lens), n_kv * group, D), np.float32)
    q[..., 0] = size * 8
    for order in ("first", "last", "turn"):
        kc, vc = (x[0].float().cpu().numpy() for x in c)
        kc[:] = 0.0
        kn = np.zeros_like(vn)
        want, mass, n_keys = np.zeros((len(lens), n_kv, D)), np.zeros((len(lens), n_kv, D)), []
        for i, L in enumerate(lens):
            big = {"first": np.arange(L + 1) <= L // 2, "last": np.arange(L + 1) >= L // 2,
                   "turn": np.arange(L + 1) % 2 == 0}[order]
            at = KV.keys_of(pool, i, L)
            vs = np.zeros((L + 1, n_kv, D))
            for x in range(L + 1):
                if x < L:
                    kc[at[x][0], :, at[x][1], 0] = 1 + big[x] / 64
                    vs[x] = vc[at[x][0], :, at[x][1]]
            kn[i, :, 0], vs[L] = 1 + big[L] / 64, vn[i]
            p = np.exp(size * (1 + big / 64) - (size * (1 + big / 64)).max())
            p = (p / p.sum())[:, None, None]
            want[i], mass[i] = (p * vs).sum(0), (p * np.abs(vs)).sum(0)
            n_keys.append(L + 1)
        c[0][0].copy_(torch.from_numpy(kc))
        out = torch.empty((len(lens), n_kv * group * D), device="cuda")
        s.kv_attend(mod.Sampler.kv_attn(mod.Sampler.kv_cache(*c), d.streams, r, t(q), out, k=t(kn), v=t(vn)))
        got = out.cpu().numpy().reshape(len(lens), n_kv, group, D)
        near = 2.0 if size == 1.0 else 0.0
        lim = bound(np.full((len(lens), n_kv), near), mass, np.array(n_keys))[:, :, None]
        worst = (np.abs(got - want[:, :, None]) / lim).max((1, 2, 3))
        assert worst.max() <= 1.0, (order, worst[:5])


# ------------------------------------------------------------------ queries and keys that are not finite


@pytest.mark.parametrize("what", ["query", "key"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("form", ["few", "many", "shared"])
@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_queries_and_keys_that_are_not_finite_stay(cbx, dtype, group, form, bad, what):  # noqa: F811
    """One query, or one key, reaches its own row, or the rows that see it, alone:
    all others are bit for bit the same."""
    torch, mod, s = cbx
    n_kv, H = 2, 2 * group
    n = [40, 21] if form == "few" else [90] * 60 if form == "many" else [1] * 9
    say("not finite", what, bad, form, group, dtype)
    out = []
    for plant in (False, True):
        rng = np.random.default_rng(5)
        n0 = 1 if form == "shared" else 0
        lens = [40] * n0 + [4 * n0] * len(n)
        share = [(40, 37, 12, 9)[i % 4] for i in range(len(n))]
        pool = KV.Pool(n0 + len(n), 8, 16, 500, n_prefix=n0, parent=[-1] * n0 + [n0 - 1] * len(n),
                       prefix_len=[0] * n0 + share)
        d = Dev(torch, mod, pool)
        c = caches(torch, rng, pool, n_kv, getattr(torch, dtype))
        if n0:
            d.plan(s, d.rows(False, sum(lens)), n_new=lens)
            store(torch, rng, pool, c, 0, lens)
        r = d.rows(bool(n0), sum(n), tile_rows=64 // group)
        d.plan(s, r, n_new=[0] * n0 + n)
        x = torch.from_numpy(rng.standard_normal((r.n_rows, (H + 2 * n_kv) * D)).astype(np.float32)).cuda()
        if n0:
            row, pos = 1 + 2, 12  # the third stream's query; the prefix's key 12, that two of four see
            hit = [row] if what == "query" else [1 + i for i in range(len(n)) if share[i] > pos]
            if plant and what == "key":
                c[0][0, int(pool.tables[0, 0]), 0, pos, 7] = bad
        else:
            row = n[0] + 9        # the second stream's tenth position
            hit = [row] if what == "query" else list(range(row, n[0] + n[1]))
            if plant and what == "key":
                x[row, H * D + 7] = bad
        if plant and what == "query":
            x[row, 7] = bad
        o = torch.empty((r.n_rows, H * D), device="cuda")
        q, k, v = x[:, :H * D], x[:, H * D:(H + n_kv) * D], x[:, (H + n_kv) * D:]
        s.kv_attend(mod.Sampler.kv_attn(mod.Sampler.kv_cache(*c), d.streams, r, q, o, k=k, v=v))
        torch.cuda.synchronize()
        out.append(o.cpu().numpy().reshape(-1, H, D))
    same = np.ones(out[0].shape[:2], bool)
    same[hit, :1 if what == "query" else group] = False
    assert np.isfinite(out[0]).all() and np.array_equal(out[0][same], out[1][same])


# ------------------------------------------------------------------ offsets past 32 bits


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_offsets_past_32_bits(cbx, dtype):  # noqa: F811
    """A pool of more than 2^32 values a layer, its second layer's last pages used."""
    torch, mod, s = cbx
    n_kv, page, used = 4, 256, 12
    n_pages = (1 << 32) // (n_kv * page * D) + 300
    say("past 32 bits", dtype)
    assert n_pages * n_kv * page < 2 ** 32 - 1 and n_pages * page < 2 ** 31
    k, v = (torch.empty((2, n_pages, n_kv, page, D), dtype=getattr(torch, dtype), device="cuda")
            for _ in range(2))
    rng = np.random.default_rng(1)
    lens = [300, 20, 511]
    for form in ("step", "shared", "prompt"):
        n0 = 1 if form == "shared" else 0
        pool = KV.Pool(3, 4, page, n_pages, n_prefix=n0, parent=[-1] + [n0 - 1] * 2,
                       prefix_len=[0, 300, 270] if n0 else [0] * 3)
        d = Dev(torch, mod, pool)  # the stack's top: the last pages
        d.plan(s, d.rows(False, sum(lens)), n_new=lens)
        r = d.rows(form != "prompt", 90, tiles=form != "step")
        plan = d.plan(s, r, n_new=[0 if n0 else 1, 1, 1] if form != "prompt" else [40, 30, 20])
        first = n_pages - used
        host = [rng.standard_normal((used, n_kv, page, D)).astype(dtype) for _ in range(2)]
        for t, x in zip((k, v), host):
            t[1, first:] = torch.from_numpy(x).cuda()
        x = rng.standard_normal((r.n_rows, 3 * n_kv * D)).astype(np.float32)
        rows = torch.from_numpy(x).cuda()
        q, kn, vn = rows.split(n_kv * D, dim=1)
        out = torch.empty((r.n_rows, n_kv * D), device="cuda")
        s.kv_attend(mod.Sampler.kv_attn(mod.Sampler.kv_cache(k, v), d.streams, r, q, out, layer=1, k=kn, v=vn))
        torch.cuda.synchronize()
        for row, sl in enumerate(plan["slot"]):
            if sl >= 0:
                for h, t in zip(host, (kn, vn)):
                    h[sl // page - first, :, sl % page] = t[row].reshape(n_kv, D).to(k.dtype).cpu().numpy()
        for t, h in zip((k, v), host):
            assert np.array_equal(t[1, first:].cpu().numpy(), h)
        small_pool = KV.Pool(3, 4, page, used, n_prefix=n0, parent=pool.parent, prefix_len=pool.prefix_len)
        small_pool.tables[:] = pool.tables - first
        stream = plan.get("stream", np.arange(3))
        want, size, mass, n_keys = KV.attend(small_pool, *[h.astype(np.float32) for h in host], stream,
                                             plan["position"], q.cpu().numpy(), 0.125)
        lim = bound(size, mass, n_keys).reshape(want.shape)
        assert (np.abs(out.cpu().numpy() - want) <= lim).all(), form
    del k, v
    torch.cuda.empty_cache()
