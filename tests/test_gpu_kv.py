"""GPU tests of the paged cache (include/cbx_kv.h) against its oracle
(oracle/cbx_kv_oracle.py): plans exactly, attention within a bound worked out
per row from the operations.

Bound (u = 2^-24, one rounding of binary32; S the largest sum |q||k| scale of a
row, A_d = sum p |v_d|, n its keys):
 * a score is a sum of 64 products, rounded at most 64 + 3 times (q scaled, the
   products, the adds, whatever their order): off by at most 67 u S, and the
   difference to the row's maximum by twice that and one rounding of at most 2 S;
 * e^x as 2^(x log2 e): log2 e and the product rounded (2 u times |x| <= 2 S),
   the function to 1 ulp (2 u); rescalings as the maximum grows or parts are
   joined multiply by such values again: at most n / 24 + 100 of them in a row's
   chain, but their exponents add up to at most 2 S, so they add 2 u a time and
   4 u S in all;
 * the sums of n terms, theirs and the weights', n u each, a product and a
   division more.
So |out - ref| <= A_d u ((2 * 67 + 2 + 4 + 4) S + 2 n + 4 (n / 24 + 100) + 10),
first order, doubled for the higher orders and for weights off in numerator and
denominator both.  Weights under the smallest normal number (2^-126 of the
largest) are lost: far below.
Where the values are fp16 (cache or matrix-core operands in two fp16 parts,
2^-22 = 4 u of each q and p), 8 u S + 8 u more.
"""
import numpy as np
import pytest

import pkg
from oracle import cbx_kv_oracle as KV

pytestmark = pytest.mark.gpu
U, D = 2.0 ** -24, 64


def bound(size, mass, n_keys):
    per = (144 + 8) * size + 2 * n_keys[:, None] + 4 * (n_keys[:, None] / 24 + 100) + 18
    return 2 * U * per[:, :, None] * mass + 1e-37


@pytest.fixture(scope="module")
def cbx():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    mod = pkg.load()
    s = mod.Sampler(device=0, max_vocab=1024, max_history=64)
    yield torch, mod, s
    s.close()


def say(*a):
    print("[gpu-case]", *a, flush=True)


class Dev:
    """A pool on the device beside its oracle."""

    def __init__(self, torch, mod, pool):
        self.torch, self.mod, self.pool = torch, mod, pool
        t = lambda a: torch.from_numpy(np.array(a, np.int32)).cuda()
        self.tables, self.length, self.free = t(pool.tables), t(pool.length), t(pool.free)
        self.n_free = t([pool.n_free])
        self.parent, self.prefix_len = t(pool.parent), t(pool.prefix_len)
        self.streams = mod.Sampler.kv_streams(self.tables, self.length, self.free, self.n_free,
                                              n_prefix=pool.n_prefix, parent=self.parent,
                                              prefix_len=self.prefix_len)

    def rows(self, step, n_rows=None, tiles=True, tile_rows=64):
        torch, n = self.torch, self.pool.n
        n_rows = n if step else n_rows
        full = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")
        b = dict(position=full(n_rows), slot=full(n_rows), row_start=full(n + 1),
                 page_start=full(n + 1), counts=full(4))
        if not step:
            b["stream"] = full(n_rows)
        if tiles:
            b["tiles"] = full(max(1, n_rows // tile_rows + (self.pool.n_prefix if step else n)), 4)
            if step:
                b["order"] = full(n_rows)
        r = self.mod.Sampler.kv_rows(**b, tile_rows=tile_rows)
        r.b = b
        return r

    def ints(self, a):
        return None if a is None else self.torch.from_numpy(np.array(a, np.int32)).cuda()

    def plan(self, s, r, in_place=True, stream=None, **kw):
        """Builds r on the device and with the oracle; compares everything."""
        torch, pool = self.torch, self.pool
        kw = {k: v for k, v in kw.items() if v is not None}
        out = {} if in_place else dict(len_out=torch.full_like(self.length, -7),
                                       n_free_out=torch.full_like(self.n_free, -7))
        before = (self.length.clone(), self.n_free.clone())
        p = self.mod.Sampler.kv_plan(self.streams, r, page_size=pool.page, **out,
                                     **{k: self.ints(v) for k, v in kw.items()})
        s.kv_build(p, stream=stream)
        torch.cuda.synchronize()
        if not in_place:
            assert torch.equal(self.length, before[0]) and torch.equal(self.n_free, before[1])
            self.length.copy_(out["len_out"])
            self.n_free.copy_(out["n_free_out"])
        step = "stream" not in r.b
        want = KV.build(pool, n_rows=len(r.b["position"]),
                        n_tiles=len(r.b["tiles"]) if "tiles" in r.b else 0,
                        tile_rows=r.tile_rows, step=step, **kw)
        for k, w in want.items():
            got = r.b[k].cpu().numpy()
            assert np.array_equal(got, w), (k, np.nonzero((got != w).reshape(len(w), -1).any(1))[0][:8],
                                            got[:8], w[:8])
        for k, got, w in (("tables", self.tables, pool.tables), ("length", self.length, pool.length),
                          ("n_free", self.n_free, [pool.n_free]), ("free", self.free, pool.free)):
            assert np.array_equal(got.cpu().numpy(), w), k
        return want


# ------------------------------------------------------------------ plans

PLANS = [  # streams, page, max_pages, pages, prefixes, tile rows
    (1, 16, 3, 4, 0, 64), (5, 16, 4, 12, 2, 1), (63, 32, 9, 300, 1, 7), (64, 16, 30, 900, 3, 64),
    (65, 256, 2, 70, 65, 64), (1000, 64, 5, 2500, 17, 21), (1024, 16, 12, 5000, 1, 64),
    (1025, 16, 12, 5000, 1000, 64), (4097, 32, 8, 9000, 40, 16), (16384, 16, 6, 40000, 16384, 64),
    (16384, 128, 2, 20000, 9000, 3),
]


@pytest.mark.parametrize("n,page,max_pages,n_pages,n_prefix,T", PLANS)
@pytest.mark.parametrize("in_place", [True, False])
def test_plans_match_oracle(cbx, n, page, max_pages, n_pages, n_prefix, T, in_place):
    """Prompts, steps, streams that end and give their pages back, refusals by
    every rule, in turn on one pool; lengths that are not ones among them."""
    torch, mod, s = cbx
    rng = np.random.default_rng(n * 31 + page)
    cap = max_pages * page
    pool = KV.Pool(n, max_pages, page, n_pages, n_prefix=n_prefix,
                   parent=rng.integers(-2, max(1, n_prefix) + 2, n),
                   prefix_len=rng.integers(-3, cap + 9, n), free=rng.permutation(n_pages))
    say("plans", n, page, n_prefix, in_place)
    if n > 8:
        pool.length[3], pool.length[5] = -4, cap + 1
        pool.free[2] = n_pages + 7  # a page that is not one
    d = Dev(torch, mod, pool)
    room = n_pages * page
    for turn in range(7):
        step = turn % 2 == 1
        ask = rng.integers(-1, 3, n) if step else \
            np.where(rng.random(n) < 0.5, rng.integers(-1, cap + 3, n), 0)
        if turn == 2:
            ask[:] = 0
        release = (rng.random(n) < 0.3).astype(np.int32) if turn > 1 else None
        state = rng.integers(0, 2, n) if turn in (3, 4) else None
        n_rows = None if step else int(max(1, min(room, rng.integers(1, room + 1) if turn == 4 else room)))
        if not step and turn == 6:
            n_rows = 4097  # the first size that takes a second launch
        d.plan(s, d.rows(step, n_rows, tiles=turn != 5, tile_rows=T), in_place=in_place,
               n_new=None if turn == 3 else ask, state=state, release=release)


def test_plan_on_another_stream_and_captured(cbx):
    """A captured step plan replayed: the streams grow by one each replay."""
    torch, mod, s = cbx
    pool = KV.Pool(9, 4, 16, 40, n_prefix=1, parent=[-1] + [0] * 8, prefix_len=[0] + [5] * 8)
    d = Dev(torch, mod, pool)
    d.plan(s, d.rows(False, 99), n_new=[7] + [13] * 8)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        d.plan(s, d.rows(True), state=[1] + [0] * 8)
    r = d.rows(True)
    state = d.ints([1] + [0] * 8)
    p = mod.Sampler.kv_plan(d.streams, r, page_size=16, state=state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.kv_build(p)
    for _ in range(6):
        graph.replay()
        torch.cuda.synchronize()
        want = KV.build(pool, n_tiles=len(r.b["tiles"]), tile_rows=64, state=[1] + [0] * 8)
        for k, w in want.items():
            assert np.array_equal(r.b[k].cpu().numpy(), w), k
        assert np.array_equal(d.tables.cpu().numpy(), pool.tables)
        assert np.array_equal(d.length.cpu().numpy(), pool.length)


# ------------------------------------------------------------------ attention


def caches(torch, rng, pool, n_kv, dtype, n_layer=1):
    """Pages that hold NaN wherever nothing was stored."""
    shape = (n_layer, len(pool.free), n_kv, pool.page, D)
    k, v = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    return k, v


def store(torch, rng, pool, caches_, layer, upto):
    """Random keys and values at the streams' positions [0, upto[i])."""
    for c in caches_:
        host = c.cpu()
        for i in range(pool.n):
            for j in range(-(-int(upto[i]) // pool.page)):
                pg, m = int(pool.tables[i, j]), min(pool.page, int(upto[i]) - j * pool.page)
                if 0 <= pg < len(pool.free):
                    x = rng.standard_normal((c.shape[2], m, D)).astype(np.float32)
                    host[layer, pg, :, :m] = torch.from_numpy(x).to(c.dtype)
        c.copy_(host)


def run(cbx, d, r, plan, cache, n_kv, group, rng, *, layer=0, sd=1.0, strided=True, new=True, q=None,
        kn=None, vn=None, stream=None, attn=None):
    """One call on planned rows, its outputs and stored rows checked.  Returns
    out, and everything that the call was made of."""
    torch, mod, s = cbx
    n_rows, H = r.n_rows, n_kv * group
    wide = (H + 2 * n_kv) * D + (8 if strided else 0)
    x = rng.standard_normal((n_rows, wide)).astype(np.float32)
    x[:, :H * D] *= sd
    rows = torch.from_numpy(x).cuda()
    if q is not None:
        rows[:, :H * D] = q
    qd, kd, vd = rows[:, :H * D], rows[:, H * D:(H + n_kv) * D], rows[:, (H + n_kv) * D:(H + 2 * n_kv) * D]
    if kn is not None:
        kd.copy_(kn)
        vd.copy_(vn)
    guard = 12
    buf = torch.full((n_rows + 1, H * D + guard), 3.0, device="cuda")
    out = buf[:n_rows, :H * D]
    k, v = cache
    before = [c.clone() for c in cache]
    a = mod.Sampler.kv_attn(mod.Sampler.kv_cache(k, v), d.streams, r, qd, out, layer=layer,
                            k=kd if new else None, v=vd if new else None, scale=0.125)
    s.kv_attend(a, stream=stream)
    torch.cuda.synchronize()
    # stored: the new rows at their slots, nothing else anywhere
    for c, b, n in ((k, before[0], kd), (v, before[1], vd)):
        if new:
            for row in range(n_rows):
                sl = int(plan["slot"][row])
                if sl >= 0:
                    b[layer, sl // d.pool.page, :, sl % d.pool.page] = n[row].reshape(n_kv, D).to(c.dtype)
        assert torch.equal(c.view(torch.int32 if c.element_size() == 4 else torch.int16),
                           b.view(torch.int32 if c.element_size() == 4 else torch.int16))
    assert torch.all(buf[:, H * D:] == 3.0) and torch.all(buf[n_rows] == 3.0)
    got = out.cpu().numpy()
    stream_of = plan.get("stream", np.arange(n_rows))
    host = [c[layer].float().cpu().numpy() for c in cache]
    want, size, mass, n_keys = KV.attend(d.pool, *host, stream_of, plan["position"],
                                         qd.cpu().numpy(), 0.125)
    b = bound(size, mass, n_keys).reshape(n_rows, -1)
    err = np.abs(got - want)
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine)
    worst = np.nanmax(np.where(fine, err / b, 0.0))
    assert worst <= 1.0, (worst, np.unravel_index(np.nanargmax(np.where(fine, err / b, 0)), err.shape))
    dead = plan["position"] < 0
    assert np.all(got[dead] == 0.0)
    return got, dict(q=qd.clone(), kn=kd.clone(), vn=vd.clone(), attn=a, out=out, want=want)


LENS = [
    [0], [1], [15], [16], [17], [31, 0, 33, 64, 65], [127, 128, 129, 383], [1000], [2049, 3],
    list(range(0, 300, 7)),
]


@pytest.mark.parametrize("lens", LENS, ids=[f"{len(x)}x{x[-1]}" for x in LENS])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("n_kv,group,page", [(4, 1, 16), (2, 2, 32), (1, 3, 16), (3, 5, 64)])
def test_step_matches_oracle(cbx, lens, dtype, n_kv, group, page):
    torch, mod, s = cbx
    rng = np.random.default_rng(len(lens) * 1000 + lens[-1] + group)
    say("step", lens[:4], dtype, n_kv, group, page)
    n = len(lens)
    max_pages = -(-(max(lens) + 1) // page)
    n_pages = sum(-(-(x + 1) // page) for x in lens) + 2
    pool = KV.Pool(n, max_pages, page, n_pages, free=rng.permutation(n_pages))
    d = Dev(torch, mod, pool)
    if sum(lens):
        d.plan(s, d.rows(False, sum(lens)), n_new=lens)
    c = caches(torch, rng, pool, n_kv, getattr(torch, dtype), n_layer=2)
    store(torch, rng, pool, c, 1, lens)
    r = d.rows(True, tiles=False)
    state = [1 if i % 5 == 4 else 0 for i in range(n)]  # some streams sit the step out
    plan = d.plan(s, r, state=state)
    run(cbx, d, r, plan, c, n_kv, group, rng, layer=1, sd=2.0)
    # the same again without new rows: they are in the cache now
    run(cbx, d, r, plan, c, n_kv, group, rng, layer=1, new=False)


SHARED = [  # prefixes' lengths, streams as (prefix or -1, positions shared, own)
    ([40], [(0, 40, 0), (0, 40, 5), (0, 33, 100), (-1, 0, 20), (0, 1, 16), (0, 0, 7)]),
    ([377], [(0, 377, x) for x in range(0, 70)]),
    ([16, 129, 700], [(i % 3, (16, 129, 650)[i % 3] - i % 2, 3 * i % 200) for i in range(41)]),
    ([64, 31], [(1, 31, 31)] * 3),
]


@pytest.mark.parametrize("prefixes,children", SHARED, ids=["mixed", "voice", "voices", "unused"])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("n_kv,group,page", [(4, 1, 16), (2, 4, 32), (1, 7, 16)])
def test_shared_prefix_matches_oracle(cbx, prefixes, children, dtype, n_kv, group, page):
    """With tiles (prefixes once for all) and without, prefixes that end inside
    a page and streams that share different parts of one."""
    torch, mod, s = cbx
    rng = np.random.default_rng(len(children) + group)
    n0 = len(prefixes)
    lens = prefixes + [x[2] for x in children]
    n = len(lens)
    say("shared", prefixes, n, dtype, n_kv, group, page)
    n_pages = sum(-(-(x + 1) // page) for x in lens) + 1
    pool = KV.Pool(n, -(-(max(lens) + 1) // page) + 1, page, n_pages, n_prefix=n0,
                   parent=[-1] * n0 + [x[0] for x in children],
                   prefix_len=[0] * n0 + [x[1] for x in children], free=rng.permutation(n_pages))
    d = Dev(torch, mod, pool)
    d.plan(s, d.rows(False, sum(lens)), n_new=lens)
    c = caches(torch, rng, pool, n_kv, getattr(torch, dtype))
    store(torch, rng, pool, c, 0, lens)
    T = mod.Sampler.kv_tile_rows(n_kv * group, n_kv)
    r = d.rows(True, tile_rows=T)
    plan = d.plan(s, r, state=[1] * n0 + [0] * (n - n0))
    got, x = run(cbx, d, r, plan, c, n_kv, group, rng, sd=2.0)
    # every row for itself
    r2 = d.rows(True, tiles=False)
    for k in ("position", "slot", "row_start"):
        r2.b[k].copy_(r.b[k])
    run(cbx, d, r2, plan, c, n_kv, group, rng, q=x["q"], kn=x["kn"], vn=x["vn"])


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("group", [1, 2, 5])
def test_many_rows_beside_prefixes(cbx, dtype, group):
    """More rows than workgroups are given one each (a wave a row and key head,
    but for fp16 with three and more query heads), some without a prefix."""
    children = [((-1, 0), (0, 140), (1, 17))[i % 3] + (i % 37,) for i in range(1040)]
    test_shared_prefix_matches_oracle(cbx, [150, 17], children, dtype, 4, group, 16)


PROMPTS = [  # prefixes, (prefix, shared, already cached, new)
    ([], [(-1, 0, 0, 1)]), ([], [(-1, 0, 0, 16)]), ([], [(-1, 0, 0, 17), (-1, 0, 0, 63)]),
    ([], [(-1, 0, 5, 64), (-1, 0, 16, 65), (-1, 0, 40, 3), (-1, 0, 0, 0), (-1, 0, 9, 129)]),
    ([45], [(0, 45, 0, 33), (0, 20, 3, 70), (-1, 0, 0, 18)]),
    ([], [(-1, 0, 0, 251)]),
    ([100], [(0, 100, 7 * i % 40, 40 + i % 50) for i in range(70)]),
    ([], [(-1, 0, 600, 130)] * 3),
]


PROMPT_CASES = [  # 64 heads to a key head: small ones, the oracle takes a head at a time
    pytest.param(p, x, *h, id=f"{len(x)}-{sum(y[3] for y in x)}-{h[0]}-{h[1]}-{h[2]}")
    for h in ((4, 1, 16), (2, 2, 32), (1, 5, 16), (1, 64, 16)) for p, x in PROMPTS
    if h[1] < 64 or sum(y[3] for y in x) < 300]


@pytest.mark.parametrize("prefixes,streams,n_kv,group,page", PROMPT_CASES)
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_prompts_match_oracle(cbx, prefixes, streams, dtype, n_kv, group, page):
    torch, mod, s = cbx
    rng = np.random.default_rng(len(streams) * 7 + group)
    n0 = len(prefixes)
    had = prefixes + [x[2] for x in streams]
    new = [0] * n0 + [x[3] for x in streams]
    n = len(had)
    say("prompt", prefixes, streams[:3], dtype, n_kv, group, page)
    total = [a + b for a, b in zip(had, new)]
    n_pages = sum(-(-x // page) for x in total) + 1
    pool = KV.Pool(n, max(-(-max(total) // page), 1) + 1, page, n_pages, n_prefix=n0,
                   parent=[-1] * n0 + [x[0] for x in streams],
                   prefix_len=[0] * n0 + [x[1] for x in streams], free=rng.permutation(n_pages))
    d = Dev(torch, mod, pool)
    if sum(had):
        d.plan(s, d.rows(False, sum(had)), n_new=had)
    c = caches(torch, rng, pool, n_kv, getattr(torch, dtype))
    store(torch, rng, pool, c, 0, had)
    r = d.rows(False, sum(new) + 5, tile_rows=mod.Sampler.kv_tile_rows(n_kv * group, n_kv))
    plan = d.plan(s, r, n_new=new)
    run(cbx, d, r, plan, c, n_kv, group, rng, sd=2.0)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_prompts_behind_long_caches(cbx, dtype):
    """Whole tiles a workgroup over many stages: cached keys, then new ones."""
    test_prompts_match_oracle(cbx, [77], [(0, 70, 523, 130), (-1, 0, 700, 129)] * 12, dtype,
                              8, 1, 16)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n", [(40, 21), (90,) * 60], ids=["few", "many"])
def test_values_that_are_not_finite_stay(cbx, dtype, bad, n):
    """A new row whose value is not finite reaches itself and the rows after it
    alone, bit for bit."""
    torch, mod, s = cbx
    rng = np.random.default_rng(5)
    n_pages = sum(-(-x // 16) for x in n)
    out = []
    for plant in (False, True):
        rng = np.random.default_rng(5)
        pool = KV.Pool(len(n), 8, 16, n_pages)
        d = Dev(torch, mod, pool)
        r = d.rows(False, sum(n))
        plan = d.plan(s, r, n_new=n)
        c = caches(torch, rng, pool, 2, getattr(torch, dtype))
        x = torch.from_numpy(rng.standard_normal((sum(n), 6 * D)).astype(np.float32)).cuda()
        if plant:
            x[n[0] + 9, 4 * D + 3] = bad   # stream 1, position 9: a value of head 0
        o = torch.empty((sum(n), 2 * D), device="cuda")
        say("not finite", dtype, bad, len(n))
        s.kv_attend(mod.Sampler.kv_attn(mod.Sampler.kv_cache(*c), d.streams, r, x[:, :2 * D], o,
                                        k=x[:, 2 * D:4 * D], v=x[:, 4 * D:]))
        torch.cuda.synchronize()
        out.append(o.cpu().numpy())
    a, b = out
    hit = np.zeros(a.shape, bool)
    hit[n[0] + 9:n[0] + n[1], 3] = True
    assert np.array_equal(a[~hit], b[~hit])
    assert not np.isfinite(b[hit]).any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_prefix_part_that_a_row_does_not_share(cbx, bad):
    """A prefix's values past a stream's share never reach it."""
    torch, mod, s = cbx
    out = []
    for plant in (False, True):
        rng = np.random.default_rng(6)
        pool = KV.Pool(5, 4, 16, 20, n_prefix=1, parent=[-1] + [0] * 4, prefix_len=[0, 40, 37, 12, 9])
        d = Dev(torch, mod, pool)
        d.plan(s, d.rows(False, 99), n_new=[40, 4, 4, 4, 4])
        c = caches(torch, rng, pool, 2, torch.float32)
        store(torch, rng, pool, c, 0, [40, 4, 4, 4, 4])
        if plant:
            c[1][0, int(pool.tables[0, 0]), 1, 12, 7] = bad  # position 12 of the prefix, head 1
        r = d.rows(True)
        d.plan(s, r, state=[1, 0, 0, 0, 0])
        x = torch.from_numpy(rng.standard_normal((5, 6 * D)).astype(np.float32)).cuda()
        o = torch.empty((5, 2 * D), device="cuda")
        say("unshared", bad)
        s.kv_attend(mod.Sampler.kv_attn(mod.Sampler.kv_cache(*c), d.streams, r, x[:, :2 * D], o,
                                        k=x[:, 2 * D:4 * D], v=x[:, 4 * D:]))
        torch.cuda.synchronize()
        out.append(o.cpu().numpy())
    hit = np.zeros(out[0].shape, bool)
    hit[1:3, D + 7] = True
    assert np.array_equal(out[0][~hit], out[1][~hit])
    assert not np.isfinite(out[1][hit]).any()


@pytest.mark.parametrize("form", ["step", "shared", "prompt"])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_pages_that_are_not_ones(cbx, form, dtype):
    """Table entries outside the pool: their positions are not seen, and nothing
    is stored there; a row that sees nothing gives zeros."""
    torch, mod, s = cbx
    rng = np.random.default_rng(9)
    pool = KV.Pool(4, 6, 16, 30, n_prefix=1, parent=[-1, 0, 0, -1], prefix_len=[0, 30, 17, 0])
    d = Dev(torch, mod, pool)
    lens = [40, 50, 10, 20]
    d.plan(s, d.rows(False, 999), n_new=lens)
    c = caches(torch, rng, pool, 2, getattr(torch, dtype))
    store(torch, rng, pool, c, 0, lens)
    pool.tables[0, 0], pool.tables[1, 1], pool.tables[1, 3] = 30, -1, 2 ** 31 - 1
    pool.tables[3, 0], pool.tables[3, 1] = -5, 1 << 20
    d.tables.copy_(torch.from_numpy(pool.tables))
    say("bad pages", form, dtype)
    step = form != "prompt"
    r = d.rows(step, 60, tiles=form != "step")
    plan = d.plan(s, r, n_new=[0, 1, 1, 1] if step else [0, 20, 3, 5])
    got, _ = run(cbx, d, r, plan, c, 2, 1, rng)
    assert np.all(got[plan["position"] < 0] == 0.0)
    last = 3 if step else 23  # stream 3 sees none of its own
    assert np.all(got[last] == 0.0)


def test_scores_all_minus_infinity(cbx):
    torch, mod, s = cbx
    rng = np.random.default_rng(2)
    pool = KV.Pool(3, 4, 16, 12)
    d = Dev(torch, mod, pool)
    d.plan(s, d.rows(False, 99), n_new=[20, 20, 20])
    c = caches(torch, rng, pool, 1, torch.float32)
    store(torch, rng, pool, c, 0, [20, 20, 20])
    c[0][0, int(pool.tables[0, 0]), 0, 3, 0] = -float("inf")   # one key of stream 0
    c[0][0, pool.tables[1, :2].tolist(), 0, :, 0] = -float("inf")  # all of stream 1's
    r = d.rows(True, tiles=False)
    d.plan(s, r)
    x = torch.from_numpy(np.abs(rng.standard_normal((3, 3 * D))).astype(np.float32)).cuda()
    x[1, D] = -float("inf")
    o = torch.empty((3, D), device="cuda")
    say("minus infinity")
    s.kv_attend(mod.Sampler.kv_attn(mod.Sampler.kv_cache(*c), d.streams, r, x[:, :D], o,
                                    k=x[:, D:2 * D], v=x[:, 2 * D:]))
    torch.cuda.synchronize()
    o = o.cpu().numpy()
    assert np.isfinite(o).all() and np.all(o[1] == 0.0) and np.all(o[0] != 0.0)


def test_long_stream(cbx):
    """More pages than a workgroup holds ids for at once, and a prefix of such a
    length read by the row itself."""
    torch, mod, s = cbx
    rng = np.random.default_rng(4)
    lens = [9001, 17, 8200]
    pool = KV.Pool(3, 570, 16, 1200, n_prefix=1, parent=[-1, 0, 0], prefix_len=[0, 9001, 8193],
                   free=rng.permutation(1200))
    d = Dev(torch, mod, pool)
    d.plan(s, d.rows(False, sum(lens)), n_new=lens)
    c = caches(torch, rng, pool, 1, torch.float32)
    store(torch, rng, pool, c, 0, lens)
    for tiles in (False, True):
        r = d.rows(True, tiles=tiles)
        plan = d.plan(s, r, n_new=[0, 1, 1])
        say("long", tiles)
        run(cbx, d, r, plan, c, 1, 1, rng)


def test_rows_do_not_depend_on_rows_beside_them(cbx):
    """A prompt's rows are bit for bit the same alone and beside other streams'
    in the same form (few rows: keys over four waves), in any place."""
    torch, mod, s = cbx
    out = []
    for lens, at in (([60], 0), ([33, 60, 7], 1), ([1, 20, 60], 2)):
        rng = np.random.default_rng(8)
        mine = rng.standard_normal((60, 6 * D)).astype(np.float32)
        pool = KV.Pool(len(lens), 4, 16, 12)
        d = Dev(torch, mod, pool)
        r = d.rows(False, sum(lens))
        d.plan(s, r, n_new=lens)
        c = caches(torch, rng, pool, 2, torch.float32)
        x = rng.standard_normal((sum(lens), 6 * D)).astype(np.float32)
        f = sum(lens[:at])
        x[f:f + 60] = mine
        x = torch.from_numpy(x).cuda()
        o = torch.empty((sum(lens), 2 * D), device="cuda")
        say("beside", lens)
        s.kv_attend(mod.Sampler.kv_attn(mod.Sampler.kv_cache(*c), d.streams, r, x[:, :2 * D], o,
                                        k=x[:, 2 * D:4 * D], v=x[:, 4 * D:]))
        torch.cuda.synchronize()
        out.append(o[f:f + 60].cpu().numpy())
    assert np.array_equal(out[0], out[1]) and np.array_equal(out[0], out[2])


def test_two_graphs_and_a_second_stream(cbx):
    """Two calls with workspaces of their own, captured and replayed at once on
    two streams, several times, against their eager results."""
    torch, mod, s = cbx
    made = []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        lens = [50] + [int(x) for x in rng.integers(1, 90, 20)]
        pool = KV.Pool(21, 7, 16, 200, n_prefix=1, parent=[-1] + [0] * 20, prefix_len=[0] + [50] * 20)
        d = Dev(torch, mod, pool)
        d.plan(s, d.rows(False, sum(lens)), n_new=lens)
        c = caches(torch, rng, pool, 4, torch.float32)
        store(torch, rng, pool, c, 0, lens)
        r = d.rows(True)
        plan = d.plan(s, r, state=[1] + [0] * 20)
        say("graphs", seed)
        got, x = run(cbx, d, r, plan, c, 4, 1, rng)
        made.append((d, r, c, got, x))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    for _, _, _, _, x in made:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.kv_attend(x["attn"])
        graphs.append(g)
    for _ in range(5):
        for _, _, _, _, x in made:
            x["out"].fill_(9.0)
        torch.cuda.synchronize()
        for st, g in zip(side, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for _, _, _, got, x in made:
            assert np.array_equal(x["out"].cpu().numpy(), got)
