"""The T3 transformer on a paged cache (cbx_t3_kv, include/cbx_t3.h) as a server
uses it: a voice's prompt stored once, requests' prompts behind it, decode steps
on tables that grow by the plan, streams that end and whose slots are given to
new requests -- every row against the binary64 oracle stepping each stream in a
dense cache of its own (oracle/cbx_t3_oracle.py), the voice's rows repeated.

Tolerance, fp32 cache: |gpu - ref| <= 5e-5 + 5e-5 |ref|, the dense step's
(tests/test_gpu_t3.py).  fp16 cache: the oracle's cache rounds to fp16 too; a
value so near a rounding border that the two round it apart is off by one step,
twice what any rounding moves one, so outputs may be off by twice what rounding
all of them changes (the largest difference between the oracle with and without
rounding), besides the fp32 tolerance.
"""
import numpy as np
import pytest

import oracle_lib as O
import pkg
from oracle import cbx_t3_oracle as T3
from test_gpu_t3_prompt import H, L_, N, V, model

pytestmark = pytest.mark.gpu
TOL = 5e-5


@pytest.fixture(scope="module")
def small():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    mod = pkg.load()
    s = mod.Sampler(device=0, max_vocab=1024, max_history=64)
    yield (torch, mod, s) + model(torch, mod, O.WTYPE_Q8_0)
    s.close()


class Server:
    """Streams of a paged pool on the device; the oracle's dense caches beside."""

    def __init__(self, torch, mod, s, dm, n, n_prefix, dtype, page=16, n_pages=90, max_pages=12):
        self.torch, self.mod, self.s, self.dm, self.n = torch, mod, s, dm, n
        z = lambda *sh: torch.zeros(sh, dtype=torch.int32, device="cuda")
        self.tables, self.length, self.n_free = z(n, max_pages), z(n), z(1) + n_pages
        self.free = torch.randperm(n_pages, device="cuda").to(torch.int32)
        self.parent, self.prefix_len = z(n) - 1, z(n)
        self.k, self.v = (torch.full((L_, n_pages, H, page, 64), float("nan"), dtype=dtype,
                                     device="cuda") for _ in range(2))
        self.cache = mod.Sampler.kv_cache(self.k, self.v)
        self.streams = mod.Sampler.kv_streams(self.tables, self.length, self.free, self.n_free,
                                              n_prefix=n_prefix, parent=self.parent,
                                              prefix_len=self.prefix_len)
        self.page, self.n_prefix = page, n_prefix

    def ints(self, a):
        return self.torch.tensor(a, dtype=self.torch.int32, device="cuda")

    def rows(self, n_rows, step, tiles=True):
        e = lambda *sh: self.torch.empty(sh, dtype=self.torch.int32, device="cuda")
        kw = {} if step else dict(stream=e(n_rows))
        if tiles:
            kw["tiles"] = e(n_rows // 64 + self.n + 1, 4)
            if step:
                kw["order"] = e(n_rows)
        self.row_start, self.counts, self.position = e(self.n + 1), e(4), e(n_rows)
        return self.mod.Sampler.kv_rows(self.position, e(n_rows), self.row_start, e(self.n + 1),
                                        self.counts, tile_rows=64, **kw)

    def plan(self, rows, **kw):
        kw = {k: self.ints(v) for k, v in kw.items()}
        self.s.kv_build(self.mod.Sampler.kv_plan(self.streams, rows, page_size=self.page, **kw))

    def prompt(self, x, n_new, room=0, **kw):
        r = self.rows(sum(n_new) + room, step=False)
        self.plan(r, n_new=n_new, **kw)
        hid = self.torch.full((r.n_rows, N), 7.0, device="cuda")
        rows = np.zeros((r.n_rows, N), np.float32)
        rows[:len(x)] = x
        self.s.t3_kv(self.dm, self.cache, self.streams, r, hid, inputs=self.torch.from_numpy(rows).cuda())
        self.torch.cuda.synchronize()
        assert self.counts.tolist()[3] == 0
        return hid.cpu().numpy()

    def step(self, tokens, state, tiles):
        r = self.rows(self.n, step=True, tiles=tiles)
        self.plan(r, state=state)
        hid = self.torch.full((self.n, N), 7.0, device="cuda")
        self.s.t3_kv(self.dm, self.cache, self.streams, r, hid, tokens=self.ints(tokens))
        self.torch.cuda.synchronize()
        return hid.cpu().numpy()


@pytest.mark.parametrize("n,tiles", [(2, False), (3, True), (7, True), (7, False), (40, True)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_serving_on_a_paged_cache(small, n, tiles, dtype):
    torch, mod, s, dm, rm = small
    print(f"[gpu-case] serving n={n} tiles={tiles} {dtype}", flush=True)
    rng = np.random.default_rng(n)
    srv = Server(torch, mod, s, dm, n, 1, getattr(torch, dtype), n_pages=30 + 8 * n)
    half = dtype == "float16"
    oracles = [T3.new_cache(n, L_, H, 160)]
    if half:
        oracles.append(tuple(c.astype(np.float16) for c in T3.new_cache(n, L_, H, 160)))
    moved = [0.0]

    def check(got, want):
        """want: the row(s) from each oracle, the plain one first."""
        if half:
            moved[0] = max(moved[0], np.abs(want[1] - want[0]).max())
        err = np.abs(got - want[-1]) - TOL * np.abs(want[-1])
        assert err.max() <= TOL + 2 * moved[0], (err.max(), moved)

    rows = lambda k: (rng.standard_normal((k, N)) * 0.7).astype(np.float32)
    voice = rows(37)
    got = srv.prompt(voice, [37] + [0] * (n - 1), room=3)
    want = [T3.prefill(rm, voice, *c, 0, 0) for c in oracles]
    check(got[:37], want)
    assert np.all(got[37:] == 0.0)
    # most requests share the whole voice, some 20 positions of it, some none
    plen = [0] + [(37, 37, 20, 0)[i % 4] for i in range(n - 1)]
    srv.prefix_len.copy_(srv.ints(plen))
    srv.parent.copy_(srv.ints([-1] + [0 if p else -1 for p in plen[1:]]))
    own = np.zeros(n, np.int64)
    filled = [37] + [0] * (n - 1)

    def admit(who):
        new, x = [0] * n, {}
        for i in who:
            new[i], own[i] = 5 + int(rng.integers(0, 40)), 0
            x[i] = rows(new[i])
            for c in oracles:  # the voice's rows in a dense cache of the stream's own
                if plen[i] and i:
                    T3.prefill(rm, voice[:plen[i]], *c, i, 0)
        got = srv.prompt(np.concatenate([x[i] for i in who]), new,
                         release=[1 if i in who else 0 for i in range(n)])
        f = 0
        for i in who:
            check(got[f:f + new[i]], [T3.prefill(rm, x[i], *c, i, plen[i]) for c in oracles])
            f, own[i] = f + new[i], new[i]

    def steps(count, state):
        for _ in range(count):
            tokens = rng.integers(0, V, n)
            active = np.array(state) == 0
            got = srv.step(tokens, state, tiles)
            want = []
            for c in oracles:
                at = np.array([plen[i] + own[i] for i in range(n)])
                want.append(T3.step(rm, tokens, at, *c, active=active))
            check(got[active], [w[active] for w in want])
            assert np.all(got[~active] == 0.0)
            own[active] += 1

    admit(list(range(1, n)))
    steps(18, [1] + [0] * (n - 1))  # over a page's end
    ended = [i for i in range(1, n) if i % 3 == 1]
    admit(ended)
    steps(3, [1] + [1 if i % 5 == 4 else 0 for i in range(1, n)])
    assert srv.length.tolist()[1:] == own[1:].tolist()
    # every page is in one table or on the stack
    held = [int(x) for i in range(n) for x in
            srv.tables[i, :-(-(37 if i == 0 else int(own[i])) // 16)].tolist()]
    free = srv.free[:int(srv.n_free)].tolist()
    assert sorted(held + free) == list(range(30 + 8 * n))


def test_rows_that_take_no_part(small):
    """A token or a position that the model does not have: zero rows, and the
    other streams' as without them."""
    torch, mod, s, dm, rm = small
    out = []
    for bad in (False, True):
        rng = np.random.default_rng(3)
        torch.manual_seed(5)
        srv = Server(torch, mod, s, dm, 6, 0, torch.float32)
        x = (rng.standard_normal((60, N)) * 0.7).astype(np.float32)
        srv.prompt(x, [10] * 6)
        tokens = rng.integers(0, V, 6)
        if bad:
            tokens[1], tokens[4] = -1, V
        print(f"[gpu-case] no part {bad}", flush=True)
        out.append([srv.step(tokens, [0] * 6, False)])
        tokens = rng.integers(0, V, 6)
        out[-1].append(srv.step(tokens, [0] * 6, False))
    keep = [0, 2, 3, 5]
    for a, b in zip(*out):
        assert np.array_equal(a[keep], b[keep])
    assert np.all(out[1][0][[1, 4]] == 0.0) and np.isfinite(out[1][1]).all()


def test_refusals(small):
    torch, mod, s, dm, rm = small
    srv = Server(torch, mod, s, dm, 4, 1, torch.float32)
    r = srv.rows(4, step=True)
    hid = torch.zeros((4, N), device="cuda")
    tok = srv.ints([0] * 4)
    two = torch.zeros((L_ + 1, 90, H, 16, 64), device="cuda")
    with pytest.raises(mod.CbxError):  # another number of layers
        s.t3_kv(dm, mod.Sampler.kv_cache(two, two.clone()), srv.streams, r, hid, tokens=tok)
    with pytest.raises(mod.CbxError):  # neither ids nor input rows
        s.t3_kv(dm, srv.cache, srv.streams, r, hid)
    with pytest.raises(ValueError):
        s.t3_kv(dm, srv.cache, srv.streams, r, hid[:3], tokens=tok)
    with pytest.raises(ValueError):
        s.t3_kv(dm, srv.cache, srv.streams, r, hid, tokens=tok.long())


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_a_step_captured_with_its_plan(small, dtype):
    """Plan and transformer in one graph, replayed past a page's end while its
    streams grow, eager calls of another server on the handle between: each
    replay's rows are the eager steps' of a server like it."""
    torch, mod, s, dm, rm = small
    made = []
    for _ in range(3):
        rng = np.random.default_rng(8)
        torch.manual_seed(9)
        srv = Server(torch, mod, s, dm, 9, 1, getattr(torch, dtype))
        srv.prompt((rng.standard_normal((21, N)) * 0.7).astype(np.float32), [21] + [0] * 8)
        srv.prefix_len.copy_(srv.ints([0] + [21] * 4 + [10] * 4))
        srv.parent.copy_(srv.ints([-1] + [0] * 8))
        srv.prompt((rng.standard_normal((72, N)) * 0.7).astype(np.float32), [0] + [9] * 8)
        made.append(srv)
    eager, captured, other = made
    state = [1] + [0] * 8
    r = captured.rows(9, step=True)
    tokens, hid = captured.ints([0] * 9), torch.zeros((9, N), device="cuda")
    plan = mod.Sampler.kv_plan(captured.streams, r, page_size=16, state=captured.ints(state))
    print(f"[gpu-case] captured step {dtype}", flush=True)
    other.step([1] * 9, state, True)  # the handle's workspace, as large as the graph's call wants it
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.kv_build(plan)
        s.t3_kv(dm, captured.cache, captured.streams, r, hid, tokens=tokens)
    for i in range(12):
        if i == 5:  # a call that wants a larger workspace than the graph's
            k = 133 if dtype == "float32" else 145
            big = Server(torch, mod, s, dm, 9, 0, torch.float32, n_pages=100)
            big.prompt((rng.standard_normal((9 * k, N)) * 0.7).astype(np.float32), [k] * 9)
        ids = rng.integers(0, V, 9)
        want = eager.step(ids, state, True)
        other.step(rng.integers(0, V, 9), state, True)
        tokens.copy_(captured.ints(ids))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(hid.cpu().numpy(), want)
    assert torch.equal(captured.length, eager.length) and captured.length.tolist()[1:] == [21] * 8


def test_a_workspace_does_not_grow_in_a_capture(small):
    torch, mod, s, dm, rm = small
    fresh = mod.Sampler(device=0, max_vocab=1024, max_history=64)
    srv = Server(torch, mod, s, dm, 9, 0, torch.float32)
    r = srv.rows(9, step=True)
    srv.plan(r)
    hid, x = torch.full((9, N), 7.0, device="cuda"), torch.zeros(8, device="cuda")
    tokens = srv.ints([1] * 9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1.0)
        with pytest.raises(mod.CbxError):
            fresh.t3_kv(dm, srv.cache, srv.streams, r, hid, tokens=tokens)
    graph.replay()
    fresh.t3_kv(dm, srv.cache, srv.streams, r, hid, tokens=tokens)
    torch.cuda.synchronize()
    assert torch.all(x == 1.0) and torch.isfinite(hid).all() and not torch.any(hid == 7.0)
    fresh.close()
