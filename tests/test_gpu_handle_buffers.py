"""A handle's buffers that a captured graph holds stay when larger calls replace
them; those that no graph holds are given back."""
import numpy as np
import pytest

import oracle_lib as O
from test_gpu_head import _problem
from test_gpu_kv_t3 import N, Server, small  # noqa: F401

pytestmark = pytest.mark.gpu


def test_only_a_captured_buffer_is_kept(small):  # noqa: F811
    """A T3 call captured, then larger and larger ones, of the T3 and of the head.
    The T3's workspace is linear in the rows (past a few), the head's too: n0 rows
    take `one` bytes.  Held at the end: the graph's and the largest, 1 + 16 of n0
    rows, and the head's largest; each allocation's rounding is far below n0 rows'."""
    torch, mod, s, dm, _ = small
    n0, most = 2000, 32000
    fresh = mod.Sampler(device=0, max_vocab=1024, max_history=64)
    srv = Server(torch, mod, s, dm, 3, 0, torch.float32)
    hid, tokens = torch.empty((most, N), device="cuda"), srv.ints([0] * most)
    rows = {}
    for n in (n0, 4 * n0, 8 * n0, 12 * n0, most):
        rows[n] = srv.rows(n, step=False)
        srv.plan(rows[n], n_new=[0, 0, 0])

    def call(n):
        fresh.t3_kv(dm, srv.cache, srv.streams, rows[n], hid[:n], tokens=tokens[:n])

    V, K = 96, 512
    blocks, bias, h = _problem(np.random.default_rng(1), V, K, 64, O.WTYPE_Q8_0)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    dW, db = t(blocks.reshape(-1)), t(bias)
    h, logits = t(h).repeat(most // 64, 1), torch.empty((most, V), device="cuda")

    def head(n):
        fresh.head_logits(mod.Sampler.head(dW, O.WTYPE_Q8_0, K, h[:n], logits[:n], bias=db), n, V, V)

    # the kernels' code is loaded by calls on another handle
    print("[gpu-case] buffers of a handle", flush=True)
    s.t3_kv(dm, srv.cache, srv.streams, rows[most], hid, tokens=tokens)
    s.head_logits(mod.Sampler.head(dW, O.WTYPE_Q8_0, K, h, logits, bias=db), most, V, V)
    torch.cuda.synchronize()

    def free():
        torch.cuda.synchronize()
        return torch.cuda.mem_get_info()[0]

    at = [free()]
    call(n0)
    one = at[0] - free()
    assert one > n0 * 10 * N * 4
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(n0)
    start = free()
    for n in (4 * n0, 8 * n0, 12 * n0, most):
        call(n)
    held = start - free()
    assert abs(held - most // n0 * one) < one, (held / one, most // n0)
    start = free()
    for n in (most // 2, most // 4 * 3, most):
        head(n)
    held = start - free()
    # the rows split into fp16 halves: 4 bytes a value, 1/32 of a scale's 4
    assert abs(held - most * K * 4 * 33 / 32) < most * K, held / (most * K * 4)
    # the graph's workspace is its own still
    hid[:n0].fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.all(hid[:n0] == 0.0)
    fresh.close()
