"""GPU tests of cbx_kv_build at the ends of its ranges."""
import numpy as np
import pytest

import pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cbx():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    mod = pkg.load()
    s = mod.Sampler(device=0, max_vocab=1024, max_history=64)
    yield torch, mod, s
    s.close()


def test_more_pages_given_back_than_32_bits_count(cbx):
    """Streams whose lengths claim more than 2^31 pages between them (no pool has
    them: the lengths are wrong, each alone is one that a stream may have): the
    stack takes pages in stream order until it is full, and nothing is written
    before it or behind it."""
    torch, mod, s = cbx
    n, max_pages, n_pages, had = 16384, 1 << 18, 1 << 18, 100
    i32 = dict(dtype=torch.int32, device="cuda")
    assert n * max_pages > 1 << 31
    tables = torch.empty((n, max_pages), **i32)
    tables[:2] = torch.arange(2 * max_pages, **i32).reshape(2, -1)
    length = torch.full((n,), max_pages * 16, **i32)
    guard = 4096
    buf = torch.full((guard + n_pages + guard,), -9, **i32)
    free = buf[guard:guard + n_pages]
    free[:had] = -3
    n_free = torch.full((1,), had, **i32)
    e = lambda *x: torch.full(x, -7, **i32)
    rows = mod.Sampler.kv_rows(e(1), e(1), e(n + 1), e(n + 1), e(4), stream=e(1))
    plan = mod.Sampler.kv_plan(mod.Sampler.kv_streams(tables, length, free, n_free), rows, page_size=16,
                               n_new=torch.zeros(n, **i32), release=torch.ones(n, **i32))
    print("[gpu-case] pages past 2^31 given back", flush=True)
    s.kv_build(plan)
    torch.cuda.synchronize()
    assert n_free.tolist() == [n_pages] and not length.any()
    want = np.full(guard + n_pages + guard, -9, np.int32)
    want[guard:guard + had] = -3
    want[guard + had:guard + n_pages] = np.arange(n_pages - had)
    assert np.array_equal(buf.cpu().numpy(), want)
    del tables, plan
    torch.cuda.empty_cache()
