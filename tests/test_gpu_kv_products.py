"""GPU: every part of a matrix-core product is there (cbx_kv_attend).  Inputs and
limits of tests/kv_products.py, under which leaving out any one product shows
(tests/test_kv_products.py); the vector units' forms are held to the same."""
import numpy as np
import pytest

import kv_products as P
from oracle import cbx_kv_oracle as KV
from test_gpu_kv import Dev, caches, cbx, run, say  # noqa: F401

pytestmark = pytest.mark.gpu
N_KV = 4


def put(torch, pool, c, i, at, x):
    """Keys and values of stream i's position at."""
    for t, y in zip(c, x):
        t[0, int(pool.tables[i, at // pool.page]), :, at % pool.page] = \
            torch.from_numpy(np.ascontiguousarray(y)).to(t.dtype).cuda()


def check(d, c, plan, got, x, dtype):
    host = [t[0].float().cpu().numpy() for t in c]
    rows = np.arange(len(got))
    want, size, mass, _ = KV.attend(d.pool, *host, plan.get("stream", rows), plan["position"],
                                    x["q"].cpu().numpy(), 0.125)
    worst = (np.abs(got - want).reshape(mass.shape) / P.limit(dtype, size, mass)).max()
    print("of the limit: %.3f" % worst, flush=True)
    assert worst <= 1.0


@pytest.mark.parametrize("X", [0.5, 100.0])
@pytest.mark.parametrize("group", [1, 2, 4])
@pytest.mark.parametrize("had", [0, 1, 2])
@pytest.mark.parametrize("n", [6, 240], ids=["few", "many"])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_prompts(cbx, dtype, n, had, group, X):  # noqa: F811
    """Two keys a stream, of which the cache holds `had` (2: a third, of zeros, is new)."""
    torch, mod, s = cbx
    rng = np.random.default_rng(group)
    say("products, prompts", dtype, n, had, group, X)
    k, v = P.keys(rng, n, N_KV, dtype)
    pool = KV.Pool(n, 1, 16, n, free=rng.permutation(n))
    d = Dev(torch, mod, pool)
    c = caches(torch, rng, pool, N_KV, getattr(torch, dtype))
    if had:
        d.plan(s, d.rows(False, had * n), n_new=[had] * n)
        for i in range(n):
            for j in range(had):
                put(torch, pool, c, i, j, (k[j, i], v[j, i]))
    new = max(2 - had, 1)
    r = d.rows(False, n * new, tile_rows=64 // group)
    plan = d.plan(s, r, n_new=[new] * n)
    q = np.repeat(P.queries(rng, k, group, X), new, 0)
    kn, vn = (np.zeros((n, new, N_KV * P.D), np.float32) for _ in range(2))
    for j in range(had, 2):
        kn[:, j - had], vn[:, j - had] = k[j].reshape(n, -1), v[j].reshape(n, -1)
    t = lambda a: torch.from_numpy(a.reshape(n * new, -1)).cuda()  # noqa: E731
    got, x = run(cbx, d, r, plan, c, N_KV, group, rng, q=t(q), kn=t(kn), vn=t(vn))
    check(d, c, plan, got, x, dtype)


@pytest.mark.parametrize("X", [0.5, 100.0])
@pytest.mark.parametrize("group", [1, 2, 4])
@pytest.mark.parametrize("shared", [0, 1, 2], ids=["own", "both", "prefix"])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_steps(cbx, dtype, shared, group, X):  # noqa: F811
    """Two keys a stream, `shared` of them a prefix's (2: a third, of zeros, is new)."""
    torch, mod, s = cbx
    rng = np.random.default_rng(group)
    say("products, steps", dtype, shared, group, X)
    n, n0 = 70, 1 if shared else 0
    k, v = P.keys(rng, n, N_KV, dtype)
    k[:shared], v[:shared] = k[:shared, :1], v[:shared, :1]
    pool = KV.Pool(n0 + n, 1, 16, n0 + n, n_prefix=n0, parent=[-1] * n0 + [n0 - 1] * n,
                   prefix_len=[0] * n0 + [shared] * n, free=rng.permutation(n0 + n))
    d = Dev(torch, mod, pool)
    c = caches(torch, rng, pool, N_KV, getattr(torch, dtype))
    own = 0 if shared else 1
    d.plan(s, d.rows(False, 2 + n), n_new=[shared] * n0 + [own] * n)
    for j in range(shared):
        put(torch, pool, c, 0, j, (k[j, 0], v[j, 0]))
    for i in range(n if own else 0):
        put(torch, pool, c, i, 0, (k[0, i], v[0, i]))
    r = d.rows(True, tiles=bool(shared), tile_rows=64 // group)
    plan = d.plan(s, r, state=[1] * n0 + [0] * n)
    t = lambda a: torch.from_numpy(np.concatenate(  # noqa: E731
        [np.zeros((n0, a[0].size), np.float32), a.reshape(n, -1)])).cuda()
    new = (k[1], v[1]) if shared < 2 else (np.zeros_like(k[1]),) * 2
    got, x = run(cbx, d, r, plan, c, N_KV, group, rng, q=t(P.queries(rng, k, group, X)),
                 kn=t(new[0]), vn=t(new[1]))
    check(d, c, plan, got, x, dtype)
