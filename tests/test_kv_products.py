"""The limit of tests/test_gpu_kv_products.py against a model of the matrix-core
products: with all parts it holds, with any one product left out it does not."""
import numpy as np
import pytest

import kv_products as P

X = [0.5, 100.0]


def made(dtype, x):
    rng = np.random.default_rng(int(x))
    k, v = P.keys(rng, 400, 4, dtype)
    q = P.queries(rng, k, 1, x).reshape(-1, P.D)
    return q, k.reshape(2, -1, P.D), v.reshape(2, -1, P.D)


def worst(dtype, x, **without):
    q, k, v = made(dtype, x)
    want, size, mass = P.exact(q, k, v)
    return (np.abs(P.model(q, k, v, dtype, **without) - want) / P.limit(dtype, size, mass)).max()


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("x", X)
def test_all_parts(dtype, x):
    assert worst(dtype, x) < 0.7


@pytest.mark.parametrize("dtype,i", [(t, i) for t in P.PRODUCTS for i in range(len(P.PRODUCTS[t]))])
def test_a_product_left_out_shows(dtype, i):
    assert worst(dtype, 100.0, scores_without=i) > 2.0
    assert worst(dtype, 0.5, values_without=i) > 2.0
