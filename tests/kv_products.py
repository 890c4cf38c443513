"""Inputs and limits that tell whether every part of a matrix-core product is
there (tests/test_kv_products.py on the CPU, tests/test_gpu_kv_products.py).

A row sees two keys, one of even dimensions alone and one of odd ones, and its
query has one dimension of each that is not zero: a score is one product of two
full mantissas of its own, and the two scores, about X, differ by 1 at most.  With u = 2^-24 (a rounding of binary32, half a step) and
2 u for each addition inside a matrix instruction, whichever way that rounds,
fp32 caches, three bf16 parts a value (each cut off: the second below 2^-7 of the
value, the third below 2^-15):
 * a score: three products of nine left out, below 2 * 2^-22 + 2^-30, 8 u of it;
   six added, the smallest first: two additions that count, 4 u, the others' sums
   are below 2^-6 of it: 12 * 2^-6 < 1 u.                          13 u
 * the scale times log2 e rounded once, the query by it once:        2 u
   so a weight is off by 15 u S, an output by twice that of A = sum p |v|.
 * w v: products left out 8 u; six additions of two keys' 12 u; the weights' sum
   three additions, 6 u; 2^x to 1 ulp in numerator and denominator, 4 u; the joins
   of four waves' sums (three factors of 0 or 1, additions) and of a prefix and a
   row's own, 4 u; the division and its product 2 u.                 36 u
   |out - ref| <= A u (30 S + 36).
fp16 caches, keys and values as they are, queries in two parts (to 2^-22, 4 u) and
weights in two (cut off, to 2^-20, 16 u, in the sum too):
 * a score: 4 u, two additions 4 u; the scale and the query 2 u:     10 u
 * w v: 2 * 16 u; two additions each of products and weights 8 u; 2^x 4 u; joins 4 u;
   the division 2 u.                                                 50 u
   |out - ref| <= A u (20 S + 50).
First order, S up to 130: the second order is below 2^-10 of it, taken as 1 %.  A third
key and value of zeros (a score of exactly 0) adds its weight to the sum, 2^x to 1 ulp
and an addition: within the joins' 4 u.
"""
import numpy as np

U, D = 2.0 ** -24, 64
LIMITS = {"float32": (30.0, 36.0), "float16": (20.0, 50.0)}


def limit(dtype, size, mass):
    """size [...]: a row's S; mass [...][64]: A."""
    s, v = LIMITS[dtype]
    return 1.01 * U * (s * size[..., None] + v) * mass + 1e-37


def keys(rng, n, n_kv, dtype):
    """Two keys and values of n streams, [2][n][n_kv][64], all bits set at random,
    the second value negative."""
    k, v = (1.0 + rng.random((2, n, n_kv, D)) for _ in range(2))
    k *= rng.choice([-1.0, 1.0], k.shape)
    k[0, ..., 1::2] = k[1, ..., 0::2] = 0.0
    v[1] *= -1.0
    return [x.astype(np.float32).astype(dtype).astype(np.float32) for x in (k, v)]


def queries(rng, k, group, X, scale=0.125):
    """Rows [n][n_kv * group * 64] whose scores with k [2][n][n_kv][64] are about X."""
    n, n_kv = k.shape[1:3]
    q = np.zeros((n, n_kv, group, D), np.float32)
    size = X * rng.uniform(0.8, 1.2, (n, n_kv, group))
    for i in range(2):
        d = 2 * rng.integers(0, D // 2, size.shape) + i
        at = np.take_along_axis(k[i][:, :, None], d[..., None], -1)[..., 0]
        x = (size + i * rng.uniform(-1.0, 1.0, size.shape)) / (scale * at)
        np.put_along_axis(q, d[..., None], x.astype(np.float32)[..., None], -1)
    return q.reshape(n, -1)


# ------------------------------------------------------------------ a model of the products

# (key or value's part, query or weight's part), in the order that they are added
PRODUCTS = {"float32": [(2, 0), (1, 1), (0, 2), (1, 0), (0, 1), (0, 0)],
            "float16": [(0, 1), (0, 0)]}


def cut(x):
    """The leading 8 bits of float32 values."""
    return (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)


def parts(x, dtype, held):
    """held: values of the cache; else queries or weights."""
    x = x.astype(np.float32)
    if dtype == "float32":
        out = []
        for _ in range(3):
            out.append(cut(x))
            x = x - out[-1]
        return out
    if held:
        return [x]
    hi = x.astype(np.float16).astype(np.float32)
    return [hi, (x - hi).astype(np.float16).astype(np.float32)]


def product(a, b, dtype, left_out, acc=np.float32(0.0)):
    """acc + a b as the parts give it, a product left out."""
    pa, pb = parts(a, dtype, True), parts(b, dtype, False)
    for i, (x, y) in enumerate(PRODUCTS[dtype]):
        if i != left_out:
            acc = (acc.astype(np.float64) + pa[x].astype(np.float64) * pb[y]).astype(np.float32)
    return acc


def model(q, k, v, dtype, scores_without=-1, values_without=-1, scale=0.125):
    """One query [m][64] each against two keys and values [2][m][64]."""
    s = (q * np.float32(scale * np.log2(np.e))).astype(np.float32)
    # to [2^14, 2^15), and the weights to 2^14: their lower parts lose nothing
    up = np.exp2(14 - np.floor(np.log2(np.abs(s).max(-1)))).astype(np.float32) if dtype == "float16" \
        else np.ones(len(q), np.float32)
    x = []
    for i in range(2):  # the one product of a score
        d = (np.abs(q) * (k[i] != 0)).argmax(-1)[:, None]
        a, b = (np.take_along_axis(t, d, -1)[:, 0] for t in (k[i], s))
        x.append(product(a, b * up, dtype, scores_without))
    x = np.stack(x)
    e = x / up
    w = np.exp2(e.astype(np.float64) - np.ceil(e.max(0))).astype(np.float32)
    w = w * np.float32(2 ** 14 if dtype == "float16" else 1)
    o = np.zeros(v.shape[1:], np.float32)
    for i in range(2):
        o = product(v[i], np.broadcast_to(w[i][:, None], o.shape).copy(), dtype, values_without, o)
    total = sum(sum(parts(w[i], dtype, False)) for i in range(2))
    return o / total[:, None]


def exact(q, k, v, scale=0.125):
    """The same in binary64, with S and A."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    x = (q * k).sum(-1) * scale
    p = np.exp(x - x.max(0))
    p /= p.sum(0)
    return (p[..., None] * v).sum(0), np.abs(x).max(0), (p[..., None] * np.abs(v)).sum(0)
