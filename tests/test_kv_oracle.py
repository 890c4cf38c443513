"""Pins of the paged cache's oracle (oracle/cbx_kv_oracle.py): plans worked out
by hand, and the attention against torch's over the same keys side by side."""
import numpy as np
import pytest

from oracle import cbx_kv_oracle as KV

torch = pytest.importorskip("torch")


def test_step_plan_by_hand():
    # pages of 16; stream 0 a prefix of 20 positions, streams 1..3 share 20, 7 and none of it
    pool = KV.Pool(4, 4, 16, 8, n_prefix=1, parent=[-1, 0, 0, -1], prefix_len=[0, 20, 7, 0])
    KV.build(pool, n_rows=99, n_new=[20, 16, 3, 0], step=False)
    assert pool.length.tolist() == [20, 16, 3, 0] and pool.n_free == 4
    # the stack's top first: page 7 and 6 to stream 0, 5 to 1, 4 to 2
    assert pool.tables[:, :2].tolist() == [[7, 6], [5, -1], [4, -1], [-1, -1]]
    r = KV.build(pool, n_tiles=2, tile_rows=64, state=[1, 0, 0, 0])
    assert pool.tables[:, :2].tolist() == [[7, 6], [5, 3], [4, -1], [2, -1]]
    assert r["position"].tolist() == [-1, 36, 10, 0]
    assert r["slot"].tolist() == [-1, 3 * 16, 4 * 16 + 3, 2 * 16]
    assert r["row_start"].tolist() == [0, 0, 1, 2, 3]
    assert r["page_start"].tolist() == [0, 0, 1, 1, 2]
    assert r["order"].tolist() == [1, 2, -1, -1]
    assert r["tiles"].tolist() == [[0, 0, 2, 20], [-1, 0, 0, 0]]
    assert r["counts"].tolist() == [3, 1, 2, 0]


def test_refusals_by_hand():
    pool = KV.Pool(4, 2, 16, 3)
    r = KV.build(pool, n_rows=40, n_tiles=9, tile_rows=8, n_new=[33, 20, 1, 17], step=False)
    # 0: past its table; 1: two pages, 20 rows; 2: the third page; 3: no page left
    assert np.diff(r["row_start"]).tolist() == [0, 20, 1, 0]
    assert r["counts"].tolist() == [21, 4, 3, 2]
    assert r["tiles"][:5].tolist() == [[1, 0, 8, 8], [1, 8, 8, 16], [1, 16, 4, 20], [2, 20, 1, 1],
                                       [-1, 0, 0, 0]]
    assert r["stream"][19:23].tolist() == [1, 2, -1, -1]
    # stream 1 gives its pages back, 3 takes them
    r = KV.build(pool, n_rows=40, n_new=[0, 0, 0, 17], release=[0, 1, 0, 0], step=False)
    assert pool.length.tolist() == [0, 0, 1, 17] and pool.n_free == 0
    assert pool.tables[3].tolist() == [1, 2]  # pushed in position order: 2, 1
    # rows past n_rows
    pool = KV.Pool(3, 4, 16, 12)
    r = KV.build(pool, n_rows=30, n_new=[20, 11, 5], step=False)
    assert np.diff(r["row_start"]).tolist() == [20, 0, 0]


@pytest.mark.parametrize("n_kv,group", [(2, 1), (1, 3)])
def test_attention_against_torch(n_kv, group):
    rng = np.random.default_rng(3)
    pool = KV.Pool(3, 5, 16, 14, n_prefix=1, parent=[-1, 0, -1], prefix_len=[0, 21, 0],
                   free=rng.permutation(14))
    KV.build(pool, n_rows=99, n_new=[25, 40, 33], step=False)
    r = KV.build(pool, n_rows=9, n_new=[0, 4, 5], step=False)
    k, v = (rng.standard_normal((14, n_kv, 16, 64)) for _ in range(2))
    q = rng.standard_normal((9, n_kv * group * 64))
    got = KV.attend(pool, k, v, r["stream"], r["position"], q, 0.125)[0]
    for i, rows in ((1, range(0, 4)), (2, range(4, 9))):
        plen = 21 if i == 1 else 0
        slots = [int(pool.tables[0, x // 16]) * 16 + x % 16 for x in range(plen)]
        slots += [int(pool.tables[i, x // 16]) * 16 + x % 16 for x in range(pool.length[i])]
        flat = [torch.from_numpy(c.transpose(0, 2, 1, 3).reshape(-1, n_kv, 64)[slots])
                .permute(1, 0, 2).repeat_interleave(group, 0) for c in (k, v)]
        Q = torch.from_numpy(q[list(rows)]).reshape(len(rows), -1, 64).permute(1, 0, 2)
        mask = torch.arange(len(slots)) <= torch.tensor(r["position"][list(rows)])[:, None]
        want = torch.nn.functional.scaled_dot_product_attention(Q, *flat, attn_mask=mask)
        want = want.permute(1, 0, 2).reshape(len(rows), -1).numpy()
        assert np.abs(got[list(rows)] - want).max() < 1e-12
        # a planted key of another stream shows
        wrong = [c.clone() for c in flat]
        wrong[0][:, 3] += 0.1
        bad = torch.nn.functional.scaled_dot_product_attention(Q, *wrong, attn_mask=mask)
        assert (bad.permute(1, 0, 2).reshape(len(rows), -1) - torch.from_numpy(want)).abs().max() > 1e-4
