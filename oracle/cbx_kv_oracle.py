"""CPU oracle of the paged cache -- test infrastructure only (imported by tests/
and nothing else; the product is chatterbox.cpp_amd/csrc/cbx_kv_plan.hip and
cbx_kv_attn.hip behind include/cbx_kv.h).

`build` restates cbx_kv_build's rules one stream at a time in Python integers;
`attend` the attention in binary64, one row and head at a time.  Pinned by
tests/test_kv_oracle.py: plans worked out by hand, and the attention of a paged
cache against torch's scaled_dot_product_attention over the same keys laid side
by side.
"""
import numpy as np

D = 64


class Pool:
    """A pool's state: tables [n][max_pages], length [n], the stack free[0,
    n_free), prefixes [0, n_prefix), parent and prefix_len [n]."""

    def __init__(self, n, max_pages, page, n_pages, n_prefix=0, parent=None, prefix_len=None,
                 free=None):
        self.n, self.max_pages, self.page, self.n_prefix = n, max_pages, page, n_prefix
        self.tables = np.full((n, max_pages), -1, np.int32)
        self.length = np.zeros(n, np.int32)
        self.free = np.arange(n_pages, dtype=np.int32) if free is None else np.array(free, np.int32)
        self.n_free = n_pages
        self.parent = np.full(n, -1, np.int32) if parent is None else np.array(parent, np.int32)
        self.prefix_len = (np.zeros(n, np.int32) if prefix_len is None
                           else np.array(prefix_len, np.int32))

    def prefix(self, i):
        """(the prefix's stream, positions shared) of stream i; (-1, 0): none."""
        p = int(self.parent[i])
        if i < self.n_prefix or not 0 <= p < self.n_prefix:
            return -1, 0
        return p, int(min(max(self.prefix_len[i], 0), self.max_pages * self.page))


def build(pool, n_rows=None, n_tiles=0, tile_rows=1, n_new=None, state=None, release=None,
          step=True):
    """One plan applied to the pool; returns the call's rows as a dict of the
    arrays that cbx_kv_rows holds."""
    n, page, cap = pool.n, pool.page, pool.max_pages * pool.page
    n_pages = len(pool.free)
    n_rows = n if step else n_rows
    up = lambda x: -(-x // page)
    for i in range(n):
        if release is not None and release[i] != 0 and 0 <= pool.length[i] <= cap:
            for j in range(up(int(pool.length[i]))):
                if pool.n_free < n_pages:
                    pool.free[pool.n_free] = pool.tables[i, j]
                    pool.n_free += 1
            pool.length[i] = 0
    rows_asked = pages_needed = refused = 0
    start, pstart, entries, top = [0], [0], [], pool.n_free
    for i in range(n):
        have = int(pool.length[i])
        ask = 1 if n_new is None else max(int(n_new[i]), 0)
        if state is not None and state[i] != 0:
            ask = 0
        if step:
            ask = min(ask, 1)
        want = ask if 0 <= have <= cap and have + ask <= cap else 0
        rows_asked += want
        if not step and rows_asked > n_rows:
            want = 0
        need = up(have + want) - up(have) if want else 0
        pages_needed += need
        if need and pages_needed > top:
            want = need = 0
        refused += ask > 0 and want == 0
        for j in range(need):
            pool.n_free -= 1
            pool.tables[i, up(have) + j] = pool.free[pool.n_free]
        pre = pool.prefix(i)[1]
        for x in range(have, have + want):
            pg = int(pool.tables[i, x // page])
            entries.append((i, pre + x, pg * page + x % page if 0 <= pg < n_pages else -1))
        start.append(start[-1] + want)
        pstart.append(pstart[-1] + need)
        pool.length[i] = have + want
    i32 = lambda a: np.array(a, np.int32)
    out = dict(row_start=i32(start), page_start=i32(pstart))
    position, slot = np.full(n_rows, -1, np.int32), np.full(n_rows, -1, np.int32)
    if step:
        for i, p, s in entries:
            position[i], slot[i] = p, s
    else:
        stream = np.full(n_rows, -1, np.int32)
        for r, e in enumerate(entries):
            stream[r], position[r], slot[r] = e
        out["stream"] = stream
    tiles = []
    if n_tiles and step:
        groups = {}
        for i, _, _ in entries:
            p, plen = pool.prefix(i)
            if plen > 0:
                groups.setdefault(p, []).append(i)
        order = []
        for p in sorted(groups):
            for f in range(0, len(groups[p]), tile_rows):
                part = groups[p][f:f + tile_rows]
                tiles.append((p, len(order), len(part), max(pool.prefix(i)[1] for i in part)))
                order += part
        out["order"] = i32(order + [-1] * (n - len(order)))
    elif n_tiles:
        for i in range(n):
            for f in range(start[i], start[i + 1], tile_rows):
                e = min(f + tile_rows, start[i + 1])
                tiles.append((i, f, e - f, int(position[e - 1]) + 1))
    if n_tiles:
        out["tiles"] = i32(tiles + [(-1, 0, 0, 0)] * (n_tiles - len(tiles)))
    out.update(position=position, slot=slot,
               counts=i32([start[-1], len(tiles), pstart[-1], refused]))
    return out


def keys_of(pool, i, last):
    """Cache rows (page, place) of positions [0, last] of stream i; None where
    the page is not one of the pool's or the stream has no such place."""
    p, plen = pool.prefix(i)
    n_pages, found = len(pool.free), []
    for j in range(last + 1):
        who, x = (p, j) if j < plen else (i, j - plen)
        pg = int(pool.tables[who, x // pool.page]) if x // pool.page < pool.max_pages else -1
        found.append((pg, x % pool.page) if 0 <= pg < n_pages else None)
    return found


def attend(pool, k, v, stream, position, q, scale):
    """Rows' attention over k, v [n_pages][n_kv][page][64] (the new rows already
    stored), q [n_rows][n_head * 64].  Returns out, and for each row and head
    what an error bound needs: the largest sum |q||k| scale, sum p |v| (both
    [n_rows][n_head], [n_rows][n_head][64]) and the number of keys."""
    n_rows, n_kv = len(position), k.shape[1]
    H = q.shape[1] // D
    out = np.zeros((n_rows, H, D))
    size, mass = np.zeros((n_rows, H)), np.zeros((n_rows, H, D))
    n_keys = np.zeros(n_rows, np.int64)
    memo = {}
    for r in range(n_rows):
        i, pos = int(stream[r]), int(position[r])
        if i < 0 or pos < 0:
            continue
        if i not in memo or len(memo[i]) <= pos:
            memo[i] = keys_of(pool, i, max(pos, max([int(position[x]) for x in range(n_rows)
                                                     if stream[x] == i])))
        at = [x for x in memo[i][:pos + 1] if x is not None]
        n_keys[r] = len(at)
        if not at:
            continue
        pg, off = np.array(at).T
        K, V = k[pg, :, off].astype(np.float64), v[pg, :, off].astype(np.float64)
        for h in range(H):
            kh, vh = K[:, h // (H // n_kv)], V[:, h // (H // n_kv)]
            qh = q[r, h * D:(h + 1) * D].astype(np.float64)
            x = kh @ qh * scale
            top = x.max()
            if top == -np.inf:
                continue
            e = np.exp(x - top)
            p = e / e.sum()
            out[r, h] = p @ vh
            size[r, h] = (np.abs(kh) @ np.abs(qh)).max() * abs(scale)
            mass[r, h] = p @ np.abs(vh)
    return out.reshape(n_rows, H * D), size, mass, n_keys
