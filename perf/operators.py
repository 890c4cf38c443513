"""The paged key/value cache of the T3 transformer, measured: page tables and slot maps built from
the streams' lengths, attention over the pages, and attention for streams that share a voice's
prompt.

Each case is one pass through one operator.  `own` chooses between the package's calls and the plain
form of the same operator in elementary torch operations; `exact` computes the attention from its
definition in 64 bits.  Inputs are synthetic, made on the GPU from the seed.  A case's lengths are
the same for every seed, in another order, so that its work is known from the case alone.
"""
import importlib.util
import math
import os
import sys

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
own = False

D = 64            # a head's dimensions (every T3 model's)
SCALE = 0.125     # 1 / sqrt(64)
TYPES = {"f32": torch.float32, "f16": torch.float16}
GOLDEN = 0.6180339887498949


def _package():
    """chatterbox.cpp_amd (a dotted directory name: loaded by path)."""
    if "cbx_amd" not in sys.modules:
        d = os.path.join(_ROOT, "chatterbox.cpp_amd")
        spec = importlib.util.spec_from_file_location(
            "cbx_amd", os.path.join(d, "__init__.py"), submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["cbx_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["cbx_amd"]


_handle = []


def _sampler():
    """The one handle that a serving program keeps for all its calls."""
    if not _handle:
        _handle.append(_package().Sampler(device=0, max_vocab=8194, max_history=64))
    return _handle[0]


# ------------------------------------------------------------------ the cases


def listed():
    def tables(name, form, streams, low, high, **kw):
        return dict(dict(name=name, kind="tables", form=form, streams=streams, low=low, high=high,
                         voices=1, voice_low=377, voice_high=377, page=16, gone=0, group=1), **kw)

    def attend(name, form, streams, low, high, **kw):
        return dict(dict(name=name, kind="attend", form=form, streams=streams, low=low, high=high,
                         voices=0, voice_low=0, voice_high=0, page=16, heads=16, kv_heads=16,
                         type="f32", have=0, shared=False), **kw)

    return [
        # a decode step's tables, every step of a 64-stream server: latency
        tables("tables_step_64", "step", 64, 129, 383),
        # 64 requests arrive at once, 5 streams that ended give their pages back
        tables("tables_prompt_64", "prompt", 64, 129, 383, gone=5),
        # a long queue admitted in one call: the largest prompt maps
        tables("tables_prompt_2048", "prompt", 2048, 1, 383, voices=16, voice_low=250,
               voice_high=500, page=32),
        # one stream decoding (latency), the engine's own case
        attend("step_1", "step", 1, 1000, 1000),
        # the 64-stream decode step, fp32 keys as the dense cache holds them
        attend("step_64", "step", 64, 129, 383),
        # long contexts of very different lengths, four query heads to a key head, half the bytes
        attend("step_256_gqa_f16", "step", 256, 64, 4001, heads=16, kv_heads=4, type="f16"),
        # one stream's prompt
        attend("prompt_251", "prompt", 1, 251, 251),
        # a batch of prompts, fp32
        attend("prompt_64", "prompt", 64, 129, 383),
        # long texts behind a voice's prompt, some of each already cached
        attend("prompt_8_voice_f16", "prompt", 8, 301, 1501, voices=1, voice_low=377,
               voice_high=377, have=100, type="f16"),
        # 64 streams of one voice: its prompt (speaker, conditioning tokens) is in the cache once
        attend("shared_64", "step", 64, 1, 300, voices=1, voice_low=377, voice_high=377,
               shared=True),
        # a server's mix of voices, half the bytes
        attend("shared_256_f16", "step", 256, 1, 400, voices=8, voice_low=250, voice_high=500,
               type="f16", page=32, shared=True),
        # many short requests behind one long prompt: the matrix cores' case
        attend("shared_512_long", "step", 512, 1, 64, voices=1, voice_low=2001, voice_high=2001,
               shared=True),
    ]


def _log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    if rng.random() < 0.25:
        form = rng.choice(["step", "prompt"])
        low = _log_int(rng, 1, 200)
        voices = rng.choice([0, 1, rng.randint(2, 16)])
        vlow = rng.randint(1, 400)
        return dict(kind="tables", form=form, streams=_log_int(rng, 1, 2048), low=low,
                    high=low + rng.randint(0, 300), voices=voices,
                    voice_low=vlow if voices else 0,
                    voice_high=vlow + rng.randint(0, 200) if voices else 0,
                    page=rng.choice([16, 32, 64]), gone=rng.randint(0, 9),
                    group=rng.choice([1, 1, 2, 3, 4]))
    form = rng.choice(["step", "step", "prompt"])
    kv_heads, group = rng.choice([(16, 1), (16, 1), (4, 4), (8, 2), (5, 3), (2, 8), (12, 1)])
    voices = rng.choice([0, 1, rng.randint(2, 8)])
    vlow = rng.randint(1, 500)
    low = _log_int(rng, 1, 1000 if form == "step" else 300)
    case = dict(kind="attend", form=form, streams=_log_int(rng, 1, 512), low=low,
                high=low + _log_int(rng, 1, 3000 if form == "step" else 1200), voices=voices,
                voice_low=vlow if voices else 0,
                voice_high=vlow + rng.randint(0, 300) if voices else 0,
                page=rng.choice([16, 16, 32, 64]), heads=kv_heads * group, kv_heads=kv_heads,
                type=rng.choice(["f32", "f16"]),
                have=rng.choice([0, rng.randint(1, 300)]) if form == "prompt" else 0,
                shared=form == "step" and voices > 0 and rng.random() < 0.75)
    most = [work(c) for c in listed()]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while case["streams"] > 1 and any(work(case)[k] > most[k] for k in most):
        case["streams"] = case["streams"] * 2 // 3
    if any(work(case)[k] > most[k] for k in most):
        case["high"] = case["low"]
    return case


def _spread(n, low, high):
    """n lengths over [low, high], the same ones every time (low-discrepancy); logarithmic where
    the range is wider than a factor of ten."""
    u = [((i + 0.5) * GOLDEN) % 1.0 for i in range(n)]
    if high > 10 * low > 0:
        return [min(high, int(low * ((high + 1) / low) ** x)) for x in u]
    return [min(high, low + int((high + 1 - low) * x)) for x in u]


def _lengths(case):
    """(voices' lengths, the streams' lengths, each stream's voice or -1, what each has cached
    before a prompt)."""
    voices = _spread(case["voices"], case["voice_low"], case["voice_high"])
    streams = _spread(case["streams"], case["low"], case["high"])
    of = [i % len(voices) if voices else -1 for i in range(len(streams))]
    have = [(7 * i + case.get("have", 0) // 2) % (case["have"] + 1) if case.get("have") else 0
            for i in range(len(streams))]
    return voices, streams, of, have


def _tile_rows(group):
    """Rows of a tile: 64 (row, query head) pairs of one key head."""
    return max(1, 64 // group)


def work(case):
    voices, streams, of, have = _lengths(case)
    n, page = len(voices) + len(streams), case["page"]
    if case["kind"] == "tables":
        step = case["form"] == "step"
        rows = n if step else _row_room(case)
        pages = (sum(-(-(x + 1) // page) - -(-x // page) for x in streams) if step
                 else sum(-(-x // page) for x in streams))
        tiles = _tiles_of(case, n)
        # lengths, counts, parents and prefixes in, lengths and the two running counts out; an id
        # read and written a page; stream, position and slot a row (prompt form), or position, slot
        # and order
        return dict(bytes=n * 4 * 7 + 8 * pages + 12 * rows + 16 * tiles, flops=0.0)
    es = 4 if case["type"] == "f32" else 2
    h, kvh = case["heads"], case["kv_heads"]
    pre = [voices[v] if v >= 0 else 0 for v in of]
    if case["form"] == "step":
        rows, cached = len(streams), sum(streams)
        pairs = sum(p + x + 1 for p, x in zip(pre, streams))
    else:
        rows, cached = sum(streams), sum(have)
        pairs = sum(x * (p + a) + x * (x + 1) // 2 for p, a, x in zip(pre, have, streams))
    cached += sum(voices[v] for v in set(of) if v >= 0)
    # q and out, the new k and v and where they go, each cached key and value once
    return dict(bytes=rows * D * 4 * 2 * h + rows * D * 2 * kvh * (4 + es) + cached * D * 2 * kvh * es,
                flops=4.0 * D * h * pairs)


# ------------------------------------------------------------------ what a program has in hand


def _row_room(case):
    """Rows that a program's prompt buffers hold: a little more than it needs."""
    return sum(_lengths(case)[1]) * 17 // 16 + 5


def _tiles_of(case, n):
    rows = n if case["form"] == "step" else _row_room(case)
    group = case.get("group") or case["heads"] // case["kv_heads"]
    more = case["voices"] if case["form"] == "step" else n
    return rows // _tile_rows(group) + more


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _empty_streams(g, case, extra):
    """n streams without pages, and a shuffled free list of the pages that they will need and a
    few more."""
    voices, streams, of, have = _lengths(case)
    n, page = len(voices) + len(streams), case["page"]
    longest = max(voices + [a + x + 1 for a, x in zip(have, streams)])
    max_pages = -(-longest // page) + 2
    need = sum(-(-x // page) for x in voices) + sum(-(-(a + x + 1) // page)
                                                    for a, x in zip(have, streams))
    n_pages = need + extra
    return dict(n=n, n_prefix=len(voices), page=page, max_pages=max_pages, n_pages=n_pages,
                tables=torch.full((n, max_pages), -1, dtype=torch.int32, device=DEV),
                length=torch.zeros(n, dtype=torch.int32, device=DEV),
                free=torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32),
                n_free=_ints([n_pages]), parent=_ints([-1] * len(voices) + of),
                prefix_len=_ints([0] * len(voices) + [voices[v] if v >= 0 else 0 for v in of]),
                len_out=torch.zeros(n, dtype=torch.int32, device=DEV), n_free_out=_ints([0]))


def _rows(st, form, n_rows, n_tiles, tile_rows):
    """The buffers of one call's rows."""
    def full(*shape):
        return torch.full(shape, -7, dtype=torch.int32, device=DEV)

    return dict(form=form, n_rows=n_rows, tile_rows=tile_rows, position=full(n_rows),
                slot=full(n_rows), row_start=full(st["n"] + 1), page_start=full(st["n"] + 1),
                counts=full(4), stream=full(n_rows) if form == "prompt" else None,
                tiles=full(n_tiles, 4) if n_tiles else None,
                order=full(n_rows) if form == "step" and n_tiles else None)


def _take(st, n_new):
    """n_new positions more for each stream (the plain form, before the measured call)."""
    rows = _rows(st, "prompt", sum(n_new), 0, 1)
    _plain_build(st, rows, _ints(n_new), None)
    st["length"].copy_(st["len_out"])
    st["n_free"].copy_(st["n_free_out"])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    voices, streams, of, have = _lengths(case)
    order = torch.randperm(len(streams), generator=g, device=DEV).tolist()
    step = case["form"] == "step"
    group = case.get("group") or case["heads"] // case["kv_heads"]
    st = _empty_streams(g, case, 24 + case.get("gone", 0) * 4)
    # this seed's order of the streams (each keeps its voice)
    pick = [len(voices) + i for i in order]
    st["parent"][len(voices):] = st["parent"][pick]
    st["prefix_len"][len(voices):] = st["prefix_len"][pick]
    length = [streams[i] for i in order]
    had = [have[i] for i in order]
    n_new = [0] * len(voices) + ([1] * len(streams) if step else list(length))
    gone = None
    before = voices + (length if step else had)
    if case["kind"] == "tables" and case["gone"]:
        # streams that ended in the call before: 37 positions each, no new rows
        at = [len(voices) + i for i in range(0, len(streams), 9)][:case["gone"]]
        gone = torch.zeros(st["n"], dtype=torch.int32, device=DEV)
        gone[at] = 1
        for i in at:
            before[i], n_new[i] = 37 if st["max_pages"] * st["page"] >= 37 else 1, 0
    _take(st, before)
    s = dict(case=case, st=st, n_new=_ints(n_new), gone=gone)
    if case["kind"] == "tables":
        s["rows"] = _rows(st, case["form"], st["n"] if step else _row_room(case),
                          _tiles_of(case, st["n"]), _tile_rows(group))
        return s
    # the rows' map is built before the call, as once for all layers of a step; tiles only where
    # the call is to share prefixes, or walks prompts
    tiles = _tiles_of(dict(case, low=1), st["n"]) if case["shared"] or not step else 0
    n_rows = st["n"] if step else sum(n_new)
    rows = s["rows"] = _rows(st, case["form"], n_rows, tiles, _tile_rows(group))
    _plain_build(st, rows, s["n_new"], None)
    t = TYPES[case["type"]]
    kvh, h = case["kv_heads"], case["heads"]

    def normal(*shape, sd=1.0):
        return torch.randn(shape, generator=g, device=DEV) * sd

    # pages hold what this and earlier requests left there
    s["k"] = normal(1, st["n_pages"], kvh, st["page"], D).to(t)
    s["v"] = normal(1, st["n_pages"], kvh, st["page"], D).to(t)
    # one product's rows, q | k | v, as the transformer's c_attn gives them
    s["qkv"] = torch.cat([normal(n_rows, h * D, sd=2.0), normal(n_rows, 2 * kvh * D)], dim=1)
    s["out"] = torch.full((n_rows, h * D), 7.0, device=DEV)
    # host numbers that the program knows: the longest context and the most rows of a stream
    pre = [voices[v] if v >= 0 else 0 for v in of]
    s["longest"] = max(p + a + x + 1 for p, a, x in zip(pre, have, streams))
    s["most"] = 1 if step else max(streams)
    return s


# ------------------------------------------------------------------ the plain forms


def _plain_build(st, rows, n_new, gone):
    """Page tables, rows and tiles by cumulative sums and lookups."""
    n, page, cap = st["n"], st["page"], st["max_pages"] * st["page"]
    at = torch.arange(n, device=DEV)
    length, free, n_free = st["length"].long(), st["free"], st["n_free"].long()
    if gone is not None:
        held = torch.where(gone != 0, (length + page - 1) // page, 0)
        back = torch.arange(st["max_pages"], device=DEV)[None] < held[:, None]
        ids = st["tables"][back]
        free[n_free + torch.arange(ids.numel(), device=DEV)] = ids
        n_free = n_free + ids.numel()
        length = torch.where(gone != 0, 0, length)
    asked = n_new.long().clamp(min=0)
    step = rows["form"] == "step"
    if step:
        asked = asked.clamp(max=1)
    want = torch.where(length + asked <= cap, asked, 0)
    want = torch.where(torch.cumsum(want, 0) <= rows["n_rows"], want, 0)
    held = (length + page - 1) // page
    need = (length + want + page - 1) // page - held
    fits = (need == 0) | (torch.cumsum(need, 0) <= n_free)
    count, take = torch.where(fits, want, 0), torch.where(fits, need, 0)
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    row_start = torch.cat([zero, torch.cumsum(count, 0)])
    page_start = torch.cat([zero, torch.cumsum(take, 0)])
    # pages from the top of the stack, in stream order
    t = torch.arange(st["n_pages"], device=DEV)
    t = t[t < page_start[-1]]
    i = torch.searchsorted(page_start[1:], t, right=True)
    st["tables"][i, held[i] + t - page_start[i]] = free[n_free - 1 - t]
    st["len_out"].copy_(length + count)
    st["n_free_out"].copy_(n_free - page_start[-1:])
    child = (at >= st["n_prefix"]) & (st["parent"] >= 0) & (st["parent"] < st["n_prefix"])
    prefix = torch.where(child, st["prefix_len"].long().clamp(0, cap), 0)
    r = torch.arange(rows["n_rows"], device=DEV)
    if step:
        i, off, real = at, length, count > 0
    else:
        real = r < row_start[-1]
        i = torch.searchsorted(row_start[1:], r, right=True).clamp(max=n - 1)
        off = length[i] + r - row_start[i]
        rows["stream"].copy_(torch.where(real, i, -1))
    inside = torch.where(real, off, 0)
    slot = st["tables"][i, inside // page].long() * page + inside % page
    rows["position"].copy_(torch.where(real, prefix[i] + off, -1))
    rows["slot"].copy_(torch.where(real, slot, -1))
    rows["row_start"].copy_(row_start)
    rows["page_start"].copy_(page_start)
    tiles = zero[0]
    if rows["tiles"] is not None:
        T, n_tiles = rows["tile_rows"], rows["tiles"].shape[0]
        t = torch.arange(n_tiles, device=DEV)
        if step:  # rows with a prefix, by prefix; a tile's keys: its longest prefix
            shares = real & (prefix > 0)
            key = torch.where(shares, st["parent"].long(), n)
            by = torch.sort(key, stable=True)
            rows["order"].copy_(torch.where(by.values < n, by.indices, -1))
            size = torch.zeros(n + 1, dtype=torch.int64, device=DEV).scatter_add_(
                0, key, torch.ones_like(key))[:n]
        else:
            size = count
        first = torch.cat([zero, torch.cumsum(size, 0)])
        begin = torch.cat([zero, torch.cumsum((size + T - 1) // T, 0)])
        k = torch.searchsorted(begin[1:], t, right=True).clamp(max=n - 1)
        used = t < begin[-1]
        f = first[k] + (t - begin[k]) * T
        c = torch.minimum(first[k] + size[k] - f, torch.full_like(f, T))
        if step:
            j = (f[:, None] + torch.arange(T, device=DEV)).clamp(max=n - 1)
            inside = torch.arange(T, device=DEV) < c[:, None]
            keys = torch.where(inside, prefix[by.indices[j.clamp(min=0)]], 0).amax(1)
        else:
            keys = prefix[k] + length[k] + f - first[k] + c
        tile = torch.stack([k, f, c, keys], 1)
        empty = torch.tensor([-1, 0, 0, 0], device=DEV)
        rows["tiles"].copy_(torch.where(used[:, None], tile, empty))
        tiles = begin[-1]
    refused = ((asked > 0) & (count == 0)).sum()
    rows["counts"].copy_(torch.stack([row_start[-1], tiles, page_start[-1], refused]))


def _built(s):
    st, rows = s["st"], s["rows"]
    out = dict(tables=st["tables"], free=st["free"], length=st["len_out"], n_free=st["n_free_out"])
    out.update({k: rows[k] for k in ("stream", "position", "slot", "row_start", "page_start",
                                     "tiles", "order", "counts") if rows[k] is not None})
    return out


def _plain_attend(s):
    """New keys and values to their slots, then every stream's keys gathered side by side, its rows
    against them in one batched product, the softmax by maximum, exponentials and sum."""
    case, st, rows, page = s["case"], s["st"], s["rows"], s["st"]["page"]
    h, kvh, n, first = case["heads"], case["kv_heads"], st["n"], st["n_prefix"]
    group, k, v = h // kvh, s["k"][0], s["v"][0]
    q, kn, vn = s["qkv"].split([h * D, kvh * D, kvh * D], dim=1)
    slot = rows["slot"].long()
    real = slot >= 0
    at = slot[real]
    k[at // page, :, at % page] = kn[real].reshape(-1, kvh, D).to(k.dtype)
    v[at // page, :, at % page] = vn[real].reshape(-1, kvh, D).to(v.dtype)
    # streams with rows (prefixes have none), their keys at [0, longest)
    j = torch.arange(s["longest"], device=DEV)
    prefix = torch.where(st["parent"] >= 0, st["prefix_len"], 0).long()[first:, None]
    mine = j - prefix
    tables = st["tables"].long().clamp(min=0)
    theirs = tables[st["parent"].long().clamp(min=0)[first:]]
    last = st["max_pages"] - 1
    ids = torch.where(mine < 0, theirs[:, (j // page).clamp(max=last)],
                      tables[first:].gather(1, (mine.clamp(min=0) // page).clamp(max=last)))
    off = torch.where(mine < 0, j, mine) % page
    K = k[ids, :, off].float().permute(0, 2, 3, 1).contiguous()   # [n, kvh, D, longest]
    V = v[ids, :, off].float().permute(0, 2, 1, 3).contiguous()   # [n, kvh, longest, D]
    R = s["most"]
    if case["form"] == "step":
        r = torch.arange(first, n, device=DEV)[:, None]
        live = real[first:, None]
    else:
        start = rows["row_start"].long()
        r = start[first:n, None] + torch.arange(R, device=DEV)
        live = r < start[first + 1:n + 1, None]
        r = r.clamp(max=rows["n_rows"] - 1)
    Q = (q[r] * SCALE).reshape(n - first, R, kvh, group, D).permute(0, 2, 3, 1, 4)
    Q = Q.reshape(n - first, kvh, group * R, D)
    score = (Q @ K).reshape(n - first, kvh, group, R, -1)
    seen = (j <= rows["position"].long()[r][..., None]) & live[..., None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    V = torch.where((j <= rows["position"].long()[r].amax(1, keepdim=True))[:, None, :, None], V, 0.0)
    o = (p.reshape(n - first, kvh, group * R, -1) @ V).reshape(n - first, kvh, group, R, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n - first, R, h * D)
    s["out"].zero_()
    s["out"][r[live]] = o[live]


# ------------------------------------------------------------------ one pass


def _bind(s):
    """The structures of device addresses that a program fills once for its buffers."""
    S, st, rows, case = _package().Sampler, s["st"], s["rows"], s["case"]
    streams = S.kv_streams(st["tables"], st["length"], st["free"], st["n_free"],
                           n_prefix=st["n_prefix"], parent=st["parent"],
                           prefix_len=st["prefix_len"])
    r = S.kv_rows(rows["position"], rows["slot"], rows["row_start"], rows["page_start"],
                  rows["counts"], stream=rows["stream"], tiles=rows["tiles"], order=rows["order"],
                  tile_rows=rows["tile_rows"])
    if case["kind"] == "tables":
        return S.kv_plan(streams, r, page_size=st["page"], n_new=s["n_new"], release=s["gone"],
                         len_out=st["len_out"], n_free_out=st["n_free_out"])
    q, k, v = s["qkv"].split([case["heads"] * D, case["kv_heads"] * D, case["kv_heads"] * D], dim=1)
    return S.kv_attn(S.kv_cache(s["k"], s["v"]), streams, r, q, s["out"], layer=0, k=k, v=v,
                     scale=SCALE)


def run(state):
    tables = state["case"]["kind"] == "tables"
    if own:
        if "bound" not in state:
            state["bound"] = _bind(state)
        if tables:
            _sampler().kv_build(state["bound"])
        else:
            _sampler().kv_attend(state["bound"])
    elif tables:
        _plain_build(state["st"], state["rows"], state["n_new"], state["gone"])
    else:
        _plain_attend(state)
    return _built(state) if tables else dict(out=state["out"], k=state["k"], v=state["v"])


# ------------------------------------------------------------------ the definition, in 64 bits


def exact(case, seed):
    """Stream by stream: softmax(scale q K^T) V over the positions each row sees, in float64."""
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    st, rows, page = s["st"], s["rows"], s["st"]["page"]
    h, kvh = case["heads"], case["kv_heads"]
    slot = rows["slot"].tolist()
    at = torch.tensor([x for x in slot if x >= 0], device=DEV)
    src = torch.tensor([r for r, x in enumerate(slot) if x >= 0], device=DEV)
    new = s["qkv"][src]
    cache = []
    for name, c in (("k", new[:, h * D:(h + kvh) * D]), ("v", new[:, (h + kvh) * D:])):
        flat = s[name][0].transpose(1, 2).reshape(-1, kvh, D).clone()  # by slot
        flat[at] = c.reshape(-1, kvh, D).to(flat.dtype)
        cache.append(flat)
    start, tables = rows["row_start"].tolist(), st["tables"].tolist()
    parent, prefix = st["parent"].tolist(), st["prefix_len"].tolist()
    pos = rows["position"].tolist()
    out = torch.zeros((rows["n_rows"], h * D), dtype=torch.float64, device=DEV)
    for i in range(st["n_prefix"], st["n"]):
        mine = [i] if case["form"] == "step" else range(start[i], start[i + 1])
        mine = [r for r in mine if pos[r] >= 0]
        if not mine:
            continue
        shared = prefix[i] if parent[i] >= 0 else 0
        keys = [tables[parent[i]][x // page] * page + x % page for x in range(shared)]
        keys += [tables[i][x // page] * page + x % page for x in range(pos[mine[-1]] + 1 - shared)]
        keys = torch.tensor(keys, device=DEV)
        K, V = (c[keys].double().permute(1, 0, 2).repeat_interleave(h // kvh, 0) for c in cache)
        Q = s["qkv"][mine[0]:mine[-1] + 1, :h * D].double().reshape(-1, h, D).permute(1, 0, 2)
        a = torch.matmul(Q.contiguous(), K.transpose(1, 2).contiguous()) * SCALE
        see = torch.tensor([pos[r] for r in mine], device=DEV)
        a = a.masked_fill(torch.arange(len(keys), device=DEV) > see[:, None], -math.inf)
        o = torch.matmul(torch.softmax(a, -1), V.contiguous())
        out[mine[0]:mine[-1] + 1] = o.permute(1, 0, 2).reshape(len(mine), h * D)
    k, v = (c.reshape(-1, page, kvh, D).transpose(1, 2)[None] for c in cache)
    return dict(out=out, k=k, v=v)
