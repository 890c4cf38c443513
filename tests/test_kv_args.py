"""Refusals of the paged cache's entry points.  CPU only: the C ABI's checks
fail before any HIP call (the handle is memory that no check reads), and the
Python view raises ValueError before the library is called."""
import ctypes

import pytest

import pkg

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    mod = pkg.load()
    return mod, mod.load_library(), ctypes.create_string_buffer(4096)


def streams(mod, **kw):
    t = mod.KvStreams()
    t.n_streams, t.n_prefix, t.max_pages, t.n_pages = 4, 1, 8, 20
    for f in ("tables", "len", "free_pages", "n_free", "parent", "prefix_len"):
        setattr(t, f, 4096)
    for f, x in kw.items():
        setattr(t, f, x)
    return t


def rows(mod, step=True, **kw):
    r = mod.KvRows()
    r.n_rows = 4 if step else 100
    r.tile_rows, r.n_tiles = 64, 2 if step else 5
    for f in ("position", "slot", "row_start", "page_start", "counts", "tiles", "order"):
        setattr(r, f, 4096)
    r.stream = None if step else 4096
    for f, x in kw.items():
        setattr(r, f, x)
    return r


def cache(mod, **kw):
    c = mod.KvCache()
    c.k = c.v = 4096
    c.type, c.n_layer, c.n_pages, c.n_head, c.page_size = 0, 2, 20, 3, 16
    for f, x in kw.items():
        setattr(c, f, x)
    return c


def refused(mod, rc, code=None):
    assert rc == (mod.CBX_ERR_INVALID if code is None else code)
    assert mod._lib.cbx_last_error()


SHARED = [
    dict(t=dict(n_streams=0)), dict(t=dict(n_streams=16385), r=dict(n_rows=16385)),
    dict(t=dict(n_prefix=-1)), dict(t=dict(n_prefix=5)), dict(t=dict(max_pages=0)),
    dict(t=dict(max_pages=1 << 26)), dict(t=dict(n_pages=0)), dict(t=dict(n_pages=1 << 27)),
    dict(t=dict(tables=None)), dict(t=dict(prefix_len=None)), dict(r=dict(n_rows=0)),
    dict(r=dict(n_rows=5)), dict(r=dict(position=None)), dict(r=dict(slot=None)),
    dict(r=dict(row_start=None)), dict(r=dict(order=None)), dict(r=dict(tiles=4100)),
    dict(r=dict(tile_rows=0)), dict(r=dict(n_tiles=0)),
    dict(step=False, r=dict(n_tiles=4)),   # 100 rows in tiles of 64 from 4 streams: 5
    dict(step=False, r=dict(n_rows=-1)),
]


@pytest.mark.parametrize("bad", SHARED + [
    dict(page=8), dict(page=24), dict(page=512), dict(t=dict(len=None)),
    dict(t=dict(free_pages=None)), dict(t=dict(n_free=None)), dict(r=dict(page_start=None)),
    dict(r=dict(counts=None)), dict(p=dict(len_out=4096)), dict(p=dict(n_free_out=4096))])
def test_build_refuses(lib, bad):
    mod, so, handle = lib
    t, r = streams(mod, **bad.get("t", {})), rows(mod, bad.get("step", True), **bad.get("r", {}))
    p = mod.KvPlan()
    p.streams, p.rows, p.page_size = ctypes.pointer(t), ctypes.pointer(r), bad.get("page", 16)
    for f, x in bad.get("p", {}).items():
        setattr(p, f, x)
    refused(mod, so.cbx_kv_build(handle, ctypes.byref(p), None))


def test_null_arguments(lib):
    mod, so, handle = lib
    p, a = mod.KvPlan(), mod.KvAttn()
    refused(mod, so.cbx_kv_build(None, ctypes.byref(p), None))
    refused(mod, so.cbx_kv_build(handle, None, None))
    refused(mod, so.cbx_kv_build(handle, ctypes.byref(p), None))
    refused(mod, so.cbx_kv_attend(None, ctypes.byref(a), None))
    refused(mod, so.cbx_kv_attend(handle, None, None))
    refused(mod, so.cbx_kv_attend(handle, ctypes.byref(a), None))
    assert so.cbx_kv_workspace_bytes(None) == 0 and so.cbx_kv_workspace_bytes(ctypes.byref(a)) == 0


def attn(mod, bad):
    c = cache(mod, **bad.get("c", {}))
    t, r = streams(mod, **bad.get("t", {})), rows(mod, bad.get("step", True), **bad.get("r", {}))
    a = mod.KvAttn()
    a.cache, a.streams, a.rows = (ctypes.pointer(x) for x in (c, t, r))
    a.layer, a.n_head, a.scale = 1, 3, 0.125
    a.q, a.ld_q, a.k, a.v, a.ld_kv, a.out, a.ld_out = 4096, 576, 4096, 4096, 576, 4096, 192
    for f, x in bad.get("a", {}).items():
        setattr(a, f, x)
    a._keep = (c, t, r)
    return a


@pytest.mark.parametrize("bad", SHARED + [
    dict(c=dict(page_size=8)), dict(c=dict(type=2)), dict(c=dict(k=None)), dict(c=dict(v=None)),
    dict(c=dict(n_layer=0)), dict(c=dict(n_pages=21)), dict(a=dict(layer=2)),
    dict(a=dict(layer=-1)), dict(a=dict(q=None)), dict(a=dict(out=None)), dict(a=dict(v=None)),
    dict(a=dict(k=None)), dict(a=dict(ld_q=188)), dict(a=dict(ld_q=577)), dict(a=dict(ld_out=190)),
    dict(a=dict(ld_out=128)), dict(a=dict(ld_kv=128)), dict(a=dict(ld_kv=193)),
    dict(a=dict(q=4100)), dict(a=dict(k=4104)), dict(a=dict(out=4097)), dict(c=dict(v=4098)),
    dict(a=dict(workspace=4100)), dict(r=dict(tile_rows=32, n_tiles=9)),
    dict(step=False, r=dict(tiles=None)),
    dict(),                                  # a step with tiles and no workspace
    dict(a=dict(workspace=4096, workspace_bytes=1000)),
])
def test_attend_refuses(lib, bad):
    mod, so, handle = lib
    refused(mod, so.cbx_kv_attend(handle, ctypes.byref(attn(mod, bad)), None))


@pytest.mark.parametrize("bad", [dict(a=dict(n_head=4)), dict(a=dict(n_head=0)),
                                 dict(a=dict(n_head=195, ld_q=195 * 64, ld_out=195 * 64)),
                                 dict(c=dict(n_pages=1 << 26, n_head=4), t=dict(n_pages=1 << 26))])
def test_attend_unsupported(lib, bad):
    mod, so, handle = lib
    refused(mod, so.cbx_kv_attend(handle, ctypes.byref(attn(mod, bad)), None),
            mod.CBX_ERR_UNSUPPORTED)


def test_tile_rows_and_workspace(lib):
    mod, so, _ = lib
    assert [mod.Sampler.kv_tile_rows(*x) for x in ((16, 16), (12, 4), (15, 3), (64, 1), (70, 1))] \
        == [64, 21, 12, 1, 1]
    assert mod.Sampler.kv_tile_rows(2, 3) == 0 and mod.Sampler.kv_tile_rows(2, 0) == 0
    a = attn(mod, {})
    assert so.cbx_kv_workspace_bytes(ctypes.byref(a)) > 4 * 3 * 65 * 4
    a = attn(mod, dict(step=False))
    assert so.cbx_kv_workspace_bytes(ctypes.byref(a)) == 0  # prompts' rows are whole


def test_grids_stay_within_a_launch(lib):
    """Rows, tiles and the parts of both in one launch: 2^24 - 1 workgroups at most."""
    mod, so, handle = lib
    n, pages = 16384, (1 << 26) - 1  # 2^30 positions a stream, near enough: 64 parts a row are wanted
    a = attn(mod, dict(t=dict(n_streams=n, n_prefix=1, max_pages=pages), r=dict(n_rows=n, n_tiles=n),
                       a=dict(n_head=960, ld_q=960 * 64, ld_kv=320 * 64, ld_out=960 * 64),
                       c=dict(n_head=320)))
    a._keep[2].tile_rows = mod.Sampler.kv_tile_rows(960, 320)
    assert n * 960 + n * 320 > 0xffffff
    refused(mod, so.cbx_kv_attend(handle, ctypes.byref(a), None), mod.CBX_ERR_UNSUPPORTED)
    assert so.cbx_kv_workspace_bytes(ctypes.byref(a)) == 0
    a.n_head, a._keep[0].n_head, a._keep[2].n_tiles = 192, 64, 1024
    a._keep[2].tile_rows = mod.Sampler.kv_tile_rows(192, 64)
    parts = so.cbx_kv_workspace_bytes(ctypes.byref(a)) // (n * 192 * (64 * 4 + 8))
    assert parts >= 2
    shared = 1  # 1024 tiles of 64 key heads fill the card with a part each
    assert 1024 * 64 * shared + (parts - shared) * n * 64 <= 0xffffff


def z(*s, dt=torch.int32):
    return torch.zeros(s, dtype=dt)


def view(mod, step=True):
    S = mod.Sampler
    f = torch.float32
    c = S.kv_cache(z(2, 20, 3, 16, 64, dt=f), z(2, 20, 3, 16, 64, dt=f))
    t = S.kv_streams(z(4, 8), z(4), z(20), z(1), n_prefix=1, parent=z(4), prefix_len=z(4))
    r = S.kv_rows(z(4), z(4), z(5), z(5), z(4), tiles=z(2, 4), order=z(4), tile_rows=64)
    return S, c, t, r


def test_python_view_refuses(lib):
    mod = lib[0]
    S, c, t, r = view(mod)
    f = torch.float32
    with pytest.raises(ValueError):
        S.kv_cache(z(2, 20, 3, 16, 64, dt=torch.bfloat16), z(2, 20, 3, 16, 64, dt=torch.bfloat16))
    with pytest.raises(ValueError):  # another head dimension
        S.kv_cache(z(2, 20, 3, 16, 128, dt=f), z(2, 20, 3, 16, 128, dt=f))
    with pytest.raises(ValueError):
        S.kv_cache(z(2, 20, 3, 16, 64, dt=f), z(2, 21, 3, 16, 64, dt=f))
    with pytest.raises(ValueError):  # parent without prefix_len
        S.kv_streams(z(4, 8), z(4), z(20), z(1), parent=z(4))
    with pytest.raises(ValueError):
        S.kv_streams(z(4, 8), z(5), z(20), z(1))
    with pytest.raises(ValueError):
        S.kv_streams(z(4, 8).long(), z(4), z(20), z(1))
    with pytest.raises(ValueError):
        S.kv_rows(z(4), z(5), z(5), z(5), z(4))
    with pytest.raises(ValueError):
        S.kv_rows(z(4), z(4), z(5), z(5), z(4), tiles=z(2, 3))
    with pytest.raises(ValueError):
        S.kv_plan(t, r, page_size=16, n_new=z(3))
    short = S.kv_rows(z(4), z(4), z(4), z(4), z(4))
    with pytest.raises(ValueError):  # row_start for another number of streams
        S.kv_plan(t, short, page_size=16)
    q, o = z(4, 192, dt=f), z(4, 192, dt=f)
    for bad in (dict(q=z(4, 100, dt=f), out=z(4, 100, dt=f)), dict(q=q, out=z(4, 128, dt=f)),
                dict(q=q.half(), out=o), dict(q=z(192, 4, dt=f).t(), out=o),
                dict(q=q, out=o, k=z(4, 192, dt=f)),
                dict(q=q, out=o, k=z(4, 192, dt=f), v=z(4, 576, dt=f)[:, :192]),
                dict(q=q, out=o, k=z(4, 128, dt=f), v=z(4, 128, dt=f))):
        with pytest.raises(ValueError):
            S.kv_attn(c, t, r, bad.pop("q"), bad.pop("out"), **bad)
    S.kv_attn(c, t, r, q, o, k=z(4, 192, dt=f), v=z(4, 192, dt=f))


def test_host_tensors_are_refused(lib):
    """Structures over host memory are made (their shapes are checked) and not run."""
    mod, so, _ = lib
    S, c, t, r = view(mod)
    s = object.__new__(S)
    s.lib, s.handle, s.device = so, None, 0
    with pytest.raises(ValueError, match="GPU 0"):
        s.kv_build(S.kv_plan(t, r, page_size=16))
    q = z(4, 192, dt=torch.float32)
    with pytest.raises(ValueError, match="GPU 0"):
        s.kv_attend(S.kv_attn(c, t, r, q, torch.empty_like(q)))
    with pytest.raises(ValueError, match="GPU 0"):
        s.t3_kv(mod.T3Model(), c, t, r, q, tokens=z(4))


def test_prompts_without_a_list_of_tiles(lib):
    """NULL tiles and n_tiles 0: found from row_start, as many as a list would
    have (n_rows / tile_rows + n_streams) within a launch's limit; the Python view
    leaves out a list that is too short, and no other."""
    mod, so, handle = lib
    a = attn(mod, dict(step=False, r=dict(tiles=None, n_tiles=0, tile_rows=0, n_rows=10),
                       t=dict(n_streams=16384), c=dict(n_head=1024, n_pages=20),
                       a=dict(n_head=1024, ld_q=65536, ld_kv=65536, ld_out=65536)))
    assert 10 * 1024 + 16384 * 1024 > 0xffffff
    refused(mod, so.cbx_kv_attend(handle, ctypes.byref(a), None), mod.CBX_ERR_UNSUPPORTED)
    S, c, t, _ = view(mod)
    q = z(100, 192, dt=torch.float32)
    for n_tiles, tile_rows, kept in ((5, 64, True), (4, 64, False), (1, 64, False), (6, 64, True),
                                     (4, 0, True)):
        r = S.kv_rows(z(100), z(100), z(5), z(5), z(4), stream=z(100), tiles=z(n_tiles, 4),
                      tile_rows=tile_rows)
        got = S.kv_attn(c, t, r, q, torch.empty_like(q)).rows.contents
        assert (got.n_tiles, bool(got.tiles)) == ((n_tiles, True) if kept else (0, False))
        assert (r.n_tiles, bool(r.tiles)) == (n_tiles, True) and got.position == r.position


@pytest.mark.parametrize("step", [True, False])
@pytest.mark.parametrize("tile_rows", [65, 2 ** 31 - 1])
def test_tiles_of_more_than_64_rows_are_refused(lib, step, tile_rows):
    """No attention takes them, and rows + tile_rows passes 32 bits in the plan."""
    mod, so, handle = lib
    t, r = streams(mod), rows(mod, step, tile_rows=tile_rows)
    p = mod.KvPlan()
    p.streams, p.rows, p.page_size = ctypes.pointer(t), ctypes.pointer(r), 16
    refused(mod, so.cbx_kv_build(handle, ctypes.byref(p), None))
