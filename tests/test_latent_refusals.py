"""What the operators of the 8-bit latent cache refuse, before anything reaches a GPU."""
import ctypes

import pytest
import torch


class Cache(ctypes.Structure):
    _fields_ = [("latent", ctypes.c_void_p), ("rope", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("n_pages", ctypes.c_int64),
                ("page_size", ctypes.c_int), ("pages", ctypes.c_void_p), ("pages_stride", ctypes.c_int64), ("pages_width", ctypes.c_int64),
                ("n_seqs", ctypes.c_int)]


def _cache(**over):
    values = dict(latent=1024, rope=2048, scale=4096, n_pages=4, page_size=64, pages=8192, pages_stride=2, pages_width=2, n_seqs=2)
    values.update(over)
    return ctypes.byref(Cache(**values))


def _lib():
    from dsv3_b200 import _lib
    i64, vp, ci, f = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    lib = ctypes.CDLL(_lib.LIB_PATH)
    lib.dsv3_latent_write.argtypes = [vp, vp, i64, vp, ci, f, vp, i64, vp, vp, i64, vp]
    lib.dsv3_latent_read.argtypes = [vp, vp, i64, vp, vp, vp]
    lib.dsv3_latent_keep.argtypes = [vp, vp, vp, i64, ci, vp, vp]
    lib.dsv3_latent_attention.argtypes = [vp, vp, i64, i64, vp, i64, i64, i64, ci, vp, vp, vp, f, vp, vp, vp, ctypes.c_size_t, vp]
    lib.dsv3_latent_attention_workspace_bytes.argtypes = [i64, ci, ci, i64]
    lib.dsv3_latent_attention_workspace_bytes.restype = ctypes.c_size_t
    return lib, _lib


def _write(lib, cache, kv=16, stride=576, tokens=1, n_positions=8, weight=16, freqs=16):
    return lib.dsv3_latent_write(cache, kv, stride, weight, 0, 1e-6, freqs, n_positions, 16, 16, tokens, None)


def _attention(lib, cache, q=16, stride=512, tokens=2, heads=1, out=16, cu=None, workspace=None, workspace_bytes=0, tree=None):
    return lib.dsv3_latent_attention(cache, q, stride, stride, q, 64, 64, tokens, heads, 16, cu, tree, 1.0, out, None, workspace, workspace_bytes, None)


@pytest.mark.parametrize("over, status", [
    (dict(page_size=8), "ERR_UNSUPPORTED"), (dict(page_size=48), "ERR_UNSUPPORTED"), (dict(page_size=0), "ERR_INVALID_ARGUMENT"),
    (dict(n_pages=-1), "ERR_INVALID_ARGUMENT"), (dict(n_pages=1 << 25), "ERR_UNSUPPORTED"), (dict(latent=None), "ERR_INVALID_ARGUMENT"),
    (dict(scale=None), "ERR_INVALID_ARGUMENT"), (dict(latent=1032), "ERR_UNSUPPORTED"), (dict(rope=2052), "ERR_UNSUPPORTED")])
def test_caches_that_every_entry_point_refuses(over, status):
    lib, names = _lib()
    want = getattr(names, status)
    assert _write(lib, _cache(**over)) == want
    assert lib.dsv3_latent_read(_cache(**over), 16, 1, 16, 16, None) == want
    assert lib.dsv3_latent_keep(_cache(**over), 16, 16, 4, 4, 16, None) == want
    assert _attention(lib, _cache(**over)) == want


@pytest.mark.parametrize("over", [dict(n_seqs=-1), dict(pages=None), dict(pages_width=-1)])
def test_page_tables_that_are_refused(over):
    lib, names = _lib()
    assert lib.dsv3_latent_read(_cache(**over), 16, 1, 16, 16, None) == names.ERR_INVALID_ARGUMENT
    assert lib.dsv3_latent_keep(_cache(**over), 16, 16, 4, 4, 16, None) == names.ERR_INVALID_ARGUMENT
    assert _attention(lib, _cache(**over)) == names.ERR_INVALID_ARGUMENT


def test_calls_that_are_refused_and_calls_of_nothing():
    lib, names = _lib()
    assert _write(lib, None) == names.ERR_INVALID_ARGUMENT
    assert _write(lib, _cache(), tokens=-1) == names.ERR_INVALID_ARGUMENT
    assert _write(lib, _cache(), kv=None) == names.ERR_INVALID_ARGUMENT
    assert _write(lib, _cache(), kv=24) == names.ERR_UNSUPPORTED
    assert _write(lib, _cache(), stride=580) == names.ERR_UNSUPPORTED
    assert _write(lib, _cache(), weight=24) == names.ERR_UNSUPPORTED
    assert _write(lib, _cache(), weight=None) == names.ERR_INVALID_ARGUMENT
    assert _write(lib, _cache(), freqs=20) == names.ERR_UNSUPPORTED
    assert _write(lib, _cache(), freqs=None) == names.ERR_INVALID_ARGUMENT
    assert _write(lib, _cache(), tokens=0) == names.OK
    assert lib.dsv3_latent_read(_cache(), 16, 1 << 31, 16, 16, None) == names.ERR_UNSUPPORTED
    assert lib.dsv3_latent_read(_cache(), 16, -1, 16, 16, None) == names.ERR_INVALID_ARGUMENT
    assert lib.dsv3_latent_read(_cache(), None, 1, 16, 16, None) == names.ERR_INVALID_ARGUMENT
    assert lib.dsv3_latent_read(_cache(), 16, 1, 24, 16, None) == names.ERR_UNSUPPORTED
    assert lib.dsv3_latent_read(_cache(), 16, 0, 16, 16, None) == names.OK
    assert lib.dsv3_latent_keep(_cache(), 16, 16, 4, -1, 16, None) == names.ERR_INVALID_ARGUMENT
    assert lib.dsv3_latent_keep(_cache(), None, 16, 4, 4, 16, None) == names.ERR_INVALID_ARGUMENT
    assert lib.dsv3_latent_keep(_cache(n_seqs=0), 16, 16, 4, 4, 16, None) == names.OK
    assert _attention(lib, _cache(), tokens=-1) == names.ERR_INVALID_ARGUMENT
    assert _attention(lib, _cache(), q=None) == names.ERR_INVALID_ARGUMENT
    assert _attention(lib, _cache(), tokens=3) == names.ERR_INVALID_ARGUMENT            # do not divide among two sequences
    assert _attention(lib, _cache(), q=24) == names.ERR_UNSUPPORTED
    assert _attention(lib, _cache(), stride=516) == names.ERR_UNSUPPORTED
    assert _attention(lib, _cache(), out=24) == names.ERR_UNSUPPORTED
    assert _attention(lib, _cache(scale=4100)) == names.ERR_UNSUPPORTED
    assert _attention(lib, _cache(n_pages=0)) == names.ERR_INVALID_ARGUMENT
    assert _attention(lib, _cache(n_seqs=0)) == names.ERR_INVALID_ARGUMENT
    assert _attention(lib, _cache(), tokens=130, tree=16) == names.ERR_UNSUPPORTED                        # 65 to a sequence
    assert b"64" in names.lib.dsv3_last_error()
    assert _attention(lib, _cache(pages_width=1 << 20), tokens=1 << 14) == names.ERR_UNSUPPORTED         # 2^14 times 2^19 tiles
    assert _attention(lib, _cache(pages_width=1 << 25)) == names.ERR_UNSUPPORTED
    need = lib.dsv3_latent_attention_workspace_bytes(2, 1, 2, 64 * 64)
    assert need > 0 and lib.dsv3_latent_attention_workspace_bytes(2, 1, 2, 128) == 0     # (one tile: nothing to cut)
    for at, size in ((None, need), (1024, need - 1), (1040, need)):
        assert _attention(lib, _cache(pages_width=64), workspace=at, workspace_bytes=size) == names.ERR_WORKSPACE
    assert _attention(lib, _cache(), heads=1025) == names.ERR_UNSUPPORTED
    assert _attention(lib, _cache(), tokens=0) == names.OK
    assert b"heads" in names.lib.dsv3_last_error()


def _planes(pages=2, page=64):
    import dsv3_b200
    return dsv3_b200.allocate_latent_cache(pages, page, device="cpu")


def test_python_entry_points_refuse_shapes_and_types():
    import dsv3_b200 as d
    c = _planes()
    kv, w = torch.zeros(3, 576, dtype=torch.bfloat16), torch.ones(512, dtype=torch.bfloat16)
    f, at = torch.zeros(8, 32, dtype=torch.complex64), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(AssertionError, match="kv must be"):
        d.latent_cache_write(c, kv[:, :512], w, f, at, at)
    with pytest.raises(AssertionError, match="2-D with contiguous rows"):
        d.latent_cache_write(c, torch.zeros(576, 3, dtype=torch.bfloat16).t(), w, f, at, at)
    with pytest.raises(AssertionError, match="norm"):
        d.latent_cache_write(c, kv, w[:500], f, at, at)
    with pytest.raises(AssertionError, match="freqs_cis"):
        d.latent_cache_write(c, kv, w, f[:, :31], at, at)
    with pytest.raises(AssertionError, match="positions and slots"):
        d.latent_cache_write(c, kv, w, f, at.int(), at)
    with pytest.raises(AssertionError, match="positions and slots"):
        d.latent_cache_write(c, kv, w, f, at, at[:2])
    with pytest.raises(AssertionError, match="a cache is latent"):
        d.latent_cache_write(d.LatentCache(c.latent, c.rope, c.scale[:1]), kv, w, f, at, at)
    with pytest.raises(AssertionError, match="planes of a cache must be contiguous"):
        d.latent_cache_write(d.LatentCache(c.latent[:, ::2], c.rope[:, ::2], c.scale[:, ::2]), kv, w, f, at, at)
    table, cu = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(AssertionError, match="a cache is latent"):
        d.latent_cache_read(d.LatentCache(c.latent[..., :256].contiguous(), c.rope, c.scale), table, cu, 1)
    ql, qr = torch.zeros(2, 4, 512, dtype=torch.bfloat16), torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        d.latent_attention(ql, qr, c, table, cu[:2], 1.0)
    with pytest.raises(TypeError):
        d.latent_attention(ql, None, c, table, cu[:2], 1.0)
    with pytest.raises(ValueError, match="power of two"):
        d.allocate_latent_cache(2, 48, device="cpu")


def test_no_cpu_path():
    import dsv3_b200 as d
    c = _planes()
    kv, w = torch.zeros(3, 576, dtype=torch.bfloat16), torch.ones(512, dtype=torch.bfloat16)
    f, at = torch.zeros(8, 32, dtype=torch.complex64), torch.zeros(3, dtype=torch.int64)
    table, cu = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        d.latent_cache_write(c, kv, w, f, at, at)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        d.latent_cache_read(c, table, cu, 1)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        d.latent_cache_keep(c, table, cu[:2], table, cu[:2])


def test_a_module_whose_cache_would_be_made_in_a_captured_graph(monkeypatch):
    import types
    import dsv3_b200 as d
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    module = types.SimpleNamespace(kv_cache=torch.zeros(2, 70, 512))
    with pytest.raises(RuntimeError, match="captured"):
        d.mla_cache(module)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    cache = d.mla_cache(module)
    assert cache.block_table.tolist() == [[0, 1], [2, 3]] and cache.pool.scale.shape == (4, 64)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert d.mla_cache(module) is cache
