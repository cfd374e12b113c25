"""What the operators of expanded attention, its parts and rotary positions refuse, before anything reaches a GPU."""
import ctypes

import pytest
import torch

i64, vp, ci, f32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float


class Args(ctypes.Structure):
    _fields_ = [("q_nope", vp), ("q_nope_token", i64), ("q_nope_head", i64), ("q_rope", vp), ("q_rope_token", i64), ("q_rope_head", i64),
                ("k_nope", vp), ("k_nope_token", i64), ("k_nope_head", i64), ("k_rope", vp), ("k_rope_token", i64), ("v", vp), ("v_token", i64), ("v_head", i64),
                ("tokens", i64), ("kv_tokens", i64), ("heads", ci), ("n_seqs", ci), ("cu_q", vp), ("cu_k", vp), ("causal", ci), ("scale", f32), ("out", vp), ("lse", vp)]


def _lib():
    from dsv3_b200 import _lib
    lib = ctypes.CDLL(_lib.LIB_PATH)
    lib.dsv3_expanded_attention.argtypes = [vp, vp, ctypes.c_size_t, vp]
    lib.dsv3_expanded_attention_workspace_bytes.argtypes = [i64, i64, ci, ci, ci, ci]
    lib.dsv3_expanded_attention_workspace_bytes.restype = ctypes.c_size_t
    lib.dsv3_attention_join.argtypes = [vp, vp, ci, i64, ci, vp, vp, vp]
    lib.dsv3_rotary_table.argtypes = [ci, ctypes.c_double, ctypes.c_double, i64, ctypes.c_double, ctypes.c_double, i64, i64, vp, vp]
    lib.dsv3_rotary.argtypes = [vp, i64, i64, vp, i64, i64, ci, i64, ci, ci, vp, i64, vp, i64, ci, ci, ci, ci, vp]
    return lib, _lib


def _args(**over):
    values = dict(q_nope=1024, q_nope_token=384, q_nope_head=192, q_rope=2048, q_rope_token=128, q_rope_head=64, k_nope=4096, k_nope_token=512, k_nope_head=256, k_rope=8192,
                  k_rope_token=64, v=16384, v_token=512, v_head=256, tokens=8, kv_tokens=8, heads=2, n_seqs=1, cu_q=None, cu_k=None, causal=1, scale=0.1, out=32768, lse=None)
    values.update(over)
    return ctypes.byref(Args(**values))


@pytest.mark.parametrize("over, status", [
    (dict(tokens=-1), "ERR_INVALID_ARGUMENT"), (dict(kv_tokens=-1), "ERR_INVALID_ARGUMENT"), (dict(heads=-1), "ERR_INVALID_ARGUMENT"), (dict(n_seqs=-1), "ERR_INVALID_ARGUMENT"),
    (dict(n_seqs=0), "ERR_INVALID_ARGUMENT"), (dict(n_seqs=3), "ERR_INVALID_ARGUMENT"), (dict(n_seqs=3, cu_q=16), "ERR_INVALID_ARGUMENT"),
    (dict(q_nope=None), "ERR_INVALID_ARGUMENT"), (dict(q_rope=None), "ERR_INVALID_ARGUMENT"), (dict(k_nope=None), "ERR_INVALID_ARGUMENT"), (dict(v=None), "ERR_INVALID_ARGUMENT"),
    (dict(k_rope=None), "ERR_INVALID_ARGUMENT"), (dict(out=None), "ERR_INVALID_ARGUMENT"), (dict(scale=0.0), "ERR_INVALID_ARGUMENT"), (dict(scale=-1.0), "ERR_INVALID_ARGUMENT"),
    (dict(scale=float("nan")), "ERR_INVALID_ARGUMENT"), (dict(scale=float("inf")), "ERR_INVALID_ARGUMENT"),
    (dict(q_nope=1032), "ERR_UNSUPPORTED"), (dict(out=8), "ERR_UNSUPPORTED"), (dict(v=16392), "ERR_UNSUPPORTED"), (dict(k_nope_token=516), "ERR_UNSUPPORTED"),
    (dict(v_head=-256), "ERR_UNSUPPORTED"), (dict(heads=1025), "ERR_UNSUPPORTED"), (dict(tokens=1 << 31), "ERR_UNSUPPORTED"), (dict(kv_tokens=1 << 31), "ERR_UNSUPPORTED"),
    (dict(tokens=1 << 30, heads=1024), "ERR_UNSUPPORTED")])
def test_attention_that_is_refused(over, status):
    lib, names = _lib()
    assert lib.dsv3_expanded_attention(_args(**over), None, 0, None) == getattr(names, status)


def test_attention_of_nothing_and_workspaces():
    lib, names = _lib()
    assert lib.dsv3_expanded_attention(None, None, 0, None) == names.ERR_INVALID_ARGUMENT
    assert lib.dsv3_expanded_attention(_args(tokens=0), None, 0, None) == names.OK
    assert lib.dsv3_expanded_attention(_args(heads=0), None, 0, None) == names.OK
    # few queries over many keys leave parts behind
    need = lib.dsv3_expanded_attention_workspace_bytes(8, 8000, 2, 1, 0, 1)
    assert need > 0 and need % (8 * 2 * 129 * 4) == 0
    assert lib.dsv3_expanded_attention(_args(kv_tokens=8000), None, 0, None) == names.ERR_WORKSPACE
    assert lib.dsv3_expanded_attention(_args(kv_tokens=8000), 256, need - 1, None) == names.ERR_WORKSPACE
    assert lib.dsv3_expanded_attention(_args(kv_tokens=8000), 264, need, None) == names.ERR_WORKSPACE
    assert lib.dsv3_expanded_attention_workspace_bytes(100000, 100000, 128, 1, 0, 1) == 0
    assert lib.dsv3_expanded_attention_workspace_bytes(0, 8000, 2, 1, 0, 1) == 0


def test_joins_that_are_refused():
    lib, names = _lib()
    outs, lses = (vp * 33)(*[1024] * 33), (vp * 33)(*[512] * 33)
    join = lambda parts=2, rows=4, dim=128, o=outs, l=lses, out=2048: lib.dsv3_attention_join(o, l, parts, rows, dim, out, None, None)  # noqa: E731, E741
    assert join(parts=0) == join(rows=-1) == join(dim=-8) == join(o=None) == join(l=None) == join(out=None) == names.ERR_INVALID_ARGUMENT
    assert join(parts=33) == join(dim=12) == join(dim=2056) == join(rows=1 << 31) == join(out=2056) == names.ERR_UNSUPPORTED
    assert join(o=(vp * 2)(1024, 1032)) == names.ERR_UNSUPPORTED and join(o=(vp * 2)(1024, None)) == names.ERR_INVALID_ARGUMENT
    assert join(rows=0) == join(dim=0) == names.OK


def test_rotations_that_are_refused():
    lib, names = _lib()

    def turn(x=1024, xt=128, xh=64, out=8192, ot=128, oh=64, dtype=0, tokens=3, heads=2, dim=64, freqs=512, n=8, positions=None, per=3, offset=0, rotated=64):
        return lib.dsv3_rotary(x, xt, xh, out, ot, oh, dtype, tokens, heads, dim, freqs, n, positions, per, offset, rotated, 0, 0, None)
    assert turn(tokens=-1) == turn(offset=-8) == turn(offset=8) == turn(per=0) == turn(x=None) == turn(out=None) == turn(freqs=None) == names.ERR_INVALID_ARGUMENT
    assert turn(out=1024, ot=256) == names.ERR_INVALID_ARGUMENT            # in place, and strides that differ
    assert turn(dtype=3) == turn(dim=60, rotated=48) == turn(rotated=24) == turn(dim=1032) == turn(x=1032) == turn(xt=132) == turn(freqs=516) == names.ERR_UNSUPPORTED
    assert turn(dim=512, rotated=272, xt=1024, xh=512, ot=1024, oh=512) == turn(tokens=1 << 31) == names.ERR_UNSUPPORTED
    assert turn(tokens=0) == turn(heads=0) == turn(dim=0, rotated=0) == names.OK
    assert turn(rotated=0, out=1024) == names.OK                           # nothing turns in place

    def table(dim=64, theta=1e4, factor=1.0, original=4096, fast=32.0, slow=1.0, start=0, length=4, out=1024):
        return lib.dsv3_rotary_table(dim, theta, factor, original, fast, slow, start, length, out, None)
    for wrong in (dict(length=-1), dict(start=-1), dict(theta=1.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(factor=0.0), dict(factor=float("inf")), dict(original=0),
                  dict(fast=0.0), dict(slow=-1.0), dict(out=None), dict(dim=-2)):
        assert table(**wrong) == names.ERR_INVALID_ARGUMENT, wrong
    assert table(dim=63) == table(dim=258) == table(length=1 << 27) == table(start=(1 << 40) + 1) == table(out=1028) == names.ERR_UNSUPPORTED
    assert table(length=0) == table(dim=0) == names.OK


def _cpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_tensors_that_python_refuses():
    """Shapes are looked at before devices; CPU tensors are then refused."""
    import dsv3_b200 as D
    q, r, k, kr, v = _cpu(4, 2, 128), _cpu(4, 2, 64), _cpu(6, 2, 128), _cpu(6, 64), _cpu(6, 2, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.expanded_attention(q, r, k, kr, v, 0.1)
    for wrong in ((q[..., :64], r, k, kr, v), (q, r[:3], k, kr, v), (q, r, k[:, :1], kr, v[:, :1]), (q, r, k, kr, v[:5]), (q, r, k, kr[:5], v), (q, r, k, kr[None], v),
                  (q.unsqueeze(0), r, k, kr, v), (q, r, k, _cpu(6, 128)[:, ::2], v), (q, r, k.transpose(0, 2).contiguous().transpose(0, 2), kr, v)):
        with pytest.raises(AssertionError):
            D.expanded_attention(*wrong, 0.1)
    with pytest.raises(TypeError):
        D.expanded_attention(q, r, k, kr, None, 0.1)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.attention_join([q], [_cpu(4, 2, dtype=torch.float32)])
    with pytest.raises(AssertionError):
        D.attention_join([], [])
    x, f = _cpu(4, 2, 64), _cpu(8, 32, dtype=torch.complex64)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.rotary(x, f)
    with pytest.raises(ValueError, match="layout"):
        D.rotary(x, f, layout="pairs")
    for wrong in (dict(x=x[0, 0]), dict(f=f[:, ::2]), dict(f=f.real), dict(offset=8), dict(offset=-8), dict(f=_cpu(8, 33, dtype=torch.complex64))):
        with pytest.raises(AssertionError):
            D.rotary(wrong.get("x", x), wrong.get("f", f), offset=wrong.get("offset", 0))
    with pytest.raises(RuntimeError, match="CUDA"):
        D.rotary_table(4, device="cpu")
    for wrong in (dict(length=-1), dict(length=1, start=-1), dict(length=1, dim=63), dict(length=1, dim=0), dict(length=1, dim=512)):
        with pytest.raises(ValueError):
            D.rotary_table(**wrong, device="cuda:0")
