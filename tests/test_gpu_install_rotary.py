"""install_rotary's apply_rotary_emb beside what it replaces: x [batch, tokens, heads, dim] by angles [tokens, dim / 2]."""
import types

import pytest
import torch

from expanded_util import check

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _apply():
    import dsv3_b200
    module = types.SimpleNamespace()
    dsv3_b200.install_rotary(module)
    return module.apply_rotary_emb


def _angles(tokens, dim):
    import dsv3_b200
    return dsv3_b200.rotary_table(tokens, dim, start=5)


def _want(x, f):
    """In 64 bits: neighbouring values as a complex number, times their angle's."""
    z = torch.view_as_complex(x.double().contiguous().unflatten(-1, (-1, 2))) * f.to(torch.complex128).view(1, x.size(1), 1, x.size(-1) // 2)
    return torch.view_as_real(z).flatten(-2)


def _check(got, x, f):
    want = _want(x, f)
    assert got.dtype == x.dtype and got.shape == x.shape
    # (two products and a sum in fp32, each rounded, and the result; a product is x's largest at most)
    most = x.double().abs().amax() if x.numel() else 0.0
    check(got, want, want.abs() * STEP[x.dtype] + 3 * 2.0 ** -24 * 2 * most + (2.0 ** -24 if x.dtype == torch.float16 else 0.0))


def test_a_table_of_other_tokens_or_another_width_is_an_error():
    apply = _apply()
    x = torch.randn(2, 30, 4, 64, device="cuda").bfloat16()
    f = _angles(64, 64)
    _check(apply(x, f[:30]), x, f[:30])
    _check(apply(x, f[:30].view(1, 30, 1, 32)), x, f[:30])
    for wrong in (f, f[:29], f[:31], f[:30, :16].contiguous(), f[:30].repeat(1, 2)):
        with pytest.raises(RuntimeError):
            apply(x, wrong)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_strides_that_the_function_it_replaces_takes(dtype):
    """Cuts from longer sequences, single tokens of them, rows at odd places, dimensions in other orders, values for several heads or sequences in one place, angles with strides."""
    apply = _apply()
    whole, f = torch.randn(3, 40, 4, 192, device="cuda").to(dtype), _angles(40, 64)
    odd = torch.randn(3 * 40 * 4 * 67 + 1, device="cuda").to(dtype)[1:].view(3, 40, 4, 67)
    cases = [(whole[..., 128:], f), (whole[:, 7:20, :, 128:], f[7:20]), (whole[:, 5:6, :, 128:], f[5:6]), (whole[1:2, 7:20, 1:3, 64:128], f[7:20]), (whole[:, ::2, :, :64], f[::2]),
             (odd[..., 3:], f), (whole.transpose(1, 2)[..., 128:], f[:4]), (whole[..., :64].transpose(1, 3).contiguous().transpose(1, 3), f), (whole[:, :, :1, 128:].expand(-1, -1, 4, -1), f),
             (whole[:1, :, :, :64].expand(3, -1, -1, -1), f), (whole[:, :0, :, :64], f[:0]), (whole[:0, :, :, :64], f)]
    for x, angles in cases:
        before = x.clone()
        _check(apply(x, angles), x, angles)
        assert torch.equal(x, before)
    _check(apply(whole[..., :64], f.t().contiguous().t()), whole[..., :64], f)


def test_what_it_does_not_take():
    apply = _apply()
    x, f = torch.randn(1, 3, 2, 64, device="cuda"), _angles(3, 64)
    with pytest.raises(NotImplementedError):
        apply(x.double(), f)
    with pytest.raises(RuntimeError, match="CUDA"):
        apply(x.cpu(), f.cpu())
    with pytest.raises(ValueError):
        apply(x[0], f)
