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
    check(got, want, want.abs() * STEP[x.dtype] + 3 * 2.0 ** -24 * 2 * x.double().abs().amax() + (2.0 ** -24 if x.dtype == torch.float16 else 0.0))


def test_a_table_of_other_tokens_or_another_width_is_an_error():
    apply = _apply()
    x = torch.randn(2, 30, 4, 64, device="cuda").bfloat16()
    f = _angles(64, 64)
    _check(apply(x, f[:30]), x, f[:30])
    _check(apply(x, f[:30].view(1, 30, 1, 32)), x, f[:30])
    for wrong in (f, f[:29], f[:31], f[:30, :16].contiguous(), f[:30].repeat(1, 2)):
        with pytest.raises(RuntimeError):
            apply(x, wrong)
