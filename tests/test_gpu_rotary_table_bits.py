"""The table of angles is rounded once: against sines and cosines in 64 bits."""
import pytest
import torch

from expanded_util import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim, start, length", [(64, 0, 163840), (128, 0, 20000), (256, 12345, 3000), (2, 0, 50000), (64, 1 << 20, 5000), (64, 1 << 31, 500)])
def test_rounded_once(dim, start, length):
    """Below 1 a rounding to fp32 is off by 2^-25 at most; the polynomials by 2^-29; frequencies and angles are rounded to 64 bits some four times, here and there: 2^-51 of the angle."""
    from dsv3_b200 import rotary_table
    got = rotary_table(length, dim, start=start)
    per = torch.tensor([10000.0 ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64, device="cuda")
    angle = torch.outer(torch.arange(start, start + length, device="cuda").double(), per)
    bound = 2.0 ** -25 + 2.0 ** -29 + angle * 2.0 ** -51
    check(got.real, angle.cos(), bound)
    check(got.imag, angle.sin(), bound)
    # ... and nearly all are the rounded ones (all but those within 2^-29 of the middle of two: of 2^-24 between two of them that is 6 %)
    near = angle < 2.0 ** 20
    for x, want in ((got.real, angle.cos()), (got.imag, angle.sin())):
        same = ((x == want.float()) | ~near | (want.abs() < 0.5)).double().mean()
        assert float(same) > 0.9
