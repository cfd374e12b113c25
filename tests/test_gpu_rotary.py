"""Rotary positions, and the joining of an attention's parts, against their definitions in 64 bits."""
import math

import pytest
import torch

from expanded_util import HALF_STEP, check

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}     # below: fewer bits


def _turned(x, f, layout, offset, inverse):
    """In 64 bits; f: complex128, broadcast over heads."""
    x = x.double().clone()
    r = 2 * f.shape[-1]
    part = x[..., offset:offset + r]
    a, b = (part[..., 0::2], part[..., 1::2]) if layout == "interleaved" else (part[..., :r // 2], part[..., r // 2:])
    s = -f.imag if inverse else f.imag
    re, im = a * f.real - b * s, a * s + b * f.real
    size = a.abs() * f.real.abs() + b.abs() * s.abs()
    size2 = a.abs() * s.abs() + b.abs() * f.real.abs()
    join = lambda u, v: torch.stack([u, v], -1).flatten(-2) if layout == "interleaved" else torch.cat([u, v], -1)  # noqa: E731
    x[..., offset:offset + r] = join(re, im)
    bound = torch.zeros_like(x)
    bound[..., offset:offset + r] = join(size, size2)
    return x, bound


def _freqs(n, pairs, seed=1):
    angle = torch.rand(n, pairs, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * 6.3
    return torch.polar(torch.ones_like(angle), angle)


def _check(got, want, size, dtype):
    # two products and a sum, each rounded to fp32, and the result to its type
    check(got, want, want.abs() * STEP[dtype] + size * 3 * 2.0 ** -24 + TINY[dtype])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens, heads, dim, offset, rotated", [(1, 1, 64, 0, 64), (3, 5, 64, 0, 64), (70, 16, 192, 128, 64), (33, 128, 64, 0, 64), (9, 3, 128, 32, 32), (65, 2, 16, 0, 16),
                                                                 (2, 300, 24, 8, 16), (7, 1, 256, 0, 256), (5, 2, 1024, 768, 256), (1031, 1, 64, 0, 32), (4, 3, 64, 16, 0)])
def test_rotation(dtype, layout, tokens, heads, dim, offset, rotated):
    from dsv3_b200 import rotary
    x = torch.randn(tokens, heads, dim, device="cuda").to(dtype)
    f = _freqs(50, rotated // 2)
    positions = torch.randint(0, 50, (tokens,), device="cuda")
    want, size = _turned(x, f.to(torch.complex128)[positions][:, None], layout, offset, False)
    before = x.clone()
    got = rotary(x, f, positions, layout=layout, offset=offset)
    assert got.is_contiguous() and torch.equal(x, before)
    _check(got, want, size, dtype)
    back, size = _turned(x, f.to(torch.complex128)[positions][:, None], layout, offset, True)
    _check(rotary(x, f, positions, layout=layout, offset=offset, inverse=True), back, size, dtype)
    # in place: the same, and the rest of the heads as it is
    y = x.clone()
    assert rotary(y, f, positions, layout=layout, offset=offset, out=y) is not None
    assert torch.equal(y, got)


def test_strides_and_batches():
    from dsv3_b200 import rotary
    wide = torch.randn(3, 20, 4, 192, device="cuda").bfloat16()
    x, f = wide[..., 128:], _freqs(20, 32)
    want, size = _turned(x, f.to(torch.complex128)[None, :, None], "interleaved", 0, False)
    got = rotary(x, f)                                       # a sequence's tokens are at 0, 1, ...
    _check(got, want, size, torch.bfloat16)
    keep = wide.clone()
    rotary(x, f, out=x)
    assert torch.equal(wide[..., 128:], got) and torch.equal(wide[..., :128], keep[..., :128])
    # heads in front, to a buffer with another layout
    fronted = keep[0, :, :, 128:].transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.zeros(20, 7, 64, dtype=torch.bfloat16, device="cuda")
    rotary(fronted, f, out=out[:, 1:5])
    assert torch.equal(out[:, 1:5], got[0]) and not out[:, 0].any() and not out[:, 5:].any()
    # one head's values for all of them
    one = keep[0, :, :1, 128:]
    assert torch.equal(rotary(one.expand(-1, 4, -1), f)[:, 3], got[0, :, 0])


def test_positions_that_the_table_does_not_hold():
    from dsv3_b200 import rotary
    x, f = torch.randn(5, 3, 192, device="cuda").bfloat16(), _freqs(4, 32)
    got = rotary(x, f, torch.tensor([0, -1, 4, 3, 1 << 40], device="cuda"), offset=128)
    lost = torch.tensor([False, True, True, False, True], device="cuda")
    assert bool(got[lost][..., 128:].isnan().all()) and not got[~lost].isnan().any() and torch.equal(got[..., :128], x[..., :128])
    nan = torch.full_like(f, complex(math.nan, math.nan))
    assert bool(rotary(x[:4], nan, offset=128)[..., 128:].isnan().all())


def test_the_gradient_is_the_inverse():
    """<g, R x> = <R^-1 g, x>, and differences of R along a direction."""
    from dsv3_b200 import rotary
    f = _freqs(6, 32)
    x, g, d = (torch.randn(6, 2, 64, device="cuda") for _ in range(3))
    for layout in ("interleaved", "half"):
        left = (g.double() * rotary(x, f, layout=layout).double()).sum()
        right = (rotary(g, f, layout=layout, inverse=True).double() * x.double()).sum()
        assert abs(float(left - right)) <= 4 * 2.0 ** -24 * float((g.abs() * x.abs().amax()).sum()) * 2
        step = rotary(x + d, f, layout=layout).double() - rotary(x - d, f, layout=layout).double()
        # (each term is rounded by 4 e of what it holds at most)
        assert abs(float((g.double() * step).sum() / 2 - (rotary(g, f, layout=layout, inverse=True).double() * d.double()).sum())) <= \
            8 * 2.0 ** -24 * float((g.abs().double() * (x.abs().amax() + d.abs().amax()).double() * 2).sum())


@pytest.mark.parametrize("dim, factor, start, length", [(64, 1.0, 0, 1), (64, 1.0, 0, 4097), (64, 40.0, 0, 163840), (64, 4.0, 100000, 33), (2, 1.0, 5, 9), (128, 2.0, 7, 1000),
                                                        (256, 1.0, 1 << 30, 50), (64, 40.0, 0, 0)])
def test_table(dim, factor, start, length):
    from dsv3_b200 import rotary_table
    got = rotary_table(length, dim, factor=factor, start=start)
    assert got.dtype == torch.complex64 and got.shape == (length, dim // 2)
    per = []
    for i in range(dim // 2):
        f = 10000.0 ** (-2.0 * i / dim)
        if factor != 1:
            low, high = (dim * math.log(4096 / (2 * math.pi * b)) / (2 * math.log(10000.0)) for b in (32, 1))
            low, high = max(math.floor(low), 0), min(math.ceil(high), dim - 1)
            smooth = 1 - min(1.0, max(0.0, (i - low) / (high - low)))
            f = f / factor * (1 - smooth) + f * smooth
        per.append(f)
    angle = torch.outer(torch.arange(start, start + length, device="cuda").double(), torch.tensor(per, dtype=torch.float64, device="cuda"))
    # an angle within an eighth of a turn in fp32 (0.8 * 2^-24), a sine and a cosine that are right to 2 ulp (2^-23 each); and the angle in 64 bits
    bound = torch.full_like(angle, 2.0 ** -24 + 2.0 ** -22) + angle.abs() * 2.0 ** -51
    check(got.real, angle.cos(), bound)
    check(got.imag, angle.sin(), bound)


@pytest.mark.parametrize("parts", [1, 2, 3, 5, 32])
@pytest.mark.parametrize("shape", [(1, 1, 128), (7, 5, 128), (3, 2, 512), (130, 8), (4, 3, 2048), (2, 9, 24)])
def test_join(parts, shape):
    from dsv3_b200 import attention_join
    gen = torch.Generator(device="cuda").manual_seed(parts)
    outs = [torch.randn(*shape, generator=gen, device="cuda").bfloat16() for _ in range(parts)]
    lses = [torch.randn(*shape[:-1], generator=gen, device="cuda") * 4 for _ in range(parts)]
    for i in range(0, parts, 2):                             # parts that see nothing hold anything
        lses[i].view(-1)[::3] = -math.inf
        outs[i].view(-1, shape[-1])[::3] = math.nan
    out, lse = attention_join(outs, lses, return_lse=True)
    all_lse = torch.stack(lses).double()
    want_lse = torch.logsumexp(all_lse, 0)
    weight = torch.exp(all_lse - torch.where(want_lse == -math.inf, 0.0, want_lse))
    terms = torch.stack([torch.where(w[..., None] > 0, o.double().nan_to_num(), 0.0) * w[..., None] for w, o in zip(weight, outs)])
    want = terms.sum(0)
    # a weight: the difference of two lses, rounded (e of each), its exponential; sums of `parts` terms
    e = 2.0 ** -24
    relative = 2 * e * (all_lse.nan_to_num(neginf=0.0).abs().amax(0) * 3 + 8 + 2 * parts)
    check(out, want, HALF_STEP * want.abs() + (1 + HALF_STEP) * relative[..., None] * terms.abs().sum(0))
    check(lse, want_lse, relative + 2 * e * want_lse.nan_to_num(neginf=0.0).abs())
    assert torch.equal(attention_join(outs, lses), out)


def test_join_of_what_is_not_finite():
    from dsv3_b200 import attention_join
    outs = [torch.ones(4, 8, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    lses = [torch.tensor([0.0, math.nan, -math.inf, 300.0], device="cuda"), torch.tensor([0.0, 1.0, -math.inf, -300.0], device="cuda")]
    outs[0][0, 3] = math.nan
    out, lse = attention_join(outs, lses, return_lse=True)
    assert bool(out[0, 3].isnan()) and not out[0, :3].isnan().any() and bool(out[1].isnan().all() and lse[1].isnan()) and not out[2].any() and float(lse[2]) == -math.inf
    assert bool((out[3] == 1).all()) and float(lse[3]) == 300.0
