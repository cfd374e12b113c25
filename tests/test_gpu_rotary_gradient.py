"""The gradient of a rotation, as autograd asks for it: against the formula in 64 bits and against differences."""
import types

import pytest
import torch

from test_gpu_rotary import _check, _freqs, _turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("tokens, heads, dim, offset, rotated", [(1, 1, 64, 0, 64), (7, 3, 192, 128, 64), (33, 16, 64, 0, 64), (5, 2, 128, 32, 32), (0, 2, 64, 0, 64)])
def test_gradient(dtype, layout, inverse, tokens, heads, dim, offset, rotated):
    from dsv3_b200 import rotary
    x, g = (torch.randn(tokens, heads, dim, device="cuda").to(dtype) for _ in range(2))
    f, positions = _freqs(50, rotated // 2), torch.randint(0, 50, (tokens,), device="cuda")
    x.requires_grad_()
    y = rotary(x, f, positions, layout=layout, offset=offset, inverse=inverse)
    with torch.no_grad():
        assert torch.equal(y, rotary(x, f, positions, layout=layout, offset=offset, inverse=inverse))
    got, = torch.autograd.grad(y, x, g)
    assert got.dtype == dtype and torch.equal(got, rotary(g, f, positions, layout=layout, offset=offset, inverse=not inverse))
    if tokens:
        _check(got, *_turned(g, f.to(torch.complex128)[positions][:, None], layout, offset, not inverse), dtype)
        # one gradient in many places
        ones, = torch.autograd.grad(rotary(x, f, positions, layout=layout, offset=offset, inverse=inverse).sum(), x)
        _check(ones, *_turned(torch.ones_like(x), f.to(torch.complex128)[positions][:, None], layout, offset, not inverse), dtype)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_against_differences(layout):
    """The rotation is linear: (R(x + d) - R(x - d)) / 2 is R d, but for what its fp32 results are rounded by."""
    from dsv3_b200 import rotary
    f = _freqs(6, 32)
    x, d, g = (torch.randn(6, 2, 192, device="cuda") for _ in range(3))
    x.requires_grad_()
    turn = lambda z: rotary(z, f, layout=layout, offset=128)  # noqa: E731
    got, = torch.autograd.grad((turn(x) * g).sum(), x)
    with torch.no_grad():
        differences = (g.double() * (turn(x + d).double() - turn(x - d).double())).sum() / 2
    # (x + d and what becomes of them: four roundings of 2^-24 of twice the largest; the gradient: three of its own)
    size = (g.double().abs() * 2 * (x.abs().amax() + d.abs().amax()).double()).sum() + (d.double().abs() * 2 * g.double().abs().amax()).sum()
    assert abs(float((got.double() * d.double()).sum() - differences)) <= 4 * 2.0 ** -24 * float(size.detach())


def test_heads_that_share_a_value_and_gradients_of_gradients():
    """As MLA's rotated part of a key, which all heads read: the heads' gradients are summed.  The gradient of <g, R x> in g is R x."""
    import dsv3_b200
    module = types.SimpleNamespace()
    dsv3_b200.install_rotary(module)
    f = _freqs(9, 32)
    kv, g = torch.randn(2, 9, 576, device="cuda", requires_grad=True), torch.randn(2, 9, 4, 64, device="cuda", requires_grad=True)
    y = module.apply_rotary_emb(kv[..., 512:].unsqueeze(2), f).expand(-1, -1, 4, -1)
    got, = torch.autograd.grad(y, kv, g, create_graph=True)
    back, size = _turned(g.detach().double().sum(2, keepdim=True), f.to(torch.complex128)[None, :, None], "interleaved", 0, True)
    assert not got[..., :512].any()
    # (three sums of four terms before the rotation)
    assert bool(((got[..., 512:].double() - back[:, :, 0]).abs() <= 2.0 ** -24 * (back.abs() + 3 * size + 8 * g.detach().double().abs().sum(2, keepdim=True).amax())[:, :, 0]).all())
    again, = torch.autograd.grad(got, g, torch.ones_like(got))
    _check(again, *_turned(torch.ones(2, 9, 4, 64, device="cuda"), f.to(torch.complex128)[None, :, None], "interleaved", 0, False), torch.float32)


def test_a_gradient_that_lies_at_an_odd_place():
    from dsv3_b200 import rotary
    f = _freqs(3, 32)
    x = torch.randn(3, 2, 64, device="cuda").bfloat16().requires_grad_()
    y = torch.cat([torch.zeros(1, device="cuda", dtype=torch.bfloat16), rotary(x, f).flatten()])
    g = torch.randn(385, device="cuda").bfloat16()
    got, = torch.autograd.grad(y, x, g)
    assert torch.equal(got, rotary(g[1:].clone().view(3, 2, 64), f, inverse=True))


def test_a_captured_forward_and_backward():
    from dsv3_b200 import rotary
    f = _freqs(30, 32)
    x, g = torch.randn(30, 4, 64, device="cuda").bfloat16(), torch.randn(30, 4, 64, device="cuda").bfloat16()
    x.requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(rotary(x, f), x, g)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = rotary(x, f)
        got, = torch.autograd.grad(y, x, g)
    for _ in range(2):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            g.copy_(torch.randn_like(g))
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(y, rotary(x, f)) and torch.equal(got, rotary(g, f, inverse=True))


def test_what_has_no_gradient():
    from dsv3_b200 import rotary
    f = _freqs(3, 32)
    x = torch.randn(3, 2, 64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="out"):
        rotary(x, f, out=torch.empty_like(x))
    with pytest.raises(RuntimeError, match="out"):
        rotary(x.detach(), f, out=torch.empty_like(x).requires_grad_())
    with pytest.raises(NotImplementedError):
        rotary(x, f.clone().requires_grad_())
    with torch.no_grad():
        assert not rotary(x, f, out=torch.empty_like(x)).requires_grad and not rotary(x, f).requires_grad
    assert not rotary(x.detach(), f).requires_grad
