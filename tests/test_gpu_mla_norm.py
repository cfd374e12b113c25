"""install_mla: a kv_norm that does more than the RMS norm of its weight is called, and what it returns is what the cache holds."""
import pytest
import torch

import latent_util as U
from test_gpu_mla_seam import _bf16_default, _freqs, _model  # noqa: F401
from test_mla_norm import Norm, OnePlus

pytestmark = pytest.mark.gpu


def _with(norm_class, m=None):
    m = m or _model(16, 0)
    norm = norm_class().cuda()
    norm.weight.data.copy_(m.kv_norm.weight)
    m.kv_norm = norm
    return m


def _stored(m, n):
    import dsv3_b200
    cache = dsv3_b200.mla_cache(m)
    return dsv3_b200.latent_cache_read(cache.pool, cache.block_table[:2], U.offsets([n, n]), 2 * n)


def _run(m, x, f):
    with torch.no_grad():
        return m(x, 0, f, torch.full((x.size(1),) * 2, float("-inf"), device="cuda").triu_(1))


def _nearest(latent):
    """What a token of these latents is stored as."""
    s = U.least_power(latent.double().abs().amax(-1, keepdim=True).clamp_min(1e-4))
    return ((latent.double() / s).float().to(torch.float8_e4m3fn).double() * s)


@pytest.fixture
def tokens():
    g = torch.Generator(device="cuda").manual_seed(6)
    return torch.randn(2, 40, 256, generator=g, device="cuda", dtype=torch.float32).bfloat16(), _freqs(40)


def test_the_plain_norm_is_part_of_the_store(tokens):
    x, f = tokens
    m = _with(Norm)
    called = []
    original = Norm.forward
    y = _run(m, x, f)
    want = [t.clone() for t in _stored(m, 40)]
    m.kv_norm.register_forward_hook(lambda mod, args, out: called.append(out))      # only looks on
    z = _run(m, x, f)
    assert len(called) == 1 and Norm.forward is original
    # One rounding to bf16 more before that to e4m3 moves a value by 2^-8 of it at most, where steps of e4m3 are 2^-4 to 2^-3 of it: below one value in ten goes to its neighbour,
    # 2^-3 of it away at most.  RMS that is below sqrt(0.1) 2^-3 = 0.04 of the latents, once as values and once through scores of about one unit's spread: sqrt(2) 0.04 < 0.06.
    got = _stored(m, 40)
    assert ((got[0].double() - want[0].double()).abs() <= 2.0 ** -3 * want[0].double().abs() + 2.0 ** -9).all() and (got[0] != want[0]).double().mean().item() < 0.1
    assert ((z.double() - y.double()).norm() / y.double().norm()).item() < 0.06


def test_a_hook_that_changes_the_result(tokens):
    x, f = tokens
    m = _with(Norm)
    m.kv_norm.register_forward_hook(lambda mod, args, out: out * 4)
    _run(m, x, f)
    with torch.no_grad():
        latent = Norm.forward(m.kv_norm, m.wkv_a(x)[..., :512]) * 4
    assert torch.equal(_stored(m, 40)[0].double(), _nearest(latent.view(80, 512)))


def test_a_forward_of_its_own_and_another_class(tokens):
    x, f = tokens
    m = _with(Norm)
    m.kv_norm.forward = lambda t: t.float() * 3                                    # (bf16 is what the cache takes)
    _run(m, x, f)
    assert torch.equal(_stored(m, 40)[0].double(), _nearest((m.wkv_a(x)[..., :512].float() * 3).bfloat16().view(80, 512)))
    m = _with(OnePlus)
    _run(m, x, f)
    with torch.no_grad():
        assert torch.equal(_stored(m, 40)[0].double(), _nearest(m.kv_norm(m.wkv_a(x)[..., :512]).view(80, 512)))


@pytest.mark.parametrize("size", [2.0 ** -60, 1e-3, 1.0, 2.0 ** 40])
def test_sizes_of_what_a_norm_returns(tokens, size):
    x, f = tokens
    m = _with(Norm)
    m.kv_norm.forward = lambda t: t * size
    _run(m, x, f)
    assert torch.equal(_stored(m, 40)[0].double(), _nearest((m.wkv_a(x)[..., :512] * size).view(80, 512)).bfloat16().double())
