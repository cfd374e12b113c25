"""install_mla: masks that are not the causal one are refused, or make the result NaN."""
import math

import pytest
import torch

from test_gpu_mla_seam import _bf16_default, _freqs, _model  # noqa: F401

pytestmark = pytest.mark.gpu


def _causal(n, end=None, low=-math.inf, dtype=torch.float32):
    end = end or n
    return torch.full((n, end), low, device="cuda", dtype=dtype).triu_(end - n + 1)


def _prompt(tokens, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(2, tokens, 256, generator=g, device="cuda", dtype=torch.float32).bfloat16()


def test_forms_of_the_causal_mask():
    m, f, x = _model(4, 0), _freqs(200), _prompt(50)
    first = m(x[:, :30], 0, f[:30], _causal(30))
    assert not torch.isnan(first).any()
    for mask in (_causal(30, dtype=torch.bfloat16), _causal(30, low=torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16), _causal(30, low=torch.finfo(torch.float32).min),
                 _causal(30).cpu()):
        assert torch.equal(m(x[:, :30], 0, f[:30], mask), first)
    chunk = m(x[:, 30:], 30, f[30:50], _causal(20))
    assert torch.equal(m(x[:, 30:], 30, f[30:50], _causal(20, 50)), chunk) and not torch.isnan(chunk).any()
    step = m(x[:, 30:31], 30, f[30:31], None)
    assert torch.equal(m(x[:, 30:31], 30, f[30:31], torch.zeros(1, 1, device="cuda")), step)
    assert torch.equal(m(x[:, 30:31], 30, f[30:31], torch.zeros(1, 31, device="cuda")), step)


@pytest.mark.parametrize("shape", [(2, 30, 30), (2, 1, 30, 30), (30,), (30, 29), (30, 60), (1, 30)])
def test_masks_of_other_shapes_are_refused(shape):
    m, f, x = _model(4, 0), _freqs(200), _prompt(30)
    with pytest.raises(NotImplementedError, match="mask of shape"):
        m(x, 0, f[:30], torch.zeros(shape, device="cuda"))


def test_masks_that_say_something_else():
    m, f, x = _model(4, 0), _freqs(200), _prompt(30)
    window = _causal(30)
    window += torch.full((30, 30), -math.inf, device="cuda").tril_(-9)
    padded = _causal(30)
    padded[:, 0] = -math.inf
    bias = _causal(30)
    bias[20, 3] = -0.5
    for mask in (window, padded, bias, torch.zeros(30, 30, device="cuda"), _causal(30) * 0.0):
        assert torch.isnan(m(x, 0, f[:30], mask)).all()
    with pytest.raises(NotImplementedError, match="neither"):
        m(x, 0, f[:30], window.cpu())
    # ... and the tokens are in the cache: the next call with the right mask is as ever
    want = _model(4, 0)(x, 0, f[:30], _causal(30))
    assert torch.equal(m(x, 0, f[:30], _causal(30)), want)
