"""install_mla's expand_tokens: how many keys and values a call holds at a time, and that its results do not depend on it."""
import pytest
import torch

from test_gpu_mla_expanded import _bf16_default, _causal, _expanding  # noqa: F401  (a fixture)
from test_gpu_mla_seam import _cached, _freqs, _off, _queries, _result

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [4, 16])
@pytest.mark.parametrize("expand_tokens", [1, 20, 100, 130, 300, 1000])
@pytest.mark.parametrize("cached, new", [(0, 300), (63, 200), (64, 130), (350, 150)])
def test_no_more_is_expanded_at_a_time(monkeypatch, heads, expand_tokens, cached, new):
    """First prompts, and chunks behind a prefix within and beyond the first page: all within the room for expand_tokens tokens, or one head of one sequence."""
    from dsv3_b200 import mla_seam
    m = _expanding(heads, 0, expand_tokens=expand_tokens, length=500)
    f, x = _freqs(500), torch.randn(2, cached + new, 256, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.float32).bfloat16()
    held, attend = [], mla_seam.expanded_attention

    def spy(q_nope, q_rope, k_nope, *rest, **more):
        held.append(k_nope.shape)
        return attend(q_nope, q_rope, k_nope, *rest, **more)
    monkeypatch.setattr(mla_seam, "expanded_attention", spy)
    if cached:
        m(x[:, :cached], 0, f[:cached], _causal(cached))
    y = m(x[:, cached:], cached, f[cached:cached + new], _causal(new))
    for sequences, tokens, some_heads, _ in held:
        assert sequences * tokens * some_heads <= heads * expand_tokens or (sequences, some_heads) == (1, 1)
    # every head of every sequence sees each of its keys
    assert sum(b * n * h for b, n, h, _ in held) == 2 * heads * (cached + cached + new)
    end = cached + new
    seen = torch.arange(end, device="cuda") <= torch.arange(cached, end, device="cuda")[:, None]
    ql, qr = _queries(m, x[:, cached:], f[cached:end])
    # (the bound of the other tests of this path: bf16 keys, values, queries, weights, results and pieces of them)
    assert _off(y, _result(m, ql, qr, *_cached(m, 2, end), seen[None])) < 2.0 ** -7


def test_memory_of_a_first_prompt():
    """2 x 4000 tokens of 16 heads, 512 tokens' keys and values at a time: 4 MB, and not 65."""
    peaks = []
    for expand_tokens in (512, 1 << 16):
        m = _expanding(16, 0, expand_tokens=expand_tokens, length=4000)
        f, x, mask = _freqs(4000), torch.randn(2, 4000, 256, device="cuda", dtype=torch.float32).bfloat16(), _causal(4000)
        m(x[:, :10], 0, f[:10], mask[:10, :10])             # (the cache)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        m(x, 0, f, mask)
        peaks.append(torch.cuda.max_memory_allocated() - before)
        del m
    # (65.5 MB against 4.2 of keys and values; the attention's result, 33 MB, is there twice at most where heads are attended to by themselves)
    assert peaks[1] - peaks[0] > 20e6, peaks
