"""install_mla with expand_from: prompts attended to with expanded keys and values; install_rotary; and the operators run one after another as a program runs them.

Against fp32 behind the same cached tokens: keys and values are rounded to bf16 (2^-9 RMS of a value at most, 2^-8 relative), as are the queries, the weights, the attention's result and the
output; together below the 2^-7 that the absorbed form is held to."""
import math
import types

import pytest
import torch

import latent_util as U
from test_gpu_mla_seam import _cached, _freqs, _model, _off, _queries, _result, _tokens
from expanded_util import check, offsets, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _bf16_default():
    import dsv3_b200
    torch.set_default_dtype(torch.bfloat16)
    yield
    torch.set_default_dtype(torch.float32)
    dsv3_b200.check_device_status()


def _expanding(heads, q_lora, expand_from=2, expand_tokens=1 << 16, **more):
    import dsv3_b200
    m = _model(heads, q_lora, **more)
    module = types.SimpleNamespace(MLA=type(m), block_size=128)
    dsv3_b200.install_mla(module, expand_from=expand_from, expand_tokens=expand_tokens)
    return m


def _causal(n):
    return torch.full((n, n), float("-inf"), device="cuda").triu_(1)


@pytest.mark.parametrize("heads, q_lora", [(4, 0), (16, 128)])
@pytest.mark.parametrize("expand_tokens", [1, 128, 1 << 16])
def test_prompt_chunks_and_steps(heads, q_lora, expand_tokens):
    """Pieces of one page to a sequence, of two pages between them, and all at once; chunks that begin inside a page."""
    m = _expanding(heads, q_lora, expand_tokens=expand_tokens, length=500)
    g = torch.Generator(device="cuda").manual_seed(1)
    f = _freqs(500)
    x = torch.randn(2, 460, 256, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    at = 0
    for n in (70, 1, 200, 17, 170, 1):
        y = m(x[:, at:at + n], at, f[at:at + n], _causal(n) if n > 1 else None)
        end = at + n
        seen = torch.arange(end, device="cuda") <= torch.arange(at, end, device="cuda")[:, None]
        ql, qr = _queries(m, x[:, at:end], f[at:end])
        assert _off(y, _result(m, ql, qr, *_cached(m, 2, end), seen[None])) < 2.0 ** -7
        assert _off(y, _result(m, ql, qr, *_tokens(m, x[:, :end], f[:end]), seen[None])) < 0.06
        at = end


def test_fewer_tokens_are_absorbed_as_before():
    plain, m = _model(4, 0), _expanding(4, 0, expand_from=51)
    f = _freqs(200)
    x = torch.randn(2, 60, 256, device="cuda", dtype=torch.float32).bfloat16()
    assert torch.equal(m(x[:, :50], 0, f[:50], _causal(50)), plain(x[:, :50], 0, f[:50], _causal(50)))
    # starts of their own, and trees, are absorbed however many tokens there are
    m = _expanding(4, 0, expand_from=1)
    plain(x[:, :50], 0, f[:50], _causal(50))
    m(x[:, :50], 0, f[:50], _causal(50))
    cached = _cached(m, 2, 50)
    assert all(torch.equal(a, b) for a, b in zip(cached, _cached(plain, 2, 50)))
    starts = torch.tensor([50, 40], device="cuda")
    angles = torch.stack([f[50:54], f[40:44]])
    mask = torch.full((4, 4), float("-inf"), device="cuda").triu_(1)
    assert torch.equal(m(x[:, 50:54], starts, angles, mask), plain(x[:, 50:54], starts, angles, mask))
    words = torch.tensor([[1, 3, 5, 9]] * 2, device="cuda")
    assert torch.equal(m(x[:, 50:54], 50, f[50:54], words), plain(x[:, 50:54], 50, f[50:54], words))


def test_angles_of_every_sequence():
    m, other = _expanding(4, 0), _expanding(4, 0)
    f = _freqs(200)
    x = torch.randn(2, 40, 256, device="cuda", dtype=torch.float32).bfloat16()
    want = m(x, 0, f[:40], _causal(40))
    assert torch.equal(other(x, 0, f[None, :40].expand(2, -1, -1), _causal(40)), want)


def test_masks_that_are_not_causal():
    m = _expanding(4, 0)
    f = _freqs(200)
    x = torch.randn(1, 30, 256, device="cuda", dtype=torch.float32).bfloat16()
    window = _causal(30)
    window[20:, :5] = float("-inf")
    assert bool(m(x, 0, f[:30], window).isnan().all())
    with pytest.raises(NotImplementedError):
        m(x, 0, f[:30], window.cpu())
    with pytest.raises(NotImplementedError):
        m(x, 0, f[:30], None)
    # the lowest number of its type instead of -inf, and a mask up to the end
    y = m(x, 0, f[:30], torch.full((30, 30), torch.finfo(torch.bfloat16).min, device="cuda", dtype=torch.bfloat16).triu_(1))
    assert not y.isnan().any()
    m(x[:, :10], 30, f[30:40], torch.full((10, 40), float("-inf"), device="cuda").triu_(31))


def test_fp8_projection_of_the_latents():
    import dsv3_b200
    m = _expanding(4, 0, seed=3)
    q, s = dsv3_b200.weight_quant(m.wkv_b.weight)
    f = _freqs(10)
    x = torch.randn(1, 5, 256, device="cuda", dtype=torch.float32).bfloat16()
    m.wkv_b.weight = dsv3_b200.weight_dequant(q, s)
    want = m(x, 0, f[:5], _causal(5))
    m.wkv_b.weight, m.wkv_b.scale = q, s
    assert torch.equal(m(x, 0, f[:5], _causal(5)), want)


def test_a_chunk_in_a_graph():
    m = _expanding(16, 128, expand_tokens=128, seed=4, length=400)
    f = _freqs(400)
    x = torch.randn(2, 300, 256, device="cuda", dtype=torch.float32).bfloat16()
    m(x[:, :200], 0, f[:200], _causal(200))
    want = m(x[:, 200:300], 200, f[200:300], _causal(100))
    static, mask = torch.zeros_like(x[:, 200:300]), _causal(100)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = m(static, 200, f[200:300], mask)
    for _ in range(3):
        static.copy_(x[:, 200:300])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_arguments_of_install_mla():
    import dsv3_b200
    for wrong in (dict(expand_from=0), dict(expand_from=-3), dict(expand_from=5, expand_tokens=0)):
        with pytest.raises(ValueError):
            dsv3_b200.install_mla(types.SimpleNamespace(MLA=object), **wrong)


@pytest.mark.parametrize("longest, factor", [(4096, 1.0), (16384, 40.0)])
def test_install_rotary(longest, factor):
    import dsv3_b200
    module = types.SimpleNamespace()
    dsv3_b200.install_rotary(module)
    args = types.SimpleNamespace(qk_rope_head_dim=64, max_seq_len=longest, beta_fast=32, beta_slow=1, rope_theta=10000.0, rope_factor=40, original_seq_len=4096)
    with torch.device("cuda"):
        f = module.precompute_freqs_cis(args)
    assert torch.equal(f, dsv3_b200.rotary_table(longest, 64, factor=factor)) and f.shape == (longest, 32)
    with pytest.raises(RuntimeError):
        module.precompute_freqs_cis(args)                   # torch's default device is the CPU
    kv = torch.randn(2, 30, 576, device="cuda")
    x = kv[..., 512:].unsqueeze(2)                          # as MLA.forward cuts it
    y = module.apply_rotary_emb(x, f[7:37])
    z = torch.view_as_complex(x.double().reshape(2, 30, 1, 32, 2)) * f[7:37].to(torch.complex128)[None, :, None]
    want = torch.view_as_real(z).flatten(-2)
    assert y.dtype == x.dtype and y.shape == x.shape
    check(y, want, want.abs() * 2.0 ** -8 + 3 * 2.0 ** -24 * 2 * x.double().abs().amax())


def test_the_operators_together():
    """A long prefix in the cache, a ragged batch of chunks behind it: table, rotation, store, read, expansion in pieces, attention, join; against the absorbed form over the same cache."""
    import dsv3_b200 as D
    heads, lens, news, page = 16, [700, 333, 64], [100, 33, 64], 64
    g = torch.Generator(device="cuda").manual_seed(5)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float32).bfloat16()  # noqa: E731
    cache = D.allocate_latent_cache(64, page)
    table = U.block_table(g, lens, page, 64)
    f = D.rotary_table(1000, 64)
    positions = torch.cat([torch.arange(n, device="cuda") for n in lens])
    seq = torch.cat([torch.full((n,), i, device="cuda") for i, n in enumerate(lens)])
    slots = table[seq, positions // page].long() * page + positions % page
    D.latent_cache_write(cache, randn(sum(lens), 576), torch.ones(512, device="cuda"), f, positions, slots)
    weight = (randn(heads, 256, 512).float() * 512 ** -0.5).bfloat16()
    q = randn(sum(news), heads, 192)
    at = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, news)])
    q_rope = D.rotary(q[..., 128:], f, at)
    cu_q, scale = offsets(news), 192 ** -0.5

    def expand(counts, first):
        latent, rope = D.latent_cache_read(cache, table[:, first // page:], offsets(counts), sum(counts))
        kv = torch.nn.functional.linear(latent, weight.flatten(0, 1)).view(-1, heads, 256)
        return kv[..., :128], rope, kv[..., 128:]

    args = expand(lens, 0)
    out, lse = D.expanded_attention(q[..., :128], q_rope, *args, scale, cu_q, offsets(lens), return_lse=True)
    want, want_lse, bound, lse_bound = reference(q[..., :128], q_rope, *args, news, lens)
    check(out, want, bound)
    check(lse, want_lse, lse_bound)
    # in two pieces: 192 tokens of each prefix (where there are as many), and the rest with the chunk
    cut = 192
    first = [min(cut, (n - m) // page * page) for n, m in zip(lens, news)]
    assert first[:2] == [cut, cut] and first[2] == 0
    a = D.expanded_attention(q[..., :128], q_rope, *expand(first, 0), scale, cu_q, offsets(first), causal=False, return_lse=True)
    shifted = table.clone()
    shifted[2] = torch.roll(table[2], cut // page)          # (the third sequence has all of its tokens in the second piece)
    latent, rope = D.latent_cache_read(cache, shifted[:, cut // page:], offsets([n - x for n, x in zip(lens, first)]), sum(lens) - sum(first))
    kv = torch.nn.functional.linear(latent, weight.flatten(0, 1)).view(-1, heads, 256)
    b = D.expanded_attention(q[..., :128], q_rope, kv[..., :128], rope, kv[..., 128:], scale, cu_q, offsets([n - x for n, x in zip(lens, first)]), return_lse=True)
    joined, joined_lse = D.attention_join([a[0], b[0]], [a[1], b[1]], return_lse=True)
    # (each part's result is rounded before they are joined)
    check(joined, want, 2 * bound + 2.0 ** -8 * want.abs() + 2.0 ** -7 * bound)
    check(joined_lse, want_lse, 4 * lse_bound + 2.0 ** -20)
    # the absorbed form: q_latent is rounded to bf16 (2^-8 of a score's terms), and so is its result before the value half of wkv_b
    q_latent = torch.einsum("thd,hdc->thc", q[..., :128], weight[:, :128])
    absorbed = D.latent_attention(q_latent, q_rope, cache, table, U.i32(lens), scale, cu_seqlens_q=cu_q)
    assert _off(torch.einsum("thc,hdc->thd", absorbed.float(), weight[:, 128:].float()), out) < 2.0 ** -6
