"""install_mla: MLA.forward on the 8-bit latent cache, prompt, steps, drafts in a tree and what is kept of them.

The module is restated here with plain bf16 Linears (model.py:396-444 for its members).  Two comparisons.  With the same 8-bit tokens: everything behind the
cache in fp32 from what the cache holds; the two differ by the roundings of bf16 at q_latent, at the attention's result and at the head's output (each 2^-9
relative RMS of values that are later summed, 2^-8 together) and the attention's own 2^-8.  Against unquantised tokens: a latent in e4m3 is off by up to 2^-4 of itself,
evenly, that is 2.6 % RMS (2^-4 / sqrt 3 over significands from 1 to 2); it enters the result once as a value and once through scores of about one unit's spread, 3.7 %
together, here held to 6 %."""
import math
import types

import pytest
import torch

import latent_util as U

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _bf16_default():
    import dsv3_b200
    torch.set_default_dtype(torch.bfloat16)
    yield
    torch.set_default_dtype(torch.float32)
    dsv3_b200.check_device_status()


class _Linear:
    def __init__(self, n, k, gen, size=None):
        self.weight = (torch.randn(n, k, generator=gen, device="cuda", dtype=torch.float32) * (size or k ** -0.5)).bfloat16()
        self.scale = None

    def __call__(self, x):
        return torch.nn.functional.linear(x, self.weight)


class _Norm:
    def __init__(self, n, gen):
        self.weight, self.eps = (1 + 0.1 * torch.randn(n, generator=gen, device="cuda", dtype=torch.float32)).bfloat16(), 1e-6

    def __call__(self, x):
        return torch.nn.functional.rms_norm(x, (x.size(-1),), self.weight, self.eps)


def _model(heads, q_lora, batch=3, length=200, seed=0):
    class MLA:
        def __init__(self):
            g = torch.Generator(device="cuda").manual_seed(seed)
            self.dim, self.n_local_heads, self.q_lora_rank, self.kv_lora_rank = 256, heads, q_lora, 512
            self.qk_nope_head_dim, self.qk_rope_head_dim, self.v_head_dim = 128, 64, 128
            if q_lora:
                self.wq_a, self.q_norm, self.wq_b = _Linear(q_lora, 256, g), _Norm(q_lora, g), _Linear(heads * 192, q_lora, g)
            else:
                self.wq = _Linear(heads * 192, 256, g)
            self.wkv_a, self.kv_norm, self.wkv_b, self.wo = _Linear(576, 256, g), _Norm(512, g), _Linear(heads * 256, 512, g), _Linear(256, heads * 128, g)
            self.softmax_scale = 192 ** -0.5
            self.kv_cache = torch.zeros(batch, length, 512, device="cuda")

        def __call__(self, *a):
            return self.forward(*a)
    module = types.SimpleNamespace(MLA=MLA, block_size=128)
    import dsv3_b200
    dsv3_b200.install_mla(module)
    return MLA()


def _freqs(n):
    angle = torch.arange(n, device="cuda", dtype=torch.float32)[:, None] * 10000.0 ** (-torch.arange(32, device="cuda", dtype=torch.float32) / 32)
    return torch.polar(torch.ones_like(angle), angle)


def _rotated(x, f):
    z = torch.view_as_complex(x.float().reshape(*x.shape[:-1], 32, 2)) * f
    return torch.view_as_real(z).flatten(-2)


def _queries(m, x, f):
    q = m.wq(x) if not m.q_lora_rank else m.wq_b(m.q_norm(m.wq_a(x)))
    q = q.view(*x.shape[:2], m.n_local_heads, 192).float()
    w = m.wkv_b.weight.view(m.n_local_heads, 256, 512).float()
    return torch.einsum("bshd,hdc->bshc", q[..., :128], w[:, :128]), _rotated(q[..., 128:], f[None, :, None])


def _result(m, ql, qr, c, k, seen):
    score = (torch.einsum("bshc,btc->bhst", ql, c) + torch.einsum("bshr,btr->bhst", qr, k)) * m.softmax_scale
    p = score.masked_fill(~seen[:, None], -math.inf).softmax(-1)
    o = torch.einsum("bhst,btc->bshc", p, c)
    w = m.wkv_b.weight.view(m.n_local_heads, 256, 512).float()
    return torch.nn.functional.linear(torch.einsum("bshc,hdc->bshd", o, w[:, 128:]).flatten(2), m.wo.weight.float())


def _tokens(m, x, f):
    kv = m.wkv_a(x).float()
    c = kv[..., :512] * torch.rsqrt(kv[..., :512].square().mean(-1, keepdim=True) + 1e-6) * m.kv_norm.weight.float()
    return c, _rotated(kv[..., 512:], f[None])


def _cached(m, batch, n):
    """The first n tokens of every sequence as the cache holds them."""
    import dsv3_b200
    cache = dsv3_b200.mla_cache(m)
    latent, rope = dsv3_b200.latent_cache_read(cache.pool, cache.block_table[:batch], U.offsets([n] * batch), batch * n)
    return latent.float().view(batch, n, 512), rope.float().view(batch, n, 64)


def _off(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("heads, q_lora", [(4, 0), (16, 128)])
def test_prompt_and_steps(heads, q_lora):
    m = _model(heads, q_lora)
    g = torch.Generator(device="cuda").manual_seed(1)
    f = _freqs(200)
    x = torch.randn(2, 90, 256, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    at = 0
    for n in (70, 1, 1, 17, 1):                                             # a prompt, steps, a chunk, a step
        mask = torch.full((n, n), float("-inf"), device="cuda").triu_(1) if n > 1 else None
        y = m(x[:, at:at + n], at, f[at:at + n], mask)
        end = at + n
        seen = torch.arange(end, device="cuda") <= torch.arange(at, end, device="cuda")[:, None]
        ql, qr = _queries(m, x[:, at:end], f[at:end])
        assert _off(y, _result(m, ql, qr, *_cached(m, 2, end), seen[None])) < 2.0 ** -7
        assert _off(y, _result(m, ql, qr, *_tokens(m, x[:, :end], f[:end]), seen[None])) < 0.06
        at = end


def test_drafts_in_a_tree_and_what_is_kept_of_them():
    import dsv3_b200
    m = _model(16, 0)
    g = torch.Generator(device="cuda").manual_seed(2)
    f = _freqs(200)
    x = torch.randn(2, 60, 256, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    m(x[:, :50], 0, f[:50], torch.full((50, 50), float("-inf"), device="cuda").triu_(1))
    parent = [-1, -1, 0, 0, 1, 2, 4]
    words, depth = [], []
    for i, p in enumerate(parent):
        words.append((words[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    d = torch.tensor(depth, device="cuda")
    drafts = torch.randn(2, 7, 256, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    y = m(drafts, 50, f[50 + d], torch.tensor([words] * 2, device="cuda"))
    seen = torch.ones(7, 57, dtype=torch.bool, device="cuda")
    seen[:, 50:] = torch.tensor([[bool(w >> j & 1) for j in range(7)] for w in words], device="cuda")
    ql, qr = _queries(m, drafts, f[50 + d])
    assert _off(y, _result(m, ql, qr, *_cached(m, 2, 57), seen[None])) < 2.0 ** -7
    # nodes 1, 4, 6 of the first sequence and 0, 3 of the second are accepted
    cache = dsv3_b200.mla_cache(m)
    before = _cached(m, 2, 57)
    dsv3_b200.latent_cache_keep(cache.pool, cache.block_table[:2], U.i32([50, 50]), U.i32([[1, 4, 6], [0, 3, 0]]), U.i32([3, 2]))
    after = _cached(m, 2, 57)
    for plane in (0, 1):
        assert torch.equal(after[plane][0, 50:53], before[plane][0, [51, 54, 56]]) and torch.equal(after[plane][1, 50:52], before[plane][1, [50, 53]])
        assert torch.equal(after[plane][:, :50], before[plane][:, :50])
    # the next token of a sequence whose accepted branch lies behind its prefix equals that of one that never drafted
    plain = _model(16, 0)
    plain(x[:1, :50], 0, f[:50], torch.full((50, 50), float("-inf"), device="cuda").triu_(1))
    plain(drafts[:1, [1, 4, 6]], 50, f[50:53], torch.full((3, 3), float("-inf"), device="cuda").triu_(1))
    a, b = m(x[:1, 50:51], 53, f[53:54], None), plain(x[:1, 50:51], 53, f[53:54], None)
    assert _off(a, b) < 2.0 ** -9


def test_fp8_projection_of_the_latents():
    """wkv_b in the checkpoint's block-scaled FP8."""
    import dsv3_b200
    m = _model(4, 0, seed=3)
    q, s = dsv3_b200.weight_quant(m.wkv_b.weight)
    f = _freqs(10)
    x = torch.randn(1, 5, 256, device="cuda", dtype=torch.float32).bfloat16()
    mask = torch.full((5, 5), float("-inf"), device="cuda").triu_(1)
    m.wkv_b.weight = dsv3_b200.weight_dequant(q, s)
    want = m(x, 0, f[:5], mask)
    m.wkv_b.weight, m.wkv_b.scale = q, s
    assert torch.equal(m(x, 0, f[:5], mask), want)


def test_a_step_in_a_graph():
    m = _model(16, 128, seed=4)
    f = _freqs(200)
    x = torch.randn(2, 66, 256, device="cuda", dtype=torch.float32).bfloat16()
    m(x[:, :64], 0, f[:64], torch.full((64, 64), float("-inf"), device="cuda").triu_(1))
    want = m(x[:, 64:65], 64, f[64:65], None)
    static = torch.zeros_like(x[:, 64:65])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = m(static, 64, f[64:65], None)
    for _ in range(3):
        static.copy_(x[:, 64:65])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_what_the_seam_refuses():
    m = _model(4, 0)
    f = _freqs(200)
    x = torch.zeros(1, 3, 256, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="mask"):
        m(x, 0, f[:3], None)
    with pytest.raises(ValueError, match="do not fit"):
        m(x[:, :1], 200, f[:1], None)
    with pytest.raises(ValueError, match="do not fit"):
        m(x[:, :1].expand(4, 1, 256), 0, f[:1], None)
    m.kv_lora_rank = 256
    with pytest.raises(NotImplementedError, match="kv_lora_rank"):
        m(x[:, :1], 0, f[:1], None)
