"""Attention over expanded keys and values, the joining of its parts and rotary positions from their definitions, in 64 bits, and how far bf16 kernels may be off."""
import math

import torch

NOPE, ROPE, VALUE = 128, 64, 128
SCALE = 192 ** -0.5
HALF_STEP = 2.0 ** -8                 # of bf16, relative to the value


def offsets(counts, device="cuda"):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def inputs(q_counts, k_counts, heads, seed=0, device="cuda"):
    """Queries, keys and values of sequences one behind the other: as a program has them, q_nope and k_nope, v cut from something wider."""
    gen = torch.Generator(device=device).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=device).bfloat16()  # noqa: E731
    q, kv = randn(sum(q_counts), heads, NOPE + ROPE), randn(sum(k_counts), heads, NOPE + VALUE)
    return q[..., :NOPE], q[..., NOPE:], kv[..., :NOPE], randn(sum(k_counts), ROPE), kv[..., NOPE:]


def reference(q_nope, q_rope, k_nope, k_rope, v, q_counts, k_counts, causal=True, scale=SCALE):
    """out, lse, and bounds for both, in 64 bits: [tokens, heads, 128], [tokens, heads].

    What bf16 results may be off by, from what is rounded where (u: a half step of bf16, e: one of fp32, 2^-24):
      scores    192 products summed in fp32, in any order: 192 e * sum |q k|; scaled: one more; the exponent's argument is rounded twice (its terms are up to 2 * |score| + |top|):
                d = softmax_scale * (193 e sum |q k| + 4 e max |x|), which a weight is off by, relatively, and twice that with its sum
      weights   u each, relative; ex2 2^-22; sums of n weights and of n products n e
      result    u of itself
    """
    e = 2.0 ** -24
    outs, lses, out_bounds, lse_bounds = [], [], [], []
    heads = q_nope.shape[1]
    a = b = 0
    for n, m in zip(q_counts, k_counts):
        q = torch.cat([q_nope[a:a + n], q_rope[a:a + n]], -1).double().transpose(0, 1)
        k = torch.cat([k_nope[b:b + m], k_rope[b:b + m, None].expand(m, heads, ROPE)], -1).double().transpose(0, 1)
        x = v[b:b + m].double().transpose(0, 1)
        score = q @ k.transpose(1, 2) * scale
        size = q.abs() @ k.abs().transpose(1, 2) * scale
        if causal:
            hidden = torch.arange(m, device=q.device)[None] > (torch.arange(n, device=q.device) + m - n)[:, None]
            score = score.masked_fill(hidden, -math.inf)
            size = size.masked_fill(hidden, 0.0)
        if m:
            top = score.amax(-1, keepdim=True)
            safe = torch.where(top == -math.inf, 0.0, top)
            weight = torch.exp(score - safe)
            total = weight.sum(-1, keepdim=True)
            weight = weight / torch.where(total == 0, 1.0, total)
            lse = (safe + total.log())[..., 0]
            d = (193 * e * size.amax(-1, keepdim=True) + 4 * e * torch.where(score == -math.inf, 0.0, score.abs()).amax(-1, keepdim=True))
            out, spread = weight @ x, weight @ x.abs()
            relative = HALF_STEP + 2 * d + 2.0 ** -21 + 2 * m * e
            out_bounds.append((HALF_STEP * out.abs() + relative * spread).transpose(0, 1))
            lse_bounds.append((d[..., 0] + 2.0 ** -21 + m * e + 4 * e * lse.abs().nan_to_num(posinf=0.0)).transpose(0, 1))
        else:
            out, lse = x.new_zeros(heads, n, VALUE), x.new_full((heads, n), -math.inf)
            out_bounds.append(torch.zeros_like(out).transpose(0, 1))
            lse_bounds.append(torch.zeros_like(lse).transpose(0, 1))
        outs.append(out.transpose(0, 1))
        lses.append(lse.transpose(0, 1))
        a, b = a + n, b + m
    return tuple(torch.cat(t) for t in (outs, lses, out_bounds, lse_bounds))


def check(got, want, bound, what="out"):
    """Equal where `want` is infinite or NaN, elsewhere within `bound` (a value below bf16's normal ones counts as zero)."""
    got = got.double()
    assert got.shape == want.shape
    odd = ~want.isfinite()
    assert torch.equal(got[odd].nan_to_num(nan=1.25), want[odd].nan_to_num(nan=1.25)), f"{what}: infinities or NaN differ"
    far = ((got - want).abs() - bound - 2.0 ** -126)[~odd]
    assert not bool((far.isnan() | (far > 0)).any()), f"{what}: {int((far > 0).sum())} values off, worst by {float(far.max()):.3g} beyond their bound; NaN {int(far.isnan().sum())}"
