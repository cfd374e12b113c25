"""The 8-bit latent cache and the attention over it, plainly and in 64 bits, for the tests of their kernels."""
import math

import torch

LATENT, ROPE = 512, 64


def dsv3():
    import dsv3_b200
    return dsv3_b200


def make_cache(gen, n_pages, page, spread=1.0):
    """A pool of tokens as latent_cache_write leaves them; `spread`: the latents' largest size against the smallest (log-uniform per token)."""
    latent = torch.randn(n_pages, page, LATENT, generator=gen, device="cuda", dtype=torch.float32)
    latent *= spread ** (torch.rand(n_pages, page, 1, generator=gen, device="cuda") - 0.5)
    rope = torch.randn(n_pages, page, ROPE, generator=gen, device="cuda", dtype=torch.float32)
    scale = least_power(latent.double().abs().amax(-1).clamp_min(1e-4)).float()
    return dsv3().LatentCache((latent / scale[..., None]).to(torch.float8_e4m3fn), (rope / scale[..., None]).bfloat16(), scale)


def least_power(top):
    """The least power of two s with top <= 448 s."""
    e = torch.floor(torch.log2(top / 448)) - 1
    s = torch.exp2(e)
    for _ in range(3):
        s = torch.where(top > 448 * s, 2 * s, s)
    return s


def block_table(gen, lens, page, n_pages, spare=0):
    """Shuffled pages; entries behind a sequence's last page name none of the pool."""
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) + spare
    names = torch.randperm(n_pages, generator=gen, device="cuda").tolist()
    assert sum(need) <= n_pages
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(names[at:at + n], dtype=torch.int32)
        at += n
    return table.cuda()


def poison_rest(cache, table, lens):
    """Everything of the pool that no sequence's tokens lie in becomes NaN bytes, values and scales."""
    page = cache.scale.shape[1]
    used = torch.zeros(cache.scale.numel(), dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(n):
            name = int(table[b, p // page])
            if 0 <= name < cache.scale.shape[0]:
                used[name * page + p % page] = True
    rest = ~used.cuda()
    cache.latent.view(torch.uint8).view(-1, LATENT)[rest] = 0x7F
    cache.rope.view(-1, ROPE)[rest] = math.nan
    cache.scale.view(-1)[rest] = math.nan


def tokens_of(cache, table, b, n):
    """Latent and rotated values of the first n tokens of sequence b in 64 bits, and which of them are there."""
    page = cache.scale.shape[1]
    p = torch.arange(n, device="cuda")
    names = table[b].long()[p // page]
    there = (names >= 0) & (names < cache.scale.shape[0])
    slot = torch.where(there, names * page + p % page, 0)
    s = cache.scale.view(-1)[slot].double()[:, None]
    c = cache.latent.view(-1, LATENT)[slot].double() * s
    k = cache.rope.view(-1, ROPE)[slot].double() * s
    return c, k, there


def attention(q_latent, q_rope, cache, table, lens, counts, scale, tree=None):
    """out, lse and a bound of what rounding may make of out, per element, for packed queries.

    The bound: a result in bf16 is off by half a step, 2^-8 of it.  A weight enters the second product with 8 significant bits, off by 2^-8 of
    itself, or, where it is small, by at most a step of 2^-13 (half of one from rounding, half from the offset before it) on a scale where the largest
    weight is at least 2^5.  The token of that weight has a latent above 224 as stored, no token one above 448: a step on any token is at most
    2^-13 * 448 / (2^5 * 224) = 2^-17 of `top`, the largest product of a weight and its token's largest latent.  n of them add up to n of that at most; the offsets
    are even over a step, which makes an error's mean zero, and then a sum of n > 64 is above 16 sqrt(n) 2^-18 with a chance of 2 exp(-32) (Hoeffding, on
    errors between -2^-17 and 2^-17: 2 exp(-2 (16 sqrt(n) 2^-18)^2 / (n (2^-16)^2))).  A score is a sum of 576
    products in fp32, off by 576 * 2^-24 of the sum of their sizes, and its error is the weight's relative one; as much again comes from the exponent's
    argument, which has 24 bits of at most the largest score.  A weight's error e comes twice, in the sum and in its divisor; 2^-14 stands for
    the exponential, the sums and the division."""
    outs, lses, bounds = [], [], []
    row = 0
    for b, (n, t) in enumerate(zip(lens, counts)):
        c, k, there = tokens_of(cache, table, b, n)
        for i in range(t):
            ql, qr = q_latent[row].double(), q_rope[row].double()
            seen = there.clone()
            p = torch.arange(n, device="cuda")
            j = p - (n - t)
            if tree is None:
                seen &= j <= i
            else:
                word = int(tree[row]) & (1 << 64) - 1
                bits = torch.tensor([bool(word >> max(0, int(v)) & 1) if int(v) < 64 else False for v in j.clamp(-1).tolist()], dtype=torch.bool, device="cuda")
                seen &= (j < 0) | bits
            row += 1
            if not bool(seen.any()):
                outs.append(torch.zeros(ql.shape[0], LATENT, dtype=torch.float64, device="cuda"))
                lses.append(torch.full((ql.shape[0],), -math.inf, dtype=torch.float64, device="cuda"))
                bounds.append(torch.zeros_like(outs[-1]))
                continue
            cs, ks = c[seen], k[seen]
            score = (ql @ cs.T + qr @ ks.T) * scale
            size = (ql.abs() @ cs.abs().T + qr.abs() @ ks.abs().T) * abs(scale)
            lse = torch.logsumexp(score, -1)
            w = torch.exp(score - lse[:, None])
            o = w @ cs
            e = 2.0 ** -14 + 2 * 576 * 2.0 ** -24 * size.amax(-1, keepdim=True)
            spread_of = w @ cs.abs()
            # small weights: a weight enters times its token's scale, so what counts is the largest product of the two
            top = (w * cs.abs().amax(-1)).amax(-1, keepdim=True)
            many = int(seen.sum())
            bounds.append(2.0 ** -8 * o.abs() + (2.0 ** -8 + 2 * e) * spread_of + min(many * 2.0 ** -17, 16 * many ** 0.5 * 2.0 ** -18) * top)
            outs.append(o)
            lses.append(lse)
    shape = (0, q_latent.shape[1])
    if not outs:
        return (torch.zeros(*shape, LATENT, dtype=torch.float64, device="cuda"), torch.zeros(shape, dtype=torch.float64, device="cuda"),
                torch.zeros(*shape, LATENT, dtype=torch.float64, device="cuda"))
    return torch.stack(outs), torch.stack(lses), torch.stack(bounds)


def assert_attention(got, lse, want, want_lse, bound):
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    fine = ~torch.isnan(want)
    over = ((g - want).abs() - bound)[fine]
    assert not over.numel() or over.max().item() <= 0, f"worst excess {over.max().item():.3e}, worst ratio {((g - want).abs() / bound.clamp_min(1e-30))[fine].max().item():.3f}"
    if lse is not None:
        a, b = lse.double(), want_lse
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(a == -math.inf, b == -math.inf)
        fin = torch.isfinite(b)
        # scores as above (here bounded at 2^-13 of ordinary sizes), and the sum's logarithm
        assert ((a - b).abs()[fin] <= 2.0 ** -12 * (1 + b.abs()[fin])).all(), (a - b).abs()[fin].max()


def causal_counts(lens, drafts):
    return [min(n, drafts) for n in lens]


def offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def random_tree(gen, nodes):
    bits = []
    for i in range(nodes):
        parent = int(torch.randint(-1, i, (1,), generator=gen)) if i else -1
        bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
    return [b - (1 << 64) if b >> 63 else b for b in bits]
