"""The latent cache of multi-head latent attention in 8 bits, and the attention that reads it, as cases that can be timed.

A cached token is 512 e4m3 values of its normalised latent, one power-of-two scale for them and 64 rotated bf16 values that are
held divided by the scale; tokens lie in pages of a pool, a sequence's pages are named by a row of its block table.

  write      norm, rotation and quantisation of new tokens into their slots of the pool
  read       the tokens of several sequences, back in bf16 and packed
  keep       after drafted tokens have been verified, the accepted ones close ranks behind their sequence's prefix
  attention  absorbed queries over the cache: one token, a chain or tree of drafted tokens, or a chunk of a prompt to a sequence

`listed` and `draw` give the cases, `prepare` what a serving program holds before the call, `run` one pass, `work` what it cannot
do without, `exact` the results from the definitions in 64 bits.  Dimensions are those of the models that bench.py and the tests use:
latents of 512 with 64 rotated values, 128 or 16 heads, and one rank's share of 128 heads under tensor parallelism.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

LATENT, ROPE = 512, 64
SOFTMAX_SCALE = 192 ** -0.5           # of heads of 128 + 64
EPS = 1e-6
FLOOR = 1e-4                          # of a token's largest latent


# ---------------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding sequence: its new token goes to the cache
        {"name": "write_1", "kind": "write", "tokens": 1, "page": 64, "weight": "bf16"},
        # a batch of prompts, with a few padded places that no slot belongs to
        {"name": "write_prefill_16001", "kind": "write", "tokens": 16001, "page": 64, "weight": "fp32"},
        # a cached prefix of one sequence is read back for the next chunk of its prompt
        {"name": "read_prefix_777", "kind": "read", "seqs": 1, "longest": 777, "page": 16},
        # the prefixes of a batch of conversations
        {"name": "read_prefixes_32", "kind": "read", "seqs": 32, "longest": 8192, "page": 64},
        # drafted tokens of one sequence have been verified
        {"name": "keep_1", "kind": "keep", "seqs": 1, "drafts": 8, "longest": 1000, "page": 64},
        # ... of a batch, trees of 64 nodes
        {"name": "keep_128", "kind": "keep", "seqs": 128, "drafts": 64, "longest": 1000, "page": 16},
        # the first tokens of an answer, one rank of eight: where latency counts
        {"name": "attention_1_short", "kind": "attention", "seqs": 1, "heads": 16, "drafts": 1, "longest": 137, "page": 64, "ragged": False,
         "mask": "causal", "lse": False},
        # an ordinary decode step of a batch, one rank of eight, ragged lengths
        {"name": "attention_decode_64", "kind": "attention", "seqs": 64, "heads": 16, "drafts": 1, "longest": 8192, "page": 64, "ragged": True,
         "mask": "causal", "lse": False},
        # trees of up to 13 drafted tokens, ragged, pages of 16
        {"name": "attention_tree_24", "kind": "attention", "seqs": 24, "heads": 16, "drafts": 13, "longest": 4001, "page": 16, "ragged": True,
         "mask": "tree", "lse": True},
        # a decode step where every rank holds all heads: the arithmetic is what counts
        {"name": "attention_heads_128", "kind": "attention", "seqs": 32, "heads": 128, "drafts": 1, "longest": 8192, "page": 64, "ragged": False,
         "mask": "causal", "lse": False},
        # one long conversation with a chain of drafted tokens
        {"name": "attention_long_131072", "kind": "attention", "seqs": 1, "heads": 16, "drafts": 4, "longest": 131072, "page": 128, "ragged": False,
         "mask": "causal", "lse": True},
        # a chunk of a prompt behind its cached beginning
        {"name": "attention_chunk_515", "kind": "attention", "seqs": 1, "heads": 16, "drafts": 515, "longest": 4099, "page": 64, "ragged": False,
         "mask": "causal", "lse": False},
    ]


def _spread(rng, low, high):
    """A whole number of the range, its logarithm evenly spread."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    kind = rng.choice(["write", "read", "keep", "attention", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "write":
        return {"kind": kind, "tokens": _spread(rng, 1, 16384), "page": page, "weight": rng.choice(["bf16", "fp32"])}
    if kind == "read":
        seqs = _spread(rng, 1, 48)
        return {"kind": kind, "seqs": seqs, "longest": _spread(rng, 1, 8192), "page": page}
    if kind == "keep":
        return {"kind": kind, "seqs": _spread(rng, 1, 128), "drafts": rng.randint(2, 64), "longest": _spread(rng, 1, 1000), "page": page}
    mask = rng.choice(["causal", "causal", "tree"])
    heads = rng.choice([5, 16, 16, 32, 64, 128])
    drafts = rng.choice([1, 1, _spread(rng, 1, 32 if mask == "tree" else 515)])
    longest = _spread(rng, drafts, 65536)
    # not more than 32 sequences of 8192 tokens with 128 queries each, nor than 2^19 tokens in the cache
    most = max(1, min(64, (1 << 25) // (longest * heads * drafts), (1 << 19) // longest))
    return {"kind": kind, "seqs": _spread(rng, 1, most), "heads": heads, "drafts": drafts, "longest": longest, "page": page,
            "ragged": rng.random() < 0.7, "mask": mask, "lse": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------------
# What a serving program holds before the call
# ---------------------------------------------------------------------------------------------------------------------
def _quantised(latent, rope):
    """The three planes of cached tokens: latent [..., 512] and rope [..., 64] in fp32."""
    top = latent.abs().amax(-1).clamp_min(FLOOR)
    m, e = torch.frexp(top / 448)
    scale = torch.ldexp(torch.ones_like(top), torch.where(m > 0.5, e, e - 1))     # least power of two with top <= 448 scale
    return (latent / scale[..., None]).to(torch.float8_e4m3fn), (rope / scale[..., None]).bfloat16(), scale


def _pool(gen, pages, page):
    """A pool full of other sequences' tokens.  (The latents of ordinary tokens are evenly sized after their norm.)"""
    latent = torch.randn(pages, page, LATENT, generator=gen, device="cuda")
    rope = torch.randn(pages, page, ROPE, generator=gen, device="cuda")
    return _quantised(latent, rope)


def _lengths(seqs, longest, ragged):
    """Lengths on the host; ragged ones spread evenly from an eighth of the longest on, the first the longest."""
    if not ragged:
        return [longest] * seqs
    return [longest] + [max(1, round(longest * (0.125 + 0.875 * (i * 0.6180339887 % 1)))) for i in range(1, seqs)]


def _block_table(gen, lens, page):
    """Pages in the order that a busy pool hands them out; one sequence's spare entries name no page."""
    width = -(-max(lens) // page)
    need = [-(-n // page) for n in lens]
    names = torch.randperm(sum(need), generator=gen, device="cuda").to(torch.int32).tolist()
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = names[at:at + n]
        at += n
    return torch.from_numpy(table).cuda(), sum(need)


def _offsets(counts):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()


def _tree(rng, nodes):
    """A tree of drafted tokens: for each node the bits of itself and its ancestors."""
    bits = []
    for i in range(nodes):
        parent = int(rng.integers(-1, i)) if i else -1          # -1: the last verified token
        bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
    return bits


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind, page = case["kind"], case["page"]
    if kind == "write":
        n = case["tokens"]
        pages = -(-(n + n // 4 + 8) // page)
        latent, rope, scale = _pool(gen, pages, page)
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:n]
        if n > 128:
            slots[5::64] = -1                                   # padded places of the batch
        angle = torch.rand(4096, ROPE // 2, generator=gen, device="cuda") * (2 * math.pi)
        weight = 1 + 0.1 * torch.randn(LATENT, generator=gen, device="cuda")
        return {"case": case, "latent": latent, "rope": rope, "scale": scale, "slots": slots,
                "kv": (torch.randn(n, LATENT + ROPE, generator=gen, device="cuda") * 1.7).bfloat16(),
                "weight": weight.bfloat16() if case["weight"] == "bf16" else weight,
                "freqs": torch.polar(torch.ones_like(angle), angle),
                "positions": torch.randint(0, 4096, (n,), generator=gen, device="cuda")}
    if kind == "read":
        lens = _lengths(case["seqs"], case["longest"], True)
        table, pages = _block_table(gen, lens, page)
        latent, rope, scale = _pool(gen, pages, page)
        return {"case": case, "latent": latent, "rope": rope, "scale": scale, "table": table, "offsets": _offsets(lens), "total": sum(lens)}
    if kind == "keep":
        lens = _lengths(case["seqs"], case["longest"], True)
        table, pages = _block_table(gen, [n + case["drafts"] for n in lens], page)
        latent, rope, scale = _pool(gen, pages, page)
        path, count = np.zeros((len(lens), case["drafts"]), np.int32), np.zeros(len(lens), np.int32)
        for i in range(len(lens)):
            n = int(rng.integers(1, max(2, case["drafts"] // 2)))             # accepted tokens: the first branch, then nodes of a later one
            straight = int(rng.integers(0, n))
            path[i, :n] = np.concatenate([np.arange(straight), np.sort(rng.choice(np.arange(n, case["drafts"]), n - straight, replace=False))])
            count[i] = n
        return {"case": case, "latent": latent, "rope": rope, "scale": scale, "table": table,
                "first": torch.tensor(lens, dtype=torch.int32, device="cuda"), "path": torch.from_numpy(path).cuda(), "count": torch.from_numpy(count).cuda()}
    seqs, heads = case["seqs"], case["heads"]
    lens = _lengths(seqs, case["longest"], case["ragged"])
    counts = [min(n, case["drafts"] if not case["ragged"] else max(1, case["drafts"] - i % 3)) for i, n in enumerate(lens)]
    table, pages = _block_table(gen, lens, page)
    latent, rope, scale = _pool(gen, pages, page)
    total = sum(counts)
    q = torch.randn(total, heads, LATENT, generator=gen, device="cuda") * 0.5
    # a sequence's first token draws a good part of many heads' attention
    lead = torch.randn(LATENT, generator=gen, device="cuda")
    q += lead * 0.15 * torch.rand(total, heads, 1, generator=gen, device="cuda")
    sink = _quantised(lead.expand(seqs, LATENT), torch.zeros(seqs, ROPE, device="cuda"))
    at = table[:, 0].long()
    latent.view(torch.uint8)[at, 0] = sink[0].view(torch.uint8)
    rope[at, 0] = sink[1]
    scale[at, 0] = sink[2]
    tree = None
    if case["mask"] == "tree":
        tree = torch.tensor([b - (1 << 64) if b >> 63 else b for n in counts for b in _tree(rng, n)], dtype=torch.int64, device="cuda")
    return {"case": case, "latent": latent, "rope": rope, "scale": scale, "table": table, "tree": tree,
            "q_latent": q.bfloat16(), "q_rope": torch.randn(total, heads, ROPE, generator=gen, device="cuda").bfloat16(),
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "offsets": _offsets(counts),
            "longest": max(lens), "drafts": max(counts)}


# ---------------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------------
def _package():
    path = os.path.join(os.getcwd(), "deepseek-v3_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import dsv3_b200
    return dsv3_b200


def _run_own(s):
    ops, kind = _package(), s["case"]["kind"]
    cache = ops.LatentCache(s["latent"], s["rope"], s["scale"])
    if kind == "write":
        ops.latent_cache_write(cache, s["kv"], s["weight"], s["freqs"], s["positions"], s["slots"], EPS)
        return cache.latent, cache.rope, cache.scale
    if kind == "read":
        return ops.latent_cache_read(cache, s["table"], s["offsets"], s["total"])
    if kind == "keep":
        ops.latent_cache_keep(cache, s["table"], s["first"], s["path"], s["count"])
        return cache.latent, cache.rope, cache.scale
    return ops.latent_attention(s["q_latent"], s["q_rope"], cache, s["table"], s["lens"], SOFTMAX_SCALE, cu_seqlens_q=s["offsets"],
                                tree_mask=s["tree"], return_lse=s["case"]["lse"])


def _write(s):
    kv = s["kv"].float()
    latent, rope = kv[:, :LATENT], kv[:, LATENT:]
    latent = latent * torch.rsqrt(latent.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    f = s["freqs"][s["positions"]]
    even, odd = rope[:, 0::2], rope[:, 1::2]
    rope = torch.stack([even * f.real - odd * f.imag, even * f.imag + odd * f.real], -1).flatten(1)
    q, r, scale = _quantised(latent, rope)
    there = s["slots"] >= 0
    at = s["slots"][there]
    s["latent"].view(torch.uint8).view(-1, LATENT)[at] = q[there].view(torch.uint8)
    s["rope"].view(-1, ROPE)[at] = r[there]
    s["scale"].view(-1)[at] = scale[there]
    return s["latent"], s["rope"], s["scale"]


def _slots_of(table, seq, position, page):
    return table[seq, position // page].long() * page + position % page


def _read(s):
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(s["offsets"].long(), row, right=True) - 1
    at = _slots_of(s["table"], seq, row - s["offsets"].long()[seq], s["case"]["page"])
    scale = s["scale"].view(-1)[at][:, None]
    return ((s["latent"].view(-1, LATENT)[at].float() * scale).bfloat16(), (s["rope"].view(-1, ROPE)[at].float() * scale).bfloat16())


def _keep(s):
    step = torch.arange(s["path"].shape[1], device="cuda")
    there = step < s["count"][:, None]
    seq = torch.arange(len(there), device="cuda")[:, None].expand_as(there)[there]
    first = s["first"].long()[:, None]
    page = s["case"]["page"]
    src = _slots_of(s["table"], seq, (first + s["path"].long())[there], page)
    dst = _slots_of(s["table"], seq, (first + step)[there], page)
    for_bytes = s["latent"].view(torch.uint8).view(-1, LATENT)
    for_bytes[dst] = for_bytes[src]
    s["rope"].view(-1, ROPE)[dst] = s["rope"].view(-1, ROPE)[src]
    s["scale"].view(-1)[dst] = s["scale"].view(-1)[src]
    return s["latent"], s["rope"], s["scale"]


def _attention(s):
    page, longest, drafts = s["case"]["page"], s["longest"], s["drafts"]
    lens, offsets = s["lens"].long(), s["offsets"].long()
    position = torch.arange(longest, device="cuda")
    seq = torch.arange(len(lens), device="cuda")[:, None]
    at = _slots_of(s["table"], seq, position.expand(len(lens), -1), page).clamp_min(0)
    scale = s["scale"].view(-1)[at][..., None]
    latent = s["latent"].view(-1, LATENT)[at].float() * scale
    rope = s["rope"].view(-1, ROPE)[at].float() * scale
    # queries padded to the same number for every sequence
    counts = offsets[1:] - offsets[:-1]
    step = torch.arange(drafts, device="cuda")
    there = step < counts[:, None]
    row = torch.where(there, offsets[:-1, None] + step, 0)
    score = torch.einsum("bthc,bsc->bths", s["q_latent"][row].float(), latent)
    score += torch.einsum("bthc,bsc->bths", s["q_rope"][row].float(), rope)
    score *= SOFTMAX_SCALE
    draft = position - (lens - counts)[:, None]                       # which drafted token a position is; below zero: the prefix
    if s["tree"] is None:
        seen = draft[:, None] <= step[:, None]
    else:
        bit = (s["tree"][row][..., None] >> draft[:, None].clamp(0, 63)) & 1
        seen = (draft[:, None] < 0) | (bit != 0)
    seen &= (position < lens[:, None])[:, None]
    score.masked_fill_(~seen[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = torch.exp(score.sub_(top))
    total = weight.sum(-1, keepdim=True)
    out = torch.einsum("bths,bsc->bthc", weight, latent) / torch.where(total == 0, 1.0, total)
    out = out[there].bfloat16()
    return (out, (top + total.log())[..., 0][there]) if s["case"]["lse"] else out


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    return _write(state) if kind == "write" else _read(state) if kind == "read" else _keep(state) if kind == "keep" else _attention(state)


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
_TOKEN = LATENT + 2 * ROPE + 4        # bytes of a cached token


def _expected(case):
    """Sum of the lengths: ragged ones are even over an eighth of the longest to all of it."""
    n, longest = case["seqs"], case["longest"]
    return longest + (n - 1) * longest * (0.5625 if case.get("ragged", True) else 1.0)


def work(case):
    kind = case["kind"]
    if kind == "write":
        n = case["tokens"]
        return {"bytes": n * (2 * (LATENT + ROPE) + 16 + 8 * (ROPE // 2) + _TOKEN), "flops": n * (8 * LATENT + 8 * ROPE)}
    if kind == "read":
        n = _expected(case)
        return {"bytes": n * (_TOKEN + 2 * (LATENT + ROPE)), "flops": n * (LATENT + ROPE)}
    if kind == "keep":
        n = case["seqs"] * max(1.0, case["drafts"] / 8)                     # about half of the accepted ones move
        return {"bytes": n * 2 * _TOKEN, "flops": 0}
    tokens = _expected(case)
    drafts = max(1, case["drafts"] - (1 if case["ragged"] else 0))
    rows = case["seqs"] * drafts * case["heads"]
    seen = max(tokens - case["seqs"] * drafts / 2, 1)
    return {"bytes": tokens * _TOKEN + rows * 2 * (2 * LATENT + ROPE), "flops": 2 * seen * drafts * case["heads"] * (2 * LATENT + ROPE)}


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits, a sequence at a time
# ---------------------------------------------------------------------------------------------------------------------
def _exact_write(s):
    x = s["kv"].double()
    c = x[:, :LATENT]
    c = c / torch.sqrt((c * c).sum(-1, keepdim=True) / LATENT + EPS) * s["weight"].double()
    z = torch.view_as_complex(x[:, LATENT:].reshape(len(x), -1, 2)) * s["freqs"].to(torch.complex128)[s["positions"]]
    r = torch.view_as_real(z).reshape(len(x), -1)
    scale = torch.exp2(torch.ceil(torch.log2(c.abs().amax(-1).clamp_min(FLOOR) / 448)))
    planes = [s["latent"].double().reshape(-1, LATENT), s["rope"].double().reshape(-1, ROPE), s["scale"].double().reshape(-1)]
    # the values that 8 and 16 bits stand for are the nearest ones: what is compared is how near
    for plane, new in zip(planes, (c / scale[:, None], r / scale[:, None], scale)):
        keep = s["slots"] >= 0
        plane[s["slots"][keep]] = new[keep]
    return tuple(p.reshape(s[k].shape) for p, k in zip(planes, ("latent", "rope", "scale")))


def _exact_tokens(s, b, n):
    """Latents and rotated values of a sequence's first n tokens."""
    page = s["case"]["page"]
    pages = s["table"][b, :-(-n // page)].long()
    scale = s["scale"][pages].double().reshape(-1)[:n, None]
    return s["latent"][pages].double().reshape(-1, LATENT)[:n] * scale, s["rope"][pages].double().reshape(-1, ROPE)[:n] * scale


def _exact_keep(s):
    planes = [s["latent"].double(), s["rope"].double(), s["scale"].double()]
    page, table = s["case"]["page"], s["table"].tolist()
    first, path, count = s["first"].tolist(), s["path"].tolist(), s["count"].tolist()
    slot = lambda b, p: table[b][p // page] * page + p % page  # noqa: E731
    src = torch.tensor([slot(b, first[b] + path[b][j]) for b in range(len(first)) for j in range(count[b])], device="cuda")
    dst = torch.tensor([slot(b, first[b] + j) for b in range(len(first)) for j in range(count[b])], device="cuda")
    for i, p in enumerate(planes):
        flat = p.reshape(len(s["scale"].reshape(-1)), -1)
        new = flat.clone()
        new[dst] = flat[src]
        planes[i] = new.reshape(p.shape)
    return tuple(planes)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "write":
        return _exact_write(s)
    if kind == "keep":
        return _exact_keep(s)
    offsets = s["offsets"].tolist()
    if kind == "read":
        parts = [_exact_tokens(s, b, offsets[b + 1] - offsets[b]) for b in range(case["seqs"])]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    outs, lses = [], []
    for b, n in enumerate(s["lens"].tolist()):
        latent, rope = _exact_tokens(s, b, n)
        t = offsets[b + 1] - offsets[b]
        for i in range(t):
            j = offsets[b] + i
            score = (s["q_latent"][j].double() @ latent.T + s["q_rope"][j].double() @ rope.T) * SOFTMAX_SCALE
            bits = (1 << (i + 1)) - 1 if s["tree"] is None else int(s["tree"][j]) & (1 << 64) - 1
            hidden = [n - t + k for k in range(t) if not bits >> k & 1]
            score[:, hidden] = -math.inf
            lse = torch.logsumexp(score, -1)
            outs.append(torch.exp(score - lse[:, None]) @ latent)
            lses.append(lse)
    out = torch.stack(outs)
    return (out, torch.stack(lses)) if case["lse"] else out
