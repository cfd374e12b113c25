"""Prompts of multi-head latent attention with expanded keys and values, and what stands around it, as cases that can be timed.

  attention  queries of a chunk of a prompt over keys and values of their own for every head, which the latents were expanded to: 128 values
             per head and 64 rotated ones that all heads share; ragged batches, chunks behind a prefix, pieces of a prefix
  join       the results of the same queries over several pieces of their keys become that over all of them
  rotary     rotation of queries (part of the head, or all of it) by the angles of their positions
  table      those angles, scaled for long contexts

`listed` and `draw` give the cases, `prepare` what a serving program holds before the call, `run` one pass, `work` what it cannot
do without, `exact` the results from the definitions in 64 bits.  Dimensions are those of the models that bench.py and the tests use: heads of
128 + 64, 128 or 16 of them, and one rank's share of 128 heads under tensor parallelism.
"""
import math
import os
import sys

import torch

own = False

NOPE, ROPE, VALUE = 128, 64, 128
SOFTMAX_SCALE = (NOPE + ROPE) ** -0.5
THETA, BETA_FAST, BETA_SLOW = 10000.0, 32, 1
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a short question, one rank of eight: where latency counts
        {"name": "attention_37", "kind": "attention", "seqs": 1, "queries": 37, "prefix": 0, "heads": 16, "ragged": False, "causal": True, "lse": False},
        # a chunk of a prompt behind its cached beginning, one rank of eight
        {"name": "attention_chunk_515", "kind": "attention", "seqs": 1, "queries": 515, "prefix": 3584, "heads": 16, "ragged": False, "causal": True,
         "lse": False},
        # a batch of prompts of different lengths, some behind a prefix of their own
        {"name": "attention_ragged_7", "kind": "attention", "seqs": 7, "queries": 2048, "prefix": 640, "heads": 32, "ragged": True, "causal": True,
         "lse": True},
        # a prompt where every rank holds all heads
        {"name": "attention_heads_128", "kind": "attention", "seqs": 1, "queries": 4096, "prefix": 0, "heads": 128, "ragged": False, "causal": True,
         "lse": False},
        # a long document, one rank of eight: the arithmetic is what counts
        {"name": "attention_long_16001", "kind": "attention", "seqs": 1, "queries": 16001, "prefix": 0, "heads": 16, "ragged": False, "causal": True,
         "lse": False},
        # a chunk's results over two pieces of its keys
        {"name": "join_chunk_515", "kind": "join", "parts": 2, "tokens": 515, "heads": 16, "dim": VALUE, "lse": False},
        # ... of a large chunk over a prefix in four pieces, all heads
        {"name": "join_pieces_4", "kind": "join", "parts": 4, "tokens": 4096, "heads": 128, "dim": VALUE, "lse": True},
        # the queries of a decode step
        {"name": "rotary_decode_64", "kind": "rotary", "tokens": 64, "heads": 16, "dim": ROPE, "beside": NOPE, "offset": 0, "rotated": ROPE,
         "layout": "interleaved", "type": "bf16", "inverse": False, "into": False},
        # ... of a prompt, all heads
        {"name": "rotary_prompt_4099", "kind": "rotary", "tokens": 4099, "heads": 128, "dim": ROPE, "beside": NOPE, "offset": 0, "rotated": ROPE,
         "layout": "interleaved", "type": "bf16", "inverse": False, "into": False},
        # whole heads, of which the last third is rotated in the layout of halves, to a buffer that the program keeps
        {"name": "rotary_half_part", "kind": "rotary", "tokens": 2047, "heads": 32, "dim": NOPE + ROPE, "beside": 0, "offset": NOPE, "rotated": ROPE,
         "layout": "half", "type": "bf16", "inverse": True, "into": True},
        # the angles of a model that is loaded for ordinary contexts
        {"name": "table_4096", "kind": "table", "length": 4096, "dim": ROPE, "factor": 1.0, "original": 4096, "start": 0},
        # ... for the longest ones
        {"name": "table_163840", "kind": "table", "length": 163840, "dim": ROPE, "factor": 40.0, "original": 4096, "start": 0},
    ]


def _spread(rng, low, high):
    """A whole number of the range, its logarithm evenly spread."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "join", "rotary", "table"])
    if kind == "table":
        factor = rng.choice([1.0, 4.0, 40.0])
        return {"kind": kind, "length": _spread(rng, 1, 163840), "dim": rng.choice([32, 64, 64, 128]) if factor == 1.0 else ROPE, "factor": factor,
                "original": 4096, "start": rng.choice([0, rng.randint(1, 100000)])}
    heads = rng.choice([1, 5, 16, 16, 32, 64, 128])
    if kind == "rotary":
        part = rng.random() < 0.5
        rotated = rng.choice([32, 64]) if part else ROPE
        return {"kind": kind, "tokens": _spread(rng, 1, 4096), "heads": heads, "dim": NOPE + ROPE if part else ROPE, "beside": 0 if part else NOPE,
                "offset": rng.choice([0, NOPE + ROPE - rotated]) if part else 0, "rotated": rotated, "layout": rng.choice(["interleaved", "half"]),
                "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "inverse": rng.random() < 0.3, "into": rng.random() < 0.3}
    if kind == "join":
        dim = rng.choice([VALUE, VALUE, 512])
        parts = rng.randint(2, 8)
        return {"kind": kind, "parts": parts, "tokens": _spread(rng, 1, 4096 * 4 * VALUE // (parts * dim)), "heads": heads, "dim": dim,
                "lse": rng.random() < 0.5}
    causal = rng.random() < 0.75
    queries = _spread(rng, 1, 8192)
    prefix = rng.choice([0, _spread(rng, 1, 16384)]) if causal else _spread(rng, 1, 16384)
    seqs = _spread(rng, 1, 24)
    # no more pairs than a prompt of 16001 tokens with 16 heads, nor more rows than one of 4096 with 128
    pairs = lambda: seqs * heads * queries * (prefix + queries / 2 if causal else prefix)  # noqa: E731
    while pairs() > 16 * 16001 ** 2 / 2 or seqs * (queries + prefix) * heads > 4096 * 128:
        if seqs > 1:
            seqs -= 1
        elif heads > 16:
            heads //= 2
        else:
            queries, prefix = max(1, queries * 3 // 4), prefix * 3 // 4
    if not causal:
        prefix = max(prefix, 1)
    return {"kind": kind, "seqs": seqs, "queries": queries, "prefix": prefix, "heads": heads, "ragged": rng.random() < 0.6, "causal": causal,
            "lse": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------------
# What a serving program holds before the call
# ---------------------------------------------------------------------------------------------------------------------
def _counts(case):
    """Queries and keys of every sequence, on the host; ragged ones spread from an eighth of the longest on, the first the longest.  Causal: the queries are
    the last keys; else the keys are those of a piece of the prefix."""
    q, k = [], []
    for i in range(case["seqs"]):
        share = 0.125 + 0.875 * (i * 0.6180339887 % 1) if case["ragged"] and i else 1.0
        other = 0.125 + 0.875 * (i * 0.7548776662 % 1) if case["ragged"] and i else 1.0
        n, before = max(1, round(case["queries"] * share)), round(case["prefix"] * other)
        q.append(n)
        k.append(before + n if case["causal"] else max(1, before))
    return q, k


def _offsets(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    kind = case["kind"]
    if kind == "table":
        # (the angles follow from a model's arguments; another seed asks for another stretch of positions)
        return {"case": case, "start": case["start"] + seed % 1000}
    if kind == "rotary":
        t, h, d, beside, r = case["tokens"], case["heads"], case["dim"], case["beside"], case["rotated"]
        dtype = TYPES[case["type"]]
        whole = randn(t, h, beside + d).to(dtype)
        angle = torch.rand(4096, r // 2, generator=gen, device="cuda") * (2 * math.pi)
        return {"case": case, "x": whole[..., beside:], "freqs": torch.polar(torch.ones_like(angle), angle),
                "positions": torch.randint(0, 4096, (t,), generator=gen, device="cuda"),
                "out": torch.zeros(t, h, d, dtype=dtype, device="cuda") if case["into"] else None}
    if kind == "join":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        outs = [randn(t, h, d).bfloat16() for _ in range(case["parts"])]
        lses = [randn(t, h) * 3 + 5 for _ in range(case["parts"])]
        # some queries see nothing of a piece
        for i, lse in enumerate(lses[1:]):
            lse[i::7] = -math.inf
            outs[i + 1][i::7] = 0
        return {"case": case, "outs": outs, "lses": lses}
    q, k = _counts(case)
    h = case["heads"]
    queries, kv = randn(sum(q), h, NOPE + ROPE), randn(sum(k), h, NOPE + VALUE)
    # a sequence's first token draws a good part of many heads' attention
    lead = randn(h, NOPE)
    queries[..., :NOPE] += lead * 0.4 * torch.rand(sum(q), h, 1, generator=gen, device="cuda")
    offsets_k = _offsets(k)
    kv[offsets_k[:-1].long(), :, :NOPE] = lead
    return {"case": case, "q": queries.bfloat16(), "q_rope": randn(sum(q), h, ROPE).bfloat16(), "kv": kv.bfloat16(), "k_rope": randn(sum(k), ROPE).bfloat16(),
            "offsets_q": _offsets(q), "offsets_k": offsets_k, "counts": (q, k)}


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
    ops, case = _package(), s["case"]
    kind = case["kind"]
    if kind == "table":
        return torch.view_as_real(ops.rotary_table(case["length"], case["dim"], THETA, factor=case["factor"], original_length=case["original"],
                                                   beta_fast=BETA_FAST, beta_slow=BETA_SLOW, start=s["start"]))
    if kind == "rotary":
        return ops.rotary(s["x"], s["freqs"], s["positions"], layout=case["layout"], offset=case["offset"], inverse=case["inverse"], out=s["out"])
    if kind == "join":
        return ops.attention_join(s["outs"], s["lses"], return_lse=case["lse"])
    return ops.expanded_attention(s["q"][..., :NOPE], s["q_rope"], s["kv"][..., :NOPE], s["k_rope"], s["kv"][..., NOPE:], SOFTMAX_SCALE,
                                  cu_seqlens_q=s["offsets_q"], cu_seqlens_k=s["offsets_k"], causal=case["causal"], return_lse=case["lse"])


def _inverse_frequencies(case):
    """Angles per position, in 64 bits: theta^(-2i/dim), and where contexts are longer than those that a model was trained on, slow ones divided by
    the factor, fast ones as they are, those in between by degrees."""
    dim = case["dim"]
    i = torch.arange(dim // 2, dtype=torch.float64, device="cuda")
    f = THETA ** (-2 * i / dim)
    if case["factor"] != 1.0:
        at = [dim * math.log(case["original"] / (b * 2 * math.pi)) / (2 * math.log(THETA)) for b in (BETA_FAST, BETA_SLOW)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        ramp = ((i - low) / (high - low if high != low else 0.001)).clamp(0, 1)
        f = f / case["factor"] * ramp + f * (1 - ramp)
    return f


def _table(s):
    case = s["case"]
    angle = torch.outer(torch.arange(s["start"], s["start"] + case["length"], dtype=torch.float64, device="cuda"), _inverse_frequencies(case))
    return torch.stack([torch.cos(angle), torch.sin(angle)], -1).float()


def _pairs(case, x):
    """First and second values of the pairs of the part that is rotated."""
    part = x[..., case["offset"]:case["offset"] + case["rotated"]]
    return (part[..., 0::2], part[..., 1::2]) if case["layout"] == "interleaved" else part.chunk(2, -1)


def _rotary(s):
    case, f = s["case"], s["freqs"][s["positions"]][:, None]
    a, b = _pairs(case, s["x"].float())
    sin = -f.imag if case["inverse"] else f.imag
    re, im = a * f.real - b * sin, a * sin + b * f.real
    turned = torch.stack([re, im], -1).flatten(-2) if case["layout"] == "interleaved" else torch.cat([re, im], -1)
    out = s["out"] if case["into"] else torch.empty_like(s["x"], memory_format=torch.contiguous_format)
    out.copy_(s["x"])
    out[..., case["offset"]:case["offset"] + case["rotated"]] = turned.to(out.dtype)
    return out


def _join(s):
    lses = torch.stack(s["lses"])
    top = lses.amax(0)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(lses - top)
    total = weights.sum(0)
    out = sum(w[..., None] * o.float() for w, o in zip(weights, s["outs"])) / torch.where(total == 0, 1.0, total)[..., None]
    out = out.bfloat16()
    return (out, top + total.log()) if s["case"]["lse"] else out


_AT_ONCE = 1 << 28                    # scores


def _attention(s):
    case = s["case"]
    q, k = s["counts"]
    out = torch.empty(sum(q), case["heads"], VALUE, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(sum(q), case["heads"], device="cuda")
    at_q = at_k = 0
    for n, m in zip(q, k):
        rows, keys = slice(at_q, at_q + n), slice(at_k, at_k + m)
        at_q, at_k = at_q + n, at_k + m
        hidden = torch.arange(m, device="cuda") > torch.arange(m - n, m, device="cuda")[:, None] if case["causal"] else None
        step = max(1, _AT_ONCE // (n * m))
        for h in range(0, case["heads"], step):
            heads = slice(h, h + step)
            kv = s["kv"][keys, heads].float()
            score = torch.einsum("thd,shd->hts", s["q"][rows, heads, :NOPE].float(), kv[..., :NOPE])
            score += torch.einsum("thd,sd->hts", s["q_rope"][rows, heads].float(), s["k_rope"][keys].float())
            score *= SOFTMAX_SCALE
            if hidden is not None:
                score.masked_fill_(hidden, -math.inf)
            top = score.amax(-1, keepdim=True)
            weight = torch.exp(score.sub_(top))
            total = weight.sum(-1, keepdim=True)
            out[rows, heads] = torch.einsum("hts,shd->thd", weight.div_(total), kv[..., NOPE:]).bfloat16()
            lse[rows, heads] = (top + total.log())[..., 0].T
    return (out, lse) if case["lse"] else out


def run(state):
    if own:
        return _run_own(state)
    return {"table": _table, "rotary": _rotary, "join": _join, "attention": _attention}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "table":
        n = case["length"] * case["dim"] // 2
        return {"bytes": 8 * n, "flops": 20 * n}
    if kind == "rotary":
        n = case["tokens"] * case["heads"]
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": 2 * n * case["dim"] * size + case["tokens"] * (8 + 4 * case["rotated"]), "flops": 3 * n * case["rotated"]}
    if kind == "join":
        n = case["tokens"] * case["heads"]
        return {"bytes": n * ((case["parts"] + 1) * case["dim"] * 2 + (case["parts"] + case["lse"]) * 4), "flops": 2 * n * case["parts"] * case["dim"]}
    q, k = _counts(case)
    h = case["heads"]
    pairs = sum(n * (m - n) + n * (n + 1) // 2 if case["causal"] else n * m for n, m in zip(q, k))
    return {"bytes": sum(q) * h * (2 * (NOPE + ROPE + VALUE) + 4 * case["lse"]) + sum(k) * 2 * (h * (NOPE + VALUE) + ROPE),
            "flops": 2 * pairs * h * (NOPE + ROPE + VALUE)}


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits, a head or a part at a time
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "table":
        dim = case["dim"]
        rows = []
        for i in range(dim // 2):
            f = math.pow(THETA, -2.0 * i / dim)
            if case["factor"] != 1.0:
                turns = lambda n: dim * math.log(case["original"] / (2 * math.pi * n)) / math.log(THETA) / 2  # noqa: E731
                low, high = max(0, math.floor(turns(BETA_FAST))), min(dim - 1, math.ceil(turns(BETA_SLOW)))
                slow = min(1.0, max(0.0, (i - low) / (high - low)))
                f = slow * f / case["factor"] + (1.0 - slow) * f
            rows.append(f)
        position = torch.arange(case["length"], device="cuda").double() + s["start"]
        z = torch.exp(1j * position[:, None] * torch.tensor(rows, dtype=torch.float64, device="cuda"))
        return torch.view_as_real(z)
    if kind == "rotary":
        x = s["x"].double().clone()
        lo, n = case["offset"], case["rotated"]
        part = x[..., lo:lo + n].clone()
        pairs = part.unflatten(-1, (n // 2, 2)) if case["layout"] == "interleaved" else part.unflatten(-1, (2, n // 2)).transpose(-1, -2)
        turn = s["freqs"].to(torch.complex128)[s["positions"]][:, None]
        z = torch.view_as_complex(pairs.contiguous()) * (turn.conj() if case["inverse"] else turn)
        pairs = torch.view_as_real(z)
        x[..., lo:lo + n] = (pairs if case["layout"] == "interleaved" else pairs.transpose(-1, -2)).flatten(-2)
        return x
    if kind == "join":
        lse = torch.stack([x.double() for x in s["lses"]]).logsumexp(0)
        out = torch.zeros(s["outs"][0].shape, dtype=torch.float64, device="cuda")
        for x, o in zip(s["lses"], s["outs"]):
            out += torch.exp(x.double() - lse)[..., None] * o.double()
        return (out, lse) if case["lse"] else out
    # (one head of one sequence at a time, in blocks of rows)
    q, k = s["counts"]
    out = torch.zeros(sum(q), case["heads"], VALUE, dtype=torch.float64, device="cuda")
    lse = torch.zeros(sum(q), case["heads"], dtype=torch.float64, device="cuda")
    first_q = first_k = 0
    for n, m in zip(q, k):
        k_rope = s["k_rope"][first_k:first_k + m].double()
        for h in range(case["heads"]):
            kv = s["kv"][first_k:first_k + m, h].double()
            keys = torch.cat([kv[:, :NOPE], k_rope], -1)
            for r in range(0, n, 4096):
                e = min(n, r + 4096)
                rows = slice(first_q + r, first_q + e)
                x = torch.cat([s["q"][rows, h, :NOPE], s["q_rope"][rows, h]], -1).double() @ keys.T * SOFTMAX_SCALE
                if case["causal"]:
                    x = x.masked_fill(torch.ones_like(x, dtype=torch.bool).triu(m - n + r + 1), -math.inf)
                lse[rows, h] = torch.logsumexp(x, -1)
                out[rows, h] = torch.softmax(x, -1) @ kv[:, NOPE:]
        first_q, first_k = first_q + n, first_k + m
    return (out, lse) if case["lse"] else out
