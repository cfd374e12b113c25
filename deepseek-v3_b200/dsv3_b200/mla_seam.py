"""Seam above the latent cache: a replacement for ``MLA.forward`` of the reference's ``model.py``.

``MLA.forward`` (model.py:446-497, ``attn_impl = "absorb"``) normalises, rotates and stores the new tokens in bf16 buffers and then runs two score
einsums, a softmax and a weighted-sum einsum over the whole prefix.  The replacement keeps the projections, the absorbed products with ``wkv_b`` and the
arguments, and does the rest with the operators of ``latent.py``: one launch stores the new tokens in the 8-bit cache, ``latent_attention`` reads it.
``kv_norm`` is part of that launch where calling it does nothing but the RMS norm of its ``weight`` and ``eps``; one with hooks, a forward of its own or another
norm is called, and its bf16 result stored.

    import model, dsv3_b200
    dsv3_b200.install_mla(model)        # model.MLA.forward = mla_forward
    dsv3_b200.install_mla(model, release_buffers=True)        # ... and the modules' bf16 buffers give their memory back
    dsv3_b200.install_mla(model, expand_from=256)             # ... and prompts of 256 tokens or more are attended to with expanded keys and values

A module's cache is made on its first call (not in a captured graph), of the size of its bf16 buffers; ``mla_cache(module)`` gives it with its block table, for
``latent_cache_keep`` and ``latent_cache_read``.  Drafted tokens: with a tree of them, ``mask`` is the int64 ``[batch, tokens]`` of
``latent_attention``'s ``tree_mask`` and ``freqs_cis`` has a row per node, that of its depth.  Sequences of which different numbers of drafts were kept are of different
lengths from then on: ``start_pos`` is then an integer tensor ``[batch]`` and ``freqs_cis`` ``[batch, tokens, 32]``.

Prompts: ``expand_from`` says from how many new tokens on (to a sequence) the keys and values of all heads are expanded from the cached latents (model.py:472-478) and
``expanded_attention`` reads those, with a third of the absorbed form's operations per token seen.  Both forms attend to the same cached tokens.
"""
from __future__ import annotations

import math
import threading
import types
from typing import NamedTuple, Optional, Union

import torch
from torch.nn.modules import module as _nn_module

from ._lib import host
from .expanded import NOPE_DIM, VALUE_DIM, attention_join, expanded_attention, rotary, rotary_table
from .latent import LATENT_DIM, ROPE_DIM, LatentCache, allocate_latent_cache, latent_attention, latent_cache_read, latent_cache_write
from .ops import weight_dequant

PAGE = 64


class MlaCache(NamedTuple):
    pool: LatentCache
    block_table: torch.Tensor       # int32 [max_batch, pages of a sequence]: sequence b has pages b * pages ... in order
    first_page_slot: int            # slots of a sequence: b * first_page_slot + position
    max_len: int


_making = threading.Lock()


def _release_buffers(module) -> None:
    """Give the memory of an MLA module's bf16 buffers back: a single zero in the buffers' shape takes their place.  ``MLA.forward`` of the reference cannot store to it
    (torch refuses to write several values to one place).  Nothing else may use the buffers' memory any more, a captured graph of that forward least of all."""
    for name in ("kv_cache", "pe_cache", "k_cache", "v_cache"):
        buffer = getattr(module, name, None)
        if buffer is not None and any(buffer.stride()):
            setattr(module, name, buffer.new_zeros(()).expand(buffer.shape))


def mla_cache(module) -> MlaCache:
    """The 8-bit cache of an MLA module, made on first use after its bf16 buffers (model.py:439-444); where those have moved to another device it goes after them."""
    cache = module.__dict__.get("_dsv3_latent")
    buffer = module.kv_cache if hasattr(module, "kv_cache") else module.k_cache
    if cache is not None and cache.block_table.device == buffer.device:
        return cache
    with _making:                                          # (one thread makes it; the others find it made)
        cache = module.__dict__.get("_dsv3_latent")
        if cache is not None and cache.block_table.device == buffer.device:
            return cache
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("an MLA module's cache is made on its first call, which cannot be a captured one: every replay would clear it")
        if cache is not None:
            cache = cache._replace(pool=LatentCache(*(t.to(buffer.device) for t in cache.pool)), block_table=cache.block_table.to(buffer.device))
        else:
            batch, length = buffer.shape[:2]
            pages = -(-length // PAGE)
            table = torch.arange(batch * pages, dtype=torch.int32, device=buffer.device).view(batch, pages)
            cache = MlaCache(allocate_latent_cache(batch * pages, PAGE, buffer.device), table, pages * PAGE, length)
        if buffer.is_cuda:
            torch.cuda.current_stream(buffer.device).synchronize()         # (the threads that find it may be on streams of their own)
        module.__dict__["_dsv3_latent"] = cache
        return cache


def _rotate(x: torch.Tensor, freqs_cis: torch.Tensor) -> torch.Tensor:
    """Neighbouring values of the last dimension as a complex number, times their angle's (model.py:378-393)."""
    z = torch.view_as_complex(x.float().view(*x.shape[:-1], -1, 2)) * freqs_cis.view(-1, x.size(1), 1, x.size(-1) // 2)
    return torch.view_as_real(z).flatten(3).to(x.dtype)


def _with_torch_alone(forward):
    """``forward`` with nothing of its surroundings but torch's modules and functions, and no builtins: code of its own (a kernel that takes its argument for device memory, say) is not
    run; or None."""
    if type(forward) is not types.FunctionType or forward.__closure__:
        return None

    def of_torch(value):
        name = value.__name__ if isinstance(value, types.ModuleType) else getattr(value, "__module__", None) if callable(value) else None
        return isinstance(name, str) and name.split(".")[0] == "torch"

    around = {name: forward.__globals__[name] for name in forward.__code__.co_names if of_torch(forward.__globals__.get(name))}
    return types.FunctionType(forward.__code__, {"__builtins__": {}, **around}, forward.__name__, forward.__defaults__)


def _norms_as_rms_norm(forward) -> bool:
    """Whether ``forward`` gives x / sqrt(mean(x^2) + eps) * weight of an object that has ``dim``, ``weight`` and ``eps`` (model.py:270-294)."""
    forward = _with_torch_alone(forward)
    if forward is None:
        return False
    x = torch.linspace(-3, 2, 2 * LATENT_DIM, dtype=torch.float32, device="cpu").view(2, LATENT_DIM).bfloat16()
    weight = torch.linspace(0.5, 2, LATENT_DIM, dtype=torch.float32, device="cpu").bfloat16()
    try:
        with torch.no_grad():
            for eps in (1e-6, 0.5):
                want = x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + eps) * weight.float()
                got = forward(types.SimpleNamespace(dim=LATENT_DIM, weight=weight, eps=eps), x)
                # (bf16 twice at most, after the norm and after the weight)
                if got.shape != want.shape or not bool(((got.float() - want).abs() <= 2.0 ** -7 * 1.01 * want.abs()).all()):
                    return False
    except Exception:                                      # (a forward that needs more than that, or a GPU)
        return False
    return True


_known_norms = {}        # class -> (its forward, the forward's code, answer)


def _is_rms_norm(norm) -> bool:
    """Whether calling ``norm`` is the RMS norm of its ``weight`` and ``eps`` and nothing else, which ``latent_cache_write`` can do in its place: a module that nothing
    intercepts, of a class whose forward gives that on a stand-in.  Kept with the class, its forward and that one's code, and found anew when one of them is another."""
    if host.intercepted(norm) or _nn_module._global_forward_hooks or _nn_module._global_forward_pre_hooks:
        return False
    cls = type(norm)
    forward = getattr(cls, "forward", None)
    if forward is None or cls.__call__ is not torch.nn.Module.__call__:
        return False
    code = getattr(forward, "__code__", None)
    known = _known_norms.get(cls)
    if known is None or known[0] is not forward or known[1] is not code:
        if len(_known_norms) >= 64:
            _known_norms.clear()
        known = _known_norms[cls] = forward, code, _norms_as_rms_norm(forward)
    return known[2]


# With this eps beside a mean of squares below 2^96, and this weight, the norm of latent_cache_write is x * 2^-60 * 2^60
_NO_NORM_EPS, _NO_NORM_WEIGHT = 2.0 ** 120, 2.0 ** 60


def _is_causal(mask: torch.Tensor, start_pos: int) -> torch.Tensor:
    """Whether an additive mask hides what lies behind each token and nothing else (Transformer.forward's, model.py:738-798; the lowest number of its type serves for -inf too)."""
    rows, columns = mask.shape
    low = torch.finfo(mask.dtype).min
    causal = mask.new_full((rows, columns), low).triu_(1 + (start_pos if columns > rows else 0))
    return (mask.clamp(min=low) == causal).all()           # (few launches: a short prompt is bound by the host)


_MOST_PARTS = 32        # of attention_join


def _steps(count: int, most: int):
    """``count`` things in equal steps of ``most`` at most (and of one at least)."""
    steps = -(-count // max(1, most))
    return [slice(count * i // steps, count * (i + 1) // steps) for i in range(steps)]


def _attend_in_steps(q_nope, q_rope, latent, k_rope, weight, room: int, softmax_scale: float, causal: bool, with_lse: bool):
    """Attention to cached tokens that are expanded for some heads, and of one head for some sequences, at a time: ``room`` tokens times heads."""
    bsz, seqlen, heads, _ = q_nope.shape
    tokens = latent.size(1)
    out = q_nope.new_empty(bsz, seqlen, heads, VALUE_DIM)
    lse = q_nope.new_empty(bsz, seqlen, heads, dtype=torch.float32) if with_lse else None
    for seqs in _steps(bsz, room // tokens):
        for some in _steps(heads, room // ((seqs.stop - seqs.start) * tokens)):
            kv = torch.nn.functional.linear(latent[seqs], weight[some].flatten(0, 1)).unflatten(-1, (-1, NOPE_DIM + VALUE_DIM))
            got = expanded_attention(q_nope[seqs, :, some], q_rope[seqs, :, some], kv[..., :NOPE_DIM], k_rope[seqs], kv[..., NOPE_DIM:], softmax_scale, causal=causal, return_lse=with_lse)
            out[seqs, :, some] = got[0] if with_lse else got
            if with_lse:
                lse[seqs, :, some] = got[1]
            del kv, got
    return (out, lse) if with_lse else out


def _attend_expanded(q_nope, q_rope, cache: MlaCache, table, start_pos: int, weight, softmax_scale: float, expand_tokens: int) -> torch.Tensor:
    """Causal attention of a chunk at ``start_pos`` to its sequences' cached tokens, expanded with ``weight`` ``[heads, 256, 512]``.  The tokens before the chunk's page are expanded and attended
    to in pieces of whole pages, ``expand_tokens`` of all sequences together to a piece, and the pieces' results joined (each is rounded to bf16 first, as a result is; the join's sums are fp32).
    Of what is more than that at a time (the chunk itself; pieces, of which there are ``_MOST_PARTS`` at most) fewer heads are expanded at once, and of one head fewer sequences: heads and sequences
    do not depend on one another, so that nothing is rounded for it."""
    bsz, seqlen, heads, _ = q_nope.shape

    def attend(first, end, causal, with_lse):
        tokens = end - first
        ends = torch.arange(0, (bsz + 1) * tokens, tokens, dtype=torch.int32, device=q_nope.device)
        latent, k_rope = latent_cache_read(cache.pool, table[:, first // PAGE:], ends, bsz * tokens)
        k_rope = k_rope.view(bsz, tokens, -1)
        if bsz * tokens > expand_tokens:
            return _attend_in_steps(q_nope, q_rope, latent.view(bsz, tokens, -1), k_rope, weight, expand_tokens * heads, softmax_scale, causal, with_lse)
        kv = torch.nn.functional.linear(latent, weight.flatten(0, 1)).view(bsz, tokens, heads, -1)
        return expanded_attention(q_nope, q_rope, kv[..., :NOPE_DIM], k_rope, kv[..., NOPE_DIM:], softmax_scale, causal=causal, return_lse=with_lse)

    before = start_pos // PAGE * PAGE                      # tokens that may be seen in pieces
    end_pos = start_pos + seqlen
    if bsz * end_pos <= expand_tokens or before == 0:
        return attend(0, end_pos, True, False)
    pages = before // PAGE
    piece = max(1, expand_tokens // (bsz * PAGE), -(-pages // (_MOST_PARTS - 1))) * PAGE
    parts = [attend(first, min(first + piece, before), False, True) for first in range(0, before, piece)] + [attend(before, end_pos, True, True)]
    return attention_join([out for out, _ in parts], [lse for _, lse in parts])


def mla_forward(self, x: torch.Tensor, start_pos: Union[int, torch.Tensor], freqs_cis: torch.Tensor, mask: Optional[torch.Tensor], *, block_size: int = 128,
                expand_from: Optional[int] = None, expand_tokens: int = 1 << 16) -> torch.Tensor:
    """``MLA.forward`` on the 8-bit latent cache.  ``mask``: None for one token, the reference's causal mask (of these tokens, or of all up to them), or
    int64 words of a tree of drafted tokens.  Masks of other shapes are refused; a floating mask that is not the causal one makes the result NaN (nothing is read back).
    ``start_pos``: one for all sequences, or an int32 or int64 tensor ``[batch]`` beside ``x``, which a captured step reads when it is replayed; a sequence whose tokens do not fit
    its cache is then not stored, and its result NaN.  ``freqs_cis``: ``[tokens, 32]``, or ``[batch, tokens, 32]``.  ``expand_from``: so many tokens, and more, of a causal mask are attended to with
    expanded keys and values where ``start_pos`` is one for all and heads are of 128 and 64 values; keys and values of ``expand_tokens`` tokens with all heads (512 bytes a token and head) are held at a time at
    most, or, if that is more, one head's of one sequence."""
    bsz, seqlen, _ = x.shape
    rope = self.qk_rope_head_dim
    if self.kv_lora_rank != LATENT_DIM or rope != ROPE_DIM:
        raise NotImplementedError(f"the latent cache holds {LATENT_DIM} + {ROPE_DIM} values a token (kv_lora_rank {self.kv_lora_rank}, qk_rope_head_dim {rope})")
    tree = mask if mask is not None and not mask.is_floating_point() else None
    if mask is None and seqlen > 1:
        raise NotImplementedError("several tokens without a mask would see one another both ways; latent_attention is causal")
    starts = start_pos if isinstance(start_pos, torch.Tensor) and start_pos.dim() == 1 else None
    if starts is not None and (starts.shape != (bsz,) or starts.dtype not in (torch.int32, torch.int64) or starts.device != x.device):
        raise ValueError(f"start_pos must be an integer, or int32 or int64 [{bsz}] on {x.device}")
    if tuple(freqs_cis.shape) not in ((seqlen, rope // 2), (bsz, seqlen, rope // 2)):
        raise ValueError(f"freqs_cis must be [{seqlen}, {rope // 2}] or [{bsz}, {seqlen}, {rope // 2}], not {list(freqs_cis.shape)}")
    end_pos = seqlen if starts is not None else start_pos + seqlen
    valid = None                                           # which sequences' results are to be had: bool [batch], or of all
    if mask is not None and tree is None:
        if mask.shape not in ((seqlen, seqlen), (seqlen, end_pos)):
            raise NotImplementedError(f"attention is causal, or that of a tree: a mask of shape {tuple(mask.shape)} is neither's ({seqlen} tokens up to position {end_pos})")
        valid = _is_causal(mask, end_pos - seqlen)
        if not mask.is_cuda and not valid:
            raise NotImplementedError("attention is causal, or that of a tree; this mask is neither's")
        valid = valid.to(x.device)
    cache = mla_cache(self)
    if bsz > cache.block_table.size(0) or end_pos > cache.max_len or end_pos < seqlen:
        raise ValueError(f"{bsz} sequences of {end_pos} tokens do not fit a cache of {cache.block_table.size(0)} of {cache.max_len}")

    q = self.wq(x) if self.q_lora_rank == 0 else self.wq_b(self.q_norm(self.wq_a(x)))
    q = q.view(bsz, seqlen, self.n_local_heads, -1)
    q_nope, q_rope = torch.split(q, [self.qk_nope_head_dim, rope], dim=-1)
    kv = self.wkv_a(x)
    step = torch.arange(seqlen, device=x.device)
    slots = (torch.arange(bsz, device=x.device) * cache.first_page_slot)[:, None] + step
    if starts is None:
        table = cache.block_table[:bsz, :-(-end_pos // PAGE)]
        lens = torch.full((bsz,), end_pos, dtype=torch.int32, device=x.device)
        slots += start_pos
    else:
        fits = (starts >= 0) & (starts <= cache.max_len - seqlen)
        valid = fits if valid is None else fits & valid
        table = cache.block_table[:bsz]
        lens = (torch.where(fits, starts, 0) + seqlen).int()
        slots = torch.where(fits[:, None], slots + starts[:, None], -1)
    positions = torch.arange(bsz * seqlen, device=x.device) if freqs_cis.dim() == 3 else step.repeat(bsz)
    norm = self.kv_norm
    if _is_rms_norm(norm):
        latent_cache_write(cache.pool, kv, norm.weight, freqs_cis.reshape(-1, ROPE_DIM // 2), positions, slots, norm.eps)
    else:
        kv = torch.cat([norm(kv[..., :LATENT_DIM]).to(kv.dtype), kv[..., LATENT_DIM:]], -1)
        latent_cache_write(cache.pool, kv, kv.new_full((LATENT_DIM,), _NO_NORM_WEIGHT, dtype=torch.float32), freqs_cis.reshape(-1, ROPE_DIM // 2), positions, slots, _NO_NORM_EPS)

    weight = self.wkv_b.weight
    scale = getattr(self.wkv_b, "scale", None)
    if scale is not None:
        weight = weight_dequant(weight, scale, block_size)
    weight = weight.view(self.n_local_heads, -1, LATENT_DIM)
    if (expand_from is not None and seqlen >= expand_from and mask is not None and tree is None and isinstance(start_pos, int)
            and (self.qk_nope_head_dim, self.v_head_dim) == (NOPE_DIM, VALUE_DIM)):
        angles = freqs_cis.reshape(-1, ROPE_DIM // 2)      # (of one sequence, or of all)
        if valid is not None:
            angles = torch.where(valid, angles, math.nan)
        # (the attention has no gradient)
        turned = rotary(q_rope.detach() if q_rope.requires_grad else q_rope, angles, None if len(angles) == seqlen else positions)
        out = _attend_expanded(q_nope, turned, cache, table, start_pos, weight, self.softmax_scale, expand_tokens)
        return self.wo(out.flatten(2))
    q_latent = torch.einsum("bshd,hdc->bshc", q_nope, weight[:, :self.qk_nope_head_dim])
    angles = freqs_cis.reshape(-1, seqlen, ROPE_DIM // 2)
    if valid is not None:
        angles = torch.where(valid.view(-1, 1, 1), angles, math.nan)
    out = latent_attention(q_latent, _rotate(q_rope, angles), cache.pool, table, lens, self.softmax_scale, tree_mask=tree)
    return self.wo(torch.einsum("bshc,hdc->bshd", out, weight[:, -self.v_head_dim:]).flatten(2))


def install_mla(model_module, release_buffers: bool = False, expand_from: Optional[int] = None, expand_tokens: int = 1 << 16) -> None:
    """Point ``model_module.MLA.forward`` at ``mla_forward``; ``model_module.block_size`` is read at call time, as in the reference.  ``release_buffers``: a module's
    bf16 buffers give their memory back at its first call; without it they stay, 1152 bytes a token beside the 644 of the 8-bit cache, for a host that goes back to the old forward.
    ``expand_from``: prompts of so many tokens and more to a sequence are attended to with expanded keys and values (None: never), with the keys and values of ``expand_tokens`` tokens at a time, cached and new
    ones of all sequences (or those of one head of one sequence, if that is more)."""
    if (expand_from is not None and expand_from < 1) or expand_tokens < 1:
        raise ValueError("expand_from and expand_tokens are numbers of tokens, from 1 on")

    def forward(self, x, start_pos, freqs_cis, mask):
        if release_buffers:
            _release_buffers(self)
        return mla_forward(self, x, start_pos, freqs_cis, mask, block_size=getattr(model_module, "block_size", 128), expand_from=expand_from, expand_tokens=expand_tokens)
    forward.__doc__ = mla_forward.__doc__
    model_module.MLA.forward = forward


def install_rotary(model_module) -> None:
    """Point ``model_module.apply_rotary_emb`` (model.py:378-393) and ``precompute_freqs_cis`` (model.py:297-375) at ``rotary`` and ``rotary_table``.

    One launch to a rotation instead of five; angles are formed in 64 bits.  ``x`` is bf16, fp16 or fp32 on a CUDA device, heads of a multiple of 16 values up to 256; of any strides, though rows that are not 16-byte aligned and
    a batch cut from longer sequences are copied first.  The table is made on torch's default device, which has to be a CUDA device
    (``with torch.device("cuda")``, as the reference's generate.py makes its model)."""
    def precompute_freqs_cis(args):
        factor = args.rope_factor if args.max_seq_len > args.original_seq_len else 1.0
        return rotary_table(args.max_seq_len, args.qk_rope_head_dim, args.rope_theta, factor=factor, original_length=args.original_seq_len, beta_fast=args.beta_fast,
                            beta_slow=args.beta_slow, device=torch.get_default_device())

    def apply_rotary_emb(x, freqs_cis):
        if not host.rotary_takes(x, freqs_cis):
            # (as there: a table that is not of x's tokens and width is an error, not a part of either)
            freqs_cis = freqs_cis.view(x.size(1), x.size(3) // 2).contiguous()
            if not host.rotary_takes(x, freqs_cis):
                x = x.clone(memory_format=torch.contiguous_format)
        return rotary(x, freqs_cis)

    model_module.precompute_freqs_cis = precompute_freqs_cis
    model_module.apply_rotary_emb = apply_rotary_emb
