"""Seam above the latent cache: a replacement for ``MLA.forward`` of the reference's ``model.py``.

``MLA.forward`` (model.py:446-497, ``attn_impl = "absorb"``) normalises, rotates and stores the new tokens in bf16 buffers and then runs two score
einsums, a softmax and a weighted-sum einsum over the whole prefix.  The replacement keeps the projections, the absorbed products with ``wkv_b`` and the
arguments, and does the rest with the operators of ``latent.py``: one launch stores the new tokens in the 8-bit cache, ``latent_attention`` reads it.
``kv_norm`` is part of that launch where calling it does nothing but the RMS norm of its ``weight`` and ``eps``; one with hooks, a forward of its own or another
norm is called, and its bf16 result stored.

    import model, dsv3_b200
    dsv3_b200.install_mla(model)        # model.MLA.forward = mla_forward
    dsv3_b200.install_mla(model, release_buffers=True)        # ... and the modules' bf16 buffers give their memory back

A module's cache is made on its first call (not in a captured graph), of the size of its bf16 buffers; ``mla_cache(module)`` gives it with its block table, for
``latent_cache_keep`` and ``latent_cache_read``.  Drafted tokens: with a tree of them, ``mask`` is the int64 ``[batch, tokens]`` of
``latent_attention``'s ``tree_mask`` and ``freqs_cis`` has a row per node, that of its depth.  Sequences of which different numbers of drafts were kept are of different
lengths from then on: ``start_pos`` is then an integer tensor ``[batch]`` and ``freqs_cis`` ``[batch, tokens, 32]``.
"""
from __future__ import annotations

import math
import threading
import types
from typing import NamedTuple, Optional, Union

import torch
from torch.nn.modules import module as _nn_module

from ._lib import host
from .latent import LATENT_DIM, ROPE_DIM, LatentCache, allocate_latent_cache, latent_attention, latent_cache_write
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


def mla_forward(self, x: torch.Tensor, start_pos: Union[int, torch.Tensor], freqs_cis: torch.Tensor, mask: Optional[torch.Tensor], *, block_size: int = 128) -> torch.Tensor:
    """``MLA.forward`` on the 8-bit latent cache.  ``mask``: None for one token, the reference's causal mask (of these tokens, or of all up to them), or
    int64 words of a tree of drafted tokens.  Masks of other shapes are refused; a floating mask that is not the causal one makes the result NaN (nothing is read back).
    ``start_pos``: one for all sequences, or an int32 or int64 tensor ``[batch]`` beside ``x``, which a captured step reads when it is replayed; a sequence whose tokens do not fit
    its cache is then not stored, and its result NaN.  ``freqs_cis``: ``[tokens, 32]``, or ``[batch, tokens, 32]``."""
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
    q_latent = torch.einsum("bshd,hdc->bshc", q_nope, weight[:, :self.qk_nope_head_dim])
    angles = freqs_cis.reshape(-1, seqlen, ROPE_DIM // 2)
    if valid is not None:
        angles = torch.where(valid.view(-1, 1, 1), angles, math.nan)
    out = latent_attention(q_latent, _rotate(q_rope, angles), cache.pool, table, lens, self.softmax_scale, tree_mask=tree)
    return self.wo(torch.einsum("bshc,hdc->bshd", out, weight[:, -self.v_head_dim:]).flatten(2))


def install_mla(model_module, release_buffers: bool = False) -> None:
    """Point ``model_module.MLA.forward`` at ``mla_forward``; ``model_module.block_size`` is read at call time, as in the reference.  ``release_buffers``: a module's
    bf16 buffers give their memory back at its first call; without it they stay, 1152 bytes a token beside the 644 of the 8-bit cache, for a host that goes back to the old forward."""
    def forward(self, x, start_pos, freqs_cis, mask):
        if release_buffers:
            _release_buffers(self)
        return mla_forward(self, x, start_pos, freqs_cis, mask, block_size=getattr(model_module, "block_size", 128))
    forward.__doc__ = mla_forward.__doc__
    model_module.MLA.forward = forward
