"""Attention of prompts over expanded keys and values, and the rotary positions around it.

``latent_attention`` multiplies absorbed queries with the cached latents: 2 * (576 + 512) operations per head, query and key, and hardly any bytes, which is what a
decoding sequence needs.  A prompt is bound by its arithmetic, and takes 2 * (192 + 128) operations where ``wkv_b`` has expanded the latents to keys and values for every
head (the ``naive`` branch of the reference's ``MLA.forward``, model.py:472-478, 486-494).

    table = rotary_table(4096, 64)                                          # once: the angles of all positions
    q_rope = rotary(q[..., 128:], table, positions)                         # the rotated part of the queries
    latent, k_rope = latent_cache_read(cache, block_table, cu_seqlens, total)              # or the new tokens' own
    kv = (latent @ wkv_b.T).view(total, heads, 256)
    out = expanded_attention(q[..., :128], q_rope, kv[..., :128], k_rope, kv[..., 128:], softmax_scale, cu_seqlens_q, cu_seqlens_k)
    out = attention_join([out_of_prefix, out_of_chunk], [lse_of_prefix, lse_of_chunk])     # a long prefix in pieces

Lengths are device memory and nothing is read back: calls can be captured in a CUDA graph.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from ._lib import host

NOPE_DIM, VALUE_DIM = 128, 128


def expanded_attention(q_nope: torch.Tensor, q_rope: torch.Tensor, k_nope: torch.Tensor, k_rope: torch.Tensor, v: torch.Tensor, softmax_scale: float,
                       cu_seqlens_q: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None, causal: bool = True,
                       return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention with keys and values for every head and a rotated part of the keys that all share (model.py:486-494): bf16 of ``q_nope``'s shape, and with
    ``return_lse`` the natural logarithms of the softmax sums, fp32.

    ``q_nope`` bf16 ``[tokens, heads, 128]``, ``q_rope`` ``[tokens, heads, 64]``, rotated; ``k_nope`` and ``v`` ``[keys, heads, 128]``, ``k_rope`` ``[keys, 64]``; or all
    with the sequences in front.  Strides of tokens and heads are free (multiples of 8).  ``cu_seqlens_q`` and ``cu_seqlens_k`` int32 ``[sequences + 1]``: where the sequences' queries
    and keys begin; without them the batch is the sequences, or all is one.  ``causal``: a sequence's queries are its last keys, and see themselves and all before; else they see all of
    its keys.  A query that sees nothing gives zeros and -inf.  A score of NaN or +inf, or a value that is
    not finite, spoils the results of the queries that see its key, and no others; a score of -inf weighs nothing."""
    return host.expanded_attention(q_nope, q_rope, k_nope, k_rope, v, softmax_scale, cu_seqlens_q, cu_seqlens_k, causal, return_lse)


def attention_join(outs: Sequence[torch.Tensor], lses: Sequence[torch.Tensor],
                   return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The results of the same queries over several pieces of their keys (up to 32), as over all of them: bf16 ``[..., dim]``, and with ``return_lse`` fp32 ``[...]``.

    ``outs`` and ``lses`` are what ``expanded_attention`` or ``latent_attention`` return with ``return_lse``.  Sums in fp32, rounded once; what a part that sees nothing (-inf) holds does not count."""
    return host.attention_join(tuple(outs), tuple(lses), return_lse)


def rotary_table(length: int, dim: int = 64, theta: float = 10000.0, factor: float = 1.0, original_length: int = 4096, beta_fast: float = 32,
                 beta_slow: float = 1, start: int = 0, device=None) -> torch.Tensor:
    """Angles of positions ``start`` ... ``start + length - 1`` as complex64 ``[length, dim / 2]`` (``precompute_freqs_cis``, model.py:297-375).

    With a ``factor`` other than 1 slow angles are divided by it, for contexts that many times as long as the ``original_length`` of the training; those that turn more than
    ``beta_fast`` times over it stay, those that turn between ``beta_slow`` and ``beta_fast`` times are divided by degrees.  Formed in 64 bits and rounded once (2^-24, and
    2^-51 of the angle), so that far positions are as exact as near ones."""
    if device is not None:
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"dsv3_b200 runs on CUDA tensors only (there is no CPU path); got a {device.type} device")
        device = device.index
    return host.rotary_table(length, dim, theta, factor, original_length, beta_fast, beta_slow, start, device)


class _Rotary(torch.autograd.Function):
    """A rotation whose gradient is the gradient turned back (and the other way round: the gradient of that is a rotation again)."""

    @staticmethod
    def forward(ctx, x, freqs_cis, positions, half, offset, inverse):
        ctx.save_for_backward(freqs_cis, positions)
        ctx.how = half, offset, inverse
        return host.rotary(x, freqs_cis, positions, half, offset, inverse, None)

    @staticmethod
    def backward(ctx, grad):
        half, offset, inverse = ctx.how
        # (a gradient may be one number in many places, or lie as whatever made it left it)
        grad = grad.contiguous() if grad.data_ptr() % 16 == 0 else grad.clone(memory_format=torch.contiguous_format)
        return _Rotary.apply(grad, *ctx.saved_tensors, half, offset, not inverse), None, None, None, None, None


def rotary(x: torch.Tensor, freqs_cis: torch.Tensor, positions: Optional[torch.Tensor] = None, layout: str = "interleaved", offset: int = 0,
           inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` with a part of every head rotated by the angles of its token's position (``apply_rotary_emb``, model.py:378-393).

    ``x`` bf16, fp16 or fp32 ``[tokens, heads, dim]`` of any strides of tokens and heads (multiples of 16 bytes), or with the sequences in front, whose tokens are then all one stride apart; ``freqs_cis`` complex64 ``[positions, rotated / 2]``:
    values ``offset`` ... ``offset + rotated - 1`` of a head turn, the others are copied.  ``layout``: ``"interleaved"`` (neighbours are a pair) or ``"half"`` (value ``i`` and value
    ``i + rotated / 2`` of the part).  ``positions`` int64, one per token; without it a sequence's tokens are at 0, 1, ...  A token at a position that the table does not hold
    becomes NaN.  ``inverse`` turns back: the gradient of the rotation, which ``x`` has where autograd asks for one (``freqs_cis`` has none).  ``out``: a tensor to write to; ``x`` itself to rotate in place, which leaves
    the rest of the heads alone; as everywhere, not where a gradient is asked for."""
    if layout not in ("interleaved", "half"):
        raise ValueError(f"layout must be 'interleaved' or 'half', not {layout!r}")
    turned = host.rotary(x, freqs_cis, positions, layout == "half", offset, inverse, out)
    if turned is None:                                      # (nothing was done: a gradient is asked for)
        if freqs_cis.requires_grad:
            raise NotImplementedError("rotary has no gradient for freqs_cis")
        if out is not None:
            raise RuntimeError("rotary: a result that is written to out has no gradient")
        return _Rotary.apply(x, freqs_cis, positions, layout == "half", offset, inverse)
    return turned
