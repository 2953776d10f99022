"""Attention of one query token per sequence over a key/value cache and a shared prefix.

Every sequence sees the prefix (keys and values that the whole batch shares:
persistent tokens, a common prompt) and the newest tokens of its own cache.
The prefix is stored once.  With 16-bit queries and heads of 64, 96 or 128 it is
read once for 16 to 128 query rows of the batch; fp32 queries and other heads
read it once for every sequence, and so does a cache of the queries' type where
the prefix has at most 128 tokens, which saves a launch.

Softmax statistics and sums are fp32; the result is rounded once to the
queries' type.  With 16-bit queries and heads of 64, 96 or 128 the weights are
rounded to the queries' type before they meet the values (beside an 8-bit cache
to fp16, as are the queries, scaled by a power of two); elsewhere they stay fp32.
``csrc/decode_attn.cu`` describes the kernels.
"""

from __future__ import annotations

import torch

from ._ext import ext, want_kernels
from .attention import NO_WINDOW
from .kv_cache import KVCache


def decode_attention_reference(q, cache, lengths, prefix_k=None, prefix_v=None, window=NO_WINDOW, scale=None):
    """PyTorch restatement: ``(out [B, Hq, d], lse [B, Hq])``."""
    B, Hq, d = q.shape
    Hkv, S = cache.k.shape[1:3]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    qg = q.to(wide).reshape(B, Hkv, Hq // Hkv, d) * scale
    k, v = cache.k.to(wide), cache.v.to(wide)
    if cache.k_scale is not None:
        k, v = k * cache.k_scale[..., None], v * cache.v_scale[..., None]
    # the position that slot j holds: the newest one that is j modulo the number of slots
    last = lengths.clamp(min=0)[:, None] - 1
    pos = last - (last - torch.arange(S, device=q.device)) % S
    seen = ((pos >= 0) & (pos > last - window))[:, None, None]
    s = torch.matmul(qg, k.transpose(2, 3)).masked_fill(~seen, float("-inf"))
    v = torch.where(seen.transpose(2, 3), v, torch.zeros((), dtype=wide, device=q.device))
    P = 0 if prefix_k is None else prefix_k.shape[0]
    if P:
        s = torch.cat([torch.einsum("bhgd,phd->bhgp", qg, prefix_k.to(wide)), s], dim=-1)
    m = s.amax(dim=-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:-1], 1), float("-inf"))
    e = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = e.sum(dim=-1, keepdim=True)
    o = torch.matmul(e[..., P:], v)
    if P:
        o = o + torch.einsum("bhgp,phd->bhgd", e[..., :P], prefix_v.to(wide))
    o = torch.where(total == 0, torch.zeros_like(o), o / total)
    lse = torch.where(total == 0, torch.full_like(m, float("-inf")), m + torch.log(total))
    return o.reshape(B, Hq, d).to(q.dtype), lse.reshape(B, Hq)


def decode_attention(q: torch.Tensor, cache: KVCache, lengths: torch.Tensor, prefix_k: torch.Tensor | None = None,
                     prefix_v: torch.Tensor | None = None, *, window: int | None = None, scale: float | None = None,
                     return_lse: bool = False, use_kernels: bool | None = None):
    """Attention output [B, Hq, d] of the queries ``q`` [B, Hq, d].

    ``lengths`` (int64 [B], on the device): tokens that each sequence has
    written to ``cache`` so far, the query's own among them; the newest
    ``min(length, slots, window)`` are visible.  ``Hq`` is a multiple of the
    cache's heads; query head h reads key head ``h // (Hq / Hkv)``.
    ``prefix_k``, ``prefix_v`` [P, Hkv, d] in the queries' type are visible to
    every sequence.  ``scale`` defaults to ``d ** -0.5``.  With ``return_lse``
    also the log-sum-exp of the scores, fp32 [B, Hq].  A sequence of length 0
    without a prefix gives zeros and ``-inf``.  No gradient flows.
    """
    if q.dim() != 3:
        raise ValueError(f"q must be [B, heads, d], not {tuple(q.shape)}")
    B, Hq, d = q.shape
    Hkv = cache.k.shape[1]
    if cache.k.shape[0] != B or cache.k.shape[3] != d or Hkv == 0 or Hq % Hkv:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {tuple(cache.k.shape)}")
    if lengths.dtype != torch.int64 or lengths.shape != (B,):
        raise ValueError(f"lengths must be int64 [{B}], not {lengths.dtype} {tuple(lengths.shape)}")
    if (prefix_k is None) != (prefix_v is None):
        raise ValueError("prefix keys and values come together")
    if prefix_k is not None:
        for t in (prefix_k, prefix_v):
            if t.dim() != 3 or t.shape != (prefix_k.shape[0], Hkv, d) or t.dtype != q.dtype:
                raise ValueError(f"the prefix must be [P, {Hkv}, {d}] of type {q.dtype}, not {t.dtype} {tuple(t.shape)}")
    window = NO_WINDOW if window is None else int(window)
    if window < 1:
        raise ValueError(f"window must be at least 1, not {window}")
    scale = d ** -0.5 if scale is None else float(scale)
    if want_kernels(q, use_kernels):
        if q.stride(-1) != 1:
            q = q.contiguous()
        out, lse = ext().decode_attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, lengths, prefix_k, prefix_v,
                                          window, scale, return_lse)
    else:
        out, lse = decode_attention_reference(q.detach(), cache, lengths, prefix_k, prefix_v, window, scale)
    return (out, lse) if return_lse else out


__all__ = ["decode_attention", "decode_attention_reference"]
