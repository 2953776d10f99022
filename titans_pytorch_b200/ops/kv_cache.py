"""Key/value cache that is quantised as it is written.

A :class:`KVCache` holds one layer's keys and values as ``[B, heads, slots, d]``
in fp32, bf16, fp16, int8 or fp8 (e4m3); the 8-bit kinds keep one fp32 scale per
(token, head).  The token at position ``p`` of a sequence lives in slot
``p mod slots``: a ring of the newest ``slots`` tokens, or a linear cache when
positions stay below ``slots``.  :func:`kv_cache_write` rotates (optionally),
quantises and stores in one pass; :func:`kv_cache_read` gives the stored tokens
back in order; :func:`~titans_pytorch_b200.ops.decode_attention.decode_attention`
reads the cache as it lies.

Quantisation of a row x (fp32, after the rotation), with ``top`` = 127 (int8) or
448 (e4m3) and amax its largest magnitude:
``stored = round(x * (top / amax))`` (to nearest, ties to even) and
``scale = amax / top``.  A row with amax < 2^-100 is stored as zeros with scale 1;
a row that holds an infinity or NaN gets the scale NaN.
"""

from __future__ import annotations

import torch

from ._ext import ext, want_kernels
from .rope import LAYOUTS, rotary_embedding_reference

KINDS = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16,
         "int8": torch.int8, "fp8": torch.float8_e4m3fn}
HEAD_DIMS = range(8, 257, 8)  # of a cache that the kernels write and read
_TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


class KVCache:
    """Keys and values ``[B, heads, slots, d]`` (and scales ``[B, heads, slots]`` of the 8-bit kinds) of one layer.

    The tensors may be views (of a stack of layers, or of part of a batch); a
    cache object owns no state besides them.  On the GPU ``d`` is a multiple of 8
    from 8 to 256.
    """

    __slots__ = ("k", "v", "k_scale", "v_scale")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None) -> None:
        if k.dtype not in KINDS.values():
            raise TypeError(f"a cache holds {', '.join(KINDS)}, not {k.dtype}")
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must be [B, heads, slots, d] of one type")
        if (k.dtype in _TOP) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise ValueError("8-bit caches, and only they, have scales for keys and values")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @classmethod
    def allocate(cls, batch: int, heads: int, slots: int, head_dim: int, kind: str = "bfloat16",
                 device=None) -> "KVCache":
        """A zeroed cache; ``kind`` is float32, bfloat16, float16, int8 or fp8."""
        if kind not in KINDS:
            raise ValueError(f"kind must be one of {tuple(KINDS)}, not {kind!r}")
        shape = (batch, heads, slots, head_dim)
        k, v = (torch.zeros(shape, dtype=KINDS[kind], device=device) for _ in range(2))
        if KINDS[kind] not in _TOP:
            return cls(k, v)
        return cls(k, v, *(torch.ones(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))

    @property
    def slots(self) -> int:
        return self.k.shape[2]

    def nbytes(self) -> int:
        ts = (self.k, self.v, self.k_scale, self.v_scale)
        return sum(t.numel() * t.element_size() for t in ts if t is not None)


def quantise_rows(x: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Stored values and scales of rows ``x`` [..., d] (PyTorch restatement)."""
    if dtype not in _TOP:
        return x.to(dtype), None
    x = x.float()
    top = x.new_full((), _TOP[dtype])  # a tensor: a Python number would be multiplied by as a reciprocal
    amax = x.abs().amax(dim=-1)
    bad = ~torch.isfinite(x).all(dim=-1)
    full = (amax >= 2.0 ** -100) & ~bad
    inv = torch.where(full, top / amax, torch.zeros_like(amax))
    scale = torch.where(full, amax / top, torch.ones_like(amax)).masked_fill(bad, float("nan"))
    y = torch.where(bad[..., None], torch.zeros_like(x), x * inv[..., None])
    return (y.round().to(dtype) if dtype == torch.int8 else y.clamp(-448.0, 448.0).to(dtype)), scale


def _check_rows(t: torch.Tensor, name: str, batch: int) -> None:
    if t.dtype != torch.int64 or t.shape != (batch,):
        raise ValueError(f"{name} must be int64 [{batch}], not {t.dtype} {tuple(t.shape)}")


def kv_cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, *,
                   counts: torch.Tensor | None = None, q: torch.Tensor | None = None,
                   inv_freq: torch.Tensor | None = None, layout: str = "interleaved", amplitude: float = 1.0,
                   rope_offset: int = 0, use_kernels: bool | None = None) -> torch.Tensor | None:
    """Store new tokens ``k``, ``v`` [B, T, heads, d] at positions ``start[b] + t``.

    ``counts`` (int64 [B]): how many of the T tokens of each sequence are real;
    the others leave the cache as it was.  Of more tokens than slots the newest
    are stored; positions below 0 are not.  With ``inv_freq`` the keys are
    rotated at position ``start[b] + t + rope_offset`` first, and so is ``q``
    [B, T, query heads, d] if given, which is returned (contiguous, in its own
    type; as given if there is no ``inv_freq``).  New tokens may be views of the
    cache: they count as they are before the call.  A cache whose own rows share
    memory (an expanded tensor, one tensor for keys and values) is refused.  No
    gradient flows: this is an inference operator.
    """
    B, H, S, d = cache.k.shape
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.shape[0] != B or tuple(k.shape[2:]) != (H, d):
        raise ValueError(f"k and v must be [{B}, T, {H}, {d}] of one type, not {tuple(k.shape)} and {tuple(v.shape)}")
    _check_rows(start, "start", B)
    if counts is not None:
        _check_rows(counts, "counts", B)
    if q is not None and (q.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != d or q.dtype != k.dtype):
        raise ValueError(f"q must be [{B}, {k.shape[1]}, heads, {d}] of the keys' type, not {tuple(q.shape)}")
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, not {layout!r}")
    if inv_freq is not None and (inv_freq.dim() != 1 or 2 * inv_freq.numel() > d):
        raise ValueError(f"inv_freq must be [n] with 2n <= {d}, not {tuple(inv_freq.shape)}")
    if want_kernels(cache.k, use_kernels):
        r = ext().kv_cache_write(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, start, counts, q,
                                 None if inv_freq is None else inv_freq.float().contiguous(), layout == "half",
                                 float(amplitude), int(rope_offset))
        return None if q is None else r
    return _write_reference(cache, k.detach(), v.detach(), start, counts, None if q is None else q.detach(), inv_freq,
                            layout, amplitude, rope_offset)


def _write_reference(cache, k, v, start, counts, q, inv_freq, layout, amplitude, rope_offset):
    """Reads no value on the host, so that a decoding step with it can be captured."""
    for x, y in ((cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        if x is not None and _shared(x, y):
            raise RuntimeError("kv_cache_write: a cache whose rows share memory cannot be written")
    B, H, S, d = cache.k.shape
    T = k.shape[1]
    at = start[:, None] + torch.arange(T, device=k.device)
    kr = k if k.dtype == torch.float64 else k.float()
    if inv_freq is not None:
        kr = rotary_embedding_reference(kr, at + rope_offset, inv_freq, layout, amplitude)
        if q is not None:
            q = rotary_embedding_reference(q, at + rope_offset, inv_freq, layout, amplitude)
    q = None if q is None else q.clone(memory_format=torch.contiguous_format)
    if T:
        n = torch.full_like(start, T) if counts is None else counts.clamp(0, T)
        # the newest min(T, S) tokens have a slot each; one that is not stored writes back what its slot held
        t = n[:, None] - min(T, S) + torch.arange(min(T, S), device=k.device)
        b, slot = torch.arange(B, device=k.device)[:, None], (start[:, None] + t) % S
        real = (t >= 0) & (start[:, None] + t >= 0)
        t = t.clamp(min=0)
        for new, data, scale in ((kr[b, t], cache.k, cache.k_scale), (v[b, t], cache.v, cache.v_scale)):
            stored, s = quantise_rows(new, data.dtype)
            if data.element_size() == 1:  # e4m3 as bytes: not every operation takes it
                stored, data = stored.view(torch.uint8), data.view(torch.uint8)
            data[b, :, slot] = torch.where(real[..., None, None], stored, data[b, :, slot])
            if scale is not None:
                scale[b, :, slot] = torch.where(real[..., None], s, scale[b, :, slot])
    return q


def _shared(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether rows of ``x`` or ``y`` lie in one another, for all that strides tell."""
    if any(n > 1 and s == 0 for t in (x, y) for n, s in zip(t.shape, t.stride(), strict=True)):
        return True
    begin = [t.data_ptr() for t in (x, y)]
    end = [p + t.numel() * t.element_size() for p, t in zip(begin, (x, y))]
    return x.is_contiguous() and y.is_contiguous() and x.numel() > 0 and begin[0] < end[1] and begin[1] < end[0]


def kv_cache_read(cache: KVCache, lengths: torch.Tensor, n: int | None = None, dtype: torch.dtype = torch.bfloat16,
                  use_kernels: bool | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [B, heads, n, d] of the newest ``min(lengths[b], slots, n)`` tokens, in order.

    ``lengths``: tokens each sequence has written in all (int64 [B]); ``n``
    defaults to the number of slots.  Rows behind a sequence's last token are
    zero.  Stored values times their scale, rounded once to ``dtype``.
    """
    B, _, S, _ = cache.k.shape
    n = S if n is None else int(n)
    _check_rows(lengths, "lengths", B)
    if not 0 <= n <= S:
        raise ValueError(f"n must be between 0 and the {S} slots, not {n}")
    if want_kernels(cache.k, use_kernels):
        return tuple(ext().kv_cache_read(cache.k, cache.v, cache.k_scale, cache.v_scale, lengths, n, dtype))
    held = lengths.clamp(0, min(S, n))[:, None]
    i = torch.arange(n, device=lengths.device)
    slot = ((lengths[:, None] - held + i) % S)[:, None, :]
    out = []
    for data, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = data if data.dtype == torch.float64 else data.float()
        if scale is not None:
            x = x * scale[..., None]
        x = torch.gather(x, 2, slot[..., None].expand(-1, x.shape[1], -1, x.shape[3]))
        out.append(torch.where((i < held)[:, None, :, None], x, torch.zeros((), dtype=x.dtype, device=x.device)).to(dtype))
    return out[0], out[1]


__all__ = ["KVCache", "KINDS", "HEAD_DIMS", "kv_cache_write", "kv_cache_read", "quantise_rows"]
