"""Token sampling from given uniform numbers: temperature, repetition penalty, top-k, top-p, min-p.

Per row, with scalars or one setting per row:

* ``z = logits / temperature`` in fp32 (then divided by ``repetition_penalty``
  for tokens of ``generated``, whatever their sign, as
  :func:`~titans_pytorch_b200.inference.generate.apply_repetition_penalty`); NaN counts as -inf;
* weights ``w = exp(z - max z)`` and all sums in fp64 (the kernel: in integers of 2^-F of the largest weight, with F
  from 47 up to 2^15 tokens down to 38 at 2^19, whose sums are exact; what weighs less than half a unit is never drawn,
  and a running sum is off by at most half a unit a token, 2^-33 to 2^-20 of the largest weight);
* top-k keeps ``z >=`` the k-th largest, ties included (0: off);
* top-p keeps, in descending order (ties: lower index first), tokens while the
  weight in front of them is at most ``top_p`` of what top-k left (1: off);
* min-p keeps ``w >= min_p``, i.e. at least ``min_p`` of the likeliest token's probability (0: off);
* the token is the first, by index, whose running sum of kept weights exceeds ``uniform`` times their sum.

``temperature <= 0`` takes the largest (lowest index on ties).  The same
uniform number gives the same token whatever else is in the batch.  A row whose
logits are all -inf or NaN gives token 0 and the log-probability NaN.
"""

from __future__ import annotations

import torch

from ._ext import ext, want_kernels


def _row(value, like: torch.Tensor, dtype: torch.dtype, name: str):
    """(tensor [B] or None, scalar) of a setting."""
    if not torch.is_tensor(value):
        return None, value
    if value.dim() == 0:
        value = value.expand(like.shape[0])
    if value.shape != like.shape[:1] or value.device != like.device:
        raise ValueError(f"{name} must be a number or [{like.shape[0]}] on the logits' device, "
                         f"not {tuple(value.shape)} on {value.device}")
    return (value if value.dtype == dtype else value.to(dtype)).contiguous(), 0


def sample_tokens_reference(logits, uniform, temperature, top_k, top_p, min_p, generated, repetition_penalty):
    """PyTorch restatement; settings are tensors [B].  ``(tokens [B], logprob [B])``."""
    V = logits.shape[1]
    greedy = ~(temperature > 0)
    z = logits.float() / torch.where(greedy, torch.ones_like(temperature), temperature)[:, None]
    if generated is not None and generated.shape[1]:
        inside = (generated >= 0) & (generated < V)
        seen = torch.zeros(z.shape[0], V + 1, dtype=torch.bool, device=z.device)
        seen.scatter_(1, torch.where(inside, generated, torch.full_like(generated, V)), True)
        z = torch.where(seen[:, :V], z / repetition_penalty[:, None], z)
    low = torch.full((), float("-inf"), device=z.device)
    z = torch.where(torch.isnan(z), low, z)
    down, order = torch.sort(z, dim=1, descending=True, stable=True)
    top = down[:, :1]
    k = torch.where((top_k <= 0) | (top_k > V), torch.full_like(top_k, V), top_k)
    w = torch.where(z == top, torch.ones((), dtype=torch.float64, device=z.device),
                    torch.exp(z.double() - top.double()))
    w = torch.where(z >= torch.gather(down, 1, (k - 1)[:, None]), w, torch.zeros_like(w))
    ranked = torch.gather(w, 1, order)
    ahead = torch.cumsum(ranked, dim=1) - ranked
    nucleus = torch.where(top_p < 1, top_p.double() * ranked.sum(dim=1), torch.full_like(ranked[:, 0], float("inf")))
    keep = torch.zeros_like(w, dtype=torch.bool).scatter_(1, order, ahead <= nucleus.clamp(min=0)[:, None])
    min_p = torch.where(min_p > 0, min_p, torch.zeros_like(min_p)).clamp(max=1)
    w = torch.where(keep & (w >= min_p.double()[:, None]), w, torch.zeros_like(w))
    reach = torch.cumsum(w, dim=1)
    uniform = torch.where(uniform > 0, uniform, torch.zeros_like(uniform))
    token = (reach <= uniform.double()[:, None] * reach[:, -1:]).sum(dim=1)
    last = torch.where(w > 0, torch.arange(V, device=z.device), -1).amax(dim=1)
    token = torch.minimum(token, last)
    empty = top[:, 0] == low
    token = torch.where(greedy | empty, order[:, 0], token)
    logprob = torch.log(torch.gather(w, 1, token[:, None])[:, 0] / reach[:, -1])
    logprob = torch.where(greedy, torch.zeros_like(logprob), logprob.masked_fill(empty, float("nan")))
    return torch.where(empty, torch.zeros_like(token), token), logprob.float()


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  generated: torch.Tensor | None = None, repetition_penalty=1.0, return_logprob: bool = False,
                  use_kernels: bool | None = None):
    """Token ids (int64 [B]) drawn from ``logits`` [B, V] with the numbers ``uniform`` (fp32 [B], in [0, 1)).

    Every setting is a number or a tensor [B]; V is at most 2^19.  In a tensor,
    ``top_p`` and ``min_p`` out of [0, 1] count as the nearest and NaN as off
    (``temperature``: as 0); a ``uniform`` below 0 or NaN counts as 0, one from
    1 on gives the last token that is kept.  ``generated`` (int64 [B, n]):
    tokens that ``repetition_penalty`` applies to; ids outside the vocabulary
    (padding) are passed over.  With ``return_logprob`` also the log-probability
    of each token among those kept (fp32 [B]; 0 where ``temperature <= 0``).
    """
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be [B, V], not {tuple(logits.shape)}")
    B = logits.shape[0]
    if uniform.shape != (B,) or uniform.dtype != torch.float32 or uniform.device != logits.device:
        raise ValueError(f"uniform must be float32 [{B}] on the logits' device, "
                         f"not {uniform.dtype} {tuple(uniform.shape)} on {uniform.device}")
    if generated is not None and (generated.dim() != 2 or generated.shape[0] != B or generated.dtype != torch.int64):
        raise ValueError(f"generated must be int64 [{B}, n], not {generated.dtype} {tuple(generated.shape)}")
    rows = [_row(v, logits, t, n) for v, t, n in (
        (temperature, torch.float32, "temperature"), (top_k, torch.int64, "top_k"), (top_p, torch.float32, "top_p"),
        (min_p, torch.float32, "min_p"), (repetition_penalty, torch.float32, "repetition_penalty"))]
    for (t, s), name in zip(rows[2:4], ("top_p", "min_p")):
        if t is None and not 0.0 <= s <= 1.0:
            raise ValueError(f"{name} must be between 0 and 1, not {s}")
    if rows[4][0] is None and not rows[4][1] > 0:
        raise ValueError(f"repetition_penalty must be positive, not {rows[4][1]}")
    if want_kernels(logits, use_kernels):
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        if generated is not None and generated.stride(1) != 1:
            generated = generated.contiguous()
        flat = [x for pair in rows for x in pair]
        token, logprob = ext().sample_tokens(logits, uniform.contiguous(), *flat, generated)
    else:
        full = [t if t is not None else torch.full((B,), s, dtype=d, device=logits.device)
                for (t, s), d in zip(rows, (torch.float32, torch.int64) + (torch.float32,) * 3)]
        token, logprob = sample_tokens_reference(logits.detach(), uniform, full[0], full[1], full[2], full[3], generated,
                                                 full[4])
    return (token, logprob) if return_logprob else token


__all__ = ["sample_tokens", "sample_tokens_reference"]
