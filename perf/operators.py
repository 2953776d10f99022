"""Serving operators on real work: rotary positions, the quantised key/value cache, single-token attention
over that cache (with a prefix that the whole batch shares) and token sampling.

``listed()`` names the cases, ``draw(rng)`` gives another one of the same ranges, ``prepare(case, seed)``
makes the inputs, ``run(state)`` does one pass.  With ``own`` false a pass is written in elementary torch
operations (fp32, or fp64 where fp32 loses what matters); with ``own`` true it calls the package's operators.
``exact(case, seed)`` is the definition in fp64.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"


# ------------------------------------------------------------------------- cases
def listed():
    return [
        # q | k of one layer of the ~170M training configuration (12 heads of 64, 8 x 4096 tokens), both directions
        dict(name="rope_train", op="rope", batch=8, tokens=4096, heads=24, dim=64, rotary=64, layout="interleaved",
             scaling="none", factor=1.0, start=0, dtype="bf16", train=True),
        # a shard of a very long context: half layout, half of a head of 96 rotated, frequencies scaled
        dict(name="rope_long_half", op="rope", batch=1, tokens=16384, heads=32, dim=96, rotary=48, layout="half",
             scaling="yarn", factor=32.0, start=1000000, dtype="fp32", train=False),
        # one decoding step of a batch, every sequence at its own position
        dict(name="rope_step", op="rope", batch=64, tokens=1, heads=24, dim=64, rotary=64, layout="interleaved",
             scaling="ntk", factor=4.0, start=5000, dtype="fp16", train=False),
        # one decoding step into a 512-slot ring of 12 heads: rotate, quantise, store; the ring read back
        dict(name="cache_step_int8", op="cache", batch=8, tokens=1, heads=12, dim=64, slots=512, kind="int8",
             layout="interleaved", rotary=64, start=700, dtype="bf16", ragged=True),
        # prompts of unequal lengths (padded batch) written into a long cache of 16 heads of 96
        dict(name="cache_prompt_fp8", op="cache", batch=4, tokens=4096, heads=16, dim=96, slots=8192, kind="fp8",
             layout="half", rotary=96, start=0, dtype="bf16", ragged=True),
        # one user, window 512, 4 persistent tokens: latency
        dict(name="attn_one", op="attend", batch=1, heads=12, kv_heads=12, dim=64, slots=512, longest=900,
             shortest=900, prefix=4, kind="bf16", dtype="bf16", lse=False),
        # a full batch of unequal lengths, some past the ring's end, int8 cache, 16 persistent tokens
        dict(name="attn_ragged_int8", op="attend", batch=64, heads=12, kv_heads=12, dim=64, slots=8192, longest=12000,
             shortest=1, prefix=16, kind="int8", dtype="bf16", lse=False),
        # many users behind one long shared prompt, a short text of their own each
        dict(name="attn_shared_prefix", op="attend", batch=128, heads=12, kv_heads=12, dim=64, slots=512, longest=512,
             shortest=1, prefix=16384, kind="bf16", dtype="bf16", lse=True),
        # long contexts, four query heads to a key head of 128, fp8 cache
        dict(name="attn_long_grouped_fp8", op="attend", batch=16, heads=32, kv_heads=8, dim=128, slots=32768,
             longest=32768, shortest=9000, prefix=0, kind="fp8", dtype="fp16", lse=True),
        # one user, the defaults of text generation
        dict(name="sample_one", op="sample", batch=1, vocab=32000, dtype="bf16", top_k=50, top_p=0.9, min_p=0.0,
             temperature=1.0, penalty=1.0, history=0, mixed=False),
        # a batch whose requests each bring their own settings, with a repetition penalty
        dict(name="sample_mixed", op="sample", batch=64, vocab=32000, dtype="bf16", top_k=50, top_p=0.9, min_p=0.05,
             temperature=0.8, penalty=1.2, history=400, mixed=True),
        # a large vocabulary, nucleus and min-p alone
        dict(name="sample_large", op="sample", batch=256, vocab=131072, dtype="fp32", top_k=0, top_p=0.95, min_p=0.001,
             temperature=1.0, penalty=1.0, history=0, mixed=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "cache", "attend", "attend", "sample"])
    if op == "rope":
        dim = rng.choice([32, 64, 80, 96, 128])
        heads = rng.randint(1, 40)
        batch = _log(rng, 1, 64)
        tokens = _log(rng, 1, max(1, min(32768, 48_000_000 // (batch * heads * dim))))
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return dict(op=op, batch=batch, tokens=tokens, heads=heads, dim=dim,
                    rotary=dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2),
                    layout=rng.choice(["interleaved", "half"]), scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 8.0, 32.0]), start=_log(rng, 1, 2000000) - 1,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), train=rng.random() < 0.5)
    if op == "cache":
        dim = rng.choice([32, 64, 96, 128])
        heads = rng.randint(1, 32)
        batch = _log(rng, 1, 64)
        slots = _log(rng, 8, max(8, min(16384, 48_000_000 // (batch * heads * dim))))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return dict(op=op, batch=batch, tokens=1 if rng.random() < 0.4 else _log(rng, 1, slots + slots // 4), heads=heads,
                    dim=dim, slots=slots, kind="fp32" if dtype == "fp32" else rng.choice(["int8", "fp8", dtype]),
                    layout=rng.choice(["interleaved", "half"]), rotary=rng.choice([0, dim, dim // 2]),
                    start=_log(rng, 1, 20000) - 1, dtype=dtype, ragged=rng.random() < 0.7)
    if op == "attend":
        dim = rng.choice([64, 64, 96, 128])
        kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
        batch = _log(rng, 1, 128)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        kind = rng.choice([dtype, dtype, "int8", "fp8"])
        slots = _log(rng, 16, max(16, min(65536, 200_000_000 // (batch * kv_heads * dim))))
        longest = _log(rng, 1, slots + slots // 2)
        prefix = rng.choice([0, 4, 16, _log(rng, 1, max(1, min(16384, 128 * 12 * 16384 // (batch * heads))))])
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, slots=slots, longest=longest,
                    shortest=rng.choice([longest, 1, (longest + 1) // 2]), prefix=prefix, kind=kind, dtype=dtype,
                    lse=rng.random() < 0.5)
    mixed = rng.random() < 0.5
    vocab = rng.choice([32000, _log(rng, 100, 131072)])
    return dict(op=op, batch=_log(rng, 1, 256), vocab=vocab, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                top_k=rng.choice([0, 1, 40, min(vocab, 1000)]), top_p=rng.choice([1.0, 0.9, 0.5]),
                min_p=rng.choice([0.0, 0.02, 0.2]), temperature=rng.choice([0.7, 1.0, 1.5]),
                penalty=rng.choice([1.0, 1.3]), history=rng.choice([0, 1, 300]), mixed=mixed)


def _lengths(case):
    """Sequence lengths between ``shortest`` and ``longest``, spread evenly, the first one the longest."""
    lo, hi = case["shortest"], case["longest"]
    return [hi - int((hi - lo) * ((0.6180339887498949 * i) % 1.0)) for i in range(case["batch"])]


def _counts(case):
    """How many of the padded batch's new tokens are real."""
    t = case["tokens"]
    if not case["ragged"] or t == 1:
        return [t] * case["batch"]
    return [t - int(0.75 * t * ((0.6180339887498949 * i) % 1.0)) for i in range(case["batch"])]


def _starts(case):
    step = 7 if case["ragged"] else 0
    return [case["start"] + step * i for i in range(case["batch"])]


def _kind_size(kind):
    return {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1, "fp8": 1}[kind]


def work(case):
    op, b = case["op"], case["batch"]
    if op == "rope":
        n, size = b * case["tokens"] * case["heads"] * case["dim"], _kind_size(case["dtype"])
        passes = 2 if case["train"] else 1
        return {"bytes": 2 * passes * n * size, "flops": 3 * passes * n * case["rotary"] // case["dim"]}
    if op == "cache":
        n = case["heads"] * case["dim"]
        s = case["slots"]
        new = sum(min(c, s) for c in _counts(case))
        held = sum(min(p + c, s) for p, c in zip(_starts(case), _counts(case)))
        row = n * _kind_size(case["kind"]) + (4 * case["heads"] if case["kind"] in ("int8", "fp8") else 0)
        size = _kind_size(case["dtype"])
        q = 2 * n * size * b * case["tokens"]
        return {"bytes": q + 2 * new * (n * size + row) + 2 * held * row + 2 * b * s * n * size, "flops": 6 * n * new + 2 * n * held}
    if op == "attend":
        d, h, hk = case["dim"], case["heads"], case["kv_heads"]
        seen = sum(min(n, case["slots"]) for n in _lengths(case))
        row = d * _kind_size(case["kind"]) + (4 if case["kind"] in ("int8", "fp8") else 0)
        size = _kind_size(case["dtype"])
        return {"bytes": 2 * hk * seen * row + 2 * hk * case["prefix"] * d * size + 2 * b * h * d * size,
                "flops": 4 * d * h * (seen + b * case["prefix"])}
    return {"bytes": b * case["vocab"] * _kind_size(case["dtype"]) + 8 * b * case["history"] + 28 * b,
            "flops": 4 * b * case["vocab"]}


# ------------------------------------------------------------------------- inputs
def _frequencies(rotary, scaling, factor, base=10000.0, original=8192):
    """Rotation per position of each pair, and the amplitude of the rotated part (host, once per model)."""
    i = torch.arange(0, rotary, 2, dtype=torch.float64)
    amplitude = 1.0
    if scaling == "ntk":
        base = base * factor ** (rotary / max(rotary - 2, 1))
    f = base ** (-i / rotary)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        turns = original * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    return f.float().to(DEVICE), amplitude


def _quantise(x, kind):
    """Stored values and the scale of each row of the last dimension."""
    if kind in DTYPES:
        return x.to(DTYPES[kind]), None
    top = 127.0 if kind == "int8" else 448.0
    amax = x.abs().amax(dim=-1)
    full = amax >= 2.0 ** -100
    inv = torch.where(full, top / amax, torch.zeros_like(amax))
    scale = torch.where(full, amax / top, torch.ones_like(amax))
    y = x * inv[..., None]
    q = y.round().to(torch.int8) if kind == "int8" else y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op, b = case["op"], case["batch"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    s = dict(case)
    if op == "rope":
        h, d, dt = case["heads"], case["dim"], DTYPES[case["dtype"]]
        # q | k are two thirds of the fused projection's output
        fused = randn(b, case["tokens"], h + (h + 1) // 2, d).to(dt)
        s["x"] = fused[:, :, :h].detach().requires_grad_(case["train"])
        s["positions"] = (torch.arange(case["tokens"], device=DEVICE)[None] + case["start"]
                          + 13 * torch.arange(b, device=DEVICE)[:, None])
        s["inv_freq"], s["amplitude"] = _frequencies(case["rotary"], case["scaling"], case["factor"])
        if case["train"]:
            s["dy"] = randn(b, case["tokens"], h, d).to(dt)
    elif op == "cache":
        h, d, n, dt = case["heads"], case["dim"], case["slots"], DTYPES[case["dtype"]]
        qkv = randn(b, case["tokens"], 3 * h, d).to(dt)
        s["q"], s["new_k"], s["new_v"] = qkv[:, :, :h], qkv[:, :, h:2 * h], qkv[:, :, 2 * h:]
        for name in ("k", "v"):
            s[name], s[name + "_scale"] = _quantise(randn(b, h, n, d), case["kind"])
        s["starts"] = torch.tensor(_starts(case), device=DEVICE)
        s["counts"] = torch.tensor(_counts(case), device=DEVICE)
        s["after"] = s["starts"] + s["counts"]
        s["inv_freq"] = _frequencies(case["rotary"], "none", 1.0)[0] if case["rotary"] else None
    elif op == "attend":
        h, hk, d, n, dt = case["heads"], case["kv_heads"], case["dim"], case["slots"], DTYPES[case["dtype"]]
        s["q"] = (1.5 * randn(b, h, d)).to(dt)
        channel = 0.5 + torch.rand(hk, 1, d, generator=g, device=DEVICE)
        for name in ("k", "v"):
            s[name], s[name + "_scale"] = _quantise(randn(b, hk, n, d) * channel, case["kind"])
        s["lengths"] = torch.tensor(_lengths(case), device=DEVICE)
        s["prefix_k"] = (randn(case["prefix"], hk, d) * channel[None, :, 0]).to(dt) if case["prefix"] else None
        s["prefix_v"] = randn(case["prefix"], hk, d).to(dt) if case["prefix"] else None
    else:
        v, dt = case["vocab"], DTYPES[case["dtype"]]
        # logits of a language model: a broad body, and a few tokens far above it
        lift = torch.zeros(b, v, device=DEVICE).scatter_(
            1, torch.randint(0, v, (b, 24), generator=g, device=DEVICE), 6 + 1.5 * randn(b, 24))
        s["logits"] = (2.2 * randn(b, v) + lift).to(dt)
        s["uniform"] = torch.rand(b, generator=g, device=DEVICE)
        row = torch.arange(b, device=DEVICE)
        if case["mixed"]:  # each request its own settings, switched off for some
            s["temps"] = case["temperature"] * (0.5 + 0.25 * (row % 5).float()) * (row % 11 != 10)
            s["ks"] = torch.where(row % 3 == 0, 0, case["top_k"] + 7 * (row % 4))
            s["ps"] = torch.where(row % 4 == 1, 1.0, case["top_p"] - 0.05 * (row % 3).float())
            s["mins"] = case["min_p"] * (row % 2).float()
            s["penalties"] = 1.0 + (case["penalty"] - 1.0) * (row % 3).float()
        else:
            s["temps"] = torch.full((b,), case["temperature"], device=DEVICE)
            s["ks"] = torch.full((b,), case["top_k"], device=DEVICE)
            s["ps"] = torch.full((b,), case["top_p"], device=DEVICE)
            s["mins"] = torch.full((b,), case["min_p"], device=DEVICE)
            s["penalties"] = torch.full((b,), case["penalty"], device=DEVICE)
        s["generated"] = torch.randint(0, v, (b, case["history"]), generator=g, device=DEVICE) if case["history"] else None
    return s


# ------------------------------------------------------------------------- plain forms
def _turn(x, positions, inv_freq, layout, amplitude=1.0, back=False):
    """Rotate the first ``2 * len(inv_freq)`` of the last dimension of ``x`` [B, T, H, d] (fp32 out)."""
    x = x.float()
    n = inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq.double()
    cos, sin = (amplitude * angle.cos()).float()[:, :, None], (amplitude * angle.sin()).float()[:, :, None]
    if back:
        sin = -sin
    part = x[..., :2 * n]
    if layout == "interleaved":
        a, c = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - c * sin, a * sin + c * cos], dim=-1).flatten(-2)
    else:
        a, c = part[..., :n], part[..., n:]
        part = torch.cat([a * cos - c * sin, a * sin + c * cos], dim=-1)
    return torch.cat([part, x[..., 2 * n:]], dim=-1)


def _plain_rope(s):
    y = _turn(s["x"].detach(), s["positions"], s["inv_freq"], s["layout"], s["amplitude"]).to(s["x"].dtype)
    if not s["train"]:
        return {"y": y}
    dx = _turn(s["dy"], s["positions"], s["inv_freq"], s["layout"], s["amplitude"], back=True)
    return {"y": y, "dx": dx.to(y.dtype)}


def _plain_cache(s):
    n, dt = s["slots"], s["q"].dtype
    at = s["starts"][:, None] + torch.arange(s["tokens"], device=DEVICE)
    q, k = s["q"], s["new_k"].float()
    if s["inv_freq"] is not None:
        q = _turn(q, at, s["inv_freq"], s["layout"]).to(dt)
        k = _turn(k, at, s["inv_freq"], s["layout"])
    # the newest token that each slot holds, and whether it is one of the new ones
    slot = torch.arange(n, device=DEVICE)
    last = s["after"][:, None] - 1
    t = last - (last - slot) % n - s["starts"][:, None]
    hit = (t >= 0) & (t < s["counts"][:, None])
    index = t.clamp(0, s["tokens"] - 1)[:, :, None, None].expand(-1, -1, s["heads"], s["dim"])
    held = s["after"].clamp(max=n)[:, None]
    first = (s["after"] - n).clamp(min=0)[:, None]
    order = (first + slot) % n
    out = {"q": q.contiguous()}
    for name, new in (("k", k), ("v", s["new_v"].float())):
        stored, scale = _quantise(torch.gather(new, 1, index).transpose(1, 2), s["kind"])
        place = hit[:, None, :, None]
        s[name].copy_(torch.where(place, stored.float(), s[name].float()).to(stored.dtype))
        value = s[name].float()
        if scale is not None:
            s[name + "_scale"].copy_(torch.where(hit[:, None], scale, s[name + "_scale"]))
            value = value * s[name + "_scale"][..., None]
            out[name + "_scale"] = s[name + "_scale"]
        value = torch.gather(value, 2, order[:, None, :, None].expand_as(value))
        out[name] = torch.where((slot < held)[:, None, :, None], value, 0.0).to(dt)
    return out


def _plain_attend(s):
    b, h, d = s["q"].shape
    hk, n = s["kv_heads"], s["slots"]
    q = s["q"].float().reshape(b, hk, h // hk, d) * d ** -0.5
    k, v = s["k"].float(), s["v"].float()
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][..., None], v * s["v_scale"][..., None]
    slot = torch.arange(n, device=DEVICE)
    seen = (slot < s["lengths"][:, None])[:, None, None]
    score = torch.matmul(q, k.transpose(2, 3)).masked_fill(~seen, float("-inf"))
    if s["prefix_k"] is not None:
        pk, pv = s["prefix_k"].float().permute(1, 2, 0), s["prefix_v"].float().transpose(0, 1)
        rows = q.transpose(0, 1).reshape(hk, -1, d)  # the queries of the whole batch, by key head
        ahead = torch.matmul(rows, pk).reshape(hk, b, h // hk, -1).transpose(0, 1)
        score = torch.cat([score, ahead], dim=-1)
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    e = torch.exp(score - top)
    total = e.sum(dim=-1, keepdim=True)
    o = torch.matmul(e[..., :n], torch.where(seen.transpose(2, 3), v, 0.0))
    if s["prefix_k"] is not None:
        rows = e[..., n:].transpose(0, 1).reshape(hk, b * (h // hk), -1)
        o = o + torch.matmul(rows, pv).reshape(hk, b, h // hk, d).transpose(0, 1)
    out = {"out": torch.where(total > 0, o / total, 0.0).reshape(b, h, d).to(s["q"].dtype)}
    if s["lse"]:
        out["lse"] = (top + torch.log(total)).reshape(b, h)
    return out


def _plain_sample(s):
    logits = s["logits"].float()
    b, v = logits.shape
    greedy = s["temps"] <= 0
    z = logits / torch.where(greedy, 1.0, s["temps"])[:, None]
    if s["generated"] is not None:
        seen = torch.zeros_like(z, dtype=torch.bool).scatter_(1, s["generated"], True)
        z = torch.where(seen, z / s["penalties"][:, None], z)
    z = torch.where(torch.isnan(z), float("-inf"), z)
    down, order = torch.sort(z, dim=1, descending=True, stable=True)
    k = torch.where((s["ks"] <= 0) | (s["ks"] > v), v, s["ks"])
    kth = torch.gather(down, 1, (k - 1)[:, None])
    weight = torch.exp(z.double() - down[:, :1].double())
    weight = torch.where(z >= kth, weight, 0.0)
    ranked = torch.gather(weight, 1, order)
    ahead = torch.cumsum(ranked, dim=1) - ranked
    nucleus = torch.where(s["ps"] >= 1, float("inf"), s["ps"].double() * ranked.sum(dim=1))
    keep = torch.zeros_like(z, dtype=torch.bool).scatter_(1, order, ahead <= nucleus[:, None])
    weight = torch.where(keep & (weight >= s["mins"].double()[:, None]), weight, 0.0)
    run_sum = torch.cumsum(weight, dim=1)
    total = run_sum[:, -1:]
    token = (run_sum <= s["uniform"].double()[:, None] * total).sum(dim=1)
    place = torch.arange(v, device=DEVICE)
    token = torch.minimum(token, torch.where(weight > 0, place, -1).amax(dim=1))
    token = torch.where(greedy, order[:, 0], token)
    logprob = torch.log(torch.gather(weight, 1, token[:, None]) / total)[:, 0]
    return {"token": token, "logprob": torch.where(greedy, 0.0, logprob).float()}


def run(s):
    op = s["op"]
    if not own:
        return {"rope": _plain_rope, "cache": _plain_cache, "attend": _plain_attend, "sample": _plain_sample}[op](s)
    from titans_pytorch_b200 import ops

    if op == "rope":
        y = ops.rotary_embedding(s["x"], s["positions"], s["inv_freq"], layout=s["layout"], amplitude=s["amplitude"])
        if not s["train"]:
            return {"y": y}
        dx, = torch.autograd.grad(y, s["x"], s["dy"])
        return {"y": y.detach(), "dx": dx}
    if op == "cache":
        cache = ops.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        q = ops.kv_cache_write(cache, s["new_k"], s["new_v"], s["starts"], counts=s["counts"], q=s["q"],
                               inv_freq=s["inv_freq"], layout=s["layout"])
        k, v = ops.kv_cache_read(cache, s["after"], dtype=s["q"].dtype)
        out = {"q": q, "k": k, "v": v}
        if s["k_scale"] is not None:
            out.update(k_scale=cache.k_scale, v_scale=cache.v_scale)
        return out
    if op == "attend":
        cache = ops.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        r = ops.decode_attention(s["q"], cache, s["lengths"], s["prefix_k"], s["prefix_v"], return_lse=s["lse"])
        return {"out": r[0], "lse": r[1]} if s["lse"] else {"out": r}
    token, logprob = ops.sample_tokens(s["logits"], s["uniform"], temperature=s["temps"], top_k=s["ks"], top_p=s["ps"],
                                       min_p=s["mins"], generated=s["generated"], repetition_penalty=s["penalties"],
                                       return_logprob=True)
    return {"token": token, "logprob": logprob}


# ------------------------------------------------------------------------- the definition in fp64
def _exact_turn(x, positions, inv_freq, layout, amplitude, sign):
    n = inv_freq.numel()
    first = torch.arange(n, device=x.device) * 2 if layout == "interleaved" else torch.arange(n, device=x.device)
    second = first + (1 if layout == "interleaved" else n)
    z = torch.polar(torch.full((), float(amplitude), dtype=torch.float64, device=x.device).expand(positions.shape + (n,)).contiguous(),
                    sign * positions.double().unsqueeze(-1) * inv_freq.double())
    pair = torch.complex(x.double()[..., first], x.double()[..., second]) * z.unsqueeze(2)
    y = x.double().clone()
    y[..., first], y[..., second] = pair.real, pair.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        args = (s["positions"], s["inv_freq"], case["layout"], s["amplitude"])
        out = {"y": _exact_turn(s["x"].detach(), *args, 1.0)}
        if case["train"]:
            out["dx"] = _exact_turn(s["dy"], *args, -1.0)
        return out
    if op == "cache":
        n, h, d = case["slots"], case["heads"], case["dim"]
        q, k = s["q"].double(), s["new_k"].double()
        if s["inv_freq"] is not None:
            at = torch.stack([torch.arange(p, p + case["tokens"], device=DEVICE) for p in _starts(case)])
            q, k = (_exact_turn(x, at, s["inv_freq"], case["layout"], 1.0, 1.0) for x in (q, k))
        top = {"int8": 127.0, "fp8": 448.0}.get(case["kind"])
        out = {"q": q}
        for name, new in (("k", k), ("v", s["new_v"].double())):
            value, scale = s[name].double(), s[name + "_scale"]
            scale = None if scale is None else scale.double()
            read = torch.zeros(case["batch"], h, n, d, dtype=torch.float64, device=DEVICE)
            for i, (p, c) in enumerate(zip(_starts(case), _counts(case))):
                tokens = torch.arange(max(0, c - n), c, device=DEVICE)
                place, rows = (p + tokens) % n, new[i, tokens].transpose(0, 1)
                if top is None:
                    value[i, :, place] = rows.to(DTYPES[case["kind"]]).double()
                else:
                    step = rows.abs().amax(-1) / top
                    level = rows / step.unsqueeze(-1)
                    level = level.round() if case["kind"] == "int8" else level.to(torch.float8_e4m3fn).double()
                    value[i, :, place], scale[i, :, place] = level, step
                full = value[i] if scale is None else value[i] * scale[i].unsqueeze(-1)
                held = torch.arange(max(0, p + c - n), p + c, device=DEVICE) % n
                read[i, :, :held.numel()] = full[:, held]
            out[name] = read
            if scale is not None:
                out[name + "_scale"] = scale
        return out
    if op == "attend":
        group = case["heads"] // case["kv_heads"]
        outs, lses = [], []
        for i, length in enumerate(_lengths(case)):
            m = min(length, case["slots"])
            k, v = s["k"][i, :, :m].double(), s["v"][i, :, :m].double()
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][i, :, :m, None].double(), v * s["v_scale"][i, :, :m, None].double()
            if s["prefix_k"] is not None:
                k = torch.cat([s["prefix_k"].double().transpose(0, 1), k], dim=1)
                v = torch.cat([s["prefix_v"].double().transpose(0, 1), v], dim=1)
            q = s["q"][i].double().reshape(case["kv_heads"], group, -1)
            score = torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(case["dim"])
            lses.append(torch.logsumexp(score, dim=-1).reshape(-1))
            outs.append(torch.einsum("hgn,hnd->hgd", torch.softmax(score, dim=-1), v).reshape(case["heads"], -1))
        out = {"out": torch.stack(outs)}
        return {**out, "lse": torch.stack(lses)} if case["lse"] else out
    # sampling: the probability of the token that the definition picks
    tokens, probs = [], []
    z32 = s["logits"].float() / torch.where(s["temps"] > 0, s["temps"], 1.0)[:, None]
    for i in range(case["batch"]):
        z = z32[i].clone()
        if s["generated"] is not None:
            at = s["generated"][i].unique()
            z[at] = z[at] / s["penalties"][i]
        if float(s["temps"][i]) <= 0:
            tokens.append(int(torch.nonzero(z == z.max())[0]))
            probs.append(0.0)
            continue
        values, order = torch.sort(z, descending=True, stable=True)
        w = torch.exp(values.double() - values[0].double())
        k = int(s["ks"][i])
        if 0 < k < w.numel():
            w = w * (values >= values[k - 1])
        p = float(s["ps"][i])
        if p < 1:
            before = torch.cat([w.new_zeros(1), torch.cumsum(w, 0)[:-1]])
            w = w * (before <= p * w.sum())
        w = w * (w >= float(s["mins"][i]))
        by_index = torch.empty_like(w)
        by_index[order] = w
        reach = torch.cumsum(by_index, 0)
        t = int(torch.searchsorted(reach, s["uniform"][i].double() * reach[-1], right=True))
        t = min(t, int(torch.nonzero(by_index)[-1]))
        tokens.append(t)
        probs.append(float(torch.log(by_index[t] / reach[-1])))
    return {"token": torch.tensor(tokens, device=DEVICE), "logprob": torch.tensor(probs, dtype=torch.float64, device=DEVICE)}
