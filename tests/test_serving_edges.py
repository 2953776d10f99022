"""Inputs at the edges of the serving operators: values of very unequal size, infinities and NaN that are visible, settings
out of range, tensors that share memory, forward-mode derivatives, captured restatements."""

from __future__ import annotations

import pytest
import torch

from titans_pytorch_b200 import ops
from titans_pytorch_b200.ops.decode_attention import decode_attention_reference
from titans_pytorch_b200.ops.kv_cache import KINDS, quantise_rows

gpu = pytest.mark.gpu
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


def _gen(seed=0, device="cpu"):
    return torch.Generator(device=device).manual_seed(seed)


# ------------------------------------------------------------------------- attention: values of unequal size
def _sink_case(kind, dtype, d, keys, nats, amplitude, batch=2, heads=2, seed=41):
    """One key whose score is ``nats`` above the largest other one and whose value row is zero; values of ``amplitude``."""
    g = _gen(seed)
    q = (1.5 * torch.randn(batch, heads, d, generator=g)).to(dtype)
    k = torch.randn(batch, heads, keys, d, generator=g)
    v = amplitude * torch.randn(batch, heads, keys, d, generator=g)
    qd = q.double()
    top = torch.einsum("bhd,bhkd->bhk", qd, k.double()).amax(-1) * d ** -0.5 + nats
    k[:, :, keys // 3] = (qd * (top / (d ** -0.5 * qd.square().sum(-1)))[..., None]).float()
    v[:, :, keys // 3] = -0.0
    (k, ks), (v, vs) = (quantise_rows(x, KINDS[kind]) for x in (k, v))
    return q.cuda(), ops.KVCache(*(t if t is None else t.cuda() for t in (k, v, ks, vs)))


def _sink_bound(q, cache, ref):
    """|error| of each output element.
    Scores: d products and sums in fp32 of |q||k| and queries in fp16 (2 d 2^-24 together, as elements below 2^-14 of the
    row's largest are off by 2^-25 of that), two roundings of a score after that and one of its difference to the
    maximum (4 * 2^-24 of it); the exponential 2^-20.  Numerator and denominator: twice.
    Weights: half a step of fp16 (bf16 beside a bf16 cache) of each; in fp16 one that is subnormal by 2^-25, where the
    largest weight times value scale is 2^7 at least: 2^-32 of that times the stored value.  A row without magnitude has
    the weight 2^97 at least, so that weights beside it are off by 2^-122 of its own too.
    Sums of n keys in fp32; the result rounded once.  Steps of subnormals: 2^-149 of an fp32 weight and of the result
    in fp32, 2^-133 and 2^-24 of a result in bf16 and fp16."""
    d, n = q.shape[-1], cache.slots
    k, v, unit, p = cache.k.double(), cache.v.double(), 1.0, None
    ks = 1.0 if cache.k_scale is None else cache.k_scale.double()[..., None]
    vs = torch.ones(k.shape[:3], device=k.device, dtype=torch.float64) if cache.v_scale is None else cache.v_scale.double()
    s = torch.einsum("bhd,bhkd->bhk", q.double(), k * ks) * d ** -0.5
    p = torch.softmax(s, -1)
    seen = torch.einsum("bhk,bhkd->bhd", p, (v * vs[..., None]).abs())
    scores = 2 * d * 2.0 ** -24 * q.double().abs().sum(-1) * (k * ks).abs().amax((-2, -1)) * d ** -0.5 \
        + 4 * 2.0 ** -24 * s.abs().amax(-1) + 2.0 ** -20
    exact_bf16 = q.dtype == torch.bfloat16 and cache.v_scale is None
    half = 0.0 if q.dtype == torch.float32 else HALF[torch.bfloat16] if exact_bf16 else HALF[torch.float16]
    low = torch.zeros_like(seen)
    if half and not exact_bf16:
        # (16-bit caches: of the largest weight, with magnitude or without)
        sized = v.abs().amax(-1) > 0 if cache.v_scale is not None else torch.ones_like(vs, dtype=torch.bool)
        unit = (p * vs * sized).amax(-1)
        low = (2.0 ** -32 * unit[..., None] + (0.0 if cache.v_scale is None else 2.0 ** -122)) * v.abs().sum(-2)
    return ((2 * scores[..., None] + half + n * 2.0 ** -23) * seen + low) * 1.01 + HALF[q.dtype] * 1.01 * ref.abs() \
        + 2.0 ** -149 * ((v * vs[..., None]).abs().sum(-2) + 1) \
        + {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 0.0}[q.dtype]


@gpu
@pytest.mark.parametrize("nats,amplitude", [(10.0, 1.0), (6.0, 1e-2), (4.0, 1e-3), (0.0, 1e-5), (15.0, 1e-4), (25.0, 1.0),
                                            (90.0, 1.0), (0.0, 1e-28), (2.0, 1e20)])
@pytest.mark.parametrize("d", [64, 96, 128, 40])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_zero_value_rows_leave_the_other_rows_their_precision(kind, d, nats, amplitude):
    """A zero row has the scale 1, far above that of small values, and adds nothing."""
    _cuda()
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        if dtype == torch.float16 and amplitude > 1e4:  # the result does not fit
            continue
        for keys in (300, 1100):
            q, cache = _sink_case(kind, dtype, d, keys, nats, amplitude)
            n = torch.full((2,), keys, device="cuda")
            out, lse = ops.decode_attention(q, cache, n, return_lse=True)
            ref, rl = decode_attention_reference(q.double(), cache, n, scale=d ** -0.5)
            bad = (out.double() - ref).abs() - _sink_bound(q, cache, ref)
            assert (bad <= 0).all(), (dtype, keys, float(bad.max()), float(ref.abs().max()))
            assert ((lse.double() - rl).abs() <= 2.0 ** -14 + 2.0 ** -20 * rl.abs()).all()


@gpu
@pytest.mark.parametrize("nats", [10.0, 15.0, 20.0])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_zero_value_rows_fp16(d, nats):
    """fp16 weights beside fp16 keys, in the cache and in a prefix, for few query rows and for many."""
    _cuda()
    q, cache = _sink_case("float16", torch.float16, d, 300, nats, 1000.0)
    n = torch.full((2,), 300, device="cuda")
    ref, _ = decode_attention_reference(q.double(), cache, n, scale=d ** -0.5)
    bound = _sink_bound(q, cache, ref)
    assert ((ops.decode_attention(q, cache, n).double() - ref).abs() <= bound).all()
    # the first sequence's keys as a prefix, and its query for every row
    pk, pv = (t[0].transpose(0, 1).contiguous() for t in (cache.k, cache.v))
    for rows in (3, 40):
        empty = ops.KVCache.allocate(rows, 2, 8, d, "float16", "cuda")
        out = ops.decode_attention(q[:1].expand(rows, -1, -1), empty, torch.zeros(rows, dtype=torch.int64, device="cuda"), pk, pv)
        assert ((out.double() - ref[:1]).abs() <= bound[:1]).all()


@gpu
@pytest.mark.parametrize("d", [64, 96, 128, 40])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_visible_value_rows_that_are_not_finite(kind, d):
    """They make the output NaN (not zero), and leave the log-sum-exp as it is."""
    _cuda()
    g = _gen(43)
    S, H = 70, 2
    for dtype in (torch.bfloat16, torch.float32):
        cache = ops.KVCache.allocate(3, H, S, d, kind, "cuda")
        new = torch.randn(3, S, H, d, generator=g).to(dtype).cuda()
        v = torch.randn(3, S, H, d, generator=g).to(dtype).cuda()
        v[0, :, :, 3] = float("inf")          # every row of the first sequence
        v[1, 17, 0, 5] = float("nan")         # one row of one head of the second
        ops.kv_cache_write(cache, new, v, torch.zeros(3, dtype=torch.int64, device="cuda"))
        q = torch.randn(3, H, d, generator=g).to(dtype).cuda()
        pk, pv = (torch.randn(5, H, d, generator=g).to(dtype).cuda() for _ in range(2))
        for lengths in ([1, 18, S], [S, S, 1]):
            n = torch.tensor(lengths, device="cuda")
            for prefix in ((None, None), (pk, pv)):
                out, lse = ops.decode_attention(q, cache, n, *prefix, return_lse=True)
                ref, rl = decode_attention_reference(q.double(), cache, n, *(None if t is None else t.double() for t in prefix),
                                                     scale=d ** -0.5)
                assert torch.equal(torch.isnan(out), torch.isnan(ref))
                assert torch.isnan(out[0]).all() and torch.isnan(out[1, 0]).all() and torch.isfinite(out[1, 1]).all()
                assert ((lse.double() - rl).abs() <= 2.0 ** -14).all()


@gpu
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_value_scales_of_zero_and_infinity(kind):
    """A cache of the caller's own may hold them: zero adds nothing, whatever the score; infinity is not a number."""
    _cuda()
    g = _gen(47)
    B, H, S, d = 2, 2, 90, 64
    k, ks = quantise_rows(torch.randn(B, H, S, d, generator=g), KINDS[kind])
    v, vs = quantise_rows(torch.randn(B, H, S, d, generator=g), KINDS[kind])
    q = (40 * torch.randn(B, H, d, generator=g)).to(torch.bfloat16).cuda()
    n = torch.tensor([S, 50], device="cuda")
    vs[0] = 0.0
    s = torch.einsum("bhd,bhkd->bhk", q.double().cpu(), k.double() * ks.double()[..., None])[1, :, :50]
    vs[1].scatter_(1, s.argsort(dim=1, descending=True)[:, :3], 0.0)    # the three likeliest keys of the second
    cache = ops.KVCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    out, lse = ops.decode_attention(q, cache, n, return_lse=True)
    ref, rl = decode_attention_reference(q.double(), cache, n, scale=d ** -0.5)
    assert (out[0] == 0).all() and torch.isfinite(out).all() and torch.isfinite(lse).all()
    assert ((lse.double() - rl).abs() <= 2.0 ** -14 + 2.0 ** -20 * rl.abs()).all()
    assert ((out.double() - ref).abs() <= 2.0 ** -6 * ref.abs().amax()).all()
    vs[0, :, 4] = float("inf")
    cache = ops.KVCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    out, lse = ops.decode_attention(q, cache, n, return_lse=True)
    assert not torch.isfinite(out[0]).any() and torch.isfinite(out[1]).all()
    assert ((lse.double() - rl).abs() <= 2.0 ** -14 + 2.0 ** -20 * rl.abs()).all()


# ------------------------------------------------------------------------- the part of a head that is not rotated
def _tail_case(d, rotary, dtype, device):
    g = _gen(53)
    x = torch.randn(2, 3, 4, d, generator=g)
    if rotary < d:
        x[0, 0, :, rotary] = float("inf")
        x[0, 1, :, d - 1] = float("nan")
        x[1, 0, :, rotary] = -0.0
        x[1, 1, :, rotary:] = -0.0
    return x.to(dtype).to(device)


@gpu
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,rotary", [(96, 20), (64, 2), (64, 8), (128, 64), (96, 94), (20, 6), (96, 48), (64, 0)])
def test_rope_copies_the_tail(d, rotary, dtype, layout):
    """Bit for bit, whatever it holds, and without an effect on what is rotated."""
    _cuda()
    x = _tail_case(d, rotary, dtype, "cuda")
    freq = ops.rope_frequencies(max(rotary, 2), device="cuda")[0][:rotary // 2]
    pos = torch.arange(3, device="cuda") + 7
    y = ops.rotary_embedding(x, pos, freq, layout=layout)
    words = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(y[..., rotary:].contiguous().view(words), x[..., rotary:].contiguous().view(words))
    clean = x.clone()
    clean[..., rotary:] = 1.0
    assert torch.isfinite(y[..., :rotary]).all()
    assert torch.equal(y[..., :rotary], ops.rotary_embedding(clean, pos, freq, layout=layout)[..., :rotary])


@gpu
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,rotary", [(96, 20), (64, 2), (64, 8), (128, 6), (96, 94), (40, 12)])
def test_cache_write_copies_the_tail(d, rotary, dtype, layout):
    _cuda()
    x = _tail_case(d, rotary, dtype, "cuda")
    freq = ops.rope_frequencies(rotary, device="cuda")[0]
    start = torch.tensor([0, 5], device="cuda")
    kind = {torch.bfloat16: "bfloat16", torch.float32: "float32"}[dtype]
    cache = ops.KVCache.allocate(2, 4, 16, d, kind, "cuda")
    q = ops.kv_cache_write(cache, x, x, start, q=x, inv_freq=freq, layout=layout)
    k = torch.stack([cache.k[b, :, int(start[b]):int(start[b]) + 3] for b in range(2)]).transpose(1, 2)
    words = torch.int32 if dtype == torch.float32 else torch.int16
    for y in (q, k):
        tail, want = y[..., rotary:].contiguous(), x[..., rotary:].contiguous()
        assert torch.equal(torch.isnan(tail), torch.isnan(want))
        live = ~torch.isnan(want)  # (a NaN may change its payload on the way through fp32)
        assert torch.equal(tail.view(words)[live], want.view(words)[live])
        assert torch.isfinite(y[..., :rotary]).all()


# ------------------------------------------------------------------------- forward-mode derivatives
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_rope_carries_tangents(device, layout):
    """The rotation is linear: its directional derivative is the rotation of the direction, with and without a backward."""
    from torch.autograd import forward_ad

    if device == "cuda":
        _cuda()
    freq, amp = ops.rope_frequencies(16, scaling="yarn", factor=4.0, device=device)
    x, t = (torch.randn(2, 3, 2, 32, generator=_gen(s)).to(device) for s in (59, 61))
    pos = torch.arange(3, device=device) + 9
    kw = dict(layout=layout, amplitude=amp)
    want = ops.rotary_embedding(t, pos, freq, **kw)
    for leaf in (x, x.clone().requires_grad_(True)):
        with forward_ad.dual_level():
            y = ops.rotary_embedding(forward_ad.make_dual(leaf, t), pos, freq, **kw)
            primal, tangent = forward_ad.unpack_dual(y)
            assert tangent is not None and torch.equal(tangent, want)
            assert torch.equal(primal, ops.rotary_embedding(x, pos, freq, **kw))
            with torch.no_grad():
                assert torch.equal(forward_ad.unpack_dual(ops.rotary_embedding(forward_ad.make_dual(leaf, t), pos, freq, **kw))[1], want)
    # the tangent of the gradient: of <dy, y> it is zero (y is linear), of |y|^2 / 2 the back-rotated, rotated direction
    leaf = x.clone().requires_grad_(True)
    with forward_ad.dual_level():
        y = ops.rotary_embedding(forward_ad.make_dual(leaf, t), pos, freq, **kw)
        (g,) = torch.autograd.grad(y.square().sum() / 2, leaf)
        out = ops.rotary_embedding(forward_ad.unpack_dual(y)[1].detach(), -pos, freq, **kw)
        assert (forward_ad.unpack_dual(g)[1] - out).abs().max() <= 4 * amp ** 2 * 2.0 ** -20 * float(t.abs().max())


# ------------------------------------------------------------------------- the decoders' settings
def _model(**kw):
    import titans_pytorch_b200 as T

    torch.manual_seed(0)
    fields = dict(dim=64, num_heads=2, num_layers=1, vocab_size=128, window_size=8, chunk_size=16, num_persistent_tokens=4,
                  dropout=0.0, max_seq_len=256, ffn_mult=2.0, memory_hidden_mult=2.0)
    return T.TitansMAG(T.TitansConfig(**{**fields, **kw})).eval()


@pytest.mark.parametrize("dim,heads", [(24, 2), (1024, 2)])
def test_ring_head_dim_is_checked_before_the_first_step(dim, heads, monkeypatch):
    """Where the kernels run, head dims that they do not take are refused at once; the restatement takes any."""
    from titans_pytorch_b200.inference import decode

    model = _model(dim=dim, num_heads=heads)
    dec = decode.StreamingDecoder(model, kv_cache="int8")
    assert torch.isfinite(dec.step(torch.zeros(1, 1, dtype=torch.long))).all()
    monkeypatch.setattr(decode, "want_kernels", lambda t, flag=None: True)
    with pytest.raises(ValueError, match="multiple of 8"):
        decode.StreamingDecoder(model, kv_cache="int8")


@gpu
def test_ring_head_dim_is_checked_on_the_gpu():
    _cuda()
    from titans_pytorch_b200.inference.decode import StreamingDecoder

    model = _model(dim=24).cuda()
    with pytest.raises(ValueError, match="multiple of 8"):
        StreamingDecoder(model, kv_cache="int8")


class _Uniforms:
    """Stands for ``sample_tokens`` in the batcher and keeps the numbers that it is given."""

    def __init__(self, monkeypatch):
        from titans_pytorch_b200.inference import generate

        self.seen, real = [], generate.sample_tokens

        def sample(logits, uniform, **kw):
            self.seen.append(uniform.clone())
            return real(logits, uniform, **kw)

        monkeypatch.setattr(generate, "sample_tokens", sample)


def _serve(requests, model=None):
    from titans_pytorch_b200.inference.generate import ContinuousBatcher

    batcher = ContinuousBatcher(model or _model(), max_batch_size=4)
    for ids, kw in requests:
        batcher.add_request(ids, **{"max_new_tokens": 4, **kw})
    return batcher.run()


def test_requests_without_a_seed_follow_the_global_one():
    """``min_p`` alone: the request's numbers follow ``torch.manual_seed``, as those of every other request."""
    prompt = torch.arange(6)
    runs = []
    for seed in (3, 3, 4):
        torch.manual_seed(seed)
        model = _model()
        torch.manual_seed(seed)
        runs.append([r["ids"].tolist() for r in _serve([(prompt, dict(min_p=1e-6, top_k=0, top_p=1.0)) for _ in range(3)], model)])
    assert runs[0] == runs[1] and runs[0] != runs[2]
    assert runs[0][0] != runs[0][1]  # each request has numbers of its own


@pytest.mark.parametrize("min_p", [-0.1, 1.5, float("nan")])
def test_request_min_p_is_checked(min_p):
    from titans_pytorch_b200.inference.generate import ContinuousBatcher

    for seed in (None, 1):
        with pytest.raises(ValueError, match="min_p"):
            ContinuousBatcher(_model()).add_request(torch.arange(3), min_p=min_p, seed=seed)


def test_request_top_p_out_of_range_is_the_nearest():
    """As :func:`sample_next` takes it."""
    prompt = torch.arange(6)
    for far, near in ((7.0, 1.0), (-2.0, 0.0)):
        a, b = (_serve([(prompt, dict(seed=5, top_p=p, top_k=0))])[0]["ids"].tolist() for p in (far, near))
        assert a == b


def test_uniform_numbers_do_not_follow_the_default_type(monkeypatch):
    from titans_pytorch_b200.inference.generate import sample_next

    logits = torch.randn(3, 50, generator=_gen(67))
    want = sample_next(logits, torch.zeros(3, 1, dtype=torch.int64), generator=_gen(1), fused=True)
    model, prompt = _model(), torch.arange(6)
    numbers = _Uniforms(monkeypatch)
    served = _serve([(prompt, dict(seed=5, top_k=0))], model)[0]["ids"].tolist()
    before = torch.get_default_dtype()
    for dtype in (torch.float64, torch.bfloat16):
        try:
            torch.set_default_dtype(dtype)
            assert torch.equal(sample_next(logits, torch.zeros(3, 1, dtype=torch.int64), generator=_gen(1), fused=True), want)
            numbers.seen.clear()
            assert _serve([(prompt, dict(seed=5, top_k=0))], model)[0]["ids"].tolist() == served
            assert all(u.dtype == torch.float32 for u in numbers.seen)
            assert float(numbers.seen[0]) == float(torch.rand((), generator=_gen(5), dtype=torch.float32))
        finally:
            torch.set_default_dtype(before)


@gpu
def test_seeded_requests_with_a_default_device():
    _cuda()
    model, prompt = _model(dim=128, window_size=16).cuda().to(torch.bfloat16), torch.arange(6)
    want = _serve([(prompt, dict(seed=5, top_k=0)), (prompt, dict(min_p=0.02))], model)[0]["ids"].tolist()
    try:
        torch.set_default_device("cuda")
        assert _serve([(prompt, dict(seed=5, top_k=0)), (prompt, dict(min_p=0.02))], model)[0]["ids"].tolist() == want
    finally:
        torch.set_default_device(None)


# ------------------------------------------------------------------------- sampling settings out of range
def _odd_settings(device):
    nan, inf = float("nan"), float("inf")
    g = _gen(79)
    logits = 2 * torch.randn(12, 200, generator=g)
    u = torch.rand(12, generator=g)
    odd = dict(top_p=(nan, 2.0, -1.0, inf), min_p=(nan, 3.0, -0.5, -inf))
    near = dict(top_p=(1.0, 1.0, 0.0, 1.0), min_p=(0.0, 1.0, 0.0, 0.0))
    for name in odd:
        for base in (dict(), dict(top_k=30), dict(temperature=0.7, top_p=0.8, min_p=0.01)):
            a, b = ({**base, name: torch.tensor(v * 3, device=device)} for v in (odd[name], near[name]))
            yield logits.to(device), u.to(device), u.to(device), a, b
    # uniform numbers: NaN and negative ones count as 0, those from 1 on give the last token that is kept
    bad = torch.tensor([nan, -0.3, -inf, 1.0, 1.5, inf] * 2)
    good = torch.tensor([0.0, 0.0, 0.0] + [1.0 - 2.0 ** -24] * 3).repeat(2)
    flat = torch.zeros(12, 200)
    flat[:, :5] = -inf
    flat[:, 190:] = -inf
    for kw in (dict(), dict(top_p=0.5), dict(min_p=0.5)):
        yield flat.to(device), bad.to(device), good.to(device), kw, kw


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_sampling_settings_out_of_range_count_as_the_nearest(device):
    if device == "cuda":
        _cuda()
    for logits, u, v, odd, near in _odd_settings(device):
        a = ops.sample_tokens(logits, u, return_logprob=True, **odd)
        b = ops.sample_tokens(logits, v, return_logprob=True, **near)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.isfinite(a[1]).all()
    # a temperature that is NaN: the largest, as 0
    hot = torch.tensor([float("nan"), 0.0, -1.0] * 4, device=device)
    tok, lp = ops.sample_tokens(2 * logits + torch.arange(200, device=device) % 7, u, temperature=hot, return_logprob=True)
    assert (tok == 6).all() and (lp == 0).all()


# ------------------------------------------------------------------------- the restatement in a captured step
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_cache_write_restatement_leaves_the_rest_as_it_was(kind, device):
    """Bits of every slot that no new token goes to, NaN among them, with tokens before position 0 and past the counts."""
    if device == "cuda":
        _cuda()
    B, T, H, S, d = 4, 11, 2, 6, 8
    g = _gen(83)
    cache = ops.KVCache.allocate(B, H, S, d, kind, device)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None:
            t.copy_(torch.randn(t.shape, generator=g).to(device))
    if cache.k_scale is None:
        cache.k[:, :, 1] = float("nan")
    old = [t if t is None else t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    k, v = (torch.randn(B, T, H, d, generator=g).to(device) for _ in range(2))
    start, counts = torch.tensor([-3, 2, 100, -20], device=device), torch.tensor([5, 3, 11, 7], device=device)
    ops.kv_cache_write(cache, k, v, start, counts=counts, use_kernels=False)
    bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}
    for data, scale, was, scale_was, new in ((cache.k, cache.k_scale, old[0], old[2], k), (cache.v, cache.v_scale, old[1], old[3], v)):
        row, s = quantise_rows(new, KINDS[kind])
        for b in range(B):
            held = {}
            for t in range(int(counts[b])):
                p = int(start[b]) + t
                if p >= 0:
                    held[p % S] = t
            for slot in range(S):
                want = row[b, held[slot]] if slot in held else was[b, :, slot]
                word = bits[want.element_size()]
                assert torch.equal(data[b, :, slot].contiguous().view(word), want.contiguous().view(word))
                if scale is not None:
                    assert torch.equal(scale[b, :, slot], s[b, held[slot]] if slot in held else scale_was[b, :, slot])


@gpu
@pytest.mark.parametrize("kind", ["bfloat16", "int8", "fp8"])
def test_restatement_decodes_in_a_graph(kind):
    """A model with ``use_kernels=False`` on the GPU: the captured step of the decoder, with the cache operators in it."""
    _cuda()
    from titans_pytorch_b200.inference.decode import StreamingDecoder

    model = _model(dim=128, window_size=16, use_kernels=False).cuda()
    ids = torch.randint(0, 128, (2, 24), generator=_gen(89)).cuda()
    a, b = (StreamingDecoder(model, batch=2, graph=g, kv_cache=kind) for g in (False, True))
    for t in range(ids.shape[1]):
        x, y = a.step(ids[:, t:t + 1]).float(), b.step(ids[:, t:t + 1]).float()
        assert torch.isfinite(y).all() and (x - y).norm() <= 1e-4 * x.norm()


# ------------------------------------------------------------------------- tensors that share memory
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_cache_write_of_its_own_rows(device):
    """New tokens that are views of the cache: what is stored is what they were before the call."""
    if device == "cuda":
        _cuda()
    B, H, S, d = 2, 3, 64, 64
    freq = ops.rope_frequencies(32, device=device)[0]
    for kind in ("bfloat16", "float32"):
        base = [torch.randn(B, H, S, d, generator=_gen(s)).to(KINDS[kind]).to(device) for s in (91, 93)]
        for shift, T in ((1, 60), (32, 32), (-1, 50)):
            start = torch.full((B,), 2 + shift, device=device)
            results = []
            for own in (True, False):
                cache = ops.KVCache(*(t.clone() for t in base))
                k, v = ((t if own else t.clone())[:, :, 2:2 + T].transpose(1, 2)[:, :S - 2 - max(shift, 0)] for t in (cache.k, cache.v))
                # keys from the values' rows and the other way round too
                for a, b in ((k, v), (v, k)):
                    q = ops.kv_cache_write(cache, a, b, start, q=a, inv_freq=freq)
                    results.append((own, cache.k.clone(), cache.v.clone(), q))
                    cache.k.copy_(base[0])
                    cache.v.copy_(base[1])
            for i in range(2):
                assert all(torch.equal(x, y) for x, y in zip(results[i][1:], results[2 + i][1:]))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_cache_whose_rows_share_memory_is_not_written(device):
    """Refused before anything is stored; such a cache can be read."""
    if device == "cuda":
        _cuda()
    S, d = 4, 8
    one = torch.zeros(1, 2, S, d, device=device)
    scale = torch.ones(3, 2, S, device=device)
    k = torch.ones(3, 2, 2, d, device=device)
    start = torch.zeros(3, dtype=torch.int64, device=device)
    full = torch.zeros(3, 2, S, d, device=device)
    eight = full.to(torch.int8)
    wide = torch.zeros(4 * 2 * S * d, device=device)
    for cache in (ops.KVCache(one.expand(3, -1, -1, -1), full), ops.KVCache(full, one.expand(3, -1, -1, -1)),
                  ops.KVCache(full, full), ops.KVCache(wide[:3 * 2 * S * d].view_as(full), wide[2 * S * d:].view_as(full)),
                  ops.KVCache(eight, eight.clone(), scale[:1].expand(3, -1, -1), scale),
                  ops.KVCache(eight, eight.clone(), scale, scale)):
        with pytest.raises(RuntimeError, match="share memory"):
            ops.kv_cache_write(cache, k, k, start)
        assert all((t == 0).all() for t in (one, full, eight, wide)) and (scale == 1).all()
        ops.kv_cache_read(cache, start + 2)
    # keys and values side by side in one tensor are two caches
    pair = torch.zeros(3, 2, S, 2 * d, device=device)
    ops.kv_cache_write(ops.KVCache(pair[..., :d], pair[..., d:]), k, 2 * k, start)
    assert (pair[:, :, :2, :d] == 1).all() and (pair[:, :, :2, d:] == 2).all() and (pair[:, :, 2:] == 0).all()


# ------------------------------------------------------------------------- dimensions of size one
@gpu
def test_sampling_takes_any_stride_of_a_dimension_of_one():
    _cuda()
    logits = torch.randn(1, 40, device="cuda")
    u = torch.full((1,), 0.5, device="cuda")
    tokens = torch.tensor([[3, 9, 4]], device="cuda")
    one = tokens[:, ::2][:, :1]
    assert one.stride(1) == 2 and one.is_contiguous()
    kw = dict(repetition_penalty=1.5, return_logprob=True)
    a, b = (ops.sample_tokens(logits, u, generated=t, **kw) for t in (one, tokens[:, :1].clone()))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    single = logits[:, ::3][:, :1]
    assert single.stride(1) == 3 and int(ops.sample_tokens(single, u)) == 0


# ------------------------------------------------------------------------- what sampling without the operator keeps drawing
def test_default_sampling_is_the_filtered_multinomial():
    """``sample_next`` without ``fused`` or ``min_p`` draws what ``torch.multinomial`` draws from the filtered softmax."""
    from titans_pytorch_b200.inference.generate import sample_next, top_k_filter, top_p_filter

    logits = 3 * torch.randn(4, 90, generator=_gen(71))
    prompt = torch.randint(0, 90, (4, 7), generator=_gen(72))
    for seed, temperature, k, p, penalty in ((6, 1.0, 50, 0.9, 1.0), (7, 0.6, 0, 0.8, 1.0), (8, 1.4, 20, 1.0, 1.3)):
        z = logits / temperature
        if penalty != 1.0:
            z = z.clone()
            for b in range(4):
                at = prompt[b].unique()
                z[b, at] = z[b, at] / penalty
        z = top_p_filter(top_k_filter(z, k), p)
        want = torch.multinomial(torch.softmax(z, -1), 1, generator=_gen(seed))
        got = sample_next(logits, prompt, temperature, k, p, penalty, generator=_gen(seed))
        assert torch.equal(got, want)


def test_seeded_request_has_the_same_numbers_whatever_else_is_served(monkeypatch):
    g = _gen(73)
    prompts = [torch.randint(0, 128, (6,), generator=g) for _ in range(3)]
    numbers = _Uniforms(monkeypatch)
    model = _model()
    alone = []
    for i in range(3):
        numbers.seen.clear()
        _serve([(prompts[i], dict(seed=100 + i, top_k=0))], model)
        alone.append(torch.cat(numbers.seen))
    assert len({tuple(a.tolist()) for a in alone}) == 3
    numbers.seen.clear()
    # beside one another, and beside one that draws from the global generator
    _serve([(prompts[i], dict(seed=100 + i, top_k=0)) for i in range(3)] + [(prompts[0], {})], model)
    for i in range(3):
        assert torch.equal(torch.stack([u[i] for u in numbers.seen]), alone[i])


@gpu
@pytest.mark.parametrize("kind,dtype", [("float32", torch.float32), ("float16", torch.float16), ("fp8", torch.float16),
                                        ("fp8", torch.bfloat16), ("int8", torch.float32), ("bfloat16", torch.float16)])
@pytest.mark.parametrize("window,d", [(1, 64), (7, 96), (64, 128), (90, 40), (200, 64)])
def test_window_below_the_ring(kind, dtype, window, d):
    """Every kind of cache with every kernel that reads it; the visible slots wrap around the ring's end."""
    _cuda()
    g = _gen(97)
    B, Hq, H, S = 6, 4, 2, 96
    (k, ks), (v, vs) = (quantise_rows(torch.randn(B, H, S, d, generator=g), KINDS[kind]) for _ in range(2))
    cache = ops.KVCache(*(t if t is None else t.cuda() for t in (k, v, ks, vs)))
    n = torch.tensor([S + 5, S + 95, 300, 50, 3, 0], device="cuda")
    q = torch.randn(B, Hq, d, generator=g).to(dtype).cuda()
    pk, pv = (torch.randn(5, H, d, generator=g).to(dtype).cuda() for _ in range(2))
    for prefix in ((None, None), (pk, pv)):
        out, lse = ops.decode_attention(q, cache, n, *prefix, window=window, return_lse=True)
        wide = [None if t is None else t.double() for t in prefix]
        ref, rl = decode_attention_reference(q.double(), cache, n, *wide, window=window, scale=d ** -0.5)
        # scores of order one (|q||k| d^-1/2 2^-24 2 d < 2^-14), weights and queries rounded once, values below 5
        tol = 5 * (2.0 ** -13 + (0.0 if dtype == torch.float32 else HALF[dtype])) + HALF[dtype] * ref.abs() + 2.0 ** -24
        assert ((out.double() - ref).abs() <= tol).all()
        live = torch.isfinite(rl)
        assert torch.equal(live, torch.isfinite(lse)) and ((lse.double() - rl)[live].abs() <= 2.0 ** -12).all()


@gpu
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("factor", [1e-37, 1e-31, 1e31, 1e35])
def test_queries_of_any_size_beside_8_bit_keys(kind, factor):
    """bf16 reaches further than the fp16 in which they meet the keys: tiny ones weigh all keys alike, huge ones take one."""
    _cuda()
    g = _gen(101)
    B, H, S, d = 2, 2, 50, 64
    (k, ks), (v, vs) = (quantise_rows(torch.randn(B, H, S, d, generator=g), KINDS[kind]) for _ in range(2))
    cache = ops.KVCache(*(t.cuda() for t in (k, v, ks, vs)))
    n = torch.full((B,), S, device="cuda")
    q = (factor * torch.randn(B, H, d, generator=g)).to(torch.bfloat16).cuda()
    out, lse = ops.decode_attention(q, cache, n, return_lse=True)
    ref, rl = decode_attention_reference(q.double(), cache, n, scale=d ** -0.5)
    assert ((out.double() - ref).abs() <= 5 * 2.0 ** -10 + 2.0 ** -8 * ref.abs()).all()
    assert ((lse.double() - rl).abs() <= 2.0 ** -14 + 2.0 ** -14 * rl.abs()).all()


