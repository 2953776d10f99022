"""Rotary positions, the quantised key/value cache, single-token attention over it and token sampling:
restatements against independent fp64 loops (CPU), kernels against the restatements in fp64 (GPU)."""

from __future__ import annotations

import math

import pytest
import torch

from titans_pytorch_b200 import ops
from titans_pytorch_b200.ops.decode_attention import decode_attention_reference
from titans_pytorch_b200.ops.kv_cache import KINDS, quantise_rows
from titans_pytorch_b200.ops.rope import rotary_embedding_reference
from titans_pytorch_b200.ops.sampling import sample_tokens_reference

gpu = pytest.mark.gpu
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


def _gen(seed=0, device="cpu"):
    return torch.Generator(device=device).manual_seed(seed)


# ------------------------------------------------------------------------- rotary: CPU
def _rope_loop(x, positions, freq, layout, amplitude):
    """One pair at a time, in Python floats."""
    y = x.double().clone()
    n = freq.numel()
    B, T, H, _ = x.shape
    pos = positions if positions.dim() == 2 else positions[None].expand(B, -1)
    for b in range(B):
        for t in range(T):
            for i in range(n):
                a = int(pos[b, t]) * float(freq[i])
                c, s = amplitude * math.cos(a), amplitude * math.sin(a)
                i0, i1 = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + n)
                u, w = x[b, t, :, i0].double(), x[b, t, :, i1].double()
                y[b, t, :, i0], y[b, t, :, i1] = u * c - w * s, u * s + w * c
    return y


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("rotary,scaling", [(8, "none"), (6, "linear"), (2, "ntk"), (8, "yarn")])
def test_rope_restatement_is_the_formula(layout, rotary, scaling):
    freq, amp = ops.rope_frequencies(rotary, scaling=scaling, factor=1.0 if scaling == "none" else 4.0)
    x = torch.randn(2, 3, 2, 8, dtype=torch.float64, generator=_gen())
    pos = torch.tensor([[0, 5, 100000], [7, 2, 999999]])
    y = ops.rotary_embedding(x, pos, freq, layout=layout, amplitude=amp)
    torch.testing.assert_close(y, _rope_loop(x, pos, freq, layout, amp), atol=1e-9, rtol=0)


def test_rope_interleaved_is_the_models_rotation():
    """The same rotation as the models' attention applies (positions small enough for its fp32 angles)."""
    from titans_pytorch_b200.models.attention import RotaryPositionEmbedding

    rope = RotaryPositionEmbedding(16)
    x = torch.randn(2, 9, 3, 16, generator=_gen())
    ref, _ = rope(x.transpose(1, 2), x.transpose(1, 2))
    y = rope.rotate(x, torch.arange(9))
    torch.testing.assert_close(y, ref.transpose(1, 2), atol=1e-5, rtol=0)


def test_rope_frequencies_scalings():
    f0, a0 = ops.rope_frequencies(64)
    assert a0 == 1.0 and f0[0] == 1.0
    lin, _ = ops.rope_frequencies(64, scaling="linear", factor=4.0)
    torch.testing.assert_close(lin, f0 / 4)
    ntk, _ = ops.rope_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0
    torch.testing.assert_close(ntk[-1], f0[-1] / 4)
    yarn, amp = ops.rope_frequencies(64, scaling="yarn", factor=4.0, original_max_position=4096)
    assert amp == pytest.approx(0.1 * math.log(4) + 1)
    turns = 4096 * f0 / (2 * math.pi)
    torch.testing.assert_close(yarn[turns >= 32], f0[turns >= 32])
    torch.testing.assert_close(yarn[turns <= 1], f0[turns <= 1] / 4)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="x"),
                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, fast_turns=1.0)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(**bad)


def test_rope_gradient_cpu():
    freq, amp = ops.rope_frequencies(6, scaling="yarn", factor=8.0)
    x = torch.randn(1, 3, 2, 8, dtype=torch.float64, generator=_gen(), requires_grad=True)
    pos = torch.tensor([3, 1, 70])
    for layout in ("interleaved", "half"):
        assert torch.autograd.gradcheck(
            lambda t: ops.rotary_embedding(t, pos, freq, layout=layout, amplitude=amp), (x,))


def test_rope_refusals():
    f, _ = ops.rope_frequencies(8)
    x, pos = torch.zeros(2, 3, 1, 8), torch.arange(3)
    with pytest.raises(ValueError):
        ops.rotary_embedding(x, pos, f, layout="other")
    with pytest.raises(ValueError):
        ops.rotary_embedding(x[0], pos, f)
    with pytest.raises(TypeError):
        ops.rotary_embedding(x, pos.float(), f)
    with pytest.raises(ValueError):
        ops.rotary_embedding(x, torch.arange(4), f)
    with pytest.raises(ValueError):
        ops.rotary_embedding(x[..., :6], pos, f)


# ------------------------------------------------------------------------- rotary: GPU
def _rope_bound(x, y, dtype, amplitude):
    """|error| of one output element: the angle is reduced in fp64 and rounded to fp32 (|r| <= pi: 2^-23), cos and sin
    are off by at most 2 ulp more (2^-22 with the amplitude's rounding), and two products and a sum round three
    times (3 * 2^-24); each times |a| + |b| <= 2 max|x|.  Then one rounding to the type."""
    top = 2 * amplitude * x.abs().amax(dim=-1, keepdim=True).double()
    return 2.0 ** -20 * top + HALF[dtype] * 1.01 * y.abs() + (2.0 ** -24 if dtype == torch.float16 else 0.0)


ROPE_CASES = [
    # batch, tokens, heads, dim, rotary, layout, start
    (1, 1, 1, 8, 8, "interleaved", 0),
    (2, 33, 3, 64, 64, "interleaved", 17),
    (3, 5, 24, 64, 64, "half", 1000003),
    (1, 257, 2, 96, 48, "half", 5),
    (2, 7, 5, 96, 20, "interleaved", 123456),   # the rotated part ends inside a vector
    (2, 7, 5, 80, 20, "half", 9),               # not a multiple of the vector: one element at a time
    (1, 3, 2, 20, 6, "half", 2),
    (1, 3, 2, 7, 4, "interleaved", 2),
    (1, 2, 1, 128, 2, "half", 50),
    (4, 1, 40, 128, 128, "half", 40000),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", ROPE_CASES)
def test_rope_kernel(case, dtype):
    _cuda()
    B, T, H, d, rotary, layout, start = case
    freq, amp = ops.rope_frequencies(rotary, scaling="yarn", factor=4.0, device="cuda")
    fused = torch.randn(B, T, 2 * H + 1, d, generator=_gen(1), dtype=torch.float32).to(dtype).cuda()
    for x in (fused[:, :, :H], fused[:, :, 1:H + 1].contiguous(), fused.transpose(1, 2)[:, :H].transpose(1, 2)):
        x = x.detach().requires_grad_(True)
        pos = start + torch.arange(T, device="cuda")
        pos = pos[None] + 11 * torch.arange(B, device="cuda")[:, None] if B > 1 else pos
        y = ops.rotary_embedding(x, pos, freq, layout=layout, amplitude=amp)
        ref = rotary_embedding_reference(x.detach().double(), pos, freq, layout, amp)
        assert y.dtype == dtype and y.is_contiguous()
        assert ((y.double() - ref).abs() <= _rope_bound(x.detach(), ref, dtype, amp)).all()
        dy = torch.randn(B, T, H, d, generator=_gen(2)).to(dtype).cuda()
        (dx,) = torch.autograd.grad(y, x, dy)
        xd = x.detach().double().requires_grad_(True)
        (rx,) = torch.autograd.grad(rotary_embedding_reference(xd, pos, freq, layout, amp), xd, dy.double())
        assert ((dx.double() - rx).abs() <= _rope_bound(dy, rx, dtype, amp)).all()


@gpu
def test_rope_kernel_edges():
    _cuda()
    freq, _ = ops.rope_frequencies(64, device="cuda")
    x = torch.randn(2, 4, 3, 64, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(4, device="cuda")
    assert ops.rotary_embedding(x[:, :0], pos[:0], freq).shape == (2, 0, 3, 64)
    assert ops.rotary_embedding(x[:, :, :0], pos, freq).shape == (2, 4, 0, 64)
    # no frequency at all: a copy; a broadcast input and a broadcast gradient
    assert torch.equal(ops.rotary_embedding(x, pos, freq[:0]), x)
    wide = x[:, :, :1].expand(-1, -1, 5, -1)
    assert torch.equal(ops.rotary_embedding(wide, pos, freq), ops.rotary_embedding(wide.contiguous(), pos, freq))
    leaf = torch.randn(1, 4, 1, 64, device="cuda", requires_grad=True)
    ops.rotary_embedding(leaf.expand(2, 4, 3, 64), pos, freq).sum().backward()
    one = torch.ones(1, 4, 1, 64, device="cuda", dtype=torch.float64)
    want = 6 * rotary_embedding_reference(one, -pos, freq)
    assert (leaf.grad.double() - want).abs().max() <= 6 * 2 * 2.0 ** -20
    # infinities and NaN stay in their pair
    y = x.clone()
    y[0, 0, 0, 5] = float("nan")
    r = ops.rotary_embedding(y, pos, freq)
    assert int(torch.isnan(r).sum()) == 2 and torch.isnan(r[0, 0, 0, 4:6]).all()
    # the rotation by p and then by -p is the identity
    far = pos + 123456789
    back = ops.rotary_embedding(ops.rotary_embedding(x.float(), far, freq), -far, freq)
    assert (back - x.float()).abs().max() <= 2 * 2.0 ** -20 * 2 * float(x.abs().max())
    with pytest.raises(RuntimeError):
        ops.rotary_embedding(x.double(), pos, freq)
    with pytest.raises(RuntimeError):
        ops.rotary_embedding(x, pos.cpu(), freq)


@gpu
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_kernel_widest_heads(layout):
    """Enough tokens of the widest head that a block's tables reach the limit of its shared memory."""
    _cuda()
    freq, _ = ops.rope_frequencies(1024, device="cuda")
    x = torch.randn(1, 12000, 1, 1024, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(12000, device="cuda")
    y = ops.rotary_embedding(x, pos, freq, layout=layout)
    ref = rotary_embedding_reference(x.double(), pos, freq, layout)
    assert ((y.double() - ref).abs() <= _rope_bound(x, ref, torch.bfloat16, 1.0)).all()
    with pytest.raises(RuntimeError):
        ops.rotary_embedding(torch.zeros(1, 1, 1, 1032, device="cuda"), pos[:1], freq)


@gpu
def test_rope_double_backward_and_graph():
    _cuda()
    freq, _ = ops.rope_frequencies(32, device="cuda")
    x = torch.randn(1, 3, 2, 32, device="cuda", requires_grad=True)
    pos = torch.arange(3, device="cuda")
    y = ops.rotary_embedding(x, pos, freq)
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y, requires_grad=True), create_graph=True)
    assert g.requires_grad
    s = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    ops.rotary_embedding(s, pos, freq)
    with torch.cuda.graph(graph):
        out = ops.rotary_embedding(s, pos, freq)
    s.copy_(x.detach())
    pos.add_(5)
    graph.replay()
    assert torch.equal(out, ops.rotary_embedding(x.detach(), pos, freq))


# ------------------------------------------------------------------------- cache: CPU
def _cache_loop(S, k, v, start, counts, kind):
    """What the cache holds, token by token: {(b, slot): (k row, v row)}."""
    held = {}
    for b in range(k.shape[0]):
        for t in range(int(counts[b])):
            p = int(start[b]) + t
            if p >= 0:
                held[b, p % S] = (k[b, t], v[b, t])
    return held


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("T,S", [(1, 8), (5, 8), (8, 8), (19, 8)])
def test_cache_restatement(kind, T, S):
    B, H, d = 3, 2, 8
    g = _gen(3)
    k, v = torch.randn(B, T, H, d, generator=g), torch.randn(B, T, H, d, generator=g)
    start, counts = torch.tensor([0, 6, 13]), torch.tensor([T, max(T - 2, 0), T])
    cache = ops.KVCache.allocate(B, H, S, d, kind)
    cache.k.copy_(torch.full((), 3.0))
    before = cache.k.clone()
    ops.kv_cache_write(cache, k, v, start, counts=counts)
    held = _cache_loop(S, k, v, start, counts, kind)
    step = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "int8": 0.5 / 127, "fp8": 2.0 ** -4}[kind]
    for b in range(B):
        for s in range(S):
            if (b, s) not in held:
                assert torch.equal(cache.k[b, :, s].float(), before[b, :, s].float())
                continue
            for data, scale, row in ((cache.k, cache.k_scale, held[b, s][0]), (cache.v, cache.v_scale, held[b, s][1])):
                x = data[b, :, s].float()
                x = x if scale is None else x * scale[b, :, s, None]
                # int8: half a step of amax / 127; the others half a step of the value (fp8: of the smallest normal at least)
                top = row.abs().amax(-1, keepdim=True)
                tol = step * (top if kind == "int8" else torch.maximum(row.abs(), top * 2.0 ** -14)) * 1.001
                assert ((x - row).abs() <= tol).all()
    lengths = start + counts
    rk, rv = ops.kv_cache_read(cache, lengths, dtype=torch.float32)
    for b in range(B):
        n = min(int(lengths[b]), S)
        for i in range(S):
            p = int(lengths[b]) - n + i
            if i >= n:
                assert (rk[b, :, i] == 0).all() and (rv[b, :, i] == 0).all()
            elif (b, p % S) in held:
                x = cache.v[b, :, p % S].float()
                x = x if cache.v_scale is None else x * cache.v_scale[b, :, p % S, None]
                assert torch.equal(rv[b, :, i], x)
    short, _ = ops.kv_cache_read(cache, lengths, n=3, dtype=torch.float32)
    for b in range(B):
        n = min(int(lengths[b]), S)
        m = min(n, 3)
        assert torch.equal(short[b, :, :m], rk[b, :, n - m:n]) and (short[b, :, m:] == 0).all()


def test_quantise_special_rows():
    x = torch.tensor([[0.0] * 4, [1e-40, 0, 0, 0], [float("inf"), 1, 0, 0], [float("nan"), 1, 0, 0], [3e38, -3e38, 1, 0]])
    for t in (torch.int8, torch.float8_e4m3fn):
        q, s = quantise_rows(x, t)
        y = q.float() * s[:, None]
        assert (y[0] == 0).all() and (y[1] == 0).all() and s[0] == 1
        assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
        assert y[4, 0] > 2.9e38 and y[4, 1] < -2.9e38 and torch.isfinite(y[4]).all()


def test_cache_refusals():
    c = ops.KVCache.allocate(2, 3, 4, 8, "int8")
    k = torch.zeros(2, 1, 3, 8)
    start = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError):
        ops.KVCache.allocate(1, 1, 1, 8, "int4")
    with pytest.raises(ValueError):
        ops.KVCache(c.k, c.v)
    with pytest.raises(ValueError):
        ops.KVCache(c.k.float(), c.v.float(), c.k_scale, c.v_scale)
    with pytest.raises(TypeError):
        ops.KVCache(c.k.long(), c.v.long())
    with pytest.raises(ValueError):
        ops.KVCache(c.k, c.v[:, :, :2], c.k_scale, c.v_scale)
    for bad in (dict(k=k[:1]), dict(v=k[..., :4]), dict(start=start.int()), dict(start=start[:1]),
                dict(counts=start[:1]), dict(q=k[:, :, :, :4]), dict(q=k.half()), dict(layout="x"),
                dict(inv_freq=torch.ones(5))):
        args = dict(k=k, v=k, start=start, counts=None, q=None, layout="half", inv_freq=None, **{})
        args.update(bad)
        with pytest.raises(ValueError):
            ops.kv_cache_write(c, args.pop("k"), args.pop("v"), args.pop("start"), **args)
    with pytest.raises(ValueError):
        ops.kv_cache_read(c, start, n=5)
    with pytest.raises(ValueError):
        ops.kv_cache_read(c, start.float())


def test_extension_errors_with_numbers_are_exceptions():
    """A check of the compiled library whose message formats a number raises (it needs the process's one libstdc++)."""
    from titans_pytorch_b200.ops._ext import available, ext

    if not available():
        pytest.skip("extension not built")
    c = torch.zeros(1, 1, 4, 12, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="multiple of 8 from 8 to 256, not 12"):
        ext().kv_cache_read(c, c, None, None, torch.zeros(1, dtype=torch.int64), 4, torch.bfloat16)


# ------------------------------------------------------------------------- cache: GPU
CACHE_CASES = [
    # batch, tokens, heads, dim, slots, rotary, layout
    (1, 1, 1, 8, 1, 8, "interleaved"),
    (3, 1, 12, 64, 16, 64, "interleaved"),
    (2, 40, 3, 96, 16, 96, "half"),        # more new tokens than slots
    (2, 9, 5, 128, 33, 32, "half"),
    (2, 9, 5, 72, 33, 20, "half"),         # partners that are no whole vector apart
    (2, 9, 2, 256, 40, 0, "interleaved"),
    (5, 17, 2, 40, 100, 30, "interleaved"),
]


def _fresh_cache(B, H, S, d, kind, seed=5):
    g = _gen(seed)
    x = [torch.randn(B, H, S, d, generator=g) for _ in range(2)]
    parts = [quantise_rows(t, KINDS[kind]) for t in x]
    return ops.KVCache(parts[0][0].cuda(), parts[1][0].cuda(),
                       *(None if p[1] is None else p[1].cuda() for p in parts))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("case", CACHE_CASES)
def test_cache_kernel(case, kind, dtype):
    _cuda()
    B, T, H, d, S, rotary, layout = case
    g = _gen(7)
    Hq = 2 * H
    fused = torch.randn(B, T, Hq + 2 * H, d, generator=g).to(dtype).cuda()
    q, k, v = fused[:, :, :Hq], fused[:, :, Hq:Hq + H], fused[:, :, Hq + H:]
    start = torch.tensor([3 * S + 7 * b for b in range(B)], device="cuda")
    start[0] = 0
    counts = torch.tensor([max(T - 3 * b, 0) for b in range(B)], device="cuda")
    freq = ops.rope_frequencies(rotary, device="cuda")[0] if rotary else None
    cache, want = _fresh_cache(B, H, S, d, kind), _fresh_cache(B, H, S, d, kind)
    got_q = ops.kv_cache_write(cache, k, v, start, counts=counts, q=q, inv_freq=freq, layout=layout, rope_offset=4)
    ops.kv_cache_write(want, k, v, start, counts=counts, q=q, inv_freq=freq, layout=layout, rope_offset=4,
                       use_kernels=False)
    pos = start[:, None] + torch.arange(T, device="cuda") + 4
    if freq is None:
        assert torch.equal(got_q, q)
    else:
        ref = rotary_embedding_reference(q.double(), pos, freq, layout)
        assert ((got_q.double() - ref).abs() <= _rope_bound(q, ref, dtype, 1.0)).all()
    # values are copied or quantised from equal fp32 numbers: bit for bit
    assert torch.equal(cache.v.view(torch.uint8) if cache.v.element_size() == 1 else cache.v,
                       want.v.view(torch.uint8) if want.v.element_size() == 1 else want.v)
    if kind in ("int8", "fp8"):
        assert torch.equal(cache.v_scale, want.v_scale)
        # the rotated keys differ by fp32 rounding: the scale by that much, a stored value by one step at a border
        amax = 2.0 ** -20 * 2 * float(k.abs().max()) / (127.0 if kind == "int8" else 448.0)
        assert ((cache.k_scale - want.k_scale).abs() <= amax + 2.0 ** -23 * want.k_scale).all()
        a, b = cache.k.float() * cache.k_scale[..., None], want.k.float() * want.k_scale[..., None]
        step = want.k_scale[..., None] * (1.01 if kind == "int8" else 32.0)
        near = (a - b).abs() <= (step if kind == "int8" else torch.maximum(step * 2.0 ** -10, 0.13 * b.abs()))
        assert near.all()
        assert float(((a - b).abs() > 1e-5 * want.k_scale[..., None] * 448).float().mean()) < 1e-2
    else:
        tol = 2.0 ** -20 * 2 * k.abs().amax().double() + 2 * HALF[KINDS[kind]] * want.k.double().abs() + 2.0 ** -24
        assert ((cache.k.double() - want.k.double()).abs() <= tol).all()
    lengths = start + counts
    for n in (None, max(1, S // 2), 0):
        for t in (torch.bfloat16, torch.float32):
            rk, rv = ops.kv_cache_read(cache, lengths, n, t)
            wk, wv = ops.kv_cache_read(cache, lengths, n, t, use_kernels=False)
            assert torch.equal(rk, wk) and torch.equal(rv, wv)


@gpu
def test_cache_kernel_edges():
    _cuda()
    B, H, S, d = 2, 3, 8, 64
    start = torch.zeros(B, dtype=torch.int64, device="cuda")
    k = torch.randn(B, 4, H, d, device="cuda", dtype=torch.bfloat16)
    # no new token, no row of the cache touched
    c = _fresh_cache(B, H, S, d, "int8")
    before = c.k.clone()
    ops.kv_cache_write(c, k[:, :0], k[:, :0], start)
    ops.kv_cache_write(c, k, k, start, counts=start)
    ops.kv_cache_write(c, k, k, start - 100)
    assert torch.equal(c.k, before)
    none = ops.KVCache.allocate(B, 0, S, d, "int8", device="cuda")
    assert ops.kv_cache_write(none, k[:, :, :0], k[:, :, :0], start) is None
    assert ops.kv_cache_read(none, start)[0].shape == (B, 0, S, d)
    # rows that are not aligned, and a layer of a stack whose neighbours stay as they were
    stack = [torch.zeros(3, B, H, S, d, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.ones(3, B, H, S, device="cuda") for _ in range(2)]
    layer = ops.KVCache(stack[0][1], stack[1][1], scales[0][1], scales[1][1])
    odd = torch.zeros(B, 4, H, d + 1, device="cuda", dtype=torch.bfloat16)
    odd[..., 1:] = k
    ops.kv_cache_write(layer, odd[..., 1:], odd[..., 1:], start)
    plain = ops.KVCache.allocate(B, H, S, d, "int8", device="cuda")
    ops.kv_cache_write(plain, k, k, start)
    assert torch.equal(layer.k, plain.k) and torch.equal(layer.v_scale, plain.v_scale)
    assert (stack[0][0] == 0).all() and (stack[0][2] == 0).all()
    # slots further apart than a row, heads in front of the batch
    base = torch.zeros(H, B, S, 2 * d, dtype=torch.bfloat16, device="cuda")
    view = base[..., :d].transpose(0, 1)
    c2 = ops.KVCache(view, torch.zeros(B, H, S, d, dtype=torch.bfloat16, device="cuda"))
    ops.kv_cache_write(c2, k, k, start)
    assert torch.equal(view[:, :, :4], k.transpose(1, 2)) and (base[..., d:] == 0).all()
    # special rows
    x = torch.zeros(1, 4, 1, d, device="cuda")
    x[0, 0, 0, 0], x[0, 1, 0, 3], x[0, 2, 0, 1], x[0, 3, 0, :2] = 1e-40, float("inf"), float("nan"), torch.tensor([3e38, -3e38])
    for kind in ("int8", "fp8"):
        c = ops.KVCache.allocate(1, 1, 4, d, kind, device="cuda")
        ops.kv_cache_write(c, x, x, start[:1])
        r = ops.kv_cache_read(c, start[:1] + 4, dtype=torch.float32)[0][0, 0]
        assert (r[0] == 0).all() and torch.isnan(r[1:3]).all() and r[3, 0] > 2.9e38 and r[3, 1] < -2.9e38
    with pytest.raises(RuntimeError):  # head_dim that is no multiple of 8
        ops.kv_cache_read(ops.KVCache.allocate(1, 1, 4, 12, device="cuda"), start[:1])
    with pytest.raises(RuntimeError):
        ops.kv_cache_write(plain, k.cpu(), k.cpu(), start)
    with pytest.raises(RuntimeError):
        ops.kv_cache_write(plain, k, k, start.cpu())


# ------------------------------------------------------------------------- attention: CPU
def _attend_loop(q, cache, lengths, pk, pv, window, scale):
    B, Hq, d = q.shape
    Hkv, S = cache.k.shape[1:3]
    out = torch.zeros(B, Hq, d, dtype=torch.float64)
    lse = torch.full((B, Hq), float("-inf"), dtype=torch.float64)
    for b in range(B):
        n = min(int(lengths[b]), S, window)
        slots = [p % S for p in range(int(lengths[b]) - n, int(lengths[b]))]
        for h in range(Hq):
            hk = h // (Hq // Hkv)
            ks, vs = [], []
            for p in range(0 if pk is None else pk.shape[0]):
                ks.append(pk[p, hk].double())
                vs.append(pv[p, hk].double())
            for s in slots:
                ks.append(cache.k[b, hk, s].double() * (1 if cache.k_scale is None else float(cache.k_scale[b, hk, s])))
                vs.append(cache.v[b, hk, s].double() * (1 if cache.v_scale is None else float(cache.v_scale[b, hk, s])))
            if ks:
                s = torch.stack(ks) @ q[b, h].double() * scale
                out[b, h] = torch.softmax(s, 0) @ torch.stack(vs)
                lse[b, h] = torch.logsumexp(s, 0)
    return out, lse


@pytest.mark.parametrize("kind", ["float32", "int8"])
@pytest.mark.parametrize("P,window", [(0, None), (3, None), (2, 4), (0, 1)])
def test_attention_restatement(kind, P, window):
    B, Hq, Hkv, S, d = 4, 4, 2, 8, 8
    g = _gen(11)
    cache = ops.KVCache(*(t for t in [quantise_rows(torch.randn(B, Hkv, S, d, generator=g), KINDS[kind])[0] for _ in range(2)]),
                        *((torch.rand(B, Hkv, S, generator=g) * 0.02 for _ in range(2)) if kind == "int8" else ()))
    q = torch.randn(B, Hq, d, generator=g, dtype=torch.float64)
    lengths = torch.tensor([0, 1, 8, 21])
    pk, pv = (torch.randn(P, Hkv, d, generator=g, dtype=torch.float64) for _ in range(2)) if P else (None, None)
    out, lse = ops.decode_attention(q, cache, lengths, pk, pv, window=window, return_lse=True)
    ref, rl = _attend_loop(q, cache, lengths, pk, pv, window or 1 << 30, d ** -0.5)
    torch.testing.assert_close(out, ref, atol=1e-9, rtol=0)
    torch.testing.assert_close(lse, rl, atol=1e-9, rtol=0)


def test_attention_refusals():
    c = ops.KVCache.allocate(2, 2, 4, 8, "float32")
    q, n = torch.zeros(2, 4, 8), torch.ones(2, dtype=torch.int64)
    p = torch.zeros(3, 2, 8)
    for args, kw in (((q[0], c, n), {}), ((q[:1], c, n), {}), ((q[:, :3], c, n), {}), ((q, c, n.int()), {}), ((q, c, n[:1]), {}),
                     ((q, c, n, p), {}), ((q, c, n, p, p[:2]), {}), ((q, c, n, p.half(), p.half()), {}),
                     ((q, c, n), dict(window=0))):
        with pytest.raises(ValueError):
            ops.decode_attention(*args, **kw)


# ------------------------------------------------------------------------- attention: GPU
def _attention_bound(q, cache, lengths, pk, pv, window, scale, ref):
    """|error| of an output element.  Scores: d fp32 products and sums of |q||k| (2^-24 each, twice: products may be
    split between units) and the exponential's 2^-22, relative to the weight; weights rounded to the type of the
    values' product (half a step each) times sum p|v| / sum p; the result rounded once.  The 8-bit kinds use fp16
    weights whatever the queries' type, and fp16 queries (relative to the row's largest element: 2^-24 of it)."""
    d = q.shape[-1]
    mag = ops.KVCache(cache.k, cache.v.float().abs().to(cache.v.dtype), cache.k_scale,
                      None if cache.v_scale is None else cache.v_scale)
    a, _ = decode_attention_reference(q.double(), mag, lengths, pk, None if pv is None else pv.abs(), window, scale)
    kmax = (cache.k.float() if cache.k_scale is None else cache.k.float() * cache.k_scale[..., None])
    kmax = torch.nan_to_num(kmax, 0.0, 0.0, 0.0).abs().amax()
    if pk is not None and pk.numel():
        kmax = torch.maximum(kmax, pk.float().abs().amax())
    scores = 2 * d * 2.0 ** -24 * float(q.double().abs().sum(-1).max() * kmax) * scale + 2.0 ** -20
    # (a prefix beside an 8-bit cache is in the queries' type)
    weight = 0.0 if q.dtype == torch.float32 else (HALF[torch.float16] if cache.k_scale is not None and pk is None else HALF[q.dtype])
    return (2 * scores + weight) * a + HALF[q.dtype] * 1.01 * ref.abs() + 2.0 ** -24, scores


def _attention_case(B, Hq, Hkv, d, S, lengths, P, kind, dtype, window=None, stale=True, seed=13):
    g = _gen(seed)
    cache = _fresh_cache(B, Hkv, S, d, kind, seed)
    q = (1.5 * torch.randn(B, Hq, d, generator=g)).to(dtype).cuda()
    n = torch.tensor([lengths[b % len(lengths)] for b in range(B)])
    if stale:  # slots that are not visible hold anything
        for b in range(B):
            if int(n[b]) < S:
                for data, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                    if scale is None:
                        data[b, :, int(n[b]):] = float("nan")
                    else:
                        scale[b, :, int(n[b]):] = float("inf")
    pk = pv = None
    if P:
        pk, pv = (torch.randn(P, Hkv, d, generator=g).to(dtype).cuda() for _ in range(2))
    return q, cache, n.cuda(), pk, pv


def _check_attention(q, cache, n, pk, pv, window=None):
    scale = q.shape[-1] ** -0.5
    out, lse = ops.decode_attention(q, cache, n, pk, pv, window=window, return_lse=True)
    w = (1 << 30) if window is None else window
    wide = lambda t: None if t is None else t.double()  # noqa: E731
    clean = ops.KVCache(*(torch.nan_to_num(t.float(), 0.0).to(t.dtype) for t in (cache.k, cache.v)),
                        *((torch.nan_to_num(t, 1.0, 1.0) for t in (cache.k_scale, cache.v_scale)) if cache.k_scale is not None else ()))
    ref, rl = decode_attention_reference(q.double(), clean, n, wide(pk), wide(pv), w, scale)
    bound, scores = _attention_bound(q, clean, n, wide(pk), wide(pv), w, scale, ref)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    bad = (out.double() - ref).abs() > bound
    assert not bad.any() and torch.isfinite(out).all(), (int(bad.sum()), float((out.double() - ref).abs().max()))
    assert torch.equal(lse == float("-inf"), rl == float("-inf"))
    live = torch.isfinite(rl)
    # lse: the scores' error, the relative error of a sum of positive fp32 numbers in pieces, one rounding
    assert ((lse.double() - rl)[live].abs() <= scores + 2.0 ** -18 + 2.0 ** -22 * rl[live].abs()).all()
    return out


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [8, 64, 96, 128, 200])
def test_attention_kernel(kind, dtype, d):
    _cuda()
    _check_attention(*_attention_case(5, 4, 4, d, 70, [0, 1, 33, 70, 501], 0, kind, dtype))
    _check_attention(*_attention_case(5, 6, 2, d, 129, [0, 1, 64, 129, 300], 5, kind, dtype))


@gpu
@pytest.mark.parametrize("dtype,kind", [(torch.bfloat16, "bfloat16"), (torch.bfloat16, "int8"), (torch.bfloat16, "fp8"),
                                        (torch.float16, "float16"), (torch.float16, "fp8"), (torch.float32, "float32"),
                                        (torch.bfloat16, "float32")])
@pytest.mark.parametrize("B,Hq,Hkv,d,S,P", [(1, 1, 1, 64, 1, 0), (1, 12, 12, 64, 512, 4), (3, 16, 1, 64, 2100, 1),
                                            (2, 40, 2, 128, 1000, 33), (2, 8, 8, 96, 5000, 130), (33, 3, 1, 64, 65, 257),
                                            (70, 4, 2, 64, 40, 1000), (9, 64, 2, 128, 300, 129)])
def test_attention_kernel_shapes(B, Hq, Hkv, d, S, P, dtype, kind):
    _cuda()
    _check_attention(*_attention_case(B, Hq, Hkv, d, S, [S, 1, S // 2 + 1, 0, 3 * S + 5], P, kind, dtype))


@gpu
@pytest.mark.parametrize("kind", ["bfloat16", "int8"])
@pytest.mark.parametrize("window", [1, 7, 64, 200])
def test_attention_kernel_window(kind, window):
    """A window below the ring: the visible slots wrap around its end."""
    _cuda()
    q, cache, n, pk, pv = _attention_case(6, 4, 2, 64, 96, [96 + 5, 96 + 95, 300, 50, 3, 0], 2, kind, torch.bfloat16)
    _check_attention(q, cache, n, pk, pv, window)
    _check_attention(q, cache, n, None, None, window)


@gpu
@pytest.mark.parametrize("kind,dtype", [("bfloat16", torch.bfloat16), ("int8", torch.bfloat16), ("float32", torch.float32)])
def test_attention_kernel_edges(kind, dtype):
    _cuda()
    q, cache, n, pk, pv = _attention_case(4, 4, 2, 64, 300, [300, 17, 0, 120], 20, kind, dtype)
    want = ops.decode_attention(q, cache, n, pk, pv)
    # repeated calls agree bit for bit; strided queries, lengths and prefix; another stream
    assert torch.equal(ops.decode_attention(q, cache, n, pk, pv), want)
    fat = torch.stack([q, q], dim=2)[:, :, 1]
    two = torch.stack([n, n + 1], dim=1)[:, 0]
    pk2, pv2 = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (pk, pv))
    assert torch.equal(ops.decode_attention(fat, cache, two, pk2, pv2), want)
    shifted = torch.zeros(q.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(q).copy_(q)
    off = torch.zeros(pk.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(pk).copy_(pk)
    assert torch.equal(ops.decode_attention(shifted, cache, n, off, pv), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.decode_attention(q, cache, n, pk, pv)
    side.synchronize()
    assert torch.equal(other, want)
    # rows without a key
    out, lse = ops.decode_attention(q, cache, n, return_lse=True)
    assert (out[2] == 0).all() and (lse[2] == float("-inf")).all() and torch.isfinite(out).all()
    # huge scores: the largest key wins; a NaN query spoils its own row only
    big = q * 1e4
    assert torch.isfinite(ops.decode_attention(big, cache, n, pk, pv)).all()
    q2 = q.clone()
    q2[1, 2, 5] = float("nan")
    got = ops.decode_attention(q2, cache, n, pk, pv)
    assert torch.isnan(got[1, 2]).all()
    got[1, 2] = want[1, 2]
    assert torch.equal(got, want)
    # an empty batch, an empty prefix
    assert ops.decode_attention(q[:0], ops.KVCache(*(None if t is None else t[:0] for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))), n[:0]).shape == (0, 4, 64)
    assert torch.equal(ops.decode_attention(q, cache, n, pk[:0], pv[:0]), ops.decode_attention(q, cache, n))
    with pytest.raises(RuntimeError):
        ops.decode_attention(q, cache, n.cpu())
    # two captured graphs, replayed with new lengths and queries, one on each of two streams
    graphs = []
    for _ in range(2):
        gq, gn = q.clone(), n.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            go = ops.decode_attention(gq, cache, gn, pk, pv)
        graphs.append((graph, gq, gn, go))
    fewer = (n - 5).clamp(min=0)
    graphs[0][1].copy_(q.flip(0))
    graphs[1][2].copy_(fewer)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][3], ops.decode_attention(q.flip(0), cache, n, pk, pv))
    assert torch.equal(graphs[1][3], ops.decode_attention(q, cache, fewer, pk, pv))


@gpu
def test_attention_kernel_large_offsets():
    """Slots beyond 2^31 bytes from the start of the cache."""
    _cuda()
    B, H, S, d = 3, 4, 700_000, 128
    cache = ops.KVCache(*(torch.zeros(B, H, S, d, dtype=torch.int8, device="cuda") for _ in range(2)),
                        *(torch.ones(B, H, S, device="cuda") for _ in range(2)))
    start = torch.full((B,), S - 2, device="cuda")
    new = torch.randn(B, 2, H, d, device="cuda", dtype=torch.bfloat16)
    ops.kv_cache_write(cache, new, new, start)
    k, _ = ops.kv_cache_read(cache, start + 2, n=2)
    assert ((k.float() - new.transpose(1, 2).float()).abs() <= new.float().abs().amax(-1).transpose(1, 2)[..., None] * (0.51 / 127 + 2.0 ** -8)).all()
    q = torch.randn(B, H, d, device="cuda", dtype=torch.bfloat16)
    out = ops.decode_attention(q, cache, start + 2, window=2)
    small = ops.KVCache(*(t[:, :, -2:].contiguous() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    want = ops.decode_attention(q, small, torch.full((B,), 2, device="cuda"))
    assert torch.equal(out, want)


# ------------------------------------------------------------------------- sampling: CPU
def _sample_loop(z, u, k, p, m):
    """One row, plain Python: the definition."""
    z = [(-math.inf if math.isnan(x) else x) for x in z]
    top = max(z)
    order = sorted(range(len(z)), key=lambda i: (-z[i], i))
    w = [math.exp(x - top) for x in z]
    if 0 < k < len(z):
        limit = z[order[k - 1]]
        w = [a if x >= limit else 0.0 for a, x in zip(w, z)]
    if p < 1:
        total, ahead, keep = math.fsum(w), 0.0, set()
        for i in order:
            if ahead <= p * total:
                keep.add(i)
            ahead += w[i]
        w = [a if i in keep else 0.0 for i, a in enumerate(w)]
    w = [a if a >= m else 0.0 for a in w]
    total, run, last = math.fsum(w), 0.0, None
    for i, a in enumerate(w):
        run += a
        if a > 0:
            last = i
            if run > u * total:
                return i, math.log(a / total)
    return last, math.log(w[last] / total)


SAMPLE_SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.8, 0.0), (1.0, 0, 1.0, 0.2), (0.9, 20, 0.9, 0.05),
                   (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (2.0, 1000, 0.5, 1.0)]


@pytest.mark.parametrize("temperature,k,p,m", SAMPLE_SETTINGS)
def test_sampling_restatement(temperature, k, p, m):
    logits = 2 * torch.randn(6, 50, generator=_gen(17))
    logits[1, 7:20] = logits[1, 7]           # ties
    logits[2, ::3] = float("-inf")
    logits[3, 4] = float("nan")
    u = torch.tensor([0.0, 0.2, 0.5, 0.9, 0.999999, 0.3])
    tok, lp = ops.sample_tokens(logits, u, temperature=temperature, top_k=k, top_p=p, min_p=m, return_logprob=True)
    for b in range(6):
        z = (logits[b] / torch.tensor(temperature)).tolist()
        f32 = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
        want, wl = _sample_loop(z, float(u[b]), k, f32(p), f32(m))
        assert int(tok[b]) == want and abs(float(lp[b]) - wl) < 1e-6


def test_sampling_special_rows_cpu():
    _special_rows("cpu")


def _special_rows(device):
    inf = float("inf")
    logits = torch.tensor([[-inf, -inf, -inf, -inf], [1.0, inf, 2.0, inf], [float("nan")] * 4, [-inf, 3.0, -inf, -inf],
                           [2.0, 2.0, 2.0, 2.0], [0.0, -0.0, 0.0, -0.0]], device=device)
    u = torch.tensor([0.5, 0.5, 0.5, 0.5, 0.75, 0.3], device=device)
    tok, lp = ops.sample_tokens(logits, u, return_logprob=True)
    assert tok.tolist() == [0, 3, 0, 1, 3, 1]
    assert torch.isnan(lp[[0, 2]]).all() and float(lp[3]) == 0.0
    assert abs(float(lp[1]) + math.log(2)) < 1e-6 and abs(float(lp[4]) + math.log(4)) < 1e-6
    # ties: top-k keeps all, top-p the lowest indices, greedy the lowest
    assert ops.sample_tokens(logits, u, top_k=2).tolist()[4] == 3
    assert ops.sample_tokens(logits, torch.full_like(u, 0.99), top_p=0.5).tolist()[4] == 2  # weight in front: 0, 1, 2 <= 0.5 * 4
    assert ops.sample_tokens(logits, u, temperature=0.0).tolist() == [0, 1, 0, 1, 0, 0]
    # the penalty divides, whatever the sign; ids outside the vocabulary are padding
    gen = torch.tensor([[1, -1, 99]] * 6, device=device)
    assert ops.sample_tokens(logits[3:4], u[:1], generated=gen[:1], repetition_penalty=5.0).tolist() == [1]
    two = torch.tensor([[1.0, 1.1]], device=device)
    assert ops.sample_tokens(two, u[:1], temperature=0.0, generated=gen[:1], repetition_penalty=2.0).tolist() == [0]


def test_sampling_refusals():
    x, u = torch.zeros(2, 5), torch.zeros(2)
    for args, kw in (((x[0], u), {}), ((x[:, :0], u), {}), ((x, u[:1]), {}), ((x, u.double()), {}), ((x, u), dict(top_p=1.5)),
                     ((x, u), dict(min_p=-0.1)), ((x, u), dict(repetition_penalty=0.0)), ((x, u), dict(temperature=torch.ones(3))),
                     ((x, u), dict(generated=torch.zeros(2, 2))), ((x, u), dict(generated=torch.zeros(1, 2, dtype=torch.int64)))):
        with pytest.raises(ValueError):
            ops.sample_tokens(*args, **kw)


def test_sampling_follows_the_distribution():
    """Uniform numbers on a grid give every token its share of the grid, off by at most one point at each of its two ends."""
    logits = torch.randn(1, 12, generator=_gen(19))
    n = 4000
    u = (torch.arange(n) + 0.5) / n
    tok = ops.sample_tokens(logits.expand(n, -1), u, top_p=0.9)
    w = torch.softmax(logits[0].double(), 0)
    down, order = torch.sort(w, descending=True)
    keep = order[(torch.cumsum(down, 0) - down) <= 0.9]
    share = torch.zeros(12, dtype=torch.float64)
    share[keep] = w[keep] / w[keep].sum()
    assert (torch.bincount(tok, minlength=12) - n * share).abs().max() <= 2


# ------------------------------------------------------------------------- sampling: GPU
def _check_sampling(logits, u, generated=None, **kw):
    B = logits.shape[0]
    full = {k: torch.as_tensor(kw.get(k, d), device="cuda").to(t).expand(B) for k, d, t in (
        ("temperature", 1.0, torch.float32), ("top_k", 0, torch.int64), ("top_p", 1.0, torch.float32),
        ("min_p", 0.0, torch.float32), ("repetition_penalty", 1.0, torch.float32))}
    tok, lp = ops.sample_tokens(logits, u, generated=generated, return_logprob=True, **kw)
    rt, rl = sample_tokens_reference(logits, u, full["temperature"], full["top_k"], full["top_p"], full["min_p"], generated,
                                     full["repetition_penalty"])
    assert torch.equal(tok, rt)
    # log of an fp64 ratio, rounded once to fp32
    torch.testing.assert_close(lp, rl, atol=1e-7, rtol=2.0 ** -22, equal_nan=True)
    return tok


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 33, 1000, 4099, 32000, 131072, 400001])
@pytest.mark.parametrize("temperature,k,p,m", SAMPLE_SETTINGS)
def test_sampling_kernel(V, dtype, temperature, k, p, m):
    _cuda()
    g = _gen(V, "cuda")
    logits = (3 * torch.randn(5, V, generator=g, device="cuda")).to(dtype)
    u = torch.rand(5, generator=g, device="cuda")
    _check_sampling(logits, u, temperature=temperature, top_k=k, top_p=p, min_p=m)


@gpu
def test_sampling_kernel_per_row_and_penalty():
    _cuda()
    B, V = 64, 32000
    g = _gen(23, "cuda")
    logits = (3 * torch.randn(B, V + 8, generator=g, device="cuda")).to(torch.bfloat16)[:, 3:V + 3]  # unaligned rows
    row = torch.arange(B, device="cuda")
    gen = torch.randint(-5, V + 5, (B, 300), generator=g, device="cuda")
    kw = dict(temperature=0.3 * (row % 5).float(), top_k=(row % 4) * 30, top_p=1.0 - 0.1 * (row % 6).float(),
              min_p=0.02 * (row % 3).float(), repetition_penalty=1.0 + 0.2 * (row % 3).float())
    u = torch.rand(B, generator=g, device="cuda")
    tok = _check_sampling(logits, u, gen, **kw)
    # the same rows in another order, one by one
    some = [0, 7, 33, 63]
    for i in some:
        one = {k: v[i:i + 1] for k, v in kw.items()}
        assert int(ops.sample_tokens(logits[i:i + 1], u[i:i + 1], generated=gen[i:i + 1], **one)) == int(tok[i])


@gpu
@pytest.mark.parametrize("fill", ["equal", "two", "masked", "steps", "wide"])
def test_sampling_kernel_ties_and_masks(fill):
    """Rows of equal logits, of two values, masked to few tokens, on a coarse grid, spread over hundreds."""
    _cuda()
    B, V = 16, 5003
    g = _gen(29, "cuda")
    x = torch.randn(B, V, generator=g, device="cuda")
    if fill == "equal":
        x = torch.full_like(x, 1.25)
    elif fill == "two":
        x = (x > 0.5).float()
    elif fill == "masked":
        x = torch.where(torch.rand(B, V, generator=g, device="cuda") < 0.999, float("-inf"), x)
        x[3] = float("-inf")
        x[4] = torch.finfo(torch.float32).min
    elif fill == "steps":
        x = (x * 4).round() / 4
    else:
        x = 100 * x
    u = torch.rand(B, generator=g, device="cuda")
    for kw in (dict(), dict(top_p=0.5), dict(top_k=7), dict(top_k=40, top_p=0.3), dict(min_p=0.9), dict(top_p=0.9, min_p=0.01),
               dict(temperature=0.0), dict(temperature=1e-3), dict(temperature=50.0, top_p=0.7)):
        _check_sampling(x, u, **kw)


@gpu
@pytest.mark.parametrize("B", [1, 40, 160])
@pytest.mark.parametrize("fill", ["equal", "two", "flat"])
def test_sampling_kernel_borders_longer_than_the_list(fill, B):
    """Borders among more elements than the candidate list holds, with one block and with several a row."""
    _cuda()
    V = 131072
    g = _gen(31, "cuda")
    x = torch.randn(B, V, generator=g, device="cuda")
    x = torch.full_like(x, -3.5) if fill == "equal" else (x > 0.5).float() if fill == "two" else x / 64
    u = torch.rand(B, generator=g, device="cuda")
    for kw in (dict(top_p=0.5), dict(top_k=100000), dict(top_k=90000, top_p=0.6), dict(min_p=0.5), dict(top_p=0.7, min_p=0.9)):
        _check_sampling(x, u, **kw)


@gpu
def test_sampling_kernel_special_rows_and_graph():
    _cuda()
    _special_rows("cuda")
    x = torch.randn(3, 1000, device="cuda")
    u = torch.rand(3, device="cuda")
    ops.sample_tokens(x, u, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_tokens(x, u, top_p=0.9)
    for _ in range(3):
        x.normal_()
        u.uniform_()
        graph.replay()
        assert torch.equal(out, ops.sample_tokens(x, u, top_p=0.9))
    assert ops.sample_tokens(x[:0], u[:0]).shape == (0,)
    assert torch.equal(ops.sample_tokens(x.t().contiguous().t(), u), ops.sample_tokens(x, u))
    with pytest.raises(ValueError):
        ops.sample_tokens(x, u.cpu())
    with pytest.raises(RuntimeError):
        ops.sample_tokens(x.double(), u)
