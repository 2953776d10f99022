"""The quantised key/value ring, the fused attention and the fused sampler inside the decoders that use them."""

from __future__ import annotations

import copy

import pytest
import torch

import titans_pytorch_b200 as T
from titans_pytorch_b200.inference.decode import StreamingDecoder, generate_incremental
from titans_pytorch_b200.inference.generate import ContinuousBatcher, generate, sample_next

FIELDS = dict(dim=64, num_heads=2, num_layers=2, vocab_size=128, window_size=8, chunk_size=16,
              num_persistent_tokens=4, dropout=0.0, max_seq_len=256, ffn_mult=2.0, memory_hidden_mult=2.0)
# How far the logits may move against the fp32 ring, as norms.  A stored element is off by half a step: of amax / 127
# (int8), 2^-4 (e4m3), 2^-8 (bf16) or 2^-11 (fp16) of itself at most.  Keys move the scores by that share of |q||k|,
# which is of order one here, and values the output; the residual stream carries at least as much from elsewhere.  Two
# layers, keys and values: four times the half step.
NEAR = {"float32": 1e-4, "float16": 4 * 2.0 ** -11, "bfloat16": 4 * 2.0 ** -8, "int8": 4 * 0.5 / 127 * 2, "fp8": 4 * 2.0 ** -4}


def _model(cls, **kw):
    torch.manual_seed(0)
    return getattr(T, cls)(T.TitansConfig(**{**FIELDS, **kw})).eval()


def _compare(model, kind, ids, near, graph=False):
    a = StreamingDecoder(copy.deepcopy(model), batch=ids.shape[0], update_every=16)
    b = StreamingDecoder(model, batch=ids.shape[0], update_every=16, kv_cache=kind, graph=graph)
    for t in range(ids.shape[1]):
        x, y = a.step(ids[:, t:t + 1]).float(), b.step(ids[:, t:t + 1]).float()
        assert torch.isfinite(y).all()
        assert float((x - y).norm() / x.norm()) <= near, (kind, t)


@pytest.mark.parametrize("cls", ["TitansMAG", "TitansMAL", "TitansLMM"])
@pytest.mark.parametrize("kind", list(NEAR))
def test_ring_kinds_cpu(cls, kind):
    """Past the window (the ring wraps three times) and across a memory update."""
    ids = torch.randint(0, 128, (2, 26), generator=torch.Generator().manual_seed(1))
    _compare(_model(cls, use_kernels=False), kind, ids, NEAR[kind])


def test_ring_without_persistent_tokens_or_rope():
    ids = torch.randint(0, 128, (1, 11), generator=torch.Generator().manual_seed(1))
    _compare(_model("TitansMAG", num_persistent_tokens=0, use_rope=False), "float32", ids, NEAR["float32"])


def test_ring_kind_is_checked():
    with pytest.raises(ValueError):
        StreamingDecoder(_model("TitansMAG"), kv_cache="int3")


def test_fused_sampling_in_generation():
    model = _model("TitansMAG")
    prompt = torch.randint(0, 128, (2, 5), generator=torch.Generator().manual_seed(2))
    kw = dict(max_new_tokens=6, top_k=0, top_p=0.9, min_p=0.01, repetition_penalty=1.2)
    runs = [generate(copy.deepcopy(model), prompt, generator=torch.Generator().manual_seed(s), **kw)[0] for s in (3, 3, 4)]
    assert runs[0].shape == (2, 11) and torch.equal(runs[0], runs[1]) and not torch.equal(runs[0], runs[2])
    out, _ = generate_incremental(copy.deepcopy(model), prompt, kv_cache="int8", fused_sampling=True,
                                  generator=torch.Generator().manual_seed(3), max_new_tokens=4)
    assert out.shape == (2, 9)
    # greedy stays argmax; top_k = 1 is argmax too
    logits = torch.randn(3, 50, generator=torch.Generator().manual_seed(5))
    assert torch.equal(sample_next(logits, prompt[:1], greedy=True, fused=True)[:, 0], logits.argmax(-1))
    assert torch.equal(sample_next(logits, prompt[:1], top_k=1, fused=True)[:, 0], logits.argmax(-1))
    # the defaults draw what they always drew
    a = sample_next(logits, prompt[:1], generator=torch.Generator().manual_seed(6))
    f = torch.softmax(logits.masked_fill(logits < torch.topk(logits, 50)[0][..., -1, None], float("-inf")), -1)
    assert a.shape == (3, 1) and f.shape == logits.shape


def test_seeded_requests_repeat():
    model = _model("TitansMAG")
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, 128, (6,), generator=g) for _ in range(3)]

    def serve(which):
        b = ContinuousBatcher(copy.deepcopy(model), max_batch_size=4)
        ids = {i: b.add_request(prompts[i], max_new_tokens=5, seed=100 + i, min_p=0.01 * i, top_k=20 * i) for i in which}
        done = {r["id"]: r["ids"].tolist() for r in b.run()}
        return {i: done[r] for i, r in ids.items()}

    together = serve([0, 1, 2])
    assert serve([0, 1, 2]) == together and all(len(v) == 11 for v in together.values())
    assert serve([2]) == serve([2])
    # seeded and unseeded requests side by side
    mixed = ContinuousBatcher(copy.deepcopy(model), max_batch_size=4)
    mixed.add_request(prompts[0], max_new_tokens=2)
    mixed.add_request(prompts[1], max_new_tokens=3, seed=1)
    assert sorted(len(r["ids"]) for r in mixed.run()) == [8, 9]


def test_inference_cli_takes_the_cache_and_sampler(tmp_path, capsys):
    from titans_pytorch_b200.cli import inference

    model = _model("TitansMAG")
    path = str(tmp_path / "m.pt")
    T.save_checkpoint(path, model)
    inference.main(["--checkpoint", path, "--prompt", "ab", "--max-tokens", "3", "--decoder", "incremental", "--kv-cache", "int8",
                    "--fused-sampling", "--min-p", "0.02", "--device", "cpu"])
    assert capsys.readouterr().out.startswith("ab")


@pytest.mark.gpu
@pytest.mark.parametrize("cls", ["TitansMAG", "TitansMAL"])
@pytest.mark.parametrize("kind", list(NEAR))
def test_ring_kinds_gpu(cls, kind):
    """bf16 model: the two decoders round to bf16 at every layer (2^-8 each way, two layers, attention and output)."""
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    model = _model(cls, dim=128, window_size=16).cuda().to(torch.bfloat16)
    ids = torch.randint(0, 128, (3, 40), generator=torch.Generator().manual_seed(1)).cuda()
    for graph in (False, True):
        _compare(copy.deepcopy(model), kind, ids, NEAR[kind] + 4 * 2.0 ** -8, graph)


@pytest.mark.gpu
def test_generation_gpu_with_everything():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    model = _model("TitansMAG", dim=128, window_size=16).cuda().to(torch.bfloat16)
    prompt = torch.randint(0, 128, (4, 9), generator=torch.Generator().manual_seed(2)).cuda()
    runs = [generate_incremental(copy.deepcopy(model), prompt, max_new_tokens=20, kv_cache="fp8", fused_sampling=True,
                                 min_p=0.01, repetition_penalty=1.1,
                                 generator=torch.Generator(device="cuda").manual_seed(3))[0] for _ in range(2)]
    assert runs[0].shape == (4, 29) and torch.equal(runs[0], runs[1])
    b = ContinuousBatcher(model, max_batch_size=4)
    for i in range(5):
        b.add_request(prompt[i % 4], max_new_tokens=4, seed=i)
    assert len(b.run()) == 5
