"""The quantised decode step as a model runs it: 4-bit projections around an
8-bit paged KV cache, in prefill, decode, CUDA graphs and the batching engine."""
import pytest
import torch

from aether_b200.models.qwen import QwenConfig, QwenModel, QwenWeights
from aether_b200.ops import functional as F
from aether_b200.serving.engine import Engine
from aether_b200.serving.kv import Paged8KVCache
from aether_b200.serving.sampling import SamplingParams
from aether_b200.serving.tokenizer import ByteTokenizer

CPU_GPU = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TINY = dict(vocab=300, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, d_ff=512, max_seq=192, init_std=0.06)


def tiny(**kw):
    return QwenConfig(**dict(TINY, **kw))


def rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def decode_logits(m, prompts, toks, use_graph):
    """fp32 logits after the prompt and after each of ``toks``, teacher-forced."""
    B, S = prompts.shape
    for r in range(B):
        m.cache.release(r)
        m.cache.ensure(r, S + toks.shape[1])
    _, logits = m.prefill(prompts, return_logits=True)
    out = [logits.clone()]
    for t in range(toks.shape[1]):
        pos = torch.full((B,), S + t, dtype=torch.int32, device=m.device)
        m.decode_step(toks[:, t], pos, torch.arange(B, dtype=torch.int32, device=m.device), use_graph=use_graph, want_logits=True)
        out.append(m.buf["logits"][:B].clone())
    return torch.stack(out, 1)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("kw", [{}, dict(qkv_bias=False, qk_norm=True, sliding_window=24), dict(attn_softcap=20.0)])
@pytest.mark.parametrize("w4", [0, 64])
def test_teacher_forced_logits(dev, kw, w4):
    """Against the fp32 forward of the same (expanded) weights. The 8-bit cache
    adds rounding of 0.3 % of a block's largest value to what bf16 leaves: about
    1 % of a typical value, averaged over the keys."""
    cfg = tiny(**kw)
    w = QwenWeights(cfg, dev, seed=3)
    if w4:
        w.quantize_w4(w4)
    m = QwenModel(cfg, device=dev, max_batch=3, weights=w, kv_pages=40, page_size=16, kv_bits=8)
    assert isinstance(m.cache, Paged8KVCache) and not m.fused_decode
    g = torch.Generator().manual_seed(1)
    seq = torch.randint(0, 300, (3, 50), generator=g).to(dev)
    got = decode_logits(m, seq[:, :37], seq[:, 37:], use_graph=dev == "cuda")
    want = m.reference_logits(seq)[:, 36:]
    assert rel(got, want) < 0.03


@pytest.mark.parametrize("dev", CPU_GPU)
def test_prefill_in_chunks_reads_the_cached_prefix(dev):
    cfg = tiny()
    m = QwenModel(cfg, device=dev, seed=5, max_batch=2, kv_pages=30, page_size=16, kv_bits=8)
    seq = torch.randint(0, 300, (2, 70), generator=torch.Generator().manual_seed(2)).to(dev)
    for r in range(2):
        m.cache.ensure(r, 70)
    m.prefill(seq[:, :41])
    _, got = m.prefill(seq[:, 41:], start_pos=41, return_logits=True)
    assert rel(got, m.reference_logits(seq)[:, -1]) < 0.03


@pytest.mark.parametrize("dev", CPU_GPU)
def test_engine_with_shared_prefixes_and_reused_pages(dev):
    """More requests than slots, pages handed from one to the next: outputs are
    those of each request alone."""
    cfg = tiny()
    g = torch.Generator().manual_seed(3)
    shared = torch.randint(0, 300, (37,), generator=g).tolist()
    prompts = [shared + torch.randint(0, 300, (n,), generator=g).tolist() for n in (1, 9, 20, 3)]

    def run(model, together):
        eng = Engine(model, ByteTokenizer(), max_concurrent=2, eos_ids=[], use_graph=dev == "cuda")
        if together:
            rs = [eng.submit(p, SamplingParams(max_tokens=12)) for p in prompts]
            outs = [list(eng.stream(r, timeout=120)) for r in rs]
        else:
            outs = [list(eng.stream(eng.submit(p, SamplingParams(max_tokens=12)), timeout=120)) for p in prompts]
        eng.shutdown()
        assert not eng.errors, eng.errors
        return outs, eng

    make = lambda pages: QwenModel(cfg, device=dev, seed=4, max_batch=2, max_seq=128, kv_pages=pages, page_size=16, kv_bits=8)  # noqa: E731
    alone, eng = run(make(12), False)
    assert eng.metrics.counters["prefix_cached_tokens"] == 3 * 32
    both, _ = run(make(12), True)
    same = sum(a == b for x, y in zip(alone, both) for a, b in zip(x, y))
    assert same >= 0.9 * 48  # a tie may break differently in another batch


def test_8bit_cache_takes_half_the_memory():
    m16, m8 = (QwenModel(tiny(), device="cpu", max_batch=1, kv_pages=9, page_size=64, kv_bits=b) for b in (16, 8))
    assert m8.cache.bytes() < 0.54 * m16.cache.bytes()


def test_w4_cpu_equals_its_expanded_weights():
    """linear_w4 inside the model computes what bf16 expanded weights do."""
    cfg = tiny()
    a = QwenWeights(cfg, "cpu", seed=6).quantize_w4(128)
    assert all(isinstance(t, F.W4Weight) for ws in (a.wqkv, a.wo, a.wgu, a.wd) for t in ws)
    b = QwenWeights(cfg, "cpu", seed=6)
    for ws, wt in ((b.wqkv, a.wqkv), (b.wo, a.wo), (b.wgu, a.wgu), (b.wd, a.wd)):
        ws[:] = [t.bf16() for t in wt]
    seq = torch.randint(0, 300, (1, 20), generator=torch.Generator().manual_seed(7))
    la, lb = (QwenModel(cfg, device="cpu", max_batch=1, weights=w).reference_logits(seq) for w in (a, b))
    assert torch.equal(la, lb)
    m = QwenModel(cfg, device="cpu", max_batch=1, weights=a)
    assert m.generate(seq, 4, use_graph=False).shape == (1, 4)


def test_refusals():
    with pytest.raises(ValueError):
        QwenModel(tiny(), device="cpu", kv_bits=8)  # not paged
    with pytest.raises(ValueError):
        QwenModel(tiny(), device="cpu", kv_pages=8, kv_bits=4)
    with pytest.raises(ValueError):
        QwenModel(tiny(), device="cpu", kv_pages=8, page_size=8, kv_bits=8)
    with pytest.raises(ValueError):
        QwenModel(tiny(n_heads=8, n_kv_heads=8), device="cpu", kv_pages=8, kv_bits=8)  # head_dim 32
    w = QwenWeights(tiny(), "cpu", tp_rank=0, tp_size=2)
    with pytest.raises(ValueError):
        w.quantize_w4()
