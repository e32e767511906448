"""Expert layers of the layer-list graphs with FP8 banks: the same numbers from pairs in slots (a few tokens) and from pairs sorted by expert (prompts)."""
from dataclasses import replace

import pytest
import torch

from machx_inference_engine_b200 import ops
from machx_inference_engine_b200.formats.model_config import preset
from machx_inference_engine_b200.models import build_model
from machx_inference_engine_b200.models.sources import SynthSource, default_policy
from machx_inference_engine_b200.models.transformer import ClampedMoEFFN, MoEFFN, ScaledInputMoEFFN, TransformerModel, UnaryMoEFFN
from machx_inference_engine_b200.ops.weights import WFormat
from machx_inference_engine_b200.parallel.comm import ParallelCtx
from machx_inference_engine_b200.runtime.engine import EngineOptions, LLMEngine, SamplingParams

H, E, K, F = 160, 6, 2, 96
DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def layer(cls, dev, shared):
    src = SynthSource(dev, default_policy("", "fp8"), seed=3, gen_device="cpu")
    if cls is ClampedMoEFFN:
        return cls(src, "x", H, H, E, K, F, 1.5, shared_ffn=64 if shared else 0, shared_limit=2.5)
    return cls(src, "x", H, H, E, K, F, shared_ffn=64 if shared else 0)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("cls", [ClampedMoEFFN, ScaledInputMoEFFN])
def test_pairs_sorted_by_expert_are_the_slots_pairs(cls, shared, dev):
    m = layer(cls, dev, shared)
    assert m.gate_up.fmt == m.down.fmt == WFormat.FP8
    for T in (1, 3, 7, 40):
        h = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(dev, torch.bfloat16)
        got = {}
        for most in (0, 1000):                               # never in slots, always
            m.PAIR_GEMV_MAX_TOKENS = most
            got[most] = m(h).materialize()
        # rows rounded alike, sums in another order: bf16 borders of the hidden rows may be crossed (2^-8 of a value, then a code's step of 2^-3 of it in one of 16), and the two
        # results are rounded to bf16 once more
        assert float((got[0] - got[1000]).norm() / got[1000].norm()) < 2.0 ** -7, T
        assert float(got[1000].norm()) > 0


@pytest.mark.parametrize("dev", DEVICES)
def test_a_graph_answers_prompts_of_any_length(dev):
    """(The first tokens agree for a prompt alone and beside others; longer continuations of random weights drift at near-ties.)"""
    cfg = preset("tiny-zegelix")
    eng = LLMEngine(build_model(cfg, torch.device(dev), quant="fp8", max_ctx=512, gen_device="cpu"), EngineOptions(max_ctx=512, max_batch_tokens=256, max_seqs=4))
    ids = torch.randint(0, cfg.vocab, (150,), generator=torch.Generator().manual_seed(1)).tolist()
    for n in (1, 3, 30, 150):
        a, = eng.generate([ids[:n]], SamplingParams(max_tokens=3))
        assert len(a) == 3, n
    both = [eng.generate([ids, ids[:9], ids[:30]], SamplingParams(max_tokens=3)) for _ in range(2)]
    assert both[0] == both[1] and [len(o) for o in both[0]] == [3, 3, 3]


def test_other_formats_take_the_padded_packing():
    src = SynthSource("cpu", default_policy("", "q8_0"), seed=3)
    m = ClampedMoEFFN(src, "x", H, H, E, K, F, 1.5)
    h = torch.randn(12, H, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    s = m(h)
    assert m.gate_up.fmt == WFormat.Q8 and s.y.shape[0] % 128 == 0
    assert isinstance(s, ops.ExpertSum) and issubclass(ClampedMoEFFN, UnaryMoEFFN)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("odd", ["down", "gate_up"])
def test_banks_of_which_one_is_fp8(odd, dev):
    """A layer's rows come in one packing; where a file has FP8 codes for some of its banks only, those are decoded to bf16 and the layer takes the other formats' paths."""
    def mixed(quant):
        def policy(name):
            down = "down" in name
            if "gate_inp" in name:
                return WFormat.BF16
            return WFormat.FP8 if quant == "fp8" and down == (odd == "down") else WFormat.Q8 if down and quant == "fp8" else WFormat.BF16
        return policy

    cfg = replace(preset("tiny-qwen3moe"), hidden=128)
    m = MoEFFN(cfg, 0, SynthSource(dev, mixed("fp8"), seed=7, gen_device="cpu"), ParallelCtx(), act=ops.ACT_SWIGLU, with_bias=False)
    assert WFormat.FP8 not in (m.gate_up.fmt, m.down.fmt)
    plain = MoEFFN(cfg, 0, SynthSource(dev, mixed("bf16"), seed=7, gen_device="cpu"), ParallelCtx(), act=ops.ACT_SWIGLU, with_bias=False)
    for T in (2, 9, 40):
        h = torch.randn(T, 128, generator=torch.Generator().manual_seed(T)).to(dev, torch.bfloat16)
        got, want = (x(h, ParallelCtx()) for x in (m, plain))
        # the same weights but for the rounding of one or two banks to e4m3, half a step of 2^-4 of each value at most, and of the other to bf16 or 8 bits
        assert float((got - want).norm() / want.norm()) < 2.0 ** -3, T


@pytest.mark.parametrize("cls", [ClampedMoEFFN, ScaledInputMoEFFN])
@pytest.mark.parametrize("which", ["gate up", "down", "up down", "gate"])
def test_gated_banks_of_which_some_are_fp8(cls, which):
    policy = lambda fp8: lambda name: WFormat.FP8 if fp8 and name.rsplit(".", 1)[-1] in which.split() else WFormat.BF16
    m, plain = (cls(SynthSource("cpu", policy(fp8), seed=3), "x", H, H, E, K, F, **({"limit": 1.5} if cls is ClampedMoEFFN else {})) for fp8 in (True, False))
    assert WFormat.FP8 not in (m.gate_up.fmt, m.down.fmt)
    for T in (2, 30):
        h = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
        got, want = m(h).materialize(), plain(h).materialize()
        assert 0 < float((got - want).norm() / want.norm()) < 2.0 ** -3      # (as above)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name,tied", [("tiny-llama", False), ("tiny-llama", True)])
def test_an_embedding_in_fp8_is_decoded_while_loading(dev, name, tied):
    """Rows of it are read, not multiplied; the head stays FP8 where it is a matrix of its own."""
    cfg = replace(preset(name), tie_embeddings=tied)
    model = TransformerModel(cfg, SynthSource(dev, lambda n: WFormat.FP8, seed=1, gen_device="cpu"), dev, max_ctx=512)
    assert model.embed_w.fmt == WFormat.BF16 and model.lm_head.w.fmt == (WFormat.BF16 if tied else WFormat.FP8)
    eng = LLMEngine(model, EngineOptions(max_ctx=512, max_batch_tokens=256, max_seqs=2))
    out, = eng.generate([list(range(40))], SamplingParams(max_tokens=4))
    assert len(out) == 4
