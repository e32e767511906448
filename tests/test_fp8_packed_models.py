"""Expert layers of the layer-list graphs with FP8 banks: the same numbers from pairs in slots (a few tokens) and from pairs sorted by expert (prompts)."""
import pytest
import torch

from machx_inference_engine_b200 import ops
from machx_inference_engine_b200.formats.model_config import preset
from machx_inference_engine_b200.models import build_model
from machx_inference_engine_b200.models.sources import SynthSource, default_policy
from machx_inference_engine_b200.models.transformer import ClampedMoEFFN, ScaledInputMoEFFN, UnaryMoEFFN
from machx_inference_engine_b200.ops.weights import WFormat
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
