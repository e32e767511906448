"""FP8 layers cut over ranks: every rank's share is FP8 as well (formats choose kernels and collectives), cut on blocks of 128 where there are enough, and the ranks' sums are
what one rank computes."""
from dataclasses import replace

import pytest
import torch

from machx_inference_engine_b200.formats.model_config import preset
from machx_inference_engine_b200.models.sources import SynthSource, default_policy
from machx_inference_engine_b200.models.transformer import DenseFFN, MoEFFN, TransformerModel, _even_chunks
from machx_inference_engine_b200.ops import ACT_SWIGLU
from machx_inference_engine_b200.ops.weights import WFormat, from_fp8
from machx_inference_engine_b200.parallel.comm import ParallelCtx
from test_parallel import _run


class Rank(ParallelCtx):
    """One rank of several without a group: sums stay partial."""

    def all_reduce(self, t):
        return t


def weight(N, K, E=1, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(E, N, K, generator=g).clamp(-4, 4) * 112).to(torch.float8_e4m3fn)
    return from_fp8(codes, torch.rand(E, -(-N // 128), -(-K // 128), generator=g) + 0.5)


@pytest.mark.parametrize("lo,hi", [(0, 64), (64, 256), (32, 300), (96, 224), (300, 301), (0, 300), (130, 172), (200, 333)])
@pytest.mark.parametrize("E", [1, 3])
def test_columns_that_cut_a_block_stay_fp8(lo, hi, E):
    w = weight(40, 333, E)
    got, want = w.slice_k(lo, hi, requant=True), w.dequantize()[:, :, lo:hi]
    assert got.fmt == WFormat.FP8 and (got.N, got.K, got.E) == (40, hi - lo, E)
    assert got.p0.shape == (E, 40, -(-(hi - lo) // 128) * 128) and got.p1.shape == (E, 3, got.p0.shape[2] // 128)
    t = got.p1.repeat_interleave(16, 1)[:, :40].repeat_interleave(128, 2)[..., :hi - lo]
    # half a step of e4m3, 2^-4 of a normal value or 2^-10 of the run's scale; the products of codes and scales are fp32 on both sides
    err = (got.dequantize() - want).abs()
    assert bool((err <= torch.maximum(want.abs() * 2.0 ** -4, t * 2.0 ** -10) * (1 + 2.0 ** -20)).all())
    block = (lo + torch.arange(hi - lo)) // 128
    old = w.p1.repeat_interleave(16, 1)[:, :40][:, :, block]
    assert bool((err[old == t] == 0).all())                 # codes that keep their scale keep their bits
    with pytest.raises(ValueError):
        w.slice_k(64, 256)


def test_one_scale_is_cut_exactly():
    w = from_fp8(weight(32, 96).p0[0, :, :96].contiguous(), torch.tensor([[0.37]]))
    for lo, hi in ((0, 64), (64, 96), (17, 50)):
        assert torch.equal(w.slice_k(lo, hi, requant=True).dequantize(), w.dequantize()[:, :, lo:hi])
    z = weight(16, 256)
    z.p1.zero_()
    assert float(z.slice_k(64, 192, requant=True).dequantize().abs().max()) == 0


def test_ranges_of_ranks():
    assert _even_chunks(256, 2, 32) == [(0, 128), (128, 256)] and _even_chunks(96, 2, 32) == [(0, 64), (64, 96)]
    assert _even_chunks(2880, 2, 128) == [(0, 1536), (1536, 2880)] and _even_chunks(2880, 3, 128) == [(0, 1024), (1024, 2048), (2048, 2880)]
    for n, parts in ((10944, 8), (2880, 4), (2880, 23), (130, 2)):
        r = _even_chunks(n, parts, 128)
        assert r[0][0] == 0 and r[-1][1] == n and all(a[1] == b[0] and a[1] % 128 == 0 for a, b in zip(r, r[1:])) and all(lo < hi for lo, hi in r)


def layers(cls, cfg, world, **kw):
    made = []
    for r in range(world):
        src = SynthSource("cpu", default_policy("", "fp8"), seed=7)
        made.append(cls(cfg, 0, src, Rank(rank=r, world=world), **kw))
    return made


# (width of an expert, ranks): blocks of 128 shared out evenly, unevenly, with a last block that is a part of one; fewer blocks than ranks
@pytest.mark.parametrize("ffn,world", [(256, 2), (416, 2), (416, 3), (768, 4), (320, 2), (96, 2), (256, 4), (160, 4)])
@pytest.mark.parametrize("bias", [False, True])
def test_experts_cut_over_ranks(ffn, world, bias):
    cfg = replace(preset("tiny-qwen3moe"), n_experts=5, expert_ffn=ffn, hidden=128)
    one, = layers(MoEFFN, cfg, 1, act=ACT_SWIGLU, with_bias=bias)
    many = layers(MoEFFN, cfg, world, act=ACT_SWIGLU, with_bias=bias)
    assert {(m.gate_up.fmt, m.down.fmt) for m in many} == {(WFormat.FP8, WFormat.FP8)}
    assert sum(m.down.K for m in many) == ffn and all(m.expert_tp for m in many)
    aligned = -(-ffn // 128) >= world
    assert not aligned or all(m.down.K % 128 == 0 for m in many[:-1])
    for T in (1, 4, 9, 40):                                  # slots, and rows sorted by expert
        h = torch.randn(T, 128, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
        want = one(h, Rank())
        got = sum(m(h, Rank(rank=r, world=world)) for r, m in enumerate(many))
        # On the blocks of 128 the codes are the same: what differs is the rounding of each rank's rows to bf16, 2^-8 of rows whose squares add up to no more than a few times the
        # sum's.  Off them a rank's codes have other scales: half a step of e4m3, 2^-4, on both sides.
        assert float((got - want).norm() / want.norm()) < (2.0 ** -6 if aligned else 2.0 ** -3), T


@pytest.mark.parametrize("ffn,world", [(688, 2), (688, 3), (1376, 8), (512, 2), (144, 4)])
def test_dense_layers_cut_over_ranks(ffn, world):
    cfg = replace(preset("tiny-llama"), ffn=ffn, hidden=128)
    one, = layers(DenseFFN, cfg, 1)
    many = layers(DenseFFN, cfg, world)
    assert {m.down.w.fmt for m in many} == {WFormat.FP8} and {m.gate_up.w.fmt for m in many} == {WFormat.FP8}
    assert sum(m.down.w.K for m in many) == ffn
    h = torch.randn(6, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    want = one(h, Rank()).float()
    got = sum(m(h, Rank(rank=r, world=world)) for r, m in enumerate(many))
    # (each side: half a step of bf16 of the sum where one rank writes it; 2^-4 of each side where codes differ)
    assert float((got - want).norm() / want.norm()) < (2.0 ** -7 if -(-ffn // 128) >= world else 2.0 ** -3)


def test_other_formats_are_cut_as_before():
    src = SynthSource("cpu", default_policy("", "q8_0"), seed=7)
    w = src.matrix("x", 64, 256)
    assert w.slice_k(48, 112, requant=True).fmt == WFormat.Q8 and w.slice_k(32, 96).fmt == WFormat.Q8
    cfg = replace(preset("tiny-qwen3moe"), n_experts=5, expert_ffn=416, hidden=128)
    many = []
    for r in range(2):
        many.append(MoEFFN(cfg, 0, SynthSource("cpu", default_policy("", "q8_0"), seed=7), Rank(rank=r, world=2), act=ACT_SWIGLU, with_bias=False))
    assert [m.down.K for m in many] == [224, 192]


# Ranks in earnest, over gloo.  Both sides round every product's input to e4m3: half a step is 2^-4 of a value at most, 2^-4 / sqrt(3) of the norm, and two layouts whose blocks or
# whose partial sums differ round differently, sqrt(2) times that, 0.05, in each of at most seven products of a layer.  Two layers: 14 independent parts of at most 0.05 of
# the stream that they join, 0.19 of the norm: a cosine of 0.98.
@pytest.mark.parametrize("name,world,within", [("tiny-llama", 2, False), ("tiny-qwen3moe", 2, False), ("tiny-qwen3moe", 2, True), ("tiny-qwen3moe", 4, True)])
def test_ranks_match_a_single_one(monkeypatch, name, world, within):
    one = _run(1, name, "fp8", "cpu")
    if within:
        monkeypatch.setenv("MX_TEST_EXPERT_TP", "1")
    many = _run(world, name, "fp8", "cpu")
    a, b = one["logits"].flatten(), many["logits"].flatten()
    assert many["world"] == world and float(torch.dot(a, b) / (a.norm() * b.norm())) > 0.98


@pytest.mark.parametrize("kind", ["attn_q", "attn_v", "attn_output", "ffn_gate", "ffn_down", "none"])
def test_the_row_sharded_prefill_is_not_taken_with_any_fp8_projection(kind):
    """Its products read gathered rows and store into their peers' memory, which no FP8 product does; a file may hold codes for some of a layer's matrices only."""
    cfg = preset("tiny-llama")
    policy = lambda name: WFormat.FP8 if kind in name and name.startswith("blk.1.") else WFormat.BF16
    par = ParallelCtx()
    model = TransformerModel(cfg, SynthSource("cpu", policy, seed=1), "cpu", par, max_ctx=1024)
    par.fused, par.sharded = object(), type("All", (), {"can_shard": lambda self, T: True})()
    assert model._can_shard(type("FB", (), {"T": 640, "want_hidden": False})(), None) == (kind == "none")
