"""FP8 weights and rows on the CPU: the rounding against its definition, surgery on the runtime layout, the oracle's products, refusals."""
import pytest
import torch

import fp8_oracle as O
from machx_inference_engine_b200 import ops
from machx_inference_engine_b200.ops import fp8
from machx_inference_engine_b200.ops.weights import QuantWeight, WFormat, from_dense, from_fp8


def codes(*shape, seed=0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).clamp(-4, 4) * 112).to(torch.float8_e4m3fn)


def weight(N, K, E=1, seed=0):
    return from_fp8(codes(E, N, K, seed=seed), torch.rand(E, -(-N // 128), -(-K // 128), generator=torch.Generator().manual_seed(seed)) + 0.5)


@pytest.mark.parametrize("M,K", [(1, 1), (3, 128), (4, 200), (2, 2880)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rounding_is_the_definition(M, K, dtype):
    g = torch.Generator().manual_seed(M + K)
    x = (torch.randn(M, K, generator=g) * torch.exp(10 * torch.randn(M, 1, generator=g))).to(dtype)
    q = ops.fp8_rows(x)
    want, scale = O.rows(x)
    assert torch.equal(q.codes.float().double(), want) and torch.equal(q.scale.double(), scale) and q.shape == (M, K)
    assert torch.equal(q.dequantize().double(), O.row_values(x))


def test_rounding_of_rows_that_are_not_finite_and_through_an_index():
    x = torch.ones(4, 300)
    x[1, 130], x[2, 5] = float("nan"), float("-inf")
    q = ops.fp8_rows(x)
    assert q.scale.isnan().tolist() == [[False, False, True, False], [False, True, False, False], [False] * 4]
    q = ops.fp8_rows(x, index=torch.tensor([3, -1, 4, 0], dtype=torch.int32))
    assert q.scale.isnan().any(0).tolist() == [False, False, True, False] and float(q.codes[1].float().abs().max()) == 0


@pytest.mark.parametrize("N,K,block", [(256, 256, (128, 128)), (200, 300, (128, 128)), (130, 100, (16, 128)), (64, 512, (32, 256)), (100, 200, (None, None)), (100, 200, (16, None))])
def test_runtime_layout_holds_the_values(N, K, block):
    c = codes(2, N, K)
    rows, cols = block[0] or 10 ** 6, block[1] or 10 ** 6
    t = torch.rand(2, -(-N // rows), -(-K // cols)) + 0.1
    w = from_fp8(c, t.to(torch.bfloat16), block)
    e, n, k = torch.meshgrid(torch.arange(2), torch.arange(N), torch.arange(K), indexing="ij")
    want = c.float() * t.to(torch.bfloat16).float()[e, n // rows, k // cols]
    assert w.fmt == WFormat.FP8 and torch.equal(w.dequantize(), want) and torch.equal(O.weight_values(w), want.double().float().double())
    flat = from_fp8(c[0], t[0].to(torch.bfloat16), block)
    assert torch.equal(flat.dequantize()[0], want[0])


def test_quantised_weights_are_near():
    w = torch.randn(3, 200, 300, generator=torch.Generator().manual_seed(1))
    q = from_dense(w, WFormat.FP8)
    # half a step of e4m3 is 2^-4 of a normal value; below 2^-6 of 448 scale units the step is 2^-9 of them
    t = q.p1.repeat_interleave(16, 1)[:, :200].repeat_interleave(128, 2)[..., :300]
    assert bool(((q.dequantize() - w).abs() <= torch.maximum(w.abs() * 2.0 ** -4, t * 2.0 ** -10) * (1 + 2.0 ** -20)).all())
    assert float(from_dense(torch.zeros(1, 20, 20), WFormat.FP8).dequantize().abs().max()) == 0


def test_rows_and_columns_are_cut_and_joined():
    w = weight(320, 640)
    d = w.dequantize()
    assert torch.equal(w.slice_rows(48, 200).dequantize(), d[:, 48:200])
    assert torch.equal(w.slice_k(128, 512).dequantize(), d[:, :, 128:512]) and torch.equal(w.slice_k(512, 640).dequantize(), d[:, :, 512:])
    odd = weight(64, 300)
    assert torch.equal(odd.slice_k(128, 300).dequantize(), odd.dequantize()[:, :, 128:]) and odd.slice_k(128, 300).K == 172
    a, b = weight(48, 300, seed=1), weight(33, 300, seed=2)
    assert torch.equal(QuantWeight.cat_rows([a, b]).dequantize(), torch.cat([a.dequantize(), b.dequantize()], 1))
    g, u = weight(64, 200, 2, seed=3), weight(64, 200, 2, seed=4)
    both = QuantWeight.interleave_gate_up(g, u).dequantize().view(2, 4, 2, 16, 200)
    assert torch.equal(both[:, :, 0].reshape(2, 64, 200), g.dequantize()) and torch.equal(both[:, :, 1].reshape(2, 64, 200), u.dequantize())
    assert torch.equal(weight(32, 128, 4).slice_experts(1, 3).dequantize(), weight(32, 128, 4).dequantize()[1:3])
    perm = torch.randperm(128, generator=torch.Generator().manual_seed(0))
    one = weight(128, 256)                                    # one row of scales: any order of the rows is exact
    assert torch.equal(one.select_rows(perm).dequantize(), one.dequantize()[:, perm])
    with pytest.raises(ValueError):
        QuantWeight.cat_rows([b, a])
    with pytest.raises(ValueError):
        w.slice_k(64, 256)
    with pytest.raises(ValueError):
        w.pad_groups(rows=(1, 400))


def test_runs_of_rows_with_different_scales_are_rounded_again():
    w = weight(256, 128)
    idx = torch.tensor([0, 130] * 8 + [200] * 3)
    got, want = w.select_rows(idx), w.dequantize()[:, idx]
    t = got.p1.repeat_interleave(16, 1)[:, :19].repeat_interleave(128, 2)
    assert got.N == 19 and torch.equal(got.dequantize()[:, 16:], want[:, 16:])
    assert bool(((got.dequantize() - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, t * 2.0 ** -10) * (1 + 2.0 ** -20)).all())
    assert torch.equal(got.p1, torch.maximum(w.p1[:, :1], w.p1[:, 8:9]).expand(1, 2, 1)) or torch.equal(got.p1[:, 1], w.p1[:, 12])


def test_products_of_the_oracle():
    x, w = torch.randn(7, 300, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16), weight(96, 300, 4)
    one = w.slice_experts(1, 2)
    want = O.row_values(x) @ O.weight_values(one)[0].T
    assert O.rel(ops.linear(x, one, out_f32=True), want) < O.fp32_bound(300) + 2.0 ** -22 and ops.linear(x, one).dtype == torch.bfloat16
    assert torch.equal(ops.linear(ops.fp8_rows(x), one), ops.linear(x, one))
    idx = torch.tensor([[0, 2], [3, 1], [2, 0], [2, 3], [0, 3], [1, 2], [3, 0]], dtype=torch.int32)
    pk = ops.moe_pack(idx, 4, tile=1)
    got = ops.expert_linear(x, w, pk, x_index=pk.packed_token, act=ops.ACT_SWIGLU, out_f32=True)
    slots = ops.expert_gemv(x, w, idx.reshape(-1), x_div=2, act=ops.ACT_SWIGLU, out_f32=True)
    want = O.activate(torch.einsum("pk,pnk->pn", O.row_values(x).repeat_interleave(2, 0), O.weight_values(w)[idx.reshape(-1).long()]), "swiglu")
    assert O.rel(got[pk.pair_to_packed.long()], want) < 1e-5 and O.rel(slots, want) < 1e-5
    assert ops.expert_linear(x, w, pk, x_index=pk.packed_token).dtype == torch.bfloat16 and ops.expert_gemv(x, w, idx.reshape(-1), x_div=2).dtype == torch.bfloat16


def refused(call):
    with pytest.raises(ValueError):
        call()


def test_refusals_of_weights():
    c = codes(64, 256)
    refused(lambda: from_fp8(c.float(), torch.ones(1, 2)))
    refused(lambda: from_fp8(c, torch.ones(2, 2)))
    refused(lambda: from_fp8(c, torch.ones(1, 2, dtype=torch.int32)))
    refused(lambda: from_fp8(c, torch.ones(8, 2), (8, 128)))
    refused(lambda: from_fp8(c, torch.ones(1, 4), (128, 64)))
    refused(lambda: from_fp8(c[:0], torch.ones(0, 2)))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_refusals_of_the_operators(dev):
    w, bank = weight(96, 256).to(dev), weight(96, 256, 4).to(dev)
    x = torch.randn(6, 256, device=dev).to(torch.bfloat16)
    refused(lambda: ops.fp8_rows(x.to(torch.float16)))
    refused(lambda: ops.fp8_rows(x[0]))
    refused(lambda: ops.fp8_rows(x[:, ::2]))
    refused(lambda: ops.fp8_rows(x[:, :0]))
    refused(lambda: ops.fp8_rows(x, index=torch.zeros(3, dtype=torch.int64, device=dev)))
    refused(lambda: ops.linear(x.float(), w))
    refused(lambda: ops.linear(x[:, :255], w))
    refused(lambda: ops.linear(x, bank))
    refused(lambda: ops.linear(x, w, bias=torch.zeros(95, device=dev)))
    refused(lambda: ops.linear(x, w, bias=torch.zeros(96, device=dev, dtype=torch.bfloat16)))
    refused(lambda: ops.linear(x, w, row_scale=torch.zeros(5, device=dev)))
    refused(lambda: ops.linear(x, w, out=torch.zeros(6, 96, device=dev)))
    refused(lambda: ops.linear(x, w, out=torch.zeros(6, 95, device=dev, dtype=torch.bfloat16)))
    refused(lambda: ops.linear(x, w, out=torch.zeros(96, 6, device=dev, dtype=torch.bfloat16).t()))
    refused(lambda: ops.linear(x, w, out=torch.zeros(1, 96, device=dev, dtype=torch.bfloat16).expand(6, 96)))
    refused(lambda: ops.linear(x, weight(80, 256).to(dev), act=ops.ACT_SWIGLU))
    refused(lambda: ops.linear(ops.fp8_rows(x), from_dense(torch.zeros(96, 256, device=dev), WFormat.BF16)))
    q = ops.fp8_rows(x)
    refused(lambda: ops.linear(ops.FP8Rows(q.codes, q.scale.t(), q.K), w))
    refused(lambda: ops.linear(ops.FP8Rows(q.codes[:, :128], q.scale, q.K), w))
    idx = torch.zeros(6, 1, dtype=torch.int32, device=dev)
    pk = ops.moe_pack(idx, 4, tile=1)
    refused(lambda: ops.expert_linear(x, bank, ops.moe_pack(idx, 4)))
    refused(lambda: ops.expert_linear(x[:5], bank, pk))
    refused(lambda: ops.expert_linear(x, bank, pk, e_lo=1))
    refused(lambda: ops.expert_linear(x, bank, pk, x_index=pk.packed_token[:3]))
    refused(lambda: ops.expert_linear(x, bank, pk, x_index=pk.packed_token.long()))
    refused(lambda: ops.expert_linear(q, bank, pk, x_index=pk.packed_token))
    refused(lambda: ops.expert_linear(x, bank, pk, bias=torch.zeros(96, device=dev)))
    refused(lambda: ops.expert_linear(x, from_dense(torch.zeros(4, 96, 256, device=dev), WFormat.Q8), pk))
    refused(lambda: ops.grouped_linear(x, bank, torch.zeros(1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)))
    refused(lambda: ops.expert_gemv(x, bank, idx.reshape(-1).long()))
    refused(lambda: ops.expert_gemv(x[:5], bank, idx.reshape(-1)))
    refused(lambda: ops.expert_gemv(x, bank, idx.reshape(-1), x_div=0))
    refused(lambda: ops.expert_gemv(x, bank, idx.reshape(-1), slot_scale=torch.zeros(5, device=dev)))
    if dev != "cpu":
        refused(lambda: ops.linear(x, w.to("cpu")))
        refused(lambda: ops.linear(x, w, bias=torch.zeros(96)))
        refused(lambda: ops.fp8_rows(x, index=torch.zeros(3, dtype=torch.int32)))
