"""Element-wise activations behind FP8 products, in each kernel that writes outputs: xIELU, GELU (tanh form) and tanh against 64 bits.

Bounds, relative to the norm: an argument is off by fp32_bound of its row's size.  tanh: the slope is 1 at most, and arguments of size 2.7 (the inputs' e / 1) have outputs of 0.85: a
factor below 4.  GELU: slopes up to 1.13 for outputs of 1 / sqrt(2) of the arguments': below 2.  xIELU with a, b below 1: slope times argument over output is 2 at most on the
right, slopes below 1.4 on the left, whose outputs are smaller than the right's: below 4.  Eight covers them all, and 2^-20 the exponential, reciprocal and tanh of a few steps of 2^-23."""
import math
import zlib

import pytest
import torch

import fp8_oracle as O
from machx_inference_engine_b200 import ops
from machx_inference_engine_b200.ops.weights import from_fp8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
A, B = 0.8, 0.9
ACTS = {
    "xielu": (ops.ACT_XIELU, lambda z: torch.where(z > 0, A * z * z + z / 2, B * (torch.exp(z.clamp(max=0)) - 1 - z) + z / 2)),
    "gelu": (ops.ACT_GELU_TANH, lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))),
    "tanh": (ops.ACT_TANH, torch.tanh),
}


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


def bank(N, K, E=1):
    g = gen(N, K, E)
    codes = (torch.randn(E, N, K, generator=g).clamp(-4, 4) * 112).to(torch.float8_e4m3fn)
    return from_fp8(codes, (0.5 + torch.rand(E, -(-N // 128), -(-K // 128), generator=g)) * (K ** -0.5 / 112)).to(DEV)


def acts(M, K):
    g = gen(M, K)
    return (torch.randn(M, K, generator=g) * torch.exp(torch.randn(K, generator=g))).to(DEV, torch.bfloat16)


def tolerance(K, bf16=False):
    return 8 * O.fp32_bound(K) + 2.0 ** -20 + (2.0 ** -8 if bf16 else 0.0)


# (few-row kernel, streaming kernel with rows rounded in it and before, tiles, tiles in pieces along K)
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M,N,K", [(1, 545, 1088), (8, 1000, 300), (1, 8224, 4096), (8, 6150, 1030), (19, 545, 1088), (64, 545, 1088), (130, 1000, 515), (513, 257, 200), (100, 256, 4096)])
def test_dense(M, N, K, act):
    x, w = acts(M, K), bank(N, K)
    code, f = ACTS[act]
    g = gen(M, act)
    bias, rs = torch.randn(N, generator=g).to(DEV), torch.rand(M, generator=g).to(DEV)
    y = O.row_values(x) @ O.weight_values(w)[0].T
    kw = dict(act=code, act_alpha=A, act_limit=B)
    assert O.rel(ops.linear(x, w, out_f32=True, **kw), f(y)) < tolerance(K)
    want = f(y + bias.cpu().double()) * rs.cpu().double()[:, None]
    assert O.rel(ops.linear(x, w, bias=bias, row_scale=rs, out_f32=True, **kw), want) < tolerance(K)
    assert O.rel(ops.linear(x, w, bias=bias, row_scale=rs, **kw), want) < tolerance(K, bf16=True)
    assert O.rel(ops.linear(x.cpu(), w.to("cpu"), out_f32=True, **kw), f(y)) < tolerance(K)      # (the CPU's form)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("T,E,k", [(1, 6, 2), (3, 20, 4), (40, 8, 3), (300, 4, 2)])
def test_experts_and_slots(T, E, k, act):
    H, F = 328, 225
    x, w = acts(T, H), bank(F, H, E)
    code, f = ACTS[act]
    kw = dict(act=code, act_alpha=A, act_limit=B, out_f32=True)
    idx = torch.randn(T, E, generator=gen(T, E)).topk(k, dim=1).indices.to(torch.int32)
    want = f(torch.einsum("pk,pnk->pn", O.row_values(x).repeat_interleave(k, 0), O.weight_values(w)[idx.reshape(-1).long()]))
    pk = ops.moe_pack(idx.to(DEV), E, tile=1)
    got = ops.expert_linear(x, w, pk, x_index=pk.packed_token, **kw)[pk.pair_to_packed.long()]
    assert O.rel(got, want) < tolerance(H)
    assert O.rel(ops.expert_gemv(x, w, idx.reshape(-1).to(DEV), x_div=k, **kw), want) < tolerance(H)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M", [1, 6, 20, 140])
def test_a_row_that_is_not_finite_stays_alone(M, act):
    x, w = acts(M, 512), bank(288, 512)
    kw = dict(act=ACTS[act][0], act_alpha=A, act_limit=B)
    clean = ops.linear(x, w, **kw)
    x[M // 2, 300] = float("nan")
    got = ops.linear(x, w, **kw)
    rows = torch.arange(M) != M // 2
    assert bool(got[M // 2].isnan().all()) and torch.equal(got[rows], clean[rows])
