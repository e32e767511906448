"""FP8 products over packings: which kernel a share of a bank takes, packings without a pair, rows that are not there."""
import zlib

import pytest
import torch

import fp8_oracle as O
from machx_inference_engine_b200 import ops
from machx_inference_engine_b200.ops.weights import from_fp8

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


def bank(N, K, E, dev):
    g = gen(N, K, E)
    codes = (torch.randn(E, N, K, generator=g).clamp(-4, 4) * 112).to(torch.float8_e4m3fn)
    return from_fp8(codes, (0.5 + torch.rand(E, -(-N // 128), -(-K // 128), generator=g)) * (K ** -0.5 / 112)).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k", [(4, 64, 4), (64, 128, 8), (48, 32, 4), (300, 16, 4)])
def test_a_share_of_a_bank_takes_the_kernel_of_the_whole_one(monkeypatch, T, E, k):
    """The rule asks for the rows of an expert on average: a rank that holds some of the experts has the same."""
    from machx_inference_engine_b200.ops import cuda as K
    plans, call = [], K._fp8_call
    monkeypatch.setattr(K, "_fp8_call", lambda *a, **kw: (plans.append(a[8:11]), call(*a, **kw))[1])
    x, w = torch.randn(T, 128, generator=gen(T)).to("cuda:0", torch.bfloat16), bank(64, 128, E, "cuda:0")
    idx = torch.randn(T, E, generator=gen(T, E)).topk(k, dim=1).indices.to("cuda:0", torch.int32)
    full = ops.moe_pack(idx, E, tile=1)
    whole = ops.expert_linear(x, w, full, x_index=full.packed_token)[full.pair_to_packed.long()]
    for parts in (2, 8):
        n = E // parts
        for lo in (0, E - n):
            pk = ops.moe_pack(idx, E, lo, lo + n, tile=1)
            got = ops.expert_linear(x, w.slice_experts(lo, lo + n), pk, x_index=pk.packed_token, e_lo=lo)
            p = pk.pair_to_packed.long()
            assert torch.equal(got[p[p >= 0]], whole[p >= 0])            # (one kernel; a single block of K is never cut)
    assert len(set(plans)) == 1


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("indexed", [False, True])
def test_a_packing_without_a_pair(dev, indexed):
    """One row, which lies behind the last expert's and is nobody's."""
    w = bank(96, 256, 3, dev)
    none = torch.empty(0, 256, dtype=torch.bfloat16, device=dev)
    pk = ops.moe_pack(torch.empty(0, 2, dtype=torch.int32, device=dev), 3, tile=1)
    assert pk.max_rows == 1 and pk.pair_to_packed.numel() == 0
    kw = dict(x_index=pk.packed_token) if indexed else {}
    some = torch.ones(5, 256, dtype=torch.bfloat16, device=dev)
    for x in (none, some) if indexed else (none, some, ops.fp8_rows(none)):
        assert ops.expert_linear(x, w, pk, **kw).shape == (1, 96)
        assert ops.expert_linear(x, w, pk, bias=torch.zeros(3, 96, device=dev), act=ops.ACT_SWIGLU, out_f32=True, **kw).shape == (1, 48)
    if dev != "cpu":
        torch.cuda.synchronize()


@pytest.mark.parametrize("dev", DEVICES)
def test_no_rows_for_pairs_are_refused(dev):
    w = bank(96, 256, 3, dev)
    pk = ops.moe_pack(torch.zeros(4, 2, dtype=torch.int32, device=dev), 3, tile=1)
    none = torch.empty(0, 256, dtype=torch.bfloat16, device=dev)
    for kw in (dict(), dict(x_index=pk.packed_token)):
        with pytest.raises(ValueError):
            ops.expert_linear(none, w, pk, **kw)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("S,N", [(6, 64), (700, 96)])
def test_slots_of_more_experts_than_a_packing_takes(S, N, dev):
    """A packing's tables end at 1024 experts; a slot names its expert itself, in the few-row kernel and in the streaming one."""
    E, K = 1100, 256
    w, x = bank(N, K, E, dev), torch.randn(S, K, generator=gen(S)).to(dev, torch.bfloat16)
    slot = torch.randint(0, E, (S,), generator=gen(S, 1), dtype=torch.int32)
    slot[:2] = torch.tensor([E - 1, 1024], dtype=torch.int32)
    want = torch.einsum("pk,pnk->pn", O.row_values(x), O.weight_values(w)[slot.long()])
    assert O.rel(ops.expert_gemv(x, w, slot.to(dev), out_f32=True), want) < O.fp32_bound(K) + 2.0 ** -22      # (2^-22: the CPU's sums in another order)
    pk = ops.MoePacking(torch.zeros(E, dtype=torch.int32, device=dev), torch.zeros(E + 1, dtype=torch.int32, device=dev), torch.zeros(S, dtype=torch.int32, device=dev),
                        torch.zeros(S, dtype=torch.int32, device=dev), None, None, S, 1)
    with pytest.raises(ValueError):
        ops.expert_linear(x, w, pk)
