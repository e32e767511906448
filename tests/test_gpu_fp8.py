"""Products of e4m3 weights (csrc/cuda/fp8_*.cu) against 64 bits (tests/fp8_oracle.py).

Bounds.  fp32 results: fp8_oracle.fp32_bound.  bf16 results: half a step, 2^-8 of the element, so 2^-8 of the norm beside the fp32 bound.  Gated activations: their
slope times the argument stays below 1 + |g| <= 8 times the value at these sizes, and the exponential adds 2^-21: eight fp32 bounds and 2^-20."""
import pytest
import torch

import fp8_oracle as O
from machx_inference_engine_b200 import ops
from machx_inference_engine_b200.ops import fp8
from machx_inference_engine_b200.ops.weights import WFormat, from_dense, from_fp8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ACTS = {"none": ops.ACT_NONE, "swiglu": ops.ACT_SWIGLU, "swiglu_oai": ops.ACT_SWIGLU_OAI, "geglu": ops.ACT_GEGLU, "relu2": ops.ACT_RELU2}


def gen(*key):
    return torch.Generator().manual_seed(hash(key) % (1 << 31))


def bank(N, K, E=1, seed=0):
    g = gen(N, K, E, seed)
    codes = (torch.randn(E, N, K, generator=g).clamp(-4, 4) * 112).to(torch.float8_e4m3fn)
    return from_fp8(codes, (0.5 + torch.rand(E, -(-N // 128), -(-K // 128), generator=g)) * (K ** -0.5 / 112)).to(DEV)


def acts(M, K, seed=0):
    g = gen(M, K, seed)
    return (torch.randn(M, K, generator=g) * torch.exp(torch.randn(K, generator=g))).to(DEV, torch.bfloat16)


def tolerance(K, act="none", bf16=False):
    t = O.fp32_bound(K)
    if act != "none":
        t = 8 * t + 2.0 ** -20
    return t + (2.0 ** -8 if bf16 else 0.0)


# ------------------------------------------------------------------ rounding of rows
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (5, 129), (1, 4096), (17, 2880), (130, 200), (1000, 640), (2, 16384), (70000, 8)])
def test_rows_are_rounded_as_defined(M, K, dtype):
    g = gen(M, K)
    x = (torch.randn(M, K, generator=g) * torch.exp(8 * torch.randn(M, 1, generator=g))).to(DEV, dtype)
    q = ops.fp8_rows(x)
    codes, scale = O.rows(x)
    assert q.shape == (M, K) and torch.equal(q.codes.cpu().float().double(), codes) and torch.equal(q.scale.cpu().double(), scale)
    same = fp8.round_rows(x.cpu())
    assert torch.equal(same.codes.view(torch.uint8), q.codes.cpu().view(torch.uint8)) and torch.equal(same.scale, q.scale.cpu())


def test_rows_of_odd_strides_and_through_an_index():
    wide = torch.randn(50, 1000, generator=gen(1)).to(DEV, torch.bfloat16)
    for lo, hi in ((0, 1000), (1, 400), (8, 520), (3, 131), (999, 1000)):
        x = wide[:, lo:hi]
        want = fp8.round_rows(x.cpu())
        got = ops.fp8_rows(x)
        assert torch.equal(got.codes.cpu().view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got.scale.cpu(), want.scale)
    index = torch.tensor([49, 0, 0, -1, 7, 50, 1 << 30, -5], dtype=torch.int32)
    want, got = fp8.round_rows(wide.cpu(), index), ops.fp8_rows(wide, index=index.to(DEV))
    assert torch.equal(got.codes.cpu().view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got.scale.cpu().isnan(), want.scale.isnan())
    assert bool(got.scale[:, 5:7].isnan().all()) and float(got.codes[3].float().abs().max()) == 0 and not bool(got.scale[:, :5].isnan().any())
    row = torch.randn(1, 256, device=DEV).to(torch.bfloat16).expand(9, 256)                # a stride of zero
    assert torch.equal(ops.fp8_rows(row).codes[8].view(torch.uint8), ops.fp8_rows(row[:1]).codes[0].view(torch.uint8))
    assert ops.fp8_rows(wide[:0]).codes.shape == (0, 1024) and ops.fp8_rows(wide, index=index[:0].to(DEV)).scale.shape == (8, 0)


def test_an_index_into_no_rows():
    none = torch.empty(0, 256, dtype=torch.bfloat16, device=DEV)
    q = ops.fp8_rows(none, index=torch.tensor([-1, 0, 5], dtype=torch.int32, device=DEV))
    assert q.scale.isnan().any(0).tolist() == [False, True, True] and float(q.codes.float().abs().max()) == 0


def test_rows_at_the_edges_of_the_range():
    inf, nan = float("inf"), float("nan")
    rows = [torch.zeros(256), torch.full((256,), 448.0), torch.full((256,), 449.0), torch.full((256,), 3e38), torch.full((256,), 1e-38), torch.full((256,), -1e-45),
            torch.cat([torch.tensor([inf]), torch.ones(255)]), torch.cat([torch.ones(255), torch.tensor([nan])]), torch.linspace(-2, 2, 256),
            torch.cat([torch.tensor([448 * 2.0 ** -100]), torch.full((255,), 2.0 ** -111)]), torch.cat([torch.tensor([1.0]), torch.full((255,), 2.0 ** -19)])]
    x = torch.stack(rows)
    q = ops.fp8_rows(x.to(DEV))
    codes, scale = O.rows(x)
    assert torch.equal(q.codes.cpu().float().double(), codes) and torch.equal(q.scale.cpu().isnan(), scale.isnan())
    assert torch.equal(q.scale.cpu().double()[~scale.isnan()], scale[~scale.isnan()])
    assert [bool(v.isnan().any()) for v in q.dequantize().cpu()] == [False] * 6 + [True, True] + [False] * 3


# ------------------------------------------------------------------ dense layers
SHAPES = [(16, 128), (1, 1), (96, 96), (257, 2880), (1000, 1024), (130, 200), (2049, 515), (32, 14336), (512, 16)]


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 257, 300])
@pytest.mark.parametrize("N,K", SHAPES)
def test_dense(M, N, K):
    x, w = acts(M, K), bank(N, K)
    want = O.row_values(x) @ O.weight_values(w)[0].T
    got = ops.linear(x, w, out_f32=True)
    assert got.dtype == torch.float32 and O.rel(got, want) < tolerance(K)
    half = ops.linear(x, w)
    assert half.dtype == torch.bfloat16 and O.rel(half, want) < tolerance(K, bf16=True)
    assert torch.equal(half, got.to(torch.bfloat16))                              # rounded once, at the end
    assert torch.equal(ops.linear(x, w, out_f32=True), got)                       # the order of the sums is fixed
    assert torch.equal(ops.linear(ops.fp8_rows(x), w, out_f32=True), got)         # rows that were rounded before


@pytest.mark.parametrize("M,N,K", [(700, 4096, 640), (1025, 1536, 256), (300, 9000, 384), (4096, 512, 128), (2300, 2304, 1000)])
def test_dense_over_many_tiles(M, N, K):
    x, w = acts(M, K), bank(N, K)
    want = O.row_values(x) @ O.weight_values(w)[0].T
    assert O.rel(ops.linear(x, w, out_f32=True), want) < tolerance(K)
    assert O.rel(ops.linear(x, w), want) < tolerance(K, bf16=True)


def K_():
    from machx_inference_engine_b200.ops import cuda
    return cuda


@pytest.mark.parametrize("M", [1, 15, 64, 128, 129, 300])
@pytest.mark.parametrize("N,K", [(1, 1), (257, 2880), (1000, 1024), (544, 515), (4096, 128)])
def test_each_kernel_at_every_tile_size(M, N, K):
    """The kernels that the dense layers choose between, at sizes that the choice would give to the other one too."""
    x, w = acts(M, K), bank(N, K)
    want = O.row_values(x) @ O.weight_values(w)[0].T
    bias, rs = torch.randn(N, generator=gen(1)).to(DEV), torch.rand(M, generator=gen(2)).to(DEV)
    full = (want + bias.cpu().double()) * rs.cpu().double()[:, None]
    q = ops.fp8_rows(x)
    for rows in (x, q):
        for nt in (n for n in K_().FP8_STREAM_ROWS if n >= M):
            out = torch.empty(M, N, device=DEV)
            assert O.rel(K_()._fp8_call(rows, w, out, None, None, 0, 0.0, 0.0, nt), want) < tolerance(K), nt
            assert O.rel(K_()._fp8_call(rows, w, out, bias, rs, 0, 0.0, 0.0, nt), full) < tolerance(K), nt
        for bn, cuts in ((128, 1), (256, 1), (128, 2), (256, 3), (128, 4), (256, 5)):
            if cuts > -(-K // 128):
                continue
            out = torch.empty(M, N, device=DEV)
            assert O.rel(K_()._fp8_call(rows, w, out, None, None, 0, 0.0, 0.0, 0, bn, cuts), want) < tolerance(K), (bn, cuts)
            assert O.rel(K_()._fp8_call(rows, w, out, bias, rs, 0, 0.0, 0.0, 0, bn, cuts), full) < tolerance(K), (bn, cuts)


@pytest.mark.parametrize("act", ["none", "geglu"])
@pytest.mark.parametrize("T,E,k", [(7, 4, 2), (200, 6, 2), (500, 3, 2), (90, 40, 5)])
def test_each_kernel_over_experts(T, E, k, act):
    H, F = 392, 320
    x, w = acts(T, H), bank(F, H, E)
    idx = routing(T, E, k, "skewed")
    pk = ops.moe_pack(idx.to(DEV), E, tile=1)
    want = O.activate(torch.einsum("pk,pnk->pn", O.row_values(x).repeat_interleave(k, 0), O.weight_values(w)[idx.reshape(-1).long()]), act)
    kw = dict(counts=pk.counts, seg=pk.seg_start)
    n = F // 2 if act != "none" else F
    for rows, index in ((x, pk.packed_token), (ops.fp8_rows(x, index=pk.packed_token), None)):
        for nt in K_().FP8_STREAM_ROWS:
            got = K_()._fp8_call(rows, w, torch.empty(T * k, n, device=DEV), None, None, ACTS[act], 1.702, 7.0, nt, index=index, **kw)
            assert O.rel(got[pk.pair_to_packed.long()], want) < tolerance(H, act), nt
        for bn in (128, 256):
            got = K_()._fp8_call(rows, w, torch.empty(T * k, n, device=DEV), None, None, ACTS[act], 1.702, 7.0, 0, bn, index=index, **kw)
            assert O.rel(got[pk.pair_to_packed.long()], want) < tolerance(H, act), bn


@pytest.mark.parametrize("act", ["swiglu", "swiglu_oai", "geglu", "relu2"])
@pytest.mark.parametrize("M", [1, 8, 19, 64, 130, 513])
def test_epilogues(M, act):
    N, K = 544, 1088
    x, w = acts(M, K), bank(N, K)
    g = gen(M, act)
    bias, rs = torch.randn(N, generator=g).to(DEV), torch.rand(M, generator=g).to(DEV)
    y = O.row_values(x) @ O.weight_values(w)[0].T
    for kw in (dict(), dict(bias=bias), dict(row_scale=rs), dict(bias=bias, row_scale=rs)):
        want = O.activate(y + (bias.cpu().double() if "bias" in kw else 0), act)
        if "row_scale" in kw:
            want = want * rs.cpu().double()[:, None]
        assert O.rel(ops.linear(x, w, act=ACTS[act], out_f32=True, **kw), want) < tolerance(K, act)
        assert O.rel(ops.linear(x, w, act=ACTS[act], **kw), want) < tolerance(K, act, bf16=True)


@pytest.mark.parametrize("M", [1, 5, 40, 150])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("lo,width", [(0, 100), (8, 120), (3, 131), (5, 100)])
def test_output_into_columns_of_a_wider_matrix(M, f32, lo, width):
    x, w = acts(M, 300), bank(100, 300)
    wide = torch.full((M + 1, lo + width), 7.0, dtype=torch.float32 if f32 else torch.bfloat16, device=DEV)
    out = wide[:M, lo:lo + 100]
    assert ops.linear(x, w, out=out, out_f32=f32) is out
    assert torch.equal(out, ops.linear(x, w, out_f32=f32))
    out.fill_(7.0)
    assert bool((wide == 7.0).all())


@pytest.mark.parametrize("M", [1, 3, 33, 200])
def test_rows_in_columns_of_a_wider_matrix(M):
    wide = acts(M, 900)
    w = bank(200, 333)
    for lo in (0, 1, 8, 567):
        assert torch.equal(ops.linear(wide[:, lo:lo + 333], w), ops.linear(wide[:, lo:lo + 333].contiguous(), w))


@pytest.mark.parametrize("M", [1, 6, 20, 70, 140, 300])
def test_a_row_that_is_not_finite_stays_alone(M):
    x, w = acts(M, 512), bank(288, 512)
    clean = ops.linear(x, w)
    bad = x.clone()
    bad[M // 2, 300] = float("inf")
    if M > 2:
        bad[0, 1] = float("nan")
    got = ops.linear(bad, w)
    rows = torch.zeros(M, dtype=torch.bool)
    rows[M // 2] = True
    rows[0] |= M > 2
    assert bool(got[rows].isnan().all()) and torch.equal(got[~rows], clean[~rows])
    assert float(ops.linear(torch.zeros_like(x), w).abs().max()) == 0
    for act in ("swiglu", "swiglu_oai", "geglu", "relu2"):
        got = ops.linear(bad, w, act=ACTS[act])
        assert bool(got[rows].isnan().all()) and not bool(got[~rows].isnan().any()), act


def test_scales_of_any_size():
    g = gen(9)
    codes = (torch.randn(1, 256, 512, generator=g).clamp(-4, 4) * 112).to(torch.float8_e4m3fn)
    t = torch.tensor([[1e-9, 1e4, -3.0, 0.0], [1e-20, 1.0, 1e10, 7.0]])[None]
    w = from_fp8(codes, t).to(DEV)
    for M in (2, 20, 150):
        x = (torch.randn(M, 512, generator=g) * 10.0 ** torch.randint(-12, 12, (M, 4), generator=g).repeat_interleave(128, dim=1)).to(DEV, torch.bfloat16)
        got, want = ops.linear(x, w, out_f32=True), O.row_values(x) @ O.weight_values(w)[0].T
        # (blocks of very different size: one of them is a row's result, and each is held to its own bound)
        assert float(((got.cpu().double() - want).abs().amax(1) / want.abs().amax(1)).max()) < 16 * tolerance(512)


def test_any_row_count_gives_close_values():
    """A row's result does not depend on the rows beside it by more than the order of its sums."""
    x, w = acts(300, 1024), bank(640, 1024)
    whole = ops.linear(x, w, out_f32=True)
    for M in (1, 8, 40, 128):
        assert O.rel(ops.linear(x[:M], w, out_f32=True), whole[:M]) < 2 * tolerance(1024)


# ------------------------------------------------------------------ experts
def routing(T, E, k, kind):
    g = gen(T, E, k, kind)
    if kind == "one":                                        # every token takes the same experts
        return torch.arange(k, dtype=torch.int32).add(E - k).repeat(T, 1)
    logits = torch.randn(T, E, generator=g) + (torch.linspace(0, 6, E) if kind == "skewed" else 0.0)
    return logits.topk(k, dim=1).indices.to(torch.int32)


@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("kind", ["even", "skewed", "one"])
@pytest.mark.parametrize("T,E,k", [(1, 4, 2), (9, 16, 2), (40, 8, 3), (64, 128, 8), (300, 5, 3), (700, 3, 1), (33, 300, 8), (260, 4, 4)])
def test_experts(T, E, k, kind, act):
    H, F = 328, 224
    x, w = acts(T, H), bank(F, H, E)
    idx = routing(T, E, k, kind)
    pk = ops.moe_pack(idx.to(DEV), E, tile=1)
    bias = torch.randn(E, F, generator=gen(E)).to(DEV)
    at, e = pk.pair_to_packed.cpu().long(), idx.reshape(-1).long()
    y = torch.einsum("pk,pnk->pn", O.row_values(x).repeat_interleave(k, 0), O.weight_values(w)[e]) + bias.cpu().double()[e]
    want = O.activate(y, act)
    got = ops.expert_linear(x, w, pk, x_index=pk.packed_token, bias=bias, act=ACTS[act], out_f32=True)
    assert got.shape[0] == T * k and O.rel(got.cpu()[at], want) < tolerance(H, act)
    packed = x[pk.packed_token.long()]
    for rows in (packed, ops.fp8_rows(packed), ops.fp8_rows(x, index=pk.packed_token)):
        assert torch.equal(ops.expert_linear(rows, w, pk, bias=bias, act=ACTS[act], out_f32=True), got)
    assert torch.equal(ops.expert_linear(x, w, pk, x_index=pk.packed_token, bias=bias, act=ACTS[act]), got.to(torch.bfloat16))


@pytest.mark.parametrize("T,E,k,lo,hi", [(50, 8, 2, 2, 5), (50, 8, 2, 0, 1), (50, 8, 2, 7, 8), (3, 8, 1, 4, 8)])
def test_a_share_of_the_experts(T, E, k, lo, hi):
    x, w = acts(T, 256), bank(96, 256, E)
    idx = routing(T, E, k, "even").to(DEV)
    full = ops.moe_pack(idx, E, tile=1)
    whole = ops.expert_linear(x, w, full, x_index=full.packed_token)[full.pair_to_packed.long()]
    pk = ops.moe_pack(idx, E, lo, hi, tile=1)
    got = ops.expert_linear(x, w.slice_experts(lo, hi), pk, x_index=pk.packed_token, e_lo=lo)
    p = pk.pair_to_packed.long()
    assert int((p >= 0).sum()) == int(((idx >= lo) & (idx < hi)).sum())
    assert O.rel(got[p[p >= 0]], whole[p >= 0]) < 2.0 ** -7 if bool((p >= 0).any()) else True


def test_wide_experts_over_many_tiles():
    T, E, k, H, F = 900, 6, 2, 512, 1600
    x, w = acts(T, H), bank(F, H, E)
    idx = routing(T, E, k, "skewed")
    pk = ops.moe_pack(idx.to(DEV), E, tile=1)
    y = torch.einsum("pk,pnk->pn", O.row_values(x).repeat_interleave(k, 0).float(), O.weight_values(w).float()[idx.reshape(-1).long()])
    got = ops.expert_linear(x, w, pk, x_index=pk.packed_token)
    assert O.rel(got[pk.pair_to_packed.long()], y) < tolerance(H, bf16=True)


@pytest.mark.parametrize("act", ["none", "swiglu_oai"])
@pytest.mark.parametrize("T,k,shared", [(1, 1, True), (1, 10, True), (3, 4, True), (5, 2, False), (8, 8, True), (8, 8, False), (40, 3, True)])
@pytest.mark.parametrize("N,K", [(96, 200), (1024, 2048), (64, 1)])
def test_slots(T, k, shared, act, N, K):
    E = 20
    w = bank(N, K, E)
    slot = torch.randint(0, E, (T * k,), generator=gen(T, k), dtype=torch.int32)
    x = acts(T if shared else T * k, K)
    bias, scale = torch.randn(E, N, generator=gen(2)).to(DEV), torch.rand(T * k, generator=gen(3)).to(DEV)
    xv = O.row_values(x).repeat_interleave(k if shared else 1, 0)
    y = torch.einsum("pk,pnk->pn", xv, O.weight_values(w)[slot.long()])
    div = k if shared else 1
    got = ops.expert_gemv(x, w, slot.to(DEV), x_div=div, act=ACTS[act], out_f32=True)
    assert O.rel(got, O.activate(y, act)) < tolerance(K, act)
    want = O.activate(y + bias.cpu().double()[slot.long()], act) * scale.cpu().double()[:, None]
    assert O.rel(ops.expert_gemv(x, w, slot.to(DEV), x_div=div, act=ACTS[act], bias=bias, slot_scale=scale), want) < tolerance(K, act, bf16=True)
    assert torch.equal(ops.expert_gemv(ops.fp8_rows(x), w, slot.to(DEV), x_div=div, act=ACTS[act], out_f32=True), got)


def test_slots_of_experts_elsewhere_are_zero():
    w, x = bank(64, 256, 3), acts(6, 256)
    slot = torch.tensor([4, 5, 6, 3, 7, -1], dtype=torch.int32, device=DEV)
    got = ops.expert_gemv(x, w, slot, bias=torch.ones(3, 64, device=DEV), e_lo=4)
    alone = ops.expert_gemv(x[:3], w, slot[:3] - 4, bias=torch.ones(3, 64, device=DEV))
    assert torch.equal(got[:3], alone) and float(got[3:].abs().max()) == 0


def test_no_tokens_and_no_rows():
    w, bank3 = bank(64, 256), bank(64, 256, 3)
    none = torch.empty(0, 256, dtype=torch.bfloat16, device=DEV)
    assert ops.linear(none, w).shape == (0, 64) and ops.linear(ops.fp8_rows(none), w, act=ops.ACT_SWIGLU).shape == (0, 32)
    assert ops.expert_gemv(none, bank3, torch.empty(0, dtype=torch.int32, device=DEV), x_div=2).shape == (0, 64)
    # experts without a token, and a packing whose tokens are all elsewhere
    idx = torch.tensor([[2], [2], [2]], dtype=torch.int32, device=DEV)
    pk = ops.moe_pack(idx, 3, 0, 2, tile=1)
    assert int((pk.pair_to_packed >= 0).sum()) == 0
    ops.expert_linear(acts(3, 256), bank3.slice_experts(0, 2), pk, x_index=pk.packed_token)
    torch.cuda.synchronize()


# ------------------------------------------------------------------ streams and graphs
def test_a_stream_of_its_own_and_captured_twice():
    """Graphs that were captured one after the other and replayed at once; another stream than the tensors' own; the same row many times."""
    x, w = acts(5, 2048), bank(4096, 2048)
    want = ops.linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.linear(x, w), want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            a = ops.linear(x, w)
            b = ops.linear(x[:1].expand(40, 2048), w)
        x.copy_(x.flip(0))
        g.replay()
    side.synchronize()
    assert torch.equal(a, want.flip(0)) and torch.equal(b, ops.linear(x[:1].expand(40, 2048).contiguous(), w))


def test_two_streams_and_a_graph_share_nothing():
    cases = [(1, 6144, 1024), (12, 1024, 4096), (70, 640, 2048), (300, 1024, 512)]
    xs, ws = [acts(M, K) for M, N, K in cases], [bank(N, K) for M, N, K in cases]
    eb, ex = bank(128, 512, 16), acts(30, 512)
    idx = routing(30, 16, 4, "even").to(DEV)

    def all_of_them():
        pk = ops.moe_pack(idx, 16, tile=1)
        return [ops.linear(x, w) for x, w in zip(xs, ws)] + [ops.expert_linear(ex, eb, pk, x_index=pk.packed_token), ops.expert_gemv(ex, eb, idx.reshape(-1), x_div=4)]

    want = all_of_them()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    got = []
    for g in graphs:
        with torch.cuda.graph(g):
            got.append(all_of_them())
    side = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for s, g in zip(side, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(side[0]):
            other = all_of_them()
    torch.cuda.synchronize()
    for r in got + [other]:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_threads_on_one_stream_do_not_share_rounded_rows():
    """Calls of several threads on the same stream: launches of one may come between the two of another."""
    import threading
    cases = [(12, 512, 640), (40, 512, 640), (200, 256, 640), (12, 512, 640)]
    xs, ws = [acts(M, K, seed=i) for i, (M, N, K) in enumerate(cases)], [bank(N, K, seed=i) for i, (M, N, K) in enumerate(cases)]
    want = [ops.linear(x, w) for x, w in zip(xs, ws)]
    wrong = []

    def run(i):
        for _ in range(150):
            if not torch.equal(ops.linear(xs[i], ws[i]), want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_layer_of_experts_from_router_to_sum():
    """Route, pack, gate / up, down and sum as a model runs them, against the same steps on the CPU.  The hidden rows are rounded to bf16 and then to e4m3 in
    both; where the two differ by a bf16 step (2^-8) a code may differ by one e4m3 step, 2^-3 of the value.  A hidden value sits so near a border with a
    chance of about its own error over the e4m3 step, 2^-15 / 2^-4: with bf16 borders between, the norm moves by less than 2^-8."""
    T, E, k, H, F = 50, 12, 3, 256, 128
    x, gu, dn = acts(T, H), bank(2 * F, H, E), bank(H, F, E, 1)
    logits = torch.randn(T, E, generator=gen(5))

    def layer(dev):
        idx, wt = ops.moe_route(logits.to(dev), None, k)
        pk = ops.moe_pack(idx, E, tile=1)
        a = ops.expert_linear(x.to(dev), gu.to(dev), pk, x_index=pk.packed_token, act=ops.ACT_SWIGLU)
        return ops.moe_combine(ops.expert_linear(a, dn.to(dev), pk), pk, wt)

    assert O.rel(layer(DEV), layer("cpu")) < 2.0 ** -8 + 2.0 ** -8


# ------------------------------------------------------------------ few rows of small layers: blocks of K shared by clusters
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("N,K", [(64, 1160), (32, 9000), (1024, 8192), (2080, 2944), (4096, 4096), (8192, 4096), (8224, 4096), (640, 14336), (50, 1025), (30000, 256), (10016, 2048), (5120, 2880), (20000, 100)])
def test_few_rows(rows, N, K):
    x, w, bias, scale = acts(rows, K), bank(N, K), torch.randn(N, generator=gen(N)).to(DEV), torch.rand(rows, generator=gen(rows)).to(DEV)
    y = O.row_values(x) @ O.weight_values(w)[0].T
    got = ops.linear(x, w, out_f32=True)
    assert O.rel(got, y) < tolerance(K)
    want = torch.relu(y + bias.cpu().double()) ** 2 * scale.cpu().double()[:, None]
    assert O.rel(ops.linear(x, w, bias=bias, act=ACTS["relu2"], row_scale=scale, out_f32=True), want) < tolerance(K, "relu2")
    if N % 32 == 0:
        assert O.rel(ops.linear(x, w, act=ACTS["swiglu"], out_f32=True), O.activate(y, "swiglu")) < tolerance(K, "swiglu")
    wide = torch.full((rows, K + 3), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 1:K + 1] = x                                                           # rows of odd alignment are rounded by a launch before
    assert torch.equal(ops.linear(wide[:, 1:K + 1], w, out_f32=True), got) and torch.equal(ops.linear(ops.fp8_rows(x), w, out_f32=True), got)
    out = torch.full((rows, N + 5), 7.0, device=DEV)
    ops.linear(x, w, out_f32=True, out=out[:, 2:N + 2])
    assert torch.equal(out[:, 2:N + 2], got) and bool((out[:, :2] == 7).all()) and bool((out[:, N + 2:] == 7).all())


@pytest.mark.parametrize("N,K", [(96, 1160), (1024, 8192)])
def test_few_rows_with_nan_and_infinity(N, K):
    x, w = acts(4, K), bank(N, K)
    clean = ops.linear(x, w, out_f32=True)
    x[1, K - 1], x[3, 5] = float("nan"), float("inf")
    got = ops.linear(x, w, out_f32=True)
    assert torch.equal(got[[0, 2]], clean[[0, 2]]) and bool(got[[1, 3]].isnan().all())


def test_a_chain_of_few_rows_replays_like_eager_calls():
    """Each launch starts before the one before has ended; what it reads of that one it reads after it."""
    ws = [bank(4096, 1024, seed=1), bank(512, 4096, seed=2), bank(640, 512, seed=3), bank(1024, 640, seed=4)]
    x = acts(3, 1024)

    def chain():
        h = x
        for w in ws:
            h = ops.linear(h, w)
        return h

    want = chain()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = chain()
        for _ in range(20):
            got.zero_()
            g.replay()
            assert torch.equal(got, want)
        x.copy_(x.flip(0))
        g.replay()
    side.synchronize()
    assert torch.equal(got, want.flip(0))
