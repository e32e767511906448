"""Products in 8-bit floating point: weights in e4m3 with a scale for each block (``WFormat.FP8``), activations rounded to e4m3 as they are read.

A row of activations is cut into blocks of 128 along K, the last one filled with zeros.  With a = max |x| of a block, its scale is the smallest power of two,
2^-100 at least, for which a <= 448 scale (1 where the block is zero), and its codes are x / scale rounded to nearest e4m3.  A power of two makes the division
exact, so the codes are the same on every path, and costs a floating-point format no precision.  The floor of 2^-100 keeps the product of a row's and a
weight's scale a normal number; blocks below 448 x 2^-100 lose their smallest values to it.  A block that holds an infinity or a NaN gets the scale NaN and codes of
zero: every output of that row is NaN, the other rows are untouched.  The product is

    y[m, n] = sum over blocks b of  scale[b, m] * wscale[n, b] * (sum over k in b of  code[m, k] * wcode[n, k])

with sums, scales and the epilogue (bias, activation, row scale) in 32 bits, rounded once to the output's type.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .weights import FP8_BLOCK, QuantWeight, WFormat


@dataclass
class FP8Rows:
    """Rows rounded by :func:`ops.fp8_rows`, which the products of FP8 weights take in the place of bf16 rows (several projections then share one rounding)."""
    codes: torch.Tensor       # float8_e4m3fn [rows, KB * 128], zeros past K
    scale: torch.Tensor       # fp32 [KB, rows]
    K: int

    @property
    def shape(self) -> tuple:
        return (self.codes.shape[0], self.K)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self) -> torch.Tensor:
        """fp32 [rows, K]; a block with the scale NaN is NaN throughout."""
        t = self.scale.t().repeat_interleave(FP8_BLOCK, dim=1)
        return (self.codes.to(torch.float32) * t)[:, :self.K].contiguous()


def check_rows(x, index=None) -> None:
    """Arguments of :func:`ops.fp8_rows`."""
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float32) or x.shape[1] < 1:
        raise ValueError(f"rows to round are bf16 or fp32 [rows, K], not {x.dtype} {list(x.shape)}")
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError("rows to round need a unit stride along K")
    if index is not None and (index.dtype != torch.int32 or index.dim() != 1 or not index.is_contiguous() or index.device != x.device):
        raise ValueError("an index of rows is a contiguous int32 vector on the rows' device")


def check_product(x, w: QuantWeight, experts: bool, rows: int, bias, act_gated: bool, what: str) -> None:
    """Arguments that the products of FP8 weights share: ``x`` bf16 rows or :class:`FP8Rows`, ``bias`` [N] ([E,N] where ``experts``) of ``rows`` output rows."""
    if w.fmt != WFormat.FP8:
        raise ValueError(f"{what}: FP8 weights are wanted, not {w.fmt.name}")
    if not experts and w.E != 1:
        raise ValueError(f"{what}: one matrix is wanted, not a bank of {w.E}")
    if isinstance(x, FP8Rows):
        kb = -(-x.K // FP8_BLOCK)
        n = x.codes.shape[0]
        if x.codes.dtype != torch.float8_e4m3fn or x.codes.shape != (n, kb * FP8_BLOCK) or not x.codes.is_contiguous() or x.scale.dtype != torch.float32 \
                or x.scale.shape != (kb, n) or not x.scale.is_contiguous() or x.scale.device != x.codes.device:
            raise ValueError(f"{what}: the rounded rows are not as ops.fp8_rows makes them")
        K, dev = x.K, x.codes.get_device()
    else:
        if x.dtype != torch.bfloat16:
            raise ValueError(f"{what}: FP8 weights take bf16 rows or FP8Rows, not {x.dtype}")
        if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
            raise ValueError(f"{what}: rows [rows, K] with a unit stride along K are wanted, not {list(x.shape)} with strides {x.stride()}")
        K, dev = x.shape[1], x.get_device()
    if K != w.K:
        raise ValueError(f"{what}: rows of {K} elements, a weight of {w.K}")
    if dev != w.p0.get_device():
        raise ValueError(f"{what}: rows on {x.device}, the weight on {w.device}")
    if act_gated and w.N % 32:
        raise ValueError(f"{what}: a gated activation takes runs of 16 gate and 16 up rows, not {w.N} rows")
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != ((w.E, w.N) if experts else (w.N,)) or not bias.is_contiguous() or bias.device != x.device):
        raise ValueError(f"{what}: the bias is a contiguous fp32 {[w.E, w.N] if experts else [w.N]} on the rows' device")
    if rows >= 1 << 31 or w.N >= 1 << 30 or w.K >= 1 << 30 or w.E >= 1 << 16:
        raise ValueError(f"{what}: too large")


def check_out(out, row_scale, rows: int, n_out: int, dtype, device) -> None:
    """``out`` and ``row_scale`` of :func:`ops.linear`."""
    if out is not None and (tuple(out.shape) != (rows, n_out) or out.dtype != dtype or out.device != device or (n_out > 1 and out.stride(1) != 1)
                            or (rows > 1 and out.stride(0) < n_out)):
        raise ValueError(f"linear: the output is {dtype} [{rows}, {n_out}] with a unit column stride on the rows' device")
    if row_scale is not None and (row_scale.dtype != torch.float32 or row_scale.numel() != rows or not row_scale.is_contiguous() or row_scale.device != device):
        raise ValueError(f"linear: the row scale is a contiguous fp32 vector of {rows} on the rows' device")


def check_packing(pk, w: QuantWeight, x, x_index, e_lo: int) -> None:
    """A compact packing (``moe_pack(..., tile=1)``) for :func:`ops.expert_linear`."""
    if pk.counts is None or pk.seg_start is None or pk.max_rows != max(pk.pair_to_packed.numel(), 1):
        raise ValueError("expert_linear takes a compact packing: moe_pack(..., tile=1)")
    E = pk.counts.numel()
    if w.E > 1024:
        raise ValueError(f"expert_linear: a bank of {w.E} experts; 1024 are taken")
    if pk.seg_start.numel() != E + 1 or e_lo < 0 or e_lo + w.E > E:
        raise ValueError(f"expert_linear: experts {e_lo} to {e_lo + w.E} of a packing of {E}")
    for t, n in ((pk.counts, E), (pk.seg_start, E + 1)):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.device != x.device:
            raise ValueError("expert_linear: the packing's tables are contiguous int32 on the rows' device")
    if x_index is None:
        if x.shape[0] < pk.pair_to_packed.numel():
            raise ValueError(f"expert_linear: {x.shape[0]} rows for a packing of {pk.pair_to_packed.numel()}")
    elif x_index.dtype != torch.int32 or x_index.numel() < pk.max_rows or not x_index.is_contiguous() or x_index.device != x.device:
        raise ValueError("expert_linear: x_index is a contiguous int32 vector with an entry for every packed row")
    elif x.shape[0] == 0 and pk.pair_to_packed.numel():
        raise ValueError(f"expert_linear: no rows for a packing of {pk.pair_to_packed.numel()}")
    if x_index is not None and isinstance(x, FP8Rows):
        raise ValueError("expert_linear: rounded rows come in packed order; fp8_rows(x, index=...) puts them there")


def check_slots(x, w: QuantWeight, slot_expert, x_div: int, bias, act_gated: bool, slot_scale) -> None:
    """Arguments of :func:`ops.expert_gemv` with an FP8 bank."""
    S = slot_expert.numel()
    check_product(x, w, True, S, bias, act_gated, "expert_gemv")
    if S >= 1 << 16:
        raise ValueError(f"expert_gemv: {S} slots; expert_linear takes that many rows")
    if slot_expert.dtype != torch.int32 or not slot_expert.is_contiguous() or slot_expert.device != x.device:
        raise ValueError("expert_gemv: the slots' experts are contiguous int32 on the rows' device")
    if x_div < 1 or x.shape[0] < -(-S // x_div):
        raise ValueError(f"expert_gemv: {S} slots of {x_div} a row, but {x.shape[0]} rows")
    if slot_scale is not None and (slot_scale.dtype != torch.float32 or slot_scale.numel() != S or not slot_scale.is_contiguous() or slot_scale.device != x.device):
        raise ValueError("expert_gemv: the slots' scales are contiguous fp32 on the rows' device")


def round_rows(x: torch.Tensor, index=None) -> FP8Rows:
    """The rounding in PyTorch (see the module's text)."""
    check_rows(x, index)
    K = x.shape[1]
    kb = -(-K // FP8_BLOCK)
    bad = None
    if index is not None:
        i = index.long()
        v = torch.zeros(i.numel(), K, dtype=torch.float32, device=x.device)
        inside = (i >= 0) & (i < x.shape[0])
        v[inside] = x.to(torch.float32)[i[inside]]
        bad = i >= x.shape[0]
    else:
        v = x.to(torch.float32)
    v = torch.nn.functional.pad(v, (0, kb * FP8_BLOCK - K)).view(-1, kb, FP8_BLOCK)
    top = v.abs().amax(dim=-1)
    ok = torch.isfinite(top)
    if bad is not None:
        ok = ok & ~bad[:, None]
    m, e = torch.frexp(torch.where(ok, top, torch.zeros_like(top)))
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-100)                     # 448 = 0.875 * 2^9
    e = torch.where(ok & (top > 0), e, torch.zeros_like(e))
    scale = ((e.to(torch.int32) + 127) << 23).view(torch.float32)
    codes = (torch.where(ok[..., None], v, torch.zeros_like(v)) / scale[..., None]).to(torch.float8_e4m3fn)
    scale = torch.where(ok, scale, torch.full_like(scale, float("nan")))
    return FP8Rows(codes.reshape(-1, kb * FP8_BLOCK), scale.t().contiguous(), K)


def values(x) -> torch.Tensor:
    """fp32 values that a product sees of ``x`` (rows or :class:`FP8Rows`)."""
    return (x if isinstance(x, FP8Rows) else round_rows(x)).dequantize()
