"""The 8-bit products in 64 bits, from their definition: rounding to e4m3 by steps of eight per octave, scales by doubling, products as plain sums."""
import math

import torch


def e4m3(z: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value, ties to the even code; |z| <= 448."""
    unit = torch.full_like(z, 2.0 ** -9)
    for _ in range(15):
        unit = torch.where(z.abs() >= 16 * unit, 2 * unit, unit)
    return torch.round(z / unit) * unit


def rows(x: torch.Tensor):
    """(code values [rows, KB * 128], scales [KB, rows]) in fp64."""
    n, k = x.shape
    kb = -(-k // 128)
    v = torch.zeros(n, kb * 128, dtype=torch.float64)
    v[:, :k] = x.double().cpu()
    v = v.view(n, kb, 128)
    a = v.abs().amax(dim=2)
    bad = ~torch.isfinite(a)
    s = torch.full_like(a, 2.0 ** -100)
    for _ in range(230):
        s = torch.where((a > 448.0 * s) & ~bad, 2.0 * s, s)
    s = torch.where(a == 0, torch.ones_like(s), s)
    q = e4m3(torch.where(bad[..., None], torch.zeros_like(v), v) / s[..., None])
    return q.view(n, kb * 128), torch.where(bad, torch.full_like(s, math.nan), s).t()


def row_values(x: torch.Tensor) -> torch.Tensor:
    q, s = rows(x)
    return (q * s.t().repeat_interleave(128, dim=1))[:, :x.shape[1]]


def weight_values(w) -> torch.Tensor:
    """[E, N, K] fp64 of a runtime weight's planes."""
    t = w.p1.double().cpu().repeat_interleave(16, dim=1)[:, :w.N].repeat_interleave(128, dim=2)
    return (w.p0.cpu().float().double() * t)[..., :w.K]


def activate(y: torch.Tensor, act: str) -> torch.Tensor:
    if act == "none":
        return y
    if act == "relu2":
        return y.clamp_min(0) ** 2
    v = y.reshape(*y.shape[:-1], y.shape[-1] // 32, 2, 16)
    g, u = v[..., 0, :], v[..., 1, :]
    if act == "swiglu":
        r = g * torch.sigmoid(g) * u
    elif act == "swiglu_oai":
        g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
        r = g * torch.sigmoid(1.702 * g) * (u + 1)
    else:
        r = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
    return r.reshape(*y.shape[:-1], -1)


def fp32_bound(k: int) -> float:
    """Relative to the result's norm: within a block of 128 the tensor cores add four sums of 32 products and may cut each at 2^-23 of the running sum; the KB
    block sums are joined by fused multiply-adds, half a step (2^-24) of the running sum each; the bias one more.  Block sums of random terms have the
    result's norm together, and no running sum's is larger."""
    kb = -(-k // 128)
    return 4 * 2.0 ** -23 + (kb + 2) * 2.0 ** -24


def rel(a, b) -> float:
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / b.norm())
