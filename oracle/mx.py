"""CPU restatement of microscaled rows and the operators on them, in float64.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). The format is OCP microscaling: blocks of
32 values share the scale ``2^e``, ``e = floor(log2 max|v|) - emax`` (8 for e4m3, 2 for e2m1),
not below -127; an element is ``v / 2^e`` to the nearest value of its grid, ties to even,
saturated. A block with an infinity or a NaN is NaN. Grids are listed value by value and an
element found by distance, so that nothing here shares the kernels' bit arithmetic.
"""

from __future__ import annotations

import torch

BLOCK, PAD = 32, 128
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]


def _nearest(a: torch.Tensor, grid: list[float]) -> torch.Tensor:
    """The index of the grid value nearest to ``a >= 0``, the even one of two."""
    g = torch.tensor(grid, dtype=torch.float64)
    hi = torch.searchsorted(g, a.clamp(max=grid[-1])).clamp(1, len(grid) - 1)
    lo = hi - 1
    below, above = a - g[lo], g[hi] - a
    return torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def quantize(v: torch.Tensor, bits: int) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` uint8 of ``v (rows, cols)``: codes one per value ``(rows, pad)`` (not
    packed), scales ``(rows, pad / 32)``."""
    rows, cols = v.shape
    pad = -(-cols // PAD) * PAD
    x = torch.zeros(rows, pad, dtype=torch.float64)
    x[:, :cols] = v.double()
    x = x.view(rows, -1, BLOCK)
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], 0.0, x)
    top = x.abs().amax(-1)
    e = torch.full(top.shape, -127.0, dtype=torch.float64)
    some = top > 0
    e[some] = torch.frexp(top[some]).exponent.double() - 1 - (8 if bits == 8 else 2)
    e = e.clamp(min=-127)
    code = _nearest(x.abs() / 2.0 ** e[..., None], E4M3 if bits == 8 else E2M1)
    code = code + torch.signbit(x) * (128 if bits == 8 else 8)
    scales = torch.where(bad, 255.0, e + 127)
    return code.view(rows, pad).to(torch.uint8), scales.to(torch.uint8)


def unpack(codes: torch.Tensor, bits: int) -> torch.Tensor:
    """One code per value from the packed bytes."""
    if bits == 8:
        return codes
    return torch.stack([codes % 16, codes // 16], -1).reshape(codes.shape[0], -1)


def values(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    """Unpacked codes and scales as float64 ``(rows, pad)``."""
    grid = torch.tensor(E4M3 + [float("nan")] if bits == 8 else E2M1, dtype=torch.float64)
    half = 128 if bits == 8 else 8
    c = codes.long()
    y = torch.where(c >= half, -grid[c % half], grid[c % half])
    s = torch.where(scales == 255, float("nan"), 2.0 ** (scales.double() - 127))
    return (y.view(y.shape[0], -1, BLOCK) * s[..., None]).view(y.shape)


def gelu(x: torch.Tensor) -> torch.Tensor:
    x = x.double()
    return 0.5 * x * torch.special.erfc(-x / 2.0 ** 0.5)


def swiglu(x: torch.Tensor) -> torch.Tensor:
    gate, up = x.double().chunk(2, dim=-1)
    return gate * torch.sigmoid(gate) * up


def rms_norm(x, residual, weight, eps):
    """``(s, s * rsqrt(mean(s^2) + eps) * weight)`` with ``s = x + residual``."""
    s = x.double() if residual is None else x.double() + residual.double()
    return s, s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * weight.double()


def adaln(x, y, gate, scale, shift, eps):
    """``(s, LN(s) * (1 + scale) + shift)`` with ``s = x + gate * y``."""
    s = x.double() if y is None else x.double() + gate.double() * y.double()
    c = s - s.mean(-1, keepdim=True)
    return s, c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps) * (1 + scale.double()) + shift.double()
