"""Bounds of the microscaled operators, and how far off the tests let them be.

Where a value is computed before it is quantized (an activation, a norm) it is off by its
float32 error, which moves a code only past a midpoint: the codes must lie between the
oracle's for the value less and plus that error.

A product's bound counts the bf16 rounding (2^-8 of the result) and what the sums lose of their
absolute sum: 2^-15 for the float32 sums of groups, steps and parts (probed with single
products: a term is cut below 2^-20 of the largest of the 16 groups of a step, 16 2^-20; 160 steps
and 8 parts of 2^-23 each), and with an 8-bit operand 7 2^-13 < 2^-10 more: the instruction adds the
8 products of a group after cutting each below 2^-13 of the power of two of the group's largest
(probed likewise), so that 7 of them lose less than 2^-13 of the largest, and the largest is at
most the group's absolute sum. Products within 2^12 of each other lose nothing there.
"""

import torch

from _inputs import gen
from flashmap_amd import ops
from oracle import mx


def codes_of(q: ops.MX):
    """(codes one per value, scales) on the CPU, padding included."""
    return mx.unpack(q.codes.cpu(), q.bits), q.scales.cpu()


def activations(rows, cols, seed, dtype=torch.bfloat16):
    g = gen(seed)
    return (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g))).to(dtype)


def check_between(q: ops.MX, v: torch.Tensor, tol: torch.Tensor) -> None:
    """Every code of ``q`` is the code of some value within ``tol`` of ``v`` (float64)."""
    code, scale = codes_of(q)
    got = mx.values(code, scale, q.bits)
    (lc, ls), (hc, hs) = mx.quantize(v - tol, q.bits), mx.quantize(v + tol, q.bits)
    down, up = mx.quantize(v.abs() - tol, q.bits)[1], mx.quantize(v.abs() + tol, q.bits)[1]
    assert ((scale >= down.minimum(up)) & (scale <= down.maximum(up))).all(), "a scale away from its block's maximum"
    lo, hi = mx.values(lc, scale.minimum(ls), q.bits), mx.values(hc, scale.maximum(hs), q.bits)
    same = ((ls == scale) & (hs == scale)).repeat_interleave(32, 1)
    inside = (got >= lo) & (got <= hi)
    assert inside[same].all(), f"{int((~inside & same).sum())} codes outside their interval"
    # where the error moves the block's maximum over a power of two: within a code of it
    step = 2.0 ** (scale.double() - 127).repeat_interleave(32, 1) * (32 if q.bits == 8 else 2)
    full = torch.zeros_like(got)
    full[:, : v.shape[1]] = v
    assert ((got - full).abs() <= step)[~same].all()


def operand(kind, x):
    """What the product is given and the float64 values that it stands for."""
    if kind == "bf16":
        return x, mx.values(*mx.quantize(x.cpu(), 8), 8)
    q = ops.mx_quantize(x, kind)
    return q, mx.values(*codes_of(q), kind)


def check_product(got, xv, wv, bias, sums=2.0 ** -15 + 2.0 ** -10):
    ref = xv @ wv.T + (0 if bias is None else bias.cpu().double())
    total = xv.abs() @ wv.abs().T + (0 if bias is None else bias.cpu().double().abs())
    err = (got.cpu().double() - ref).abs()
    bad = err > 2.0 ** -8 * ref.abs() + sums * total
    assert not bad.any(), f"{int(bad.sum())} results off, by up to {(err / total)[bad].max():.2e} of the absolute sum"


def check_activation(q: ops.MX, x: torch.Tensor, activation: str) -> None:
    """``q`` against the activation of ``x`` (CPU): erfc(z) moves by 2 z^2 of its argument's
    relative error, z^2 = x^2 / 2, and exp(-g) by g."""
    want = mx.gelu(x) if activation == "gelu" else mx.swiglu(x)
    check_between(q, want, 2.0 ** -22 * (8 + x.double()[:, : want.shape[1]] ** 2) * want.abs())


def check_rms_norm(stream, q: ops.MX, x, residual, weight, eps) -> None:
    """On CPU inputs. A thread's 64 squares and the join of 256 threads: 76 roundings of positive
    terms, half of it by the root; the sum s, the root and two products."""
    s, want = mx.rms_norm(x, residual, weight, eps)
    tol = want.abs() * (38 + 8) * 2.0 ** -24
    if residual is not None:
        tol = tol + 2.0 ** -24 * (x.double().abs() + residual.double().abs()) * (want / s).abs().nan_to_num(0, 0, 0)
        assert ((stream.cpu().double() - s).abs() <= 2.0 ** -8 * s.abs() + 2.0 ** -24 * s.abs()).all()
    check_between(q, want, tol)


def check_adaln(stream, q: ops.MX, x, y, gate, scale, shift, eps) -> None:
    """On CPU inputs, ``x`` and ``gate`` expandable to the rows. The mean of a thread's 64 values
    and the join of 256 threads: 76 roundings of the absolute sum; the centred value takes its
    error and its own, the root half of 80 roundings."""
    s, want = mx.adaln(x, y, gate, scale, shift, eps)
    err_s = 2.0 ** -24 * s.abs()  # the fused multiply-add's rounding
    if y is not None:
        assert ((stream.cpu().double() - s).abs() <= 2.0 ** -8 * s.abs() + err_s).all()
    mean_err = 76 * 2.0 ** -24 * s.abs().mean(-1, keepdim=True)
    c = (s - s.mean(-1, keepdim=True)).abs()
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    centre = err_s + mean_err + 2.0 ** -24 * c
    root = 44 * 2.0 ** -24 + (centre * c + centre ** 2).mean(-1, keepdim=True) * rstd ** 2
    one = (1 + scale.double()).abs()
    check_between(q, want, one * rstd * (centre + c * (root + 4 * 2.0 ** -24)) + 2.0 ** -24 * want.abs())
