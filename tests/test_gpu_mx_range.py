"""Microscaled operators where their accuracy shows: the activations over everything that their
inputs' types hold, each value in a block of its own, and products whose sums cancel, against
float64 (oracle/mx.py)."""

import pytest
import torch

from _mx_checks import codes_of
from flashmap_amd import ops
from oracle import mx

pytestmark = pytest.mark.gpu


def _check_alone(code, scale, bits, v, off):
    """Rows of one value each: what is stored lies between what is stored for the value less and plus
    its error (a block of one value stores a value that never falls as the value rises, its
    saturation below a power of two included)."""
    got = mx.values(code, scale, bits)
    lo, hi = (mx.values(*mx.quantize(w, bits), bits) for w in (v - off, v + off))
    bad = (got < lo) | (got > hi) | torch.isnan(got)
    rows = torch.nonzero(bad.any(1))[:5, 0]
    assert not bad.any(), f"{int(bad.any(1).sum())} values off: " + ", ".join(f"{v[r, 0]:.9g} gave {got[r, 0]:.9g}" for r in rows)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_swiglu_over_the_whole_range(dev, dtype, bits):
    """Gates and factors of every size, each pair in a block of its own: the result counts, whatever
    the gate's exponential or the product of the two does by itself. A few roundings of the
    exponential, the quotient and three products: 16 of 2^-24, and half of the smallest float where
    the result is subnormal. Where float32 cannot hold it the block is NaN, as where an input is
    not finite."""
    sizes = [0.0, 1e-40, 1e-30, 1e-3, 0.5, 1.0, 9.0, 50.0, 80.0, 87.0, 87.3, 87.5, 88.0, 88.5, 89.0, 95.0, 103.0, 104.0,
             120.0, 140.0, 199.0, 201.0, 1e3, 1e4, 1e9, 1e30, 2.4e38, 3e38, float("inf")]
    gates = torch.tensor([s * v for v in sizes for s in (1, -1)] + [float("nan")])
    ups = torch.tensor([1e-40, 1e-30, 1e-10, -1.0, 300.0, -1e9, 1e30, 1e37, 3e38, 0.0, float("inf"), float("nan")])
    pairs = torch.cartesian_prod(gates, ups)
    x = torch.zeros(len(pairs), 64)
    x[:, 0], x[:, 32] = pairs[:, 0], pairs[:, 1]
    x = x.to(dtype)
    q = ops.mx_quantize(x.to(dev), bits, "swiglu")
    want = mx.swiglu(x)
    want[~torch.isfinite(want.float())] = float("nan")
    bad = torch.isnan(want[:, 0])
    code, scale = codes_of(q)
    wrong = (scale[:, 0] == 255) != bad
    assert not wrong.any(), f"{int(wrong.sum())} pairs: " + str([x[i, [0, 32]].tolist() for i in torch.nonzero(wrong)[:5, 0]])
    _check_alone(code[~bad], scale[~bad], bits, want[~bad], 2.0 ** -20 * want[~bad].abs() + 2.0 ** -150)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gelu_over_the_whole_range(dev, dtype, bits):
    """Every bf16 value (in float32 too, with values between them): x Phi(x) = max(x, 0) - h, h = |x| / 2
    erfc(|x| / sqrt 2), where h moves by x^2 of its argument's relative error and is 0 below 2^-126, and
    the difference is rounded once. NaN for what is not finite."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)[:, None].to(dtype)
    if dtype == torch.float32:
        x = torch.cat([x, torch.linspace(-16, 16, 65537)[:, None]])
    q = ops.mx_quantize(x.to(dev), bits, "gelu")
    fine = torch.isfinite(x[:, 0])
    code, scale = codes_of(q)
    assert (scale[~fine, 0] == 255).all()
    v, want = x[fine].double(), mx.gelu(x[fine])
    h = 0.5 * v.abs() * torch.special.erfc(v.abs() / 2.0 ** 0.5)
    off = 2.0 ** -22 * (8 + v.clamp(-20, 20) ** 2) * h + 2.0 ** -24 * want.abs() + 2.0 ** -126
    _check_alone(code[fine], scale[fine], bits, want, off)
    best = mx.quantize(want.float(), bits)
    differ = ((code[fine] != best[0]).any(1) | (scale[fine] != best[1]).any(1)) & (want[:, 0].abs() > 2.0 ** -126)
    print(f"gelu {dtype} bits={bits}: {int(differ.sum())} of {len(v)} codes are not those of the value rounded to float32, "
          f"at x from {x[fine][differ].abs().min():.3g}" if differ.any() else "gelu: all codes as rounded", flush=True)


@pytest.mark.parametrize("kind", ["bf16", 8, 4])
@pytest.mark.parametrize("rows,n,k", [(1, 48, 2048), (16, 40, 1024), (40, 70, 2048), (130, 64, 512)])
def test_sums_that_cancel(dev, rows, n, k, kind):
    """What the product's sums lose, not hidden by the rounding of a result of the sum's size: the
    second half of k holds the first half's values again, negated and in another order, and one
    column of its own. Per step of 128 the 16 groups of 8 products lose at most 7 2^-13 of each
    group's largest product, together of the step's 16 largest (nothing with 4-bit rows); the
    float32 sums 2^-15 of the absolute sum."""
    g = torch.Generator().manual_seed(rows + k)
    half = k // 2
    order = torch.cat([32 * b + torch.randperm(32, generator=g) for b in torch.randperm(half // 32, generator=g)])
    x = torch.randn(rows, half, generator=g) * torch.exp(torch.randn(half, generator=g))
    w = torch.randn(n, half, generator=g)
    x, w = torch.cat([x, -x[:, order]], 1).bfloat16(), torch.cat([w, w[:, order]], 1)
    x[:, -1] *= 1.25
    weight = ops.mx_quantize(w.to(dev), 4)
    given = x.to(dev) if kind == "bf16" else ops.mx_quantize(x.to(dev), kind)
    xv = mx.values(*(mx.quantize(x, 8) if kind == "bf16" else codes_of(given)), 4 if kind == 4 else 8)
    products = xv[:, None] * mx.values(*codes_of(weight), 4)[None]
    ref, size = products.sum(-1), products.abs().sum(-1)
    lost = 0 if kind == 4 else 7 * 2.0 ** -13 * products.abs().view(rows, n, -1, 128).topk(16, -1).values.sum((-1, -2))
    err = (ops.mx_linear(given, weight).cpu().double() - ref).abs()
    over = (err - 2.0 ** -8 * ref.abs()).clamp(min=0) / size
    print(f"mx_linear rows={rows} n={n} k={k} x={kind}: sums of {float((ref.abs() / size).median()):.2e} of their absolute "
          f"sum, off by {float(over.max()):.1e} of it at most, {float(over.mean()):.1e} in the mean", flush=True)
    assert (err <= 2.0 ** -8 * ref.abs() + lost + 2.0 ** -15 * size).all()
