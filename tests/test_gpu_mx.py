"""Microscaled rows on the GPU (flashmap_amd.ops.mx_*, rms_norm_mx, adaln_residual_mx) against
float64 (oracle/mx.py), with the bounds of _mx_checks.py; quantization of a tensor's own values is
one rounding of exact quotients, and its codes and scales are equal to the oracle's."""

import pytest
import torch

from _inputs import gen
from _mx_checks import (activations, check_activation, check_adaln, check_product, check_rms_norm, codes_of,
                        operand)
from flashmap_amd import ops
from oracle import mx

pytestmark = pytest.mark.gpu


SIZES = [(1, 1), (3, 31), (2, 32), (5, 33), (17, 127), (1, 128), (4, 129), (33, 200), (7, 2056), (3, 20480)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantize_is_exact(dev, rows, cols, dtype, bits):
    print(f"mx_quantize {rows} x {cols} {dtype} bits={bits}", flush=True)
    x = activations(rows, cols, rows + cols, dtype)
    q = ops.mx_quantize(x.to(dev), bits)
    code, scale = codes_of(q)
    wc, ws = mx.quantize(x, bits)
    assert q.shape == (rows, cols) and torch.equal(scale, ws) and torch.equal(code, wc)
    back = ops.mx_dequantize(q, torch.float32)
    assert torch.equal(back.cpu().double(), mx.values(wc, ws, bits)[:, :cols])
    for other in (torch.bfloat16, torch.float16):
        assert torch.equal(ops.mx_dequantize(q, other).cpu(), back.cpu().to(other))


@pytest.mark.parametrize("bits", [8, 4])
def test_quantize_edges(dev, bits):
    """Midpoints, the largest and smallest floats, infinities and NaN, zeros of both signs."""
    grid = torch.tensor(mx.E4M3 if bits == 8 else mx.E2M1)
    over = grid[-1:] * torch.tensor([1.01, 1.03, 1.06, 1.13])
    mids = torch.cat([grid, (grid[1:] + grid[:-1]) / 2, over])
    v = torch.cat([mids, -mids])
    v = torch.cat([v, torch.zeros(-len(v) % 32)])
    top = torch.full((32,), float(grid[-1]))
    rows = [torch.cat([v * 2.0 ** e, top * 2.0 ** e]) for e in (0, -5, 17, -100, 100)]
    n = len(rows[0])
    special = torch.zeros(6, n)
    special[0, 5], special[0, 40] = float("inf"), float("nan")
    special[1, :] = -0.0
    special[2, ::2] = torch.finfo(torch.float32).max
    special[3, :] = torch.linspace(-1, 1, n) * 2.0 ** -118
    special[4, 0::32], special[4, 1::32] = 2.0 ** -126, -(2.0 ** -127)
    special[5, 3], special[5, 7] = -float("inf"), 2.0 ** -149
    # a scale of 2^e puts each block's maximum on the grid's top: the grid's own points and midpoints
    x = torch.cat([torch.stack(rows), special])
    x[:, 0::32] = torch.where(x[:, 0::32].abs() < x[:, -1:].abs(), x[:, -1:], x[:, 0::32])
    q = ops.mx_quantize(x.to(dev), bits)
    wc, ws = mx.quantize(x, bits)
    code, scale = codes_of(q)
    assert torch.equal(scale, ws)
    fine = (ws != 255).repeat_interleave(32, 1)
    assert torch.equal(code[fine], wc[fine])
    back = ops.mx_dequantize(q, torch.float32).cpu().double()
    torch.testing.assert_close(back, mx.values(wc, ws, bits)[:, :n], rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("activation", ["gelu", "swiglu"])
@pytest.mark.parametrize("rows,cols,dtype", [(3, 33, torch.float32), (16, 8192, torch.bfloat16),
                                             (5, 200, torch.float16), (1, 1, torch.bfloat16), (9, 260, torch.float32)])
def test_activation(dev, rows, cols, dtype, activation, bits):
    x = activations(rows, cols * (2 if activation == "swiglu" else 1), 5 * cols, dtype).clamp(-9, 9)
    check_activation(ops.mx_quantize(x.to(dev), bits, activation), x, activation)


def test_layouts(dev):
    """Leading dimensions, strided and unaligned rows, expanded rows, no rows."""
    wide = activations(12, 520, 3).to(dev)
    want = ops.mx_quantize(wide[:, :256].contiguous())
    for x in (wide[:, :256], torch.cat([wide.new_zeros(1), wide[:, :256].reshape(-1)])[1:].view(12, 256),
              wide[:, :256].t().contiguous().t(), wide[:, :256].reshape(3, 4, 256)):
        q = ops.mx_quantize(x)
        assert q.shape == tuple(x.shape) and torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)
    odd = ops.mx_quantize(wide[:, 3:260])
    assert torch.equal(codes_of(odd)[0], mx.quantize(wide[:, 3:260].cpu(), 8)[0])
    one = ops.mx_quantize(wide[:1, :256].expand(12, 256))
    assert torch.equal(one.codes, want.codes[:1].expand(12, -1))
    empty = ops.mx_quantize(wide[:0])
    assert empty.rows == 0 and ops.mx_dequantize(empty).shape == (0, 520)
    assert ops.mx_linear(empty, ops.mx_quantize(wide, 4)).shape == (0, 12)
    assert ops.mx_quantize(wide[0]).shape == (520,)


@pytest.mark.parametrize("kind", ["bf16", 8, 4])
@pytest.mark.parametrize("rows,n,k", [
    (1, 1, 1), (1, 17, 32), (3, 15, 33), (16, 16, 128), (17, 33, 160), (16, 300, 2048), (31, 257, 129), (32, 64, 1000),
    (33, 100, 4096), (64, 130, 640), (65, 127, 256), (100, 1000, 384), (128, 128, 512), (129, 300, 2048),
    (255, 257, 1152), (256, 512, 1024), (300, 513, 896), (600, 260, 130), (1, 5000, 2048), (16, 9000, 512),
    # a stream of columns: groups that end early, odd columns, the longest rows that lie in LDS
    (16, 8200, 128), (1, 9001, 700), (7, 12288, 1408), (16, 8193, 5632), (3, 8300, 10880),
    # few rows, long sums, in parts: whole ones and a last one of less than a chunk
    (5, 100, 8192), (16, 70, 20480), (33, 64, 8320), (64, 200, 4224), (130, 72, 6272),
    # tiles of 128 and 256, more than the chip holds at once and not
    (2048, 2048, 256), (1920, 2500, 384), (3300, 4100, 128), (2048, 6144, 640), (4096, 4096, 200)])
def test_linear(dev, rows, n, k, kind):
    print(f"mx_linear rows={rows} n={n} k={k} x={kind}", flush=True)
    x = activations(rows, k, rows + n + k).to(dev)
    w = ops.mx_quantize(torch.randn(n, k, generator=gen(n)).to(dev) / k ** 0.5, 4)
    bias = torch.randn(n, generator=gen(k)).bfloat16().to(dev) if (rows + n) % 2 else None
    given, xv = operand(kind, x)
    got = ops.mx_linear(given, w, bias)
    assert got.shape == (rows, n) and got.dtype == torch.bfloat16
    check_product(got, xv, mx.values(*codes_of(w), 4), bias, 2.0 ** -15 + (0 if kind == 4 else 2.0 ** -10))


@pytest.mark.parametrize("kind", ["bf16", 8])
@pytest.mark.parametrize("rows,n,k", [(1, 300, 2048), (16, 5000, 1000), (13, 9000, 5632), (16, 100, 20480),
                                      (40, 70, 8320), (130, 1500, 384), (1024, 2048, 512), (2048, 6200, 640)])
def test_linear_of_even_magnitudes(dev, rows, n, k, kind):
    """x of magnitudes from 1 to 2 within each block: codes of one or two binades, products
    (with the weights' 0.5 to 6) within 2^6 of each other, nothing lost in the groups."""
    g = gen(rows + k)
    x = (1 + torch.rand(rows, k, generator=g)) * torch.randint(0, 2, (rows, k), generator=g).mul(2).sub(1)
    x = x * torch.randint(-6, 7, (rows, -(-k // 32)), generator=g).float().exp2().repeat_interleave(32, 1)[:, :k]
    w = ops.mx_quantize(torch.randn(n, k, generator=g).to(dev), 4)
    given, xv = operand(kind, x.bfloat16().to(dev))
    check_product(ops.mx_linear(given, w), xv, mx.values(*codes_of(w), 4), None, 2.0 ** -15)


@pytest.mark.parametrize("kind", ["bf16", 8, 4])
@pytest.mark.parametrize("rows", [2, 40, 300])
def test_linear_layouts(dev, rows, kind):
    """Leading dimensions, a strided x and out, an out that already holds values around it."""
    n, k = 100, 300
    base = activations(rows, k + 20, 7).to(dev)
    w = ops.mx_quantize(torch.randn(n, k, generator=gen(1)).to(dev), 4)
    x = base[:, 5:5 + k]
    given = x if kind == "bf16" else ops.mx_quantize(x, kind)
    want = ops.mx_linear(x.contiguous() if kind == "bf16" else given, w)
    buf = torch.full((rows, n + 9), 7.0, dtype=torch.bfloat16, device=dev)
    got = ops.mx_linear(given, w, out=buf[:, 3:3 + n])
    assert got.data_ptr() == buf[:, 3:].data_ptr() and torch.equal(got, want)
    assert (buf[:, :3] == 7).all() and (buf[:, 3 + n:] == 7).all()
    lead = given.view(2, rows // 2) if kind != "bf16" else x.reshape(2, rows // 2, k)
    assert torch.equal(ops.mx_linear(lead, w).view(rows, n), want)
    # rows of a wider code buffer, and a weight cut out of a larger one
    if kind != "bf16":
        wider = torch.zeros(rows, given.codes.shape[1] + 48, dtype=torch.uint8, device=dev)
        wider[:, 16:16 + given.codes.shape[1]] = given.codes
        cut = ops.MX(wider[:, 16:16 + given.codes.shape[1]], given.scales, given.bits, given.shape)
        assert torch.equal(ops.mx_linear(cut, w), want)
    part = ops.MX(w.codes[30:90], w.scales[30:90], 4, (60, k))
    assert torch.equal(ops.mx_linear(given, part), want[:, 30:90])


@pytest.mark.parametrize("kind", ["bf16", 8, 4])
@pytest.mark.parametrize("rows", [3, 70, 260])
def test_linear_not_finite(dev, rows, kind):
    """A block with an infinity or a NaN makes its row's (or column's) results NaN and no others."""
    n, k = 90, 416
    x, wv = activations(rows, k, 1), torch.randn(n, k, generator=gen(2))
    x[1, 77], x[2, 3] = float("nan"), float("inf")
    wv[5, 400], wv[89, 0] = -float("inf"), float("nan")
    w = ops.mx_quantize(wv.to(dev), 4)
    given, xv = operand(kind, x.to(dev))
    got = ops.mx_linear(given, w).cpu()
    bad = torch.isnan(xv).any(1)[:, None] | torch.isnan(mx.values(*codes_of(w), 4)).any(1)[None]
    assert torch.equal(torch.isnan(got), bad) and bad[:3].float().sum() == n * 2 + 2


@pytest.mark.parametrize("kind", ["bf16", 8])
def test_linear_extreme_scales(dev, kind):
    """Rows of 2^100 and 2^-100 beside each other: products stay finite where the result is."""
    rows, n, k = 20, 40, 256
    x = torch.randn(rows, k, generator=gen(1)) * 2.0 ** torch.linspace(-100, 100, rows)[:, None]
    w = ops.mx_quantize((torch.randn(n, k, generator=gen(2)) * 2.0 ** -20).to(dev), 4)
    given, xv = operand(kind, x.bfloat16().to(dev))
    check_product(ops.mx_linear(given, w), xv, mx.values(*codes_of(w), 4), None)


NORM_SIZES = [(1, 1), (5, 33), (3, 129), (16, 512), (33, 2048), (7, 2056), (2, 4100), (9, 8192), (2, 16384)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_rms_norm(dev, rows, cols, with_residual, bits):
    print(f"rms_norm_mx {rows} x {cols} residual={with_residual} bits={bits}", flush=True)
    g = gen(rows + cols)
    x, w = activations(rows, cols, cols), 0.5 + torch.rand(cols, generator=g)
    res = torch.randn(rows, cols, generator=g).bfloat16() if with_residual else None
    stream, q = ops.rms_norm_mx(x.to(dev), w.to(dev), 1e-6, None if res is None else res.to(dev))
    if bits == 4:
        q = ops.rms_norm_mx(x.to(dev), w.to(dev), 1e-6, None if res is None else res.to(dev), bits=4)[1]
    assert (stream is None) == (res is None)
    check_rms_norm(stream, q, x, res, w, 1e-6)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("part", ["norm", "residual", "per_row", "shared"])
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_adaln(dev, rows, cols, part, bits):
    print(f"adaln_residual_mx {rows} x {cols} {part} bits={bits}", flush=True)
    g = gen(rows + cols)
    x = (activations(rows, cols, cols) + 0.25)
    y = torch.randn(rows, cols, generator=g).bfloat16()
    gate, scale, shift = (0.3 * torch.randn(3, cols, generator=g)).bfloat16().unbind(0)
    gr = gate
    if part == "per_row":
        gate = torch.randn(rows, generator=g).bfloat16()
        gr = gate[:, None]
    if part == "shared":
        x = x[0]
    given_y = None if part == "norm" else y
    stream, q = ops.adaln_residual_mx(x.to(dev), None if given_y is None else y.to(dev), gate.to(dev),
                                      (scale.to(dev), shift.to(dev)), 1e-6, gate_per_row=part == "per_row", bits=bits)
    xs = x.expand(rows, cols) if part == "shared" else x
    check_adaln(stream, q, xs, given_y, gr, scale, shift, 1e-6)


def test_norms_in_place_and_strided(dev):
    rows, cols = 12, 264
    wide = activations(rows, cols + 33, 4).to(dev)
    x, y = wide[:, 1:1 + cols], torch.randn(rows, cols, generator=gen(1)).bfloat16().to(dev)
    v = [t.to(dev) for t in (0.3 * torch.randn(3, cols, generator=gen(2))).bfloat16().unbind(0)]
    w = torch.rand(cols, generator=gen(3)).to(dev)
    for call in (lambda a, o: ops.rms_norm_mx(a, w, 1e-5, y, x_out=o),
                 lambda a, o: ops.adaln_residual_mx(a, y, v[0], (v[1], v[2]), 1e-5, x_out=o)):
        stream, q = call(x.contiguous(), None)
        s2, q2 = call(x, None)  # rows at odd addresses
        assert torch.equal(s2, stream) and torch.equal(q2.codes, q.codes) and torch.equal(q2.scales, q.scales)
        held = wide.clone()
        s3, q3 = call(held[:, 1:1 + cols], held[:, 1:1 + cols])
        assert s3.data_ptr() == held[:, 1:].data_ptr() and torch.equal(s3, stream) and torch.equal(q3.codes, q.codes)
        assert torch.equal(held[:, 0], wide[:, 0]) and torch.equal(held[:, 1 + cols:], wide[:, 1 + cols:])


def test_norm_rows_that_are_not_finite(dev):
    """A NaN or an infinity in a row makes that row NaN and leaves the others."""
    x = torch.randn(5, 200, generator=gen(1)).bfloat16()
    x[1, 3], x[3, 190] = float("nan"), float("inf")
    v = torch.zeros(200).bfloat16().to(dev)
    for q in (ops.rms_norm_mx(x.to(dev), torch.ones(200, device=dev), 1e-6)[1],
              ops.adaln_residual_mx(x.to(dev), None, None, (v, v), 1e-6)[1]):
        bad = torch.isnan(ops.mx_dequantize(q)).cpu()
        assert bad[1].all() and bad[[0, 2, 4]].sum() == 0
        # an infinite sum of squares: the finite values' quotients are 0, the infinity's NaN
        assert bad[3, 190] and (bad[3].all() or not bad[3, :160].any())


def test_two_streams_and_a_graph(dev):
    """Calls on a stream of their own, two captured graphs side by side, replays with eager work
    between them."""
    n, k = 300, 1000
    w = ops.mx_quantize(torch.randn(n, k, generator=gen(1)).to(dev), 4)
    xs = [activations(r, k, r).to(dev) for r in (16, 200)]
    want = [ops.mx_linear(x, w) for x in xs]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [ops.mx_linear(x, w) for x in xs]
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.mx_linear(x, w))
        graphs.append(g)
    for _ in range(3):
        for x in xs:
            x.mul_(-0.5)
        for g in graphs:
            g.replay()
        again = [ops.mx_linear(x, w) for x in xs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, again))


def test_mlp_of_a_layer(dev):
    """The operators in a row, as a layer's last sublayer runs them: each step against float64
    on what the step before it gave."""
    rows, dim, hidden = 48, 256, 800
    g = gen(11)
    x, y = activations(rows, dim, 1).to(dev), torch.randn(rows, dim, generator=g).bfloat16().to(dev)
    gate, scale, shift = (t.to(dev) for t in (0.3 * torch.randn(3, dim, generator=g)).bfloat16().unbind(0))
    fc1 = ops.mx_quantize((torch.randn(hidden, dim, generator=g) / 16).to(dev), 4)
    fc2 = ops.mx_quantize((torch.randn(dim, hidden, generator=g) / 28).to(dev), 4)
    b1 = torch.randn(hidden, generator=g).bfloat16().to(dev)
    stream, h = ops.adaln_residual_mx(x, y, gate, (scale, shift), 1e-6)
    up = ops.mx_linear(h, fc1, b1)
    mid = ops.mx_quantize(up, activation="gelu")
    out = ops.mx_linear(mid, fc2)
    check_product(up, mx.values(*codes_of(h), 8), mx.values(*codes_of(fc1), 4), b1)
    check_activation(mid, up.cpu(), "gelu")
    check_product(out, mx.values(*codes_of(mid), 8), mx.values(*codes_of(fc2), 4), None)
    s, norm = mx.adaln(*(t.cpu() for t in (x, y, gate, scale, shift)), 1e-6)
    # end to end: e4m3 activations (2^-4 each at most) in front of both products
    ref = mx.gelu(norm @ mx.values(*codes_of(fc1), 4)[:, :dim].T + b1.cpu().double())
    ref = ref @ mx.values(*codes_of(fc2), 4)[:, :hidden].T
    assert float((out.cpu().double() - ref).norm() / ref.norm()) < 2.0 ** -4
    assert stream.shape == x.shape


def test_rows_far_into_memory(dev):
    """Weights and outputs whose last rows lie past 2^32 bytes and 2^32 values."""
    n, k = (1 << 20) + 100, 8200
    pad = -(-k // 128) * 128
    seeded = torch.Generator(dev).manual_seed(1)
    codes = torch.randint(0, 256, (n, pad // 2), dtype=torch.uint8, device=dev, generator=seeded)
    codes[:, k // 2:] = 0
    scales = torch.randint(120, 130, (n, pad // 32), dtype=torch.uint8, device=dev)
    assert codes.numel() > 1 << 32
    w = ops.MX(codes, scales, 4, (n, k))
    last = ops.MX(codes[-200:], scales[-200:], 4, (200, k))
    for rows in (1, 20, 300):
        x = ops.mx_quantize(activations(rows, k, rows).to(dev))
        check_product(ops.mx_linear(x, w)[:, -200:], mx.values(*codes_of(x), 8), mx.values(*codes_of(last), 4), None)
    # 4-bit rows as the many: x's rows far into memory too
    few = ops.MX(codes[:40], scales[:40], 4, (40, k))
    check_product(ops.mx_linear(w, few)[-200:], mx.values(*codes_of(last), 4), mx.values(*codes_of(few), 4), None)
    back = ops.mx_dequantize(w)
    assert back.numel() > 1 << 32
    want = mx.values(mx.unpack(codes[-3:].cpu(), 4), scales[-3:].cpu(), 4)[:, :k]
    assert torch.equal(back[-3:].cpu().double(), want)
    again = ops.mx_quantize(back[-1000:], 8)
    assert torch.equal(ops.mx_dequantize(again), back[-1000:])  # e2m1 values are e4m3 values
    far = ops.mx_quantize(back, 8)
    assert torch.equal(far.codes[-1000:], again.codes) and torch.equal(far.scales[-1000:], again.scales)


def test_outputs_that_overlap_inputs(dev):
    """An output over rows that the call reads is refused, but for the very same rows of a norm,
    whose results equal those into a tensor of their own."""
    buf = activations(34, 256, 5, torch.bfloat16).to(dev)
    x, y = buf[:16, :128], buf[:16, 128:]
    w = ops.mx_quantize(activations(128, 128, 6, torch.bfloat16).to(dev), 4)
    for rows in (16, 17):
        read = buf[:rows, :128]
        with pytest.raises(ValueError, match="overlaps"):
            ops.mx_linear(read, w, out=read)
        with pytest.raises(ValueError, match="overlaps"):
            ops.mx_linear(read, w, out=buf[1:rows + 1, :128])
        want = ops.mx_linear(read, w)
        side = buf.clone()
        assert torch.equal(ops.mx_linear(side[:rows, :128], w, out=side[:rows, 128:]), want)
        assert torch.equal(side[:, :128], buf[:, :128]) and torch.equal(side[rows:], buf[rows:])
    v = buf[33, :128].clone()
    for call in (lambda a, b, out: ops.rms_norm_mx(a, v, 1e-6, residual=b, x_out=out),
                 lambda a, b, out: ops.adaln_residual_mx(a, b, v, (v, v), 1e-6, x_out=out)):
        with pytest.raises(ValueError, match="overlaps"):
            call(x, y, buf[1:17, :128])
        with pytest.raises(ValueError, match="overlaps"):
            call(x, y, buf[:16, 64:192])
        s, q = call(x, y, None)
        for half in (slice(0, 128), slice(128, 256)):
            own = buf.clone()
            t, p = call(own[:16, :128], own[:16, 128:], own[:16, half])
            assert torch.equal(t, s) and torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
            assert torch.equal(own[16:], buf[16:])


@pytest.mark.parametrize("kind", [8, 4])
@pytest.mark.parametrize("rows,n,k,stride", [
    (4096, 4160, 128, 4160), (4100, 4200, 256, 4204), (1024, 16900, 128, 16902), (2050, 8193, 384, 8193),
    (1024, 16640, 640, 16640)])
def test_linear_last_round(dev, rows, n, k, stride, kind):
    """More tiles of 256 x 256 than the chip holds at once, the last ones few (their columns go
    to smaller tiles) and rows of out aligned to 16, 8, 4 and 2 bytes."""
    print(f"mx_linear rows={rows} n={n} k={k} x={kind} stride={stride}", flush=True)
    x = activations(rows, k, rows + n).to(dev)
    w = ops.mx_quantize(torch.randn(n, k, generator=gen(n)).to(dev) / k ** 0.5, 4)
    bias = torch.randn(n, generator=gen(k)).bfloat16().to(dev)
    given, xv = operand(kind, x)
    buf = torch.full((rows, stride), 7.0, dtype=torch.bfloat16, device=dev)
    got = ops.mx_linear(given, w, bias, out=buf[:, :n])
    check_product(got, xv, mx.values(*codes_of(w), 4), bias, 2.0 ** -15 + (0 if kind == 4 else 2.0 ** -10))
    assert (buf[:, n:] == 7).all()


@pytest.mark.parametrize("rows,n", [(20, 70), (70, 130), (300, 513), (1500, 2500)])
@pytest.mark.parametrize("stride", [0, 1, 2, 4])
def test_linear_rows_of_any_alignment(dev, rows, n, stride):
    """The same bits whatever the alignment of out's rows, and nothing written between them."""
    k = 300
    w = ops.mx_quantize(torch.randn(n, k, generator=gen(1)).to(dev), 4)
    x = ops.mx_quantize(activations(rows, k, n).to(dev))
    want = ops.mx_linear(x, w)
    wide = -(-n // 8) * 8 + 8 + stride
    for first in (0, stride):
        buf = torch.full((rows, wide), 7.0, dtype=torch.bfloat16, device=dev)
        got = ops.mx_linear(x, w, out=buf[:, first:first + n])
        assert torch.equal(got, want)
        assert (buf[:, :first] == 7).all() and (buf[:, first + n:] == 7).all()
