"""Microscaled rows without a GPU: what the wrappers and the C entries refuse before anything
is launched, and the sizes of what they allocate."""

import ctypes

import pytest
import torch

from flashmap_amd import _native, ops

BF = torch.bfloat16


@pytest.fixture
def host(monkeypatch):
    """The wrappers' own checks on CPU tensors; a launch fails the test."""
    monkeypatch.setattr(ops, "_check_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(ops, "call", lambda name, *a: pytest.fail(f"{name} was launched"))


def _rows(rows, cols, bits):
    return ops._mx_new((rows, cols), bits, torch.device("cpu"))


def test_cpu_tensors_are_refused():
    x, q = torch.zeros(4, 64, dtype=BF), _rows(8, 64, 4)
    for f in (lambda: ops.mx_quantize(x), lambda: ops.mx_dequantize(q), lambda: ops.mx_linear(x, q),
              lambda: ops.rms_norm_mx(x, torch.ones(64), 1e-6),
              lambda: ops.adaln_residual_mx(x, None, None, (x[0], x[0]), 1e-6)):
        with pytest.raises(ValueError, match="GPU"):
            f()


@pytest.mark.parametrize("cols,pad", [(1, 128), (127, 128), (128, 128), (129, 256), (2048, 2048)])
def test_sizes(cols, pad):
    for bits in (4, 8):
        q = _rows(3, cols, bits)
        assert q.codes.shape == (3, pad * bits // 8) and q.scales.shape == (3, pad // 32)
        assert (q.rows, q.cols, q.view(3, 1).shape) == (3, cols, (3, 1, cols))
        with pytest.raises(ValueError, match="cannot be viewed"):
            q.view(2, 2)
        with pytest.raises(TypeError, match="bytes"):
            q.to(BF)
    assert _native.lib().fm_mx_linear_workspace_bytes(0, 5, cols, 8) == 0


def test_quantize_refuses(host):
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        ops.mx_quantize(torch.zeros(2, 64, dtype=torch.float64))
    with pytest.raises(ValueError, match="4 or 8"):
        ops.mx_quantize(torch.zeros(2, 64), bits=6)
    with pytest.raises(ValueError, match="activation"):
        ops.mx_quantize(torch.zeros(2, 64), activation="relu")
    with pytest.raises(ValueError, match="two halves"):
        ops.mx_quantize(torch.zeros(2, 65), activation="swiglu")
    with pytest.raises(ValueError, match="columns"):
        ops.mx_quantize(torch.zeros(2, 0))
    with pytest.raises(ValueError, match="cols"):
        ops.mx_quantize(torch.tensor(1.0))
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.mx_quantize(torch.zeros(2, 64, requires_grad=True))
    with pytest.raises(TypeError, match="dtype"):
        ops.mx_dequantize(_rows(2, 64, 8), torch.float64)


def test_linear_refuses(host):
    w, x = _rows(8, 64, 4), torch.zeros(4, 64, dtype=BF)
    with pytest.raises(ValueError, match="in 4 bits"):
        ops.mx_linear(x, _rows(8, 64, 8))
    with pytest.raises(ValueError, match="in 4 bits"):
        ops.mx_linear(x, w.view(2, 4))
    with pytest.raises(ValueError, match="64 columns"):
        ops.mx_linear(x[:, :32], w)
    with pytest.raises(ValueError, match="64 columns"):
        ops.mx_linear(x[0, 0], w)
    with pytest.raises(TypeError, match="bfloat16 or microscaled"):
        ops.mx_linear(x.float(), w)
    with pytest.raises(ValueError, match="bias"):
        ops.mx_linear(x, w, torch.zeros(9, dtype=BF))
    with pytest.raises(ValueError, match="bias"):
        ops.mx_linear(x, w, torch.zeros(8))
    with pytest.raises(ValueError, match="x_out|out must"):
        ops.mx_linear(x, w, out=torch.zeros(4, 8))
    with pytest.raises(ValueError, match="overlap"):
        ops.mx_linear(x, w, out=torch.zeros(1, 8, dtype=BF).expand(4, 8))
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.mx_linear(x.clone().requires_grad_(True), w)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.mx_linear(_rows(4, 64, 8), w, torch.zeros(8, dtype=BF, requires_grad=True))
    for bad in (ops.MX(w.codes[:, :16], w.scales, 4, (8, 64)), ops.MX(w.codes, w.scales[:7], 4, (8, 64)),
                ops.MX(w.codes, w.scales, 4, (9, 64)), ops.MX(w.codes, w.scales, 4, (8, 200))):
        with pytest.raises(ValueError, match="holds codes|columns"):
            ops.mx_linear(torch.zeros(4, bad.cols, dtype=BF), bad)
    with pytest.raises(TypeError, match="uint8"):
        ops.mx_linear(x, ops.MX(w.codes.float(), w.scales, 4, (8, 64)))


def test_norms_refuse(host):
    x, w, v = torch.zeros(4, 64, dtype=BF), torch.ones(64), torch.zeros(64, dtype=BF)
    with pytest.raises(TypeError, match="bfloat16"):
        ops.rms_norm_mx(x.float(), w, 1e-6)
    with pytest.raises(ValueError, match="weight"):
        ops.rms_norm_mx(x, w[:32], 1e-6)
    with pytest.raises(ValueError, match="residual"):
        ops.rms_norm_mx(x, w, 1e-6, x[:2])
    with pytest.raises(ValueError, match="give one"):
        ops.rms_norm_mx(x, w, 1e-6, x_out=x)
    with pytest.raises(ValueError, match="x_out"):
        ops.rms_norm_mx(x, w, 1e-6, x, x_out=x[:2])
    with pytest.raises(ValueError, match="16384"):
        ops.rms_norm_mx(torch.zeros(1, 16385, dtype=BF), torch.ones(16385), 1e-6)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.rms_norm_mx(x, w.clone().requires_grad_(True), 1e-6)
    with pytest.raises(ValueError, match="modulation"):
        ops.adaln_residual_mx(x, None, None, None, 1e-6)
    with pytest.raises(ValueError, match="gate"):
        ops.adaln_residual_mx(x, x, None, (v, v), 1e-6)
    with pytest.raises(ValueError, match="scale"):
        ops.adaln_residual_mx(x, None, None, (v[:3], v), 1e-6)
    with pytest.raises(ValueError, match="one per row"):
        ops.adaln_residual_mx(x, x, v, (v, v), 1e-6, gate_per_row=True)
    with pytest.raises(ValueError, match="does not match"):
        ops.adaln_residual_mx(x, x[:, :32], v, (v, v), 1e-6)
    with pytest.raises(ValueError, match="shared"):
        row = torch.zeros(4, 64, dtype=BF)
        ops.adaln_residual_mx(row[0], x, v, (v, v), 1e-6, x_out=row)
    with pytest.raises(ValueError, match="give one"):
        ops.adaln_residual_mx(x, None, None, (v, v), 1e-6, x_out=x)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.adaln_residual_mx(x, x, v.clone().requires_grad_(True), (v, v), 1e-6)


def _fails(match, code, name, *args):
    with pytest.raises(_native.NativeError, match=match) as e:
        _native.call(name, *args)
    assert e.value.code == code


def test_entries_refuse_what_they_cannot_launch():
    """The C entries' own checks, which return before anything is launched."""
    at, inv, unsup = 4096, _native.FM_ERR_INVALID, _native.FM_ERR_UNSUPPORTED

    def quant(x=at, dt=0, xs=64, act=0, bits=8, c=at, cs=128, s=at, ss=4, rows=4, cols=64):
        return "fm_mx_quantize", x, dt, xs, act, bits, c, cs, s, ss, rows, cols, None

    def dq(bits=8, out=at, dt=0, os=64, rows=4, cols=64):
        return "fm_mx_dequantize", at, 128, at, 4, bits, out, dt, os, rows, cols, None

    _fails("bad sizes", inv, *quant(rows=-1))
    _fails("bad sizes", inv, *quant(cols=0))
    _fails("dtype 3", inv, *quant(dt=3))
    _fails("activation 3", inv, *quant(act=3))
    _fails("bits 5", inv, *quant(bits=5))
    _fails("NULL", inv, *quant(x=None))
    _fails("NULL codes", inv, *quant(c=None))
    _fails("overlap", inv, *quant(xs=32))
    _fails("overlap", inv, *quant(act=2, xs=127))
    _fails("rows of 128 bytes", inv, *quant(cs=64))
    _fails("rows of 128 bytes", inv, *quant(c=at + 8))
    _fails("scales must be", inv, *quant(ss=2))
    _fails("at most 2\\^26", unsup, *quant(cols=(1 << 26) + 1, xs=1 << 27))
    assert _native.call(*quant(x=None, rows=0)) is None
    _fails("NULL", inv, *dq(out=None))
    _fails("bits 16", inv, *dq(bits=16))
    _fails("overlap", inv, *dq(os=63))

    def lin(x=at, xb=8, xs=128, xsc=at, xss=4, w=at, ws=64, wss=4, out=at, os=8, rows=4, n=8, k=64, wk=None, wb=0):
        return "fm_mx_linear", x, xb, xs, xsc, xss, w, ws, at, wss, None, out, os, rows, n, k, wk, wb, None

    _fails("x_bits 5", inv, *lin(xb=5))
    _fails("bad sizes", inv, *lin(k=0))
    _fails("NULL", inv, *lin(w=None))
    _fails("w: 16-byte", inv, *lin(ws=48))
    _fails("w: 16-byte", inv, *lin(wss=2))
    _fails("x: 16-byte", inv, *lin(xs=64))
    _fails("x: 16-byte", inv, *lin(xsc=None))
    _fails("out rows", inv, *lin(os=7))
    _fails("at most 2\\^26", unsup, *lin(n=(1 << 26) + 1, os=1 << 27))
    _fails("at most 2\\^22", unsup, *lin(k=(1 << 22) + 1))
    _fails("below 2\\^24", inv, *lin(xs=1 << 24))
    _fails("below 2\\^24", inv, *lin(ws=1 << 24))
    # bf16 rows that the product's kernel does not quantize itself need room for their codes
    lib = _native.lib()
    for rows, n, k in ((17, 8, 64), (4, 8, 63), (16, 8, 8192), (16, 8200, 5640)):
        pad = -(-k // 128) * 128
        need = lib.fm_mx_linear_workspace_bytes(rows, n, k, 8) + rows * pad * 33 // 32
        assert lib.fm_mx_linear_workspace_bytes(rows, n, k, 16) == need
        w = dict(xb=16, xs=k, ws=pad // 2, wss=pad // 32, os=n, rows=rows, n=n, k=k)
        _fails(f"workspace of 0 bytes, need {need}", _native.FM_ERR_WORKSPACE, *lin(**w))
        _fails("workspace of", _native.FM_ERR_WORKSPACE, *lin(**w, wk=at, wb=need - 1))
        _fails("workspace of", _native.FM_ERR_WORKSPACE, *lin(**w, wk=at + 8, wb=need))
        _fails("overlap", inv, *lin(**dict(w, xs=k - 1), wk=at, wb=need))
    for rows, n, k in ((16, 8, 8184), (16, 8200, 5632), (1, 8192, 8)):
        assert lib.fm_mx_linear_workspace_bytes(rows, n, k, 16) == 0
    _fails("bf16 x", inv, *lin(xb=16, xs=60, k=56))
    _fails("bf16 x", inv, *lin(xb=16, xs=64, x=at + 8))
    assert _native.call(*lin(x=None, rows=0)) is None
    f = ctypes.c_float(1e-6)
    _fails("at most 16384", unsup, "fm_rms_norm_mx", at, 64, None, 0, at, f, None, 0, 8, at, 128, at, 4, 4, 16385, None)
    _fails("go together", inv, "fm_rms_norm_mx", at, 64, at, 64, at, f, None, 0, 8, at, 128, at, 4, 4, 64, None)
    _fails("cover a row", inv, "fm_rms_norm_mx", at, 63, None, 0, at, f, None, 0, 8, at, 128, at, 4, 4, 64, None)
    _fails("needs its gate", inv, "fm_adaln_residual_mx", at, 64, at, 64, None, 0, at, at, at, 64, f, 8, at, 128, at, 4,
           4, 64, None)
    _fails("shared x row", inv, "fm_adaln_residual_mx", at, 0, at, 64, at, 0, at, at, at, 64, f, 8, at, 128, at, 4, 4,
           64, None)


def test_outputs_over_rows_that_are_read():
    """ops._apart: rows of one buffer side by side and the very same rows pass, others do not."""
    from flashmap_amd import ops

    buf = torch.zeros(40, 64, dtype=torch.bfloat16)
    x = buf[:16, :32]
    for name, out, same, refused in (
        ("beside", buf[:16, 32:], False, False),
        ("the same, read first", x, True, False),
        ("the same, read by others", x, False, True),
        ("behind", buf[16:32, :32], False, False),
        ("a row on", buf[1:17, :32], True, True),
        ("some columns on", buf[:16, 16:48], True, True),
        ("from one row's end into the next", buf.view(-1)[48:48 + 16 * 64].view(16, 64)[:, :32], False, True),
        ("another stride", buf.view(-1)[: 16 * 32].view(16, 32), True, True),
    ):
        args = ("out", out, out.stride(0), 16, 32, (x, 64, 16, 32, same))
        if refused:
            with pytest.raises(ValueError, match="overlaps rows"):
                ops._apart(*args)
        else:
            ops._apart(*args)
    ops._apart("out", buf[1:2], 64, 1, 64, (buf[0:1], 64, 1, 64, False))
    with pytest.raises(ValueError):
        ops._apart("out", buf[0:1, 8:], 56, 1, 56, (buf[0:1], 64, 1, 64, False))
