"""Outputs that a caller gives over memory that the call reads, without a GPU: the wrappers refuse
each operand, and take what lies beside it."""

import pytest
import torch

from flashmap_amd import ops
from test_mx_cpu import host  # noqa: F401  (the wrappers' checks on CPU tensors)

BF = torch.bfloat16
ROWS, COLS, N = 4, 64, 8


@pytest.fixture
def launched(host, monkeypatch):  # noqa: F811
    made = []
    monkeypatch.setattr(ops, "_mx_call", lambda name, index, *args: made.append(name))
    return made


def _at(buf, first, shape, dtype):
    """A tensor of ``shape`` on the bytes of ``buf`` from ``first`` on."""
    count = torch.Size(shape).numel()
    return buf[first:first + count * dtype.itemsize].view(dtype).view(shape)


@pytest.mark.parametrize("over", ["x codes", "x scales", "weight codes", "weight scales", "bias", "bf16 x", None])
def test_linear(launched, over):
    buf = torch.zeros(1 << 14, dtype=torch.uint8)
    x = ops.MX(_at(buf, 0, (ROWS, 128), torch.uint8), _at(buf, 1024, (ROWS, 4), torch.uint8), 8, (ROWS, COLS))
    w = ops.MX(_at(buf, 2048, (N, 64), torch.uint8), _at(buf, 4096, (N, 4), torch.uint8), 4, (N, COLS))
    bias, plain = _at(buf, 5120, (N,), BF), _at(buf, 6144, (ROWS, COLS), BF)
    first = {"x codes": x.codes, "x scales": x.scales, "weight codes": w.codes, "weight scales": w.scales, "bias": bias,
             "bf16 x": plain, None: buf[8192:]}[over].data_ptr() - buf.data_ptr()
    out = _at(buf, first, (ROWS, N), BF)
    given = plain if over == "bf16 x" else x
    if over is None:
        assert ops.mx_linear(given, w, bias, out=out) is out and launched == ["fm_mx_linear"]
        return
    for at in (out, _at(buf, max(first - 48, 0), (ROWS, N), BF)):  # the same bytes, and with the last row
        with pytest.raises(ValueError, match="overlaps"):
            ops.mx_linear(given, w, bias, out=at)
    assert not launched


def test_rms_norm_weight(launched):
    """A float32 weight is read as it is; one of another type is read from a copy."""
    buf = torch.zeros(1 << 14, dtype=torch.uint8)
    x, r = _at(buf, 0, (ROWS, COLS), BF), _at(buf, 1024, (ROWS, COLS), BF)
    for first in (2048, 2048 + 2 * COLS, 2048 - 2 * COLS * (ROWS - 1)):
        with pytest.raises(ValueError, match="overlaps"):
            ops.rms_norm_mx(x, _at(buf, 2048, (COLS,), torch.float32), 1e-6, r, x_out=_at(buf, first, (ROWS, COLS), BF))
    assert not launched
    ops.rms_norm_mx(x, _at(buf, 2048, (COLS,), BF), 1e-6, r, x_out=_at(buf, 2048, (ROWS, COLS), BF))
    ops.rms_norm_mx(x, _at(buf, 2048, (COLS,), torch.float32), 1e-6, r, x_out=x)
    assert launched == ["fm_rms_norm_mx"] * 2


@pytest.mark.parametrize("over", ["gate", "per-row gate", "scale", "shift", None])
def test_adaln_vectors(launched, over):
    buf = torch.zeros(1 << 14, dtype=torch.uint8)
    x, y = _at(buf, 0, (ROWS, COLS), BF), _at(buf, 1024, (ROWS, COLS), BF)
    vectors = {"gate": _at(buf, 2048, (COLS,), BF), "per-row gate": _at(buf, 3072, (ROWS,), BF),
               "scale": _at(buf, 4096, (COLS,), BF), "shift": _at(buf, 5120, (COLS,), BF)}
    per_row = over == "per-row gate"
    gate = vectors["per-row gate" if per_row else "gate"]

    def call(out):
        return ops.adaln_residual_mx(x, y, gate, (vectors["scale"], vectors["shift"]), 1e-6, x_out=out,
                                     gate_per_row=per_row)

    if over is None:
        for out in (x, y, _at(buf, 6144, (ROWS, COLS), BF)):
            call(out)
        # rows of a wider buffer whose gap holds a vector
        wide = _at(buf, 8192, (ROWS, 2 * COLS), BF)
        vectors["scale"] = wide[1, COLS:]
        call(wide[:, :COLS])
        assert launched == ["fm_adaln_residual_mx"] * 4
        return
    at = vectors[over].data_ptr() - buf.data_ptr()
    for first in (at, at - 2 * COLS * (ROWS - 1)):
        with pytest.raises(ValueError, match="overlaps"):
            call(_at(buf, first, (ROWS, COLS), BF))
    assert not launched
