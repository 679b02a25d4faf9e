"""The microscaled oracle (oracle/mx.py) on the CPU: its grids are the formats' values, its
rounding the nearest with ties to even, and its blocks what the format says at the edges."""

import pytest
import torch

from oracle import mx


def test_grids():
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(every, torch.tensor(mx.E4M3, dtype=torch.float64))
    assert mx.E4M3[-1] == 448 and len(mx.E2M1) == 8


def test_rounding_to_eight_bits_is_the_types():
    v = torch.linspace(-448, 448, 40001)
    code = mx._nearest(v.double().abs(), mx.E4M3)
    want = v.to(torch.float8_e4m3fn).double().abs()
    assert torch.equal(torch.tensor(mx.E4M3, dtype=torch.float64)[code], want)


def test_rounding_to_four_bits():
    a = torch.tensor([0.25, 0.2501, 0.75, 0.7499, 1.25, 1.75, 2.5, 2.51, 3.5, 5.0, 5.01, 7.9])
    got = [mx.E2M1[i] for i in mx._nearest(a.double(), mx.E2M1)]
    assert got == [0.0, 0.5, 1.0, 0.5, 1.0, 2.0, 2.0, 3.0, 4.0, 4.0, 6.0, 6.0]


@pytest.mark.parametrize("bits,emax", [(8, 8), (4, 2)])
def test_blocks(bits, emax):
    v = torch.zeros(2, 161, dtype=torch.float64)
    v[0, 0], v[0, 33], v[0, 64], v[0, 100] = 1.0, float("inf"), 2.0 ** -140, -3.0
    v[1, 160] = float("nan")
    codes, scales = mx.quantize(v, bits)
    assert codes.shape == (2, 256) and scales.shape == (2, 8)
    assert scales[0].tolist() == [127 - emax, 255, 0, 128 - emax, 0, 0, 0, 0]
    assert scales[1].tolist() == [0, 0, 0, 0, 0, 255, 0, 0]
    back = mx.values(codes, scales, bits)
    assert back[0, 0] == 1 and back[0, 100] == -3 and torch.isnan(back[0, 32:64]).all()
    assert torch.isnan(back[1, 160:192]).all() and (back[1, :160] == 0).all()
