"""The ends of what log probabilities take: temperatures next to zero, tokens that are NaN, and rows that
are cut into parts of several tiles, of small and of wide ones."""

import pytest
import torch

from flashmap_amd import ops
from test_gpu_log_probs import _check, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(6, 3000), (1100, 500)])
@pytest.mark.parametrize("temp", [2e-38, 4.2e-39, 1e-39, 1e-45])
def test_cold(dev, rows, vocab, temp):
    """Positive temperatures whose reciprocal float32 does not hold: all of a row on its largest logits."""
    x, k = _logits(rows, vocab, torch.float32, 20)
    x[::2, 17] = x[::2].amax(-1) + 1
    x[1::2, [5, 19]] = x[1::2].amax(-1, keepdim=True) + 1
    k[:2] = 17
    x, k, temps = x.to(dev), k.to(dev), torch.full((rows,), temp, device=dev)
    assert (temps > 0).all()
    got = ops.log_probs_rows(x, k, 3, temps)
    want = torch.zeros(rows, dtype=torch.float64)
    want[1::2] = torch.tensor(2.0, dtype=torch.float64).log()
    assert ((got.entropy.cpu() - want).abs() <= 2.0 ** -22).all()
    # a logit below the largest by d: d / T, at least 1e-7 / 2e-38, has left the result's range or is below -1e30
    first = torch.tensor([[17], [5]], device=dev).repeat(-(-rows // 2), 1)[:rows, 0]
    assert torch.equal(got.top_ids[:, 0], first) and torch.equal(got.top_ids[1::2, 1], torch.full_like(first[1::2], 19))
    assert ((got.top[:, 0].cpu() + want).abs() <= 2.0 ** -22).all()
    assert (got.top[::2, 1:] < -1e30).all() and (got.top[1::2, 2] < -1e30).all()
    assert got.token[0] == 0 and got.token[1] < -1e30
    assert not any(t.isnan().any() for t in (got.token, got.entropy, got.top))


@pytest.mark.parametrize("rows,vocab", [(6, 3000), (1100, 500)])
@pytest.mark.parametrize("temp", [1e10, 1e30, 3e38])
def test_hot(dev, rows, vocab, temp):
    """Temperatures that leave nothing of the logits' differences: even over all that are not masked."""
    x, k = _logits(rows, vocab, torch.float32, 21)
    x[:, 1::2] = float("-inf")
    x, k, temps = x.to(dev), k.to(dev), torch.full((rows,), temp, device=dev)
    _check(x, k, 3, temps, ops.log_probs_rows(x, k, 3, temps))


@pytest.mark.parametrize("rows,vocab", [(4, 9000), (1100, 500)])
def test_infinite_and_nan_tokens(dev, rows, vocab):
    """-inf is a probability of 0 and leaves the row's others alone; a NaN is the first of its row."""
    x, _ = _logits(rows, vocab, torch.bfloat16, 22)
    x[0, 7] = float("-inf")
    x[1, 7] = float("nan")
    x[2, 7] = float("inf")
    k = torch.full((rows,), 7, device=dev)
    x = x.to(dev)
    got = ops.log_probs_rows(x, k, 4)
    _check(x, k, 4, None, got)
    assert got.token[0] == float("-inf") and got.rank[0] == vocab and got.top[0].isfinite().all()
    assert got.entropy[0].isfinite()
    assert got.token[1].isnan() and got.token[2].isnan() and got.rank[1:3].tolist() == [1, 1]
    assert got.top[1:3].isnan().all() and got.top_ids[1, 0] == 7 and got.top_ids[2, 0] == 7
    assert got.top[3:].isfinite().all()


# Rows cut into parts of several tiles: wide tiles of 4096 logits (the first four), small ones of 2048. Where rows are
# fewer than 1024, 1024 / rows parts a row at most; wide where a row has at least as many wide tiles.
CUTS = [(61, 128_257), (200, 50_257), (700, 9_000), (600, 40_000), (64, 60_000), (128, 28_000), (33, 120_001)]


def _tiles(rows, vocab):
    """(logits of a tile, tiles of a part), as rows are cut."""
    most = -(-1024 // rows)
    tile = 2048 if -(-(vocab + 7) // 4096) < most else 4096
    return tile, -(-(-(-(vocab + 7) // tile)) // most)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", CUTS)
def test_parts_of_tiles(dev, dtype, rows, vocab):
    tile, tiles = _tiles(rows, vocab)
    assert tiles > 1 and tile == (2048 if (rows, vocab) in CUTS[4:] else 4096)
    # 11 columns aside, at every alignment of a row's start
    x, k = _logits(rows, vocab + 11, dtype, 23)
    x, k = x.to(dev), (k % vocab).to(dev)
    temps = torch.linspace(0.4, 1.7, rows, device=dev)
    for at, top, t in ((0, 20, None), (3, 32, temps), (11, 0, temps), (8, 1, None)):
        y = x[:, at:at + vocab]
        _check(y, k, top, t, ops.log_probs_rows(y, k, top, t))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(61, 128_257), (700, 9_000), (64, 60_000)])
@pytest.mark.parametrize("kind", ["rising", "falling", "equal", "ties", "ends", "late", "lowest", "nan", "first part"])
def test_parts_in_order(dev, dtype, rows, vocab, kind):
    """What the lists and sums carry from tile to tile, and what parts that hold nothing leave."""
    tile, tiles = _tiles(rows, vocab)
    x, k = _logits(rows, vocab, dtype, 24)
    edges = [c + o for c in range(tile, vocab, tile) for o in (-1, 0)]  # the ends of tiles (aligned rows) and parts
    if kind in ("rising", "falling"):
        x = x.sort(-1, descending=kind == "falling").values
    elif kind == "equal":
        x = torch.full_like(x, -2.5)
    elif kind == "ties":
        x = x.round().clamp(-3, 3)
    elif kind == "ends":
        x[:, edges] = 15.0
        k[::2] = edges[-1]
    elif kind == "nan":
        x[::3, edges[len(edges) // 2]] = float("nan")
        x[1::3, [edges[0], vocab - 1]] = float("nan")
    elif kind == "first part":
        x[:, tile * tiles:] = float("-inf")
    else:
        x[:, :vocab - 37] = torch.finfo(dtype).min if kind == "lowest" else float("-inf")
        k = vocab - 1 - k % 37
    x, k = x.to(dev), k.to(dev)
    for top in (1, 9, 32):
        _check(x, k, top, None, ops.log_probs_rows(x, k, top))
