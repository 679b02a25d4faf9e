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
