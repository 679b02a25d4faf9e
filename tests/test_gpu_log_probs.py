"""Log probabilities, ranks, entropies and likeliest tokens of rows of logits, against float64.

Bounds, in nats of float32 half steps u = 2^-24. A log probability is (x - m) / T - log S: the difference
and the quotient 2 u of |x - m| / T, the subtraction u of the result. S: each exponential's argument is off by
3 u of |x - m| / T (the difference, 1 / T, the product), where it matters at most by 3 u 20 (below exp(-20) of
the maximum the terms of 2^18 logits are under 2^-10 of it together, times 3 u 100), the exponential 2 u, the
joining of lanes, wavefronts and parts 40 u, so that log S is off by about 110 u; a lane's sums in between by u for
each of up to vocab / 512 additions in a row and by 3 u for each of up to vocab / 4096 tiles with a new maximum (the
exponential and the product); its own rounding u of it.
"""

import pytest
import torch

from flashmap_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _check(logits, tokens, top, temps, got: ops.LogProbs) -> None:
    x = logits.cpu().double()
    rows, vocab = x.shape
    t = torch.ones(rows, dtype=torch.float64) if temps is None else temps.cpu().double()
    m = x.amax(-1, keepdim=True)
    lp = torch.log_softmax(x / t[:, None], -1)
    d = ((x - m) / t[:, None]).abs()
    sums = 110 + vocab / 512 + 3 * vocab / 4096
    tol = 3 * U * d + sums * U + 2 * U * lp.abs()

    def near(a, want, tol):
        a = a.cpu().double()
        same = (a == want) | (a.isnan() & want.isnan())
        assert (same | ((a - want).abs() <= tol)).all(), (a - want).abs().nan_to_num(0, 0, 0).max()

    if tokens is not None:
        k = tokens.cpu().long()
        none = (k < 0) | (k >= vocab)
        at = k.clamp(0, vocab - 1)[:, None]
        want = torch.where(none, float("nan"), lp.gather(1, at)[:, 0])
        near(got.token, want, tol.gather(1, at)[:, 0])
        rank = (x > x.gather(1, at)).sum(-1) + 1
        assert torch.equal(got.rank.cpu(), torch.where(none, 0, rank))
    else:
        assert got.token is None and got.rank is None
    entropy = torch.where(m[:, 0].isfinite() & ~x.isnan().any(-1), torch.special.entr(lp.exp()).sum(-1), float("nan"))
    # log S, and D / S: its terms (x - m) / T off by 3 u of them, as S
    near(got.entropy, entropy, (10 + 2 * sums) * U * (1 + (lp.exp() * d.nan_to_num(0, 0, 0)).sum(-1)))
    assert got.top_ids.shape == got.top.shape == (rows, top)
    if top:
        order = torch.sort(torch.where(x.isnan(), float("inf"), x), dim=-1, descending=True, stable=True)
        nan_first = torch.sort((~x.isnan()).long().gather(1, order.indices), dim=-1, stable=True).indices
        ids = order.indices.gather(1, nan_first)[:, :top]
        assert torch.equal(got.top_ids.cpu(), ids)
        near(got.top, lp.gather(1, ids), tol.gather(1, ids))


def _logits(rows, vocab, dtype, seed, sigma=3.0):
    g = torch.Generator().manual_seed(seed)
    x = sigma * torch.randn(rows, vocab, generator=g)
    x[:, torch.randint(vocab, (8,), generator=g)] += 8
    return x.to(dtype), torch.randint(vocab, (rows,), generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 7, 0), (1, 100, 32), (2, 8191, 5), (4, 8192, 20),
                                            (3, 8193, 1), (2, 50257, 32), (1, 151936, 20), (7, 128256, 8)])
def test_sizes(dev, dtype, rows, vocab, top):
    x, k = _logits(rows, vocab, dtype, 1)
    x, k = x.to(dev), k.to(dev)
    _check(x, k, top, None, ops.log_probs_rows(x, k, top))
    temps = torch.linspace(0.3, 2.0, rows, device=dev)
    _check(x, k, top, temps, ops.log_probs_rows(x, k, top, temps))
    _check(x, None, top, temps, ops.log_probs_rows(x, None, top, temps))


def test_very_wide(dev):
    """More tiles than one step puts together."""
    x, k = _logits(2, 600_001, torch.bfloat16, 2)
    x, k = x.to(dev), k.to(dev)
    _check(x, k, 32, None, ops.log_probs_rows(x, k, 32))


def test_many_rows(dev):
    x, k = _logits(40_000, 65, torch.bfloat16, 3)
    x, k = x.to(dev), k.to(dev).int()
    _check(x, k, 3, None, ops.log_probs_rows(x, k, 3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(dev, dtype):
    """Rows that start anywhere, rows in between others, columns apart, one row for all."""
    base, _ = _logits(6, 20_011, dtype, 4)
    base = base.to(dev)
    k = torch.randint(0, 9_001, (3,), device=dev)
    for x in (base[1::2, 3:9_004], base[:3, 5:9_006], base[:3, ::2][:, :9_001], base[:1, 1:9_002].expand(3, -1)):
        _check(x, k, 9, None, ops.log_probs_rows(x, k, 9))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("left", [1, 3, 40, 5000])
def test_masked(dev, dtype, left):
    """Logits at -inf and at the type's lowest value but for a few."""
    x, _ = _logits(4, 30_000, dtype, 5)
    g = torch.Generator().manual_seed(6)
    keep = torch.randperm(30_000, generator=g)[:left]
    for low in (float("-inf"), torch.finfo(dtype).min):
        y = torch.full_like(x, low)
        y[:, keep] = x[:, keep]
        k = torch.stack([keep[0], keep[-1], torch.tensor(11), torch.tensor(29_999)]).to(dev)
        y = y.to(dev)
        _check(y, k, 20, None, ops.log_probs_rows(y, k, 20))


@pytest.mark.parametrize("value", [0.0, -3.5, float("-inf"), torch.finfo(torch.bfloat16).min,
                                   torch.finfo(torch.bfloat16).max])
def test_equal(dev, value):
    """Rows of one value: the lowest indexes; of -inf: NaN."""
    x = torch.full((3, 20_000), value, dtype=torch.bfloat16, device=dev)
    k = torch.tensor([0, 19_999, 5], device=dev)
    got = ops.log_probs_rows(x, k, 32)
    assert torch.equal(got.top_ids.cpu(), torch.arange(32).expand(3, 32)) and (got.rank == 1).all()
    if value == float("-inf"):
        assert got.token.isnan().all() and got.entropy.isnan().all() and got.top.isnan().all()
    else:
        _check(x, k, 32, None, got)


def test_ties_and_zeros(dev):
    """Few different values, both zeros among them: equal logits in the order of their indexes."""
    g = torch.Generator().manual_seed(7)
    values = torch.tensor([-1.0, -0.0, 0.0, 1.0])
    x = values[torch.randint(4, (5, 25_000), generator=g)]
    x[2, :] = values[torch.randint(3, (25_000,), generator=g)]
    x[3, :] = -1
    x[3, [24_999, 300, 8191, 8192]] = torch.tensor([0.0, -0.0, 0.0, -0.0])
    k = torch.tensor([3, 24_999, 8, 300, 0])
    for dtype in (torch.bfloat16, torch.float32):
        y = x.to(dtype).to(dev)
        _check(y, k.to(dev), 32, None, ops.log_probs_rows(y, k.to(dev), 32))


def test_sorted_rows(dev):
    """Rows in rising and falling order: every tile's largest lie side by side."""
    x = torch.linspace(-8, 8, 40_000)
    y = torch.stack([x, x.flip(0)]).to(dev)
    k = torch.tensor([0, 39_999], device=dev)
    _check(y, k, 32, None, ops.log_probs_rows(y, k, 32))


def test_not_finite(dev):
    """A NaN or +inf: NaN for every probability of its row, and the list still in order; no other row."""
    x, k = _logits(5, 20_000, torch.float32, 8)
    x[0, 777] = float("nan")
    x[1, 12_345] = float("inf")
    x[2, [5, 19_999, 9_000]] = torch.tensor([float("nan"), float("nan"), float("inf")])
    x[3, 4] = -float("nan")
    x, k = x.to(dev), k.to(dev)
    got = ops.log_probs_rows(x, k, 5)
    assert got.token[:4].isnan().all() and got.entropy[:4].isnan().all() and got.top[:4].isnan().all()
    assert got.top_ids[0, 0] == 777 and got.top_ids[1, 0] == 12_345 and got.top_ids[3, 0] == 4
    assert got.top_ids[2, :3].tolist() == [5, 19_999, 9_000]
    _check(x, k, 5, None, got)


def test_tokens_outside(dev):
    x, _ = _logits(4, 1000, torch.bfloat16, 9)
    k = torch.tensor([-1, 1000, 999, -2 ** 40], device=dev)
    x = x.to(dev)
    _check(x, k, 2, None, ops.log_probs_rows(x, k, 2))


def test_sampled_tokens(dev):
    """As a server uses it: the sampler's tokens and what the logits say of them."""
    x, _ = _logits(32, 32_000, torch.bfloat16, 10)
    x = x.to(dev)
    temps = torch.full((32,), 0.8, device=dev)
    greedy = torch.arange(32, device=dev) % 2 == 0
    tokens = ops.sample_rows(x, temps, greedy, torch.tensor(5, device=dev))
    got = ops.log_probs_rows(x, tokens, 4, temps)
    _check(x, tokens, 4, temps, got)
    assert (got.rank[greedy] == 1).all() and torch.equal(got.top_ids[greedy, 0], tokens[greedy])
    assert torch.equal(got.top_ids[:, 0], ops.argmax_rows(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 20_000), (9, 70_001), (1100, 9_000)])
@pytest.mark.parametrize("kind", ["rising", "falling", "two", "late", "lowest", "nan"])
def test_orders(dev, dtype, rows, vocab, kind):
    """Rows whose lists change with every tile, or in the last one alone; many equals; whole tiles of -inf or
    of the type's lowest value; NaN in one tile."""
    x, tokens = _logits(rows, vocab, dtype, 12)
    if kind in ("rising", "falling"):
        x = x.sort(-1, descending=kind == "falling").values
    elif kind == "two":
        x = torch.where(x > 0, 1.0, -1.0).to(dtype)
    elif kind == "nan":
        x[::3, vocab // 2] = float("nan")
    else:
        x[:, :vocab - 37] = torch.finfo(dtype).min if kind == "lowest" else float("-inf")
        tokens = vocab - 1 - tokens % 37
    x, tokens = x.to(dev), tokens.to(dev)
    for top in (1, 8, 32):
        _check(x, tokens, top, None, ops.log_probs_rows(x, tokens, top))
