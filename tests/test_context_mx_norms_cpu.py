"""The bound on the 4-bit contexts' attention as a whole: the kernel's own roundings, made here in float64, pass it on
every kind of input, and one mistake at a time does not."""

import pytest
import torch

from _context_mx_checks import check, make
from _context_mx_norms import attention, check_norm

LOG2E = 1.4426950408889634


def _two_operands(x: torch.Tensor, second: bool = True) -> torch.Tensor:
    """Rows as sums of two e4m3 operands, a power of two for every 32 channels."""
    blocks = x.unflatten(-1, (-1, 32))
    unit = torch.exp2(torch.floor(torch.log2(blocks.abs().amax(-1, keepdim=True).clamp(min=1e-30))) - 7)
    hi = (blocks / unit).float().to(torch.float8_e4m3fn).double() * unit
    lo = ((blocks - hi) / unit * 32).float().to(torch.float8_e4m3fn).double() * unit / 32
    return (hi + lo if second else hi).flatten(-2)


def _attend(query, rows, lens_q, scale, mistake=None):
    at, outs, d = 0, [], query.shape[-1]
    for kv, n in zip(rows, lens_q):
        q = query[at:at + n].double()
        at += n
        if mistake == "last position":
            kv = kv[:-1]
        elif mistake == "last step":
            kv = kv[:-128]
        elif mistake == "half":
            kv = kv[:kv.shape[0] // 2]
        elif mistake == "position again":
            kv = torch.cat([kv, kv[-1:]])
        x = _two_operands(q * (scale * LOG2E * (1.02 if mistake == "scale" else 1.0)), mistake != "operand")
        out = torch.empty_like(q)
        for h in range(q.shape[1]):
            k, v = (t[:, h // (q.shape[1] // kv.shape[1])] for t in (kv[..., :d], kv[..., d:]))
            s = x[:, h] @ k.T.contiguous()
            if mistake == "mean":
                s = torch.zeros_like(s)
            if mistake == "neighbour":  # the keys of the next position
                s = s.roll(1, -1)
            p = torch.exp2(s - s.amax(-1, keepdim=True) - 7)
            p = p.to(torch.float8_e4m3fn).double() if mistake == "probabilities" else p.bfloat16().double()
            out[:, h] = p @ v / p.sum(-1, keepdim=True)
        outs.append(out * {"larger": 1.02, "zeros": 0.0}.get(mistake, 1.0))
    return torch.cat(outs).bfloat16()


KINDS = {
    "one": dict(lens=[1], lens_q=[16], hq=4, hkv=2, d=128),
    "short": dict(lens=[2, 5, 31, 33], lens_q=[4, 4, 4, 4], hq=2, hkv=2, d=64),
    "token": dict(lens=[77, 450], lens_q=[1, 1], hq=8, hkv=1, d=128),
    "blocks": dict(lens=[130, 999, 400], lens_q=[3, 16, 7], hq=4, hkv=2, d=128),
    "middle": dict(lens=[700, 1500], lens_q=[16, 16], hq=4, hkv=1, d=128),
    "narrow": dict(lens=[700, 1500], lens_q=[16, 16], hq=4, hkv=2, d=64),
    "long": dict(lens=[20_000], lens_q=[2], hq=2, hkv=1, d=128),
}


def _inputs(kind, seed):
    c = KINDS[kind]
    _, _, rows = make(c["lens"], c["hkv"], c["d"], 16, seed, "cpu")
    g = torch.Generator().manual_seed(seed + 1)
    query = torch.randn(sum(c["lens_q"]), c["hq"], c["d"], generator=g).bfloat16()
    return query, rows, c["lens_q"], c["d"] ** -0.5


@pytest.mark.parametrize("kind", KINDS)
def test_own_roundings_pass(kind):
    for seed in range(1, 2 if kind == "long" else 5):
        inputs = _inputs(kind, seed)
        worst = check_norm(_attend(*inputs), *inputs)
        assert worst == 0 if kind == "one" else 0.2 < worst < 0.95  # one position's 4-bit values: bf16 holds them
        # and the exact result, but for its own rounding
        assert check_norm(torch.cat([o for o, _ in attention(*inputs)]).bfloat16(), *inputs) < 0.65


@pytest.mark.parametrize("kind", [k for k in KINDS if k not in ("one", "short")])
@pytest.mark.parametrize("mistake", ["zeros", "larger", "mean", "half", "scale", "operand", "probabilities", "neighbour",
                                     "last step", "last position", "position again"])
def test_mistakes_do_not(kind, mistake):
    if kind == "long" and mistake in ("last position", "position again"):
        pytest.skip("one of 20000 equals")  # tests of long contexts make such positions outweigh the others
    if kind == "token" and mistake == "last step":
        pytest.skip("no such step")
    inputs = _inputs(kind, 1)
    with pytest.raises(AssertionError, match="off by"):
        check_norm(_attend(*inputs, mistake), *inputs)


@pytest.mark.parametrize("d", [128, 64])
def test_missing_positions(d):
    """Sharply scaled queries that are a position's key: the bound a value rejects a result without that position."""
    g = torch.Generator().manual_seed(3)
    n, values = 1500, torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    kv = values[torch.randint(8, (n, 1, 2 * d), generator=g)] * (2 * torch.randint(2, (n, 1, 2 * d), generator=g) - 1)
    kv[..., :d] /= 2.0 ** torch.randint(2, 4, (n, 1, d // 32), generator=g).repeat_interleave(32, -1)
    picks = [0, 31, 32, 127, 128, 640, n - 1]
    query = kv[picks, :, :d]

    def result(kv):
        return (torch.softmax(query[:, 0] @ kv[:, 0, :d].T, -1) @ kv[:, 0, d:])[:, None].bfloat16()

    check(result(kv), query, [kv], [len(picks)], 1.0)
    for p in picks:
        with pytest.raises(AssertionError, match="off"):
            check(result(torch.cat([kv[:p], kv[p + 1:]])), query, [kv], [len(picks)], 1.0)
