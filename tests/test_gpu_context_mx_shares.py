"""The attention over a 4-bit context where there is more to do than workgroups: shares of several steps and units,
units cut by them and joined, references that move, rings that are used again.

A share is one workgroup's, at most 3 a CU for up to 32 query rows a KV head and 2 for more, over the row groups of
64 rows; below that many steps of 128 positions every share is one step. Results are held to float64 by
_context_mx_norms."""

import pytest
import torch

from _context_mx_checks import BF, check
from _context_mx_norms import check_norm
from flashmap_amd import ops

pytestmark = pytest.mark.gpu


def _shares(dev, rows: int) -> int:
    """Workgroups of a row group for so many query rows a KV head, at most."""
    blocks = -(-rows // 16)
    groups = -(-blocks // 4)
    per_cu = 3 if -(-blocks // groups) <= 2 else 2
    return max(8, per_cu * torch.cuda.get_device_properties(dev).multi_processor_count // groups // 8 * 8)


def _steps(lens) -> int:
    return sum(-(-n // 128) for n in lens)


def _cache(lens, hkv, d, page, seed, dev):
    """(cache of random codes and scales, block table, contexts as float64 on the GPU)."""
    g = torch.Generator(dev).manual_seed(seed)
    pages = [-(-n // page) for n in lens]
    blocks = sum(pages) + 2
    rows = blocks * hkv * page
    codes = torch.randint(0, 256, (rows, d), dtype=torch.uint8, generator=g, device=dev)
    scales = torch.randint(122, 130, (rows, d // 16), dtype=torch.uint8, generator=g, device=dev)
    scales[:, :d // 32] = torch.randint(124, 126, (rows, d // 32), dtype=torch.uint8, generator=g, device=dev)
    order = torch.randperm(blocks, generator=g, device=dev)
    table = torch.full((len(lens), max(1, max(pages))), 10 ** 6, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    cache = ops.MX(codes, scales, 4, (blocks, hkv, page, 2 * d))
    return cache, table, [_context(cache, table[b], n) for b, n in enumerate(lens)]


VALUES = [0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6]


def _context(cache, pages, n):
    """A request's positions (n, hkv, 2 D) in float64."""
    blocks, hkv, page, d2 = cache.shape
    ids = pages[:-(-n // page)].long()
    codes, scales = (t.view(blocks, hkv, page, -1)[ids].transpose(1, 2).reshape(-1, hkv, t.shape[-1])[:n]
                     for t in (cache.codes, cache.scales))
    values = torch.tensor(VALUES, dtype=torch.float64, device=codes.device)
    y = values[torch.stack([codes & 15, codes >> 4], -1).int()].view(n, hkv, d2 // 32, 32)
    return (y * torch.exp2(scales.double() - 127)[..., None]).view(n, hkv, d2)


def _run(cache, table, lens, q_lens, hq, d, seed, dev):
    g = torch.Generator(dev).manual_seed(seed)
    query = torch.randn(sum(q_lens), hq, d, generator=g, device=dev).to(BF)
    cu = torch.tensor([0, *torch.tensor(q_lens).cumsum(0).tolist()], dtype=torch.int32, device=dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    return query, ops.block_attention_paged_mx(query, cache, cu, seq, table, max(q_lens), max(lens), d ** -0.5)


# Query rows a KV head: 1 to 4 row blocks, two row groups of 4, three of 3.
ROWS = [(1, 4), (16, 1), (16, 2), (9, 5), (16, 4), (32, 4), (48, 3)]


def _cost(dev, q_len, group, hkv, most):
    """Lengths, of no position and of one to long ones, with ``hkv`` KV heads `most` times as many steps as shares."""
    wanted = most * _shares(dev, q_len * group) // hkv
    few = [0, 1, 128, 129, 300, 40, 0, 7, 7, 7, 257, 1000]
    left = max(wanted - _steps(few), 3)
    return few[:6] + [128 * (left * 2 // 3) - 77] + few[6:] + [128 * (left // 3) + 5, 0]


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("most", [2, 5, 13, 26])
@pytest.mark.parametrize("q_len,group", ROWS)
def test_shares(dev, d, most, q_len, group):
    """Units of all lengths, several in a share and one in several, at every size of a unit's own cost."""
    hkv = 64
    lens = _cost(dev, q_len, group, hkv, most)
    assert hkv * _steps(lens) > (most - 1) * _shares(dev, q_len * group)
    cache, table, rows = _cache(lens, hkv, d, 16, most, dev)
    q_lens = [max(1, q_len - 3 * b % q_len) for b in range(len(lens))]
    q_lens[0] = q_len
    query, out = _run(cache, table, lens, q_lens, hkv * group, d, 7, dev)
    check_norm(out, query, rows, q_lens, d ** -0.5)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("q_len,group", [(1, 1), (16, 2), (16, 4), (32, 4)])
def test_few_units(dev, d, q_len, group):
    """Long contexts of few KV heads: units of many shares each, joined by several workgroups."""
    hkv, lens = 4, [50_001, 20_000, 30_123]
    most = 2 if q_len == 1 else 3
    lens = [n * (2 if q_len * group <= 32 else 1) for n in lens]
    assert hkv * _steps(lens) > most * _shares(dev, q_len * group)
    cache, table, rows = _cache(lens, hkv, d, 24, 3, dev)
    query, out = _run(cache, table, lens, [q_len] * 3, hkv * group, d, 4, dev)
    check_norm(out, query, rows, [q_len] * 3, d ** -0.5)


@pytest.mark.parametrize("d", [128, 64])
def test_edges_win(dev, d):
    """Queries that are the key of a position at a step's, a tile's or the context's end, sharply scaled: it outweighs
    all others, or nearly."""
    hkv, lens = 16, [30_000, 1, 9_217, 14_976]
    assert hkv * _steps(lens) > 8 * _shares(dev, 16)
    cache, table, rows = _cache(lens, hkv, d, 16, 5, dev)
    g = torch.Generator().manual_seed(6)
    picks = []
    for n in lens:
        step = 128 * torch.randint(max(1, n // 128), (4,), generator=g)
        tile = 32 * torch.randint(max(1, n // 32), (3,), generator=g)
        picks.append(torch.cat([step, step + 127, tile, tile + 31, torch.tensor([0, n - 1])]).clamp(max=n - 1))
    query = torch.cat([kv[at.to(dev), :, :d] for kv, at in zip(rows, picks)]).to(BF)
    # A query is exactly a key, whose few different magnitudes are rounded alike, not independently: the worst case of
    # each value holds, the norms' bound does not.
    out = ops.block_attention_paged_mx(query, cache, None, torch.tensor(lens, device=dev), table, 16, 30_000, 1.0)
    check(out, query, [kv.cpu() for kv in rows], [16] * 4, 1.0)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("q_len,group", [(16, 1), (16, 2), (12, 4), (16, 4), (32, 4)])
def test_references_move(dev, d, q_len, group):
    """Scores that pass their row's reference by more than 2^8 again and again inside a share, for half of the rows;
    for the others, scores that fall as far. A level's positions weigh as much together as the few above them."""
    hkv, n = 16, 30_000
    assert hkv * _steps([n]) > 4 * _shares(dev, q_len * group)
    g = torch.Generator(dev).manual_seed(8)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=dev)
    kv = rand(n, hkv, 2 * d)
    level = torch.where(torch.arange(n, device=dev) % 15_000 < 9_000, 0.0, 3.0)
    level[torch.randperm(n, generator=g, device=dev)[:24]] += 3.0
    kv[..., :32] = level[:, None, None]
    rows = -(-n // 16) * 16
    held = torch.zeros(rows, hkv, 2 * d, device=dev)
    held[:n] = kv
    cache = ops.mx_quantize(held.view(-1, 16, hkv, 2 * d).transpose(1, 2).contiguous(), 4)
    table = torch.arange(rows // 16, dtype=torch.int32, device=dev)[None]
    query = rand(q_len, hkv * group, d)
    # 32 channels of 0.5 to 1.5 each: a level of 3 is 32 * 3 * scale, 8 (D 128) or 12 (D 64) times log2(e)
    query[..., :32] = 0.5 + torch.rand(q_len, hkv * group, 32, generator=g, device=dev)
    query[::2, :, :32] *= -1
    query = query.to(BF)
    out = ops.block_attention_paged_mx(query, cache, None, torch.tensor([n], device=dev), table, q_len, n, d ** -0.5)
    context = [_context(cache, table[0], n)]
    for odd in (0, 1):  # rows of either kind apart
        part = slice(odd, None, 2)
        check_norm(out[part], query[part], context, [len(out[part])], d ** -0.5)


def test_captured_lengths(dev):
    """One captured call, replayed over contexts that grow, end and are cut in other places."""
    hkv, d, q_len = 32, 128, 16
    lens = [6_000, 20, 9_000, 300, 2_000]
    cache, table, _ = _cache(lens, hkv, d, 16, 9, dev)
    query = torch.randn(5 * q_len, hkv, d, generator=torch.Generator(dev).manual_seed(1), device=dev).to(BF)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    run = lambda: ops.block_attention_paged_mx(query, cache, None, seq, table, q_len, 9_000, d ** -0.5)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for now in ([6_000, 20, 9_000, 300, 2_000], [1, 0, 2, 0, 3], [5_999, 1, 8_193, 0, 128], [0, 0, 0, 0, 0],
                [64, 20, 9_000, 300, 1_024], lens):
        seq.copy_(torch.tensor(now, dtype=torch.int32))
        want = run()
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check_norm(out, query, [_context(cache, table[b], n) for b, n in enumerate(now)], [q_len] * 5, d ** -0.5)


def _rotated(query, weight, angles, at):
    """Norm and rotation in float64: what attends."""
    x = query.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.double()
    e, o, (c, s) = x[..., 0::2], x[..., 1::2], angles.double()[at][:, None].unbind(-1)
    return torch.stack([e * c - o * s, o * c + e * s], -1).flatten(-2)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("q_len,group", ROWS)
@pytest.mark.parametrize("table_of", ["interleaved", "apart"])
def test_prologue_and_query_as_out(dev, d, q_len, group, table_of):
    """The next unit's positions, rotary rows and queries fetched while one ends, and written over as results."""
    hkv, most = 16, 9
    lens = _cost(dev, q_len, group, hkv, most)
    assert hkv * _steps(lens) > (most - 1) * _shares(dev, q_len * group)
    cache, table, rows = _cache(lens, hkv, d, 8, 11, dev)
    g = torch.Generator(dev).manual_seed(12)
    q_lens = [max(1, q_len - 5 * b % q_len) for b in range(len(lens))]
    q_lens[-1] = q_len
    tokens = sum(q_lens)
    query = (3 * torch.randn(tokens, hkv * group, d, generator=g, device=dev)).to(BF)
    weight = 0.5 + torch.rand(d, generator=g, device=dev)
    angle = torch.arange(900, device=dev).double()[:, None] * 1e4 ** -(torch.arange(0, d, 2, device=dev).double() / d)
    angles = torch.stack([angle.cos(), angle.sin()], -1).float()
    at = torch.randint(0, 900, (tokens,), generator=g, device=dev)
    rope = ops.rope_from_table(angles) if table_of == "interleaved" else ops.rope_from_split(*angles.unbind(-1))
    cu = torch.tensor([0, *torch.tensor(q_lens).cumsum(0).tolist()], dtype=torch.int32, device=dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    args = cache, cu, seq, table, q_len, max(lens), d ** -0.5, ops.Prologue(weight, rope, at, 1e-6)
    out = ops.block_attention_paged_mx(query, *args)
    check_norm(out, _rotated(query, weight, angles, at), rows, q_lens, d ** -0.5)
    same = query.clone()
    assert torch.equal(ops.block_attention_paged_mx(same, *args, out=same), out)


@pytest.mark.parametrize("q_len,group", [(3, 1), (16, 4)])
def test_many_requests(dev, q_len, group):
    """More requests than a launch takes, each launch with more steps than shares."""
    hkv, d = 32, 64
    g = torch.Generator().manual_seed(13)
    lens = torch.randint(0, 700, (600,), generator=g).tolist()
    lens[255], lens[256], lens[511], lens[512], lens[599] = 600, 0, 0, 650, 1
    for first in (0, 256):
        assert hkv * _steps(lens[first:first + 256]) > 4 * _shares(dev, q_len * group)
    cache, table, rows = _cache(lens, hkv, d, 16, 14, dev)
    q_lens = [1 + b % q_len for b in range(600)]
    query, out = _run(cache, table, lens, q_lens, hkv * group, d, 15, dev)
    some = [0, 1, 2, 100, 254, 255, 256, 257, 300, 511, 512, 513, 598, 599]
    starts = [0, *torch.tensor(q_lens).cumsum(0).tolist()]
    for b in some:
        part = slice(starts[b], starts[b + 1])
        check_norm(out[part], query[part], [rows[b]], [q_lens[b]], d ** -0.5)
    # the others as calls of their own: the same terms, in another order of sums
    for first in range(0, 600, 100):
        part = slice(starts[first], starts[first + 100])
        cu = torch.tensor(starts[first:first + 101], dtype=torch.int32, device=dev) - starts[first]
        few = ops.block_attention_paged_mx(query[part], cache, cu, torch.tensor(lens[first:first + 100], device=dev),
                                           table[first:first + 100], q_len, 700, d ** -0.5)
        assert (few.float() - out[part].float()).abs().max() <= 2.0 ** -7 * out.float().abs().max()
