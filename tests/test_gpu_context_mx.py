"""Contexts in microscaled 4 bits on the GPU: appending to them and attending over them, against
float64 (the bounds stand in _context_mx_checks.py and beside the tests)."""

import pytest
import torch

from _context_mx_checks import BF, cache_of, cache_values, check, make
from _mx_checks import check_between
from flashmap_amd import ops
from oracle import mx

pytestmark = pytest.mark.gpu


def _table(positions, d, dev, theta=1e4):
    angle = torch.arange(positions).double()[:, None] * theta ** -(torch.arange(0, d, 2).double() / d)
    return torch.stack([angle.cos(), angle.sin()], -1).float().to(dev)


def _attend(cache, table, lens, lens_q, hq, d, dev, seed, scale=None, q_scale=1.0, ragged=True):
    g = torch.Generator().manual_seed(seed)
    scale = d ** -0.5 if scale is None else scale
    query = (torch.randn(sum(lens_q), hq, d, generator=g) * q_scale).to(BF).to(dev)
    cu = torch.tensor([0, *torch.tensor(lens_q).cumsum(0).tolist()], dtype=torch.int32, device=dev) if ragged else None
    seqused = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = ops.block_attention_paged_mx(query, cache, cu, seqused, table, max(lens_q), max(max(lens), 1), scale)
    return out, query, scale


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("lens", [[1], [31], [32], [33], [127, 128, 129], [0, 5, 0, 300, 0], [700, 0], [1500]])
def test_lengths(dev, d, lens):
    cache, table, rows = make(lens, 2, d, 16, 1, dev)
    out, q, scale = _attend(cache, table, lens, [16] * len(lens), 4, d, dev, 2)
    check(out, q, rows, [16] * len(lens), scale)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("hkv,group,q_len", [(1, 1, 1), (2, 1, 16), (3, 2, 16), (1, 3, 16), (2, 4, 16), (1, 5, 16),
                                             (1, 8, 1), (2, 1, 17), (1, 1, 200), (1, 16, 9), (5, 1, 3), (1, 6, 40)])
def test_rows(dev, d, hkv, group, q_len):
    lens = [77, 450, 3]
    cache, table, rows = make(lens, hkv, d, 16, 3, dev)
    out, q, scale = _attend(cache, table, lens, [q_len] * 3, hkv * group, d, dev, 4, ragged=False)
    check(out, q, rows, [q_len] * 3, scale)


@pytest.mark.parametrize("page", [1, 2, 5, 8, 16, 24, 64, 1000])
def test_pages(dev, page):
    lens = [130, 1, 999, 40]
    cache, table, rows = make(lens, 2, 128, page, 5, dev)
    out, q, scale = _attend(cache, table, lens, [3, 16, 1, 7], 4, 128, dev, 6)
    check(out, q, rows, [3, 16, 1, 7], scale)


@pytest.mark.parametrize("d", [128, 64])
def test_one_position_wins(dev, d):
    """Queries that are a stored key, sharply scaled: the output is that position's values."""
    lens = [257, 64, 640]
    cache, table, rows = make(lens, 2, d, 8, 7, dev)
    picks = [[0, 31, 32, 256], [63, 1, 5, 33], [639, 512, 127, 128]]
    query = torch.stack([rows[b][i, :, :d] for b in range(3) for i in picks[b]]).to(BF)
    out = ops.block_attention_paged_mx(query.to(dev), cache, None, torch.tensor(lens, device=dev), table, 4, 640, 1.0)
    want = torch.stack([rows[b][i, :, d:] for b in range(3) for i in picks[b]])
    # k.k is about D, k.k' about sqrt(D): exp(-(64 - 5 * 8)) of the others
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-6).all()


def test_many_requests(dev):
    """More requests than a launch takes, lengths from none to many."""
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(0, 90, (600,), generator=g).tolist()
    cache, table, rows = make(lens, 1, 64, 16, 9, dev)
    out, q, scale = _attend(cache, table, lens, [2] * 600, 2, 64, dev, 10)
    check(out, q, rows, [2] * 600, scale)
    out2, q, _ = _attend(cache, table, lens, [2] * 600, 2, 64, dev, 10, ragged=False)
    assert torch.equal(out, out2)


def test_long_context(dev):
    """A context cut over many shares, beside a short one."""
    lens = [70000, 3]
    cache, table, rows = make(lens, 1, 128, 16, 11, dev)
    out, q, scale = _attend(cache, table, lens, [2, 2], 2, 128, dev, 12)
    check(out, q, rows, [2, 2], scale)


def test_rows_behind_are_left(dev):
    lens = [100, 40]
    cache, table, rows = make(lens, 2, 128, 16, 13, dev)
    query = torch.randn(20, 2, 128, device=dev).to(BF)
    out = torch.full_like(query, 7.0)
    cu = torch.tensor([0, 5, 9], dtype=torch.int32, device=dev)
    ops.block_attention_paged_mx(query, cache, cu, torch.tensor(lens, device=dev), table, 8, 128, 0.1, out=out)
    assert (out[9:] == 7).all()
    check(out[:9], query[:9], rows, [5, 4], 0.1)
    # more rows than max_seqlen_q: the first ones
    out.fill_(7.0)
    ops.block_attention_paged_mx(query, cache, cu, torch.tensor(lens, device=dev), table, 3, 128, 0.1, out=out)
    assert (out[3:5] == 7).all() and (out[8:] == 7).all()
    check(out[[0, 1, 2, 5, 6, 7]], query[[0, 1, 2, 5, 6, 7]], rows, [3, 3], 0.1)
    # what cu_seqlens_q says past the query's rows is not read
    ops.block_attention_paged_mx(query[:9], cache, torch.tensor([0, 5, 50], dtype=torch.int32, device=dev),
                                 torch.tensor(lens, device=dev), table, 60, 128, 0.1)


def test_lengths_are_bounded(dev):
    """A length past max_seqlen_k or the table, or below 0, is cut; a page that is none is page 0."""
    cache, table, rows = make([64, 64], 2, 128, 16, 14, dev)
    out, q, scale = _attend(cache, table, [64, 64], [4, 4], 2, 128, dev, 15)
    seq = torch.tensor([10 ** 9, -5], dtype=torch.int32, device=dev)
    cut = ops.block_attention_paged_mx(q, cache, None, seq, table, 4, 10 ** 6, scale)
    assert torch.equal(cut[:4], out[:4]) and (cut[4:] == 0).all()
    cut = ops.block_attention_paged_mx(q, cache, None, seq, table, 4, 20, scale)
    check(cut, q, [rows[0][:20], rows[1][:0]], [4, 4], scale)
    bad = table.clone()
    bad[0, 1], bad[1, 0] = -7, 2 ** 31 - 1
    first = cache_values(cache)[0].transpose(0, 1)
    rows[0][16:32], rows[1][:16] = first, first
    got = ops.block_attention_paged_mx(q, cache, None, torch.tensor([64, 64], device=dev), bad, 4, 64, scale)
    check(got, q, rows, [4, 4], scale)


@pytest.mark.parametrize("d,hq,hkv,q_len", [(128, 4, 2, 16), (64, 6, 2, 9), (128, 8, 1, 16), (128, 1, 1, 1)])
def test_prologue(dev, d, hq, hkv, q_len):
    """The norm and rotation on the way, against float64: the query's 8 bits are its one rounding, 2^-8 of a
    channel (float32's own are below 2^-20)."""
    lens = [50, 333]
    cache, table, rows = make(lens, hkv, d, 16, 16, dev)
    g = torch.Generator().manual_seed(17)
    query = (3 * torch.randn(2 * q_len, hq, d, generator=g)).to(BF)
    weight = 0.5 + torch.rand(d, generator=g)
    angles = _table(400, d, "cpu")
    pos = torch.cat([n + torch.arange(q_len) for n in lens])
    seq = torch.tensor(lens, device=dev)
    x = query.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.double()

    def turned(at):
        e, o, c, s = x[..., 0::2], x[..., 1::2], *angles.double()[at][:, None].unbind(-1)
        return torch.stack([e * c - o * s, o * c + e * s], -1).flatten(-2)

    for layout in (ops.rope_from_table(angles.to(dev)), ops.rope_from_split(*angles.to(dev).unbind(-1)),
                   ops.rope_from_cat(torch.cat(angles.unbind(-1), -1).to(dev))):
        got = ops.block_attention_paged_mx(query.to(dev), cache, None, seq, table, q_len, 333, d ** -0.5,
                                           prologue=ops.Prologue(weight.to(dev), layout, pos.to(dev), 1e-6))
        check(got, turned(pos), rows, [q_len] * 2, d ** -0.5, 2.0 ** -8)
    # without positions, a query row's own table row
    got = ops.block_attention_paged_mx(query.to(dev), cache, None, seq, table, q_len, 333, d ** -0.5,
                                       prologue=ops.Prologue(weight.to(dev), layout, None, 1e-6))
    check(got, turned(torch.arange(2 * q_len)), rows, [q_len] * 2, d ** -0.5, 2.0 ** -8)


def test_query_range(dev):
    """Query channels of very different sizes: what lies within 2^13 of a block's largest is exact."""
    lens = [90]
    cache, table, rows = make(lens, 1, 128, 16, 18, dev)
    g = torch.Generator().manual_seed(19)
    query = torch.randn(16, 1, 128, generator=g) * 2.0 ** torch.randint(-12, 1, (16, 1, 128), generator=g)
    for factor in (1.0, 2.0 ** -60, 2.0 ** 60):
        q = (query * factor).to(BF).to(dev)
        out = ops.block_attention_paged_mx(q, cache, None, torch.tensor(lens, device=dev), table, 16, 90, 0.3 / factor)
        check(out, q, rows, [16], 0.3 / factor)


def test_scales_of_all_sizes(dev):
    """Blocks whose scales lie far apart, zero blocks and the smallest scale."""
    g = torch.Generator().manual_seed(20)
    values = torch.randn(4, 1, 16, 256, generator=g, dtype=torch.float64)
    values[..., 128:] *= 2.0 ** torch.randint(-40, 40, (4, 1, 16, 4), generator=g).repeat_interleave(32, -1)
    values[1, 0, :, 128:160] = 0
    values[2, 0, 3, :] = 0
    values[..., 192:224] *= 2.0 ** -100
    cache = cache_of(values, dev)
    rows = [cache_values(cache)[[2, 0, 3, 1]].permute(0, 2, 1, 3).reshape(-1, 1, 256)[:60]]
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device=dev)
    q = torch.randn(16, 1, 128, generator=g).to(BF).to(dev)
    out = ops.block_attention_paged_mx(q, cache, None, torch.tensor([60], device=dev), table, 16, 64, 0.1)
    check(out, q, rows, [16], 0.1)


def test_nan_blocks(dev):
    """A key block that is NaN makes its head's rows NaN, a value block its channels; no others."""
    lens = [40, 40]
    cache, table, rows = make(lens, 2, 128, 8, 21, dev)
    q = torch.randn(8, 2, 128, device=dev).to(BF)
    seq = torch.tensor(lens, device=dev)
    clean = ops.block_attention_paged_mx(q, cache, None, seq, table, 4, 40, 0.1)
    row = (int(table[0, 2]) * 2 + 1) * 8 + 3  # request 0, head 1, position 19
    scales = cache.scales.clone()
    scales[row, 1] = 255
    got = ops.block_attention_paged_mx(q, ops.MX(cache.codes, scales, 4, cache.shape), None, seq, table, 4, 40, 0.1)
    assert got[:4, 1].isnan().all()
    assert torch.equal(got[:4, 0], clean[:4, 0]) and torch.equal(got[4:], clean[4:])
    scales = cache.scales.clone()
    scales[row, 4 + 2] = 255
    got = ops.block_attention_paged_mx(q, ops.MX(cache.codes, scales, 4, cache.shape), None, seq, table, 4, 40, 0.1)
    assert got[:4, 1, 64:96].isnan().all()
    clean[:4, 1, 64:96] = 0
    got[:4, 1, 64:96] = 0
    assert torch.equal(got, clean)
    # positions behind a context's end may hold anything
    got = ops.block_attention_paged_mx(q, ops.MX(cache.codes, scales, 4, cache.shape), None,
                                       torch.tensor([19, 40], device=dev), table, 4, 40, 0.1)
    assert not got.isnan().any()
    # a query with an infinity or a NaN: its own rows only
    for v in (float("inf"), float("nan")):
        bad = q.clone()
        bad[1, 0, 5] = v
        got = ops.block_attention_paged_mx(bad, cache, None, seq, table, 4, 40, 0.1)
        assert got[1, 0].isnan().all() and int(got.isnan().sum()) == 128


def test_strides(dev):
    """Rows of a wider query, of a wider out, of caches inside wider rows, and the query as out."""
    lens = [200, 90]
    cache, table, rows = make(lens, 2, 128, 16, 22, dev)
    wide = torch.randn(10, 4, 256, device=dev).to(BF)
    q = wide[:, :, 128:]
    seq = torch.tensor(lens, device=dev)
    want = ops.block_attention_paged_mx(q.contiguous(), cache, None, seq, table, 5, 200, 0.1)
    codes = torch.zeros(cache.codes.shape[0], 160, dtype=torch.uint8, device=dev)
    codes[:, :128], codes[:, 144:152] = cache.codes, cache.scales
    inside = ops.MX(codes[:, :128], codes[:, 144:152], 4, cache.shape)
    out = torch.zeros(10, 4, 136, device=dev, dtype=BF)[:, :, :128]
    got = ops.block_attention_paged_mx(q, inside, None, seq, table, 5, 200, 0.1, out=out)
    assert got is out and torch.equal(out, want)
    table64 = torch.full((2, 2 * table.shape[1]), 3, dtype=torch.int64, device=dev)
    table64[:, ::2] = table
    assert torch.equal(ops.block_attention_paged_mx(q, inside, None, seq.long(), table64[:, ::2], 5, 200, 0.1), want)
    same = q.contiguous()
    assert torch.equal(ops.block_attention_paged_mx(same, cache, None, seq, table, 5, 200, 0.1, out=same), want)


def test_large_cache(dev):
    """Rows past 2^32 bytes: two pages, the first and the last of 5 GB."""
    blocks = 40_000_000 // 16
    codes = torch.zeros(blocks * 16, 128, dtype=torch.uint8, device=dev)
    scales = torch.zeros(blocks * 16, 8, dtype=torch.uint8, device=dev)
    cache = ops.MX(codes, scales, 4, (blocks, 1, 16, 256))
    g = torch.Generator().manual_seed(23)
    kv = torch.randn(32, 1, 2, 1, 128, generator=g).to(BF).to(dev)
    slots = torch.cat([torch.arange(16), blocks * 16 - 16 + torch.arange(16)]).to(dev)
    ops.write_context_kv_mx(kv, torch.zeros(32, dtype=torch.int64, device=dev), slots, torch.ones(128, device=dev),
                            ops.rope_from_table(_table(2, 128, dev)), [cache], 1e-6)
    ends = torch.cat([codes[:16], codes[-16:]]), torch.cat([scales[:16], scales[-16:]])
    assert (ends[0] != 0).any(1).all() and int((codes != 0).any(1).sum()) == 32
    rows = [cache_values(ops.MX(*ends, 4, (32, 1, 1, 256))).view(32, 1, 256)]
    q = torch.randn(4, 1, 128, generator=g).to(BF).to(dev)
    table = torch.tensor([[0, blocks - 1]], dtype=torch.int32, device=dev)
    out = ops.block_attention_paged_mx(q, cache, None, torch.tensor([32], device=dev), table, 4, 32, 0.1)
    check(out, q, rows, [4], 0.1)


# ------------------------------------------------------------------------------- appending


def _written(kv, positions, weight, table, eps):
    """Float64 rows (tokens, layers, heads, 2 D) that a write quantizes, and what float32 may move them by."""
    k, v = kv[:, :, 0].double(), kv[:, :, 1].double()
    k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + eps) * weight.double()[:, None]
    t = table.double()[positions][:, None, None]
    e, o, c, s = k[..., 0::2], k[..., 1::2], t[..., 0], t[..., 1]
    turned = torch.stack([e * c - o * s, o * c + e * s], -1).flatten(-2)
    size = torch.stack([(e * c).abs() + (o * s).abs(), (o * c).abs() + (e * s).abs()], -1).flatten(-2)
    # sum, quotient, + eps, root, reciprocal: 3 half steps of r; two products, a turn's product and sum: 4
    return torch.cat([turned, v], -1), torch.cat([8 * 2.0 ** -24 * size, torch.zeros_like(v)], -1)


@pytest.mark.parametrize("tokens,layers,heads,d,page", [(1, 1, 1, 128, 1), (1, 6, 16, 128, 16), (33, 2, 5, 64, 8),
                                                        (200, 3, 4, 128, 24), (7, 40, 1, 64, 16),
                                                        (513, 1, 20, 128, 16)])
def test_append(dev, tokens, layers, heads, d, page):
    g = torch.Generator().manual_seed(30)
    kv = (torch.randn(tokens, layers, 2, heads, d, generator=g) * torch.exp(torch.randn(d, generator=g))).to(BF)
    weight = 0.5 + torch.rand(layers, d, generator=g)
    positions = torch.randint(0, 500, (tokens,), generator=g)
    table = _table(500, d, "cpu")
    blocks = -(-tokens // page) + 2
    slots = torch.randperm(blocks * page, generator=g)[:tokens]
    if tokens > 4:
        slots[1], slots[3] = -1, blocks * page  # skipped: before and behind the cache
    cache = ops.mx_cache(blocks, heads, page, d, dev, layers)
    cache.codes.fill_(0xAB)
    cache.scales.fill_(99)
    args = kv.to(dev), positions.to(dev), slots.to(dev), weight.to(dev), ops.rope_from_table(table.to(dev))
    ops.write_context_kv_mx(*args, cache, 1e-5)
    want, tol = _written(kv, positions, weight, table, 1e-5)
    kept = ((slots >= 0) & (slots < blocks * page)).nonzero()[:, 0]
    held = [t.view(layers, blocks, heads, page, -1) for t in (cache.codes, cache.scales)]
    got = [h[:, slots[kept] // page, :, slots[kept] % page].reshape(-1, h.shape[-1]) for h in held]
    flat = [t[kept].reshape(-1, 2 * d) for t in (want, tol)]
    check_between(ops.MX(*got, 4, (got[0].shape[0], 2 * d)), *flat)
    # the values' codes are exact
    exact = mx.quantize(want[kept].reshape(-1, 2 * d), 4)
    assert torch.equal(mx.unpack(got[0].cpu(), 4)[:, d:], exact[0][:, d:])
    assert torch.equal(got[1].cpu()[:, d // 32:], exact[1][:, d // 32:])
    # nothing else was written
    untouched = torch.ones(blocks * page, dtype=torch.bool)
    untouched[slots[kept]] = False
    rows = untouched.nonzero()[:, 0]
    assert (held[0][:, rows // page, :, rows % page] == 0xAB).all()
    assert (held[1][:, rows // page, :, rows % page] == 99).all()
    # a cache a layer: the same bytes
    apart = [ops.mx_cache(blocks, heads, page, d, dev) for _ in range(layers)]
    for c in apart:
        c.codes.fill_(0xAB)
        c.scales.fill_(99)
    ops.write_context_kv_mx(*args, apart, 1e-5)
    for i in range(layers):
        assert torch.equal(apart[i].codes, cache[i].codes) and torch.equal(apart[i].scales, cache[i].scales)


def test_append_infinities(dev):
    kv = torch.randn(3, 1, 2, 1, 128)
    kv[0, 0, 1, 0, 40] = float("inf")
    kv[1, 0, 1, 0, 3] = float("nan")
    kv[2, 0, 0, 0, 3] = float("inf")
    cache = ops.mx_cache(3, 1, 1, 128, dev)
    ops.write_context_kv_mx(kv.to(BF).to(dev), torch.zeros(3, dtype=torch.int64, device=dev),
                            torch.arange(3, device=dev), torch.ones(128, device=dev),
                            ops.rope_from_table(_table(1, 128, dev)), [cache], 1e-6)
    nan = (cache.scales == 255).cpu()
    # an infinite key: inf / inf in its own block, finite / inf = 0 in the others
    assert nan.nonzero().tolist() == [[0, 5], [1, 4], [2, 0]]
    assert ops.mx_dequantize(cache).isnan().sum() == 96


def test_append_and_attend(dev):
    """Written rows are what the attention then reads, in the order of a server's step."""
    g = torch.Generator().manual_seed(31)
    layers, heads, d, page, lens = 2, 4, 128, 16, [70, 5]
    cache = ops.mx_cache(8, heads, page, d, dev, layers)
    table = torch.tensor([[3, 1, 7, 0, 4], [6, 0, 0, 0, 0]], dtype=torch.int32, device=dev)
    rope = ops.rope_from_table(_table(128, d, dev))
    weight = 0.5 + torch.rand(layers, d, generator=g)
    for first, last in ((0, 5), (5, 70)):  # a prompt in two parts
        pos = torch.cat([torch.arange(first, min(last, n)) for n in lens])
        req = torch.cat([torch.full((max(0, min(last, n) - first),), b) for b, n in enumerate(lens)])
        kv = torch.randn(len(pos), layers, 2, heads, d, generator=g).to(BF).to(dev)
        slots = table.cpu()[req, pos // page].long() * page + pos % page
        ops.write_context_kv_mx(kv, pos.to(dev), slots.to(dev), weight.to(dev), rope, cache, 1e-6)
    query = torch.randn(32, heads, d, generator=g).to(BF).to(dev)
    for i in range(layers):
        held = cache_values(cache[i])
        pages = [held[ids].permute(0, 2, 1, 3).reshape(-1, heads, 2 * d) for ids in table.cpu().long()]
        rows = [p[:n] for p, n in zip(pages, lens)]
        out = ops.block_attention_paged_mx(query, cache[i], None, torch.tensor(lens, device=dev), table, 16, 80, 0.1)
        check(out, query, rows, [16, 16], 0.1)
