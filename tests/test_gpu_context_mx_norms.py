"""The attention over a 4-bit context held to the size of its roundings (_context_mx_norms): lengths, pages, query
rows, the query's norm and rotation on the way, channels of different sizes, scales."""

import pytest
import torch

from _context_mx_checks import BF, cache_of, cache_values, make
from _context_mx_norms import check_norm
from flashmap_amd import ops
from test_gpu_context_mx import _attend, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("page", [1, 5, 16, 1000])
@pytest.mark.parametrize("lens", [[1], [2], [31, 32, 33], [127, 128, 129], [0, 5, 0, 300, 0], [1500, 700]])
def test_lengths(dev, d, page, lens):
    cache, table, rows = make(lens, 2, d, page, 1, dev)
    out, q, scale = _attend(cache, table, lens, [16] * len(lens), 4, d, dev, 2)
    check_norm(out.cpu(), q.cpu(), rows, [16] * len(lens), scale)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("hkv,group,q_len", [(1, 1, 1), (3, 2, 16), (1, 3, 16), (1, 8, 1), (2, 1, 17), (1, 1, 200),
                                             (1, 16, 9), (1, 6, 40)])
def test_rows(dev, d, hkv, group, q_len):
    lens = [77, 450, 3]
    cache, table, rows = make(lens, hkv, d, 16, 3, dev)
    out, q, scale = _attend(cache, table, lens, [q_len] * 3, hkv * group, d, dev, 4, ragged=False)
    check_norm(out.cpu(), q.cpu(), rows, [q_len] * 3, scale)


@pytest.mark.parametrize("d,hq,hkv,q_len", [(128, 4, 2, 16), (64, 6, 2, 9), (128, 8, 1, 16), (128, 1, 1, 1), (64, 8, 1, 16)])
def test_prologue(dev, d, hq, hkv, q_len):
    lens = [50, 333]
    cache, table, rows = make(lens, hkv, d, 16, 16, dev)
    g = torch.Generator().manual_seed(17)
    query = (3 * torch.randn(2 * q_len, hq, d, generator=g)).to(BF)
    weight = 0.5 + torch.rand(d, generator=g)
    angles = _table(400, d, "cpu")
    seq = torch.tensor(lens, device=dev)
    x = query.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.double()
    pos = torch.cat([n + torch.arange(q_len) for n in lens])
    for at in (pos, None):
        e, o = x[..., 0::2], x[..., 1::2]
        c, s = angles.double()[torch.arange(2 * q_len) if at is None else at][:, None].unbind(-1)
        want = torch.stack([e * c - o * s, o * c + e * s], -1).flatten(-2)
        for layout in (ops.rope_from_table(angles.to(dev)), ops.rope_from_split(*angles.to(dev).unbind(-1)),
                       ops.rope_from_cat(torch.cat(angles.unbind(-1), -1).to(dev))):
            pro = ops.Prologue(weight.to(dev), layout, None if at is None else at.to(dev), 1e-6)
            got = ops.block_attention_paged_mx(query.to(dev), cache, None, seq, table, q_len, 333, d ** -0.5, prologue=pro)
            check_norm(got.cpu(), want, rows, [q_len] * 2, d ** -0.5)


@pytest.mark.parametrize("factor", [1.0, 2.0 ** -60, 2.0 ** 60])
def test_query_range(dev, factor):
    """Blocks of query channels down to 2^-12 of the largest, with keys as much larger there."""
    g = torch.Generator().manual_seed(19)
    sizes = 2.0 ** -torch.tensor([0.0, 12.0, 3.0, 7.0]).repeat_interleave(32)
    kv = torch.randn(6, 1, 16, 256, generator=g)
    kv[..., :128] /= sizes
    cache, table = cache_of(kv, dev), torch.arange(6, dtype=torch.int32, device=dev)[None]
    held = cache_values(cache).view(96, 1, 256)[:90]
    query = (torch.randn(16, 1, 128, generator=g) * sizes * factor).to(BF)
    out = ops.block_attention_paged_mx(query.to(dev), cache, None, torch.tensor([90], device=dev), table, 16, 90,
                                       0.1 / factor)
    check_norm(out.cpu(), query, [held], [16], 0.1 / factor)


@pytest.mark.parametrize("larger", [1, 6, 12])
def test_sizes_in_a_block(dev, larger):
    """One channel of each block of 32 that is 2^larger times the others, and whose keys are 0: the others keep their
    own 8 bits."""
    g = torch.Generator().manual_seed(20)
    kv = torch.randn(25, 1, 16, 256, generator=g)
    kv[..., 0:128:32] = 0
    cache, table = cache_of(kv, dev), torch.arange(25, dtype=torch.int32, device=dev)[None]
    rows = [cache_values(cache).view(400, 1, 256)]
    query = torch.randn(16, 1, 128, generator=g)
    query[..., ::32] = 2.0 ** larger * (1 + torch.rand(16, 1, 4, generator=g))
    query = query.to(BF)
    out = ops.block_attention_paged_mx(query.to(dev), cache, None, torch.tensor([400], device=dev), table, 16, 400, 0.1)
    check_norm(out.cpu(), query, rows, [16], 0.1)


@pytest.mark.parametrize("scale", [0.0, 1e-3, 0.02, 0.2])
def test_scales(dev, scale):
    lens = [90, 400]
    cache, table, rows = make(lens, 2, 128, 16, 23, dev)
    out, q, _ = _attend(cache, table, lens, [16] * 2, 4, 128, dev, 24, scale=scale)
    check_norm(out.cpu(), q.cpu(), rows, [16] * 2, scale)
