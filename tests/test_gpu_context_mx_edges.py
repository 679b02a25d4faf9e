"""The ends of what 4-bit contexts take, on the GPU."""

import pytest
import torch

from _context_mx_checks import BF, check, make
from flashmap_amd import ops

pytestmark = pytest.mark.gpu


def test_table_without_columns(dev):
    """Contexts that are all empty: zeros, with a table of no columns and with no position allowed."""
    cache, table, _ = make([16, 16], 2, 128, 16, 1, dev)
    query = torch.randn(8, 4, 128, device=dev).to(BF)
    lens = torch.tensor([5, 0], dtype=torch.int32, device=dev)
    for columns, most in ((table[:, :0], 16), (table[:, :0], 0), (table, 0)):
        out = torch.full_like(query, 7.0)
        ops.block_attention_paged_mx(query, cache, None, lens, columns, 4, most, 0.1, out=out)
        assert (out == 0).all()


@pytest.mark.parametrize("rows", [1 << 20, 1_048_513, 1_000_003])
def test_most_query_rows(dev, rows):
    """Up to 2^20 query rows for a KV head: as calls of fewer rows, the last row and those at the launches' ends."""
    cache, table, held = make([300], 1, 64, 16, 2, dev)
    query = torch.randn(rows, 1, 64, generator=torch.Generator(dev).manual_seed(3), device=dev).to(BF)
    lens = torch.tensor([300], dtype=torch.int32, device=dev)
    out = ops.block_attention_paged_mx(query, cache, None, lens, table, rows, 300, 0.125)
    some = sorted({r for at in range(0, rows, 16384) for r in (at - 1, at)} - {-1} | {rows - 1, rows - 17, rows // 2})
    check(out[some], query[some], held, [len(some)], 0.125)
    # a row's terms do not depend on the call, their order in sums may: float32 steps, then bf16's
    for first in range(0, rows, 65536):
        part = query[first:first + 65536]
        few = ops.block_attention_paged_mx(part, cache, None, lens, table, len(part), 300, 0.125)
        assert (few.float() - out[first:first + 65536].float()).abs().max() <= 2.0 ** -7 * out.float().abs().max()


def test_sliced_requests(dev):
    """Several heads a KV head and ragged requests, their rows more than one launch takes; the query as out."""
    lens, lens_q = [300, 0, 41], [40000, 7, 12345]
    cache, table, held = make(lens, 2, 128, 16, 4, dev)
    query = torch.randn(sum(lens_q), 4, 128, generator=torch.Generator(dev).manual_seed(5), device=dev).to(BF)
    cu = torch.tensor([0, 40000, 40007, 52352], dtype=torch.int32, device=dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    want = ops.block_attention_paged_mx(query, cache, cu, seq, table, 40000, 300, 0.1)
    some = [0, 1, 16383, 16384, 25535, 25536, 39999]
    at = torch.tensor(some + [40000, 40006] + [40007 + t for t in (0, 4096, 12344)], device=dev)
    check(want[at], query[at], held, [7, 2, 3], 0.1)
    same = query.clone()
    assert torch.equal(ops.block_attention_paged_mx(same, cache, cu, seq, table, 40000, 300, 0.1, out=same), want)


def test_out_between_the_querys_values(dev):
    lens = [200, 90]
    cache, table, _ = make(lens, 2, 128, 16, 22, dev)
    wide = torch.randn(10, 4, 264, device=dev).to(BF)
    query, out, seq = wide[:, :, :128], wide[:, :, 136:], torch.tensor(lens, device=dev)
    before = wide[:, :, :136].clone()
    want = ops.block_attention_paged_mx(query.contiguous(), cache, None, seq, table, 5, 200, 0.1)
    ops.block_attention_paged_mx(query, cache, None, seq, table, 5, 200, 0.1, out=out)
    assert torch.equal(out, want) and torch.equal(wide[:, :, :136], before)
