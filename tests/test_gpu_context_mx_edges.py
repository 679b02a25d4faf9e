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
