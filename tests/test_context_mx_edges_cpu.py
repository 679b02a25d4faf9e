"""The ends of what 4-bit contexts and log probabilities take, without a GPU: calls that the C entries and the
wrappers let through to the launch, and those that they refuse."""

import ctypes

import pytest
import torch

from flashmap_amd import _native, ops
from flashmap_amd.draft_step import DraftStep

BF = torch.bfloat16
X = ctypes.c_void_p(256)


def _attend(table=X, width=4, max_k=32, q_len=4, batch=2, q_tokens=1 << 40, hq=4, hkv=2, d=64, blocks=4, page=8,
            ws_bytes=64):
    """The entry on addresses that nothing reads: a workspace of 64 bytes is the last thing that it refuses."""
    return _native.lib().fm_block_attn_paged_mx(
        X, q_tokens, hq * d, d, X, hq * d, d, None, X, d, X, d // 16, blocks, page, table, width, width, X, batch, q_len,
        max_k, hq, hkv, d, ctypes.c_float(0.1), None, None, None, 0, 0, 0, None, ctypes.c_float(1e-6), X, ws_bytes, None)


def test_table_without_columns():
    """A batch of empty contexts may come with a table of no columns, whose tensor has no address."""
    assert _attend() == _native.FM_ERR_WORKSPACE
    assert _attend(table=None) == _native.FM_ERR_INVALID and "NULL" in _native.last_error()
    assert _attend(table=None, width=0) == _native.FM_ERR_WORKSPACE
    assert _attend(table=None, max_k=0) == _native.FM_ERR_WORKSPACE


def test_query_rows():
    """2^20 query rows a KV head are taken, for a workspace that does not grow with them; more are refused."""
    size = _native.lib().fm_block_attn_paged_mx_workspace_bytes
    for rows in (1 << 20, (1 << 20) - 1, (1 << 20) - 63, 1_048_513, 1_048_512):
        assert _attend(q_len=rows, hq=2, hkv=2) == _native.FM_ERR_WORKSPACE
        assert 0 < size(rows, 2, 2, 128) < 600_000_000
    assert _attend(q_len=1 << 19, hq=4, hkv=2) == _native.FM_ERR_WORKSPACE
    assert _attend(q_len=(1 << 20) + 1, hq=2, hkv=2) == _native.FM_ERR_INVALID and "2^20" in _native.last_error()
    assert size((1 << 20) + 1, 2, 2, 128) == 0


def test_units():
    """What one launch counts in 32 bits: KV heads of its sequences, and a share's steps."""
    many = dict(batch=256, blocks=1, page=1, width=1)
    assert _attend(hq=65535, hkv=65535, **many) == _native.FM_ERR_WORKSPACE
    assert _attend(hq=65536, hkv=65536, **many) == _native.FM_ERR_INVALID and "2^24" in _native.last_error()
    long = dict(batch=256, blocks=1, page=256, width=1 << 16, max_k=1 << 24, q_len=1 << 14)
    assert _attend(hq=500, hkv=500, **long) == _native.FM_ERR_WORKSPACE
    assert _attend(hq=5000, hkv=5000, **long) == _native.FM_ERR_INVALID and "positions" in _native.last_error()


def test_parts():
    """Microscaled rows of two dimensions have no parts; those of more have their leading dimension's."""
    cache = ops.mx_cache(3, 2, 4, 64, "cpu", layers=2)
    parts = list(cache)
    assert [p.shape for p in parts] == [(3, 2, 4, 128)] * 2
    assert [p.codes.data_ptr() for p in parts] == [cache[0].codes.data_ptr(), cache[1].codes.data_ptr()]
    rows = ops.MX(cache.codes, cache.scales, 4, (48, 128))
    for use in (list, iter, lambda q: print(*q), lambda q: 1 in q):
        with pytest.raises(TypeError):
            use(rows)


def test_mixed_caches():
    """A draft step's caches are all in 4 bits or none, whichever comes first."""
    cache, plain = ops.mx_cache(2, 2, 16, 128, "cpu"), torch.zeros(2, 2, 16, 256, dtype=BF)
    for caches in ([cache, plain], [plain, cache], [plain, plain, cache]):
        with pytest.raises(TypeError, match="all be microscaled"):
            DraftStep.cache_layout(caches)
    assert DraftStep.cache_layout([cache, cache]) == [cache, cache]
    joined = ops.mx_cache(2, 2, 16, 128, "cpu", layers=3)
    assert [c.shape for c in DraftStep.cache_layout(joined)] == [(2, 2, 16, 256)] * 3


@pytest.fixture
def launched(monkeypatch):
    """The wrappers' own checks on CPU tensors: the names of the entries that a call would have launched."""
    names = []
    monkeypatch.setattr(ops, "_check_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(ops, "_mx_call", lambda name, *a: names.append(name))
    monkeypatch.setattr(ops, "_attn_mx_workspace_bytes", lambda *a: 64)
    return names


def test_one_cache_for_two_layers(launched):
    kv, idx = torch.zeros(2, 2, 2, 2, 64, dtype=BF), torch.zeros(2, dtype=torch.int64)
    caches = [ops.mx_cache(4, 2, 8, 64, "cpu") for _ in range(2)]
    rope = ops.rope_from_table(torch.zeros(8, 32, 2))
    with pytest.raises(ValueError, match="different"):
        ops.write_context_kv_mx(kv, idx, idx, torch.ones(2, 64), rope, [caches[0], caches[0]], 1e-6)
    halves = ops.MX(caches[0].codes, caches[1].scales, 4, caches[0].shape)
    with pytest.raises(ValueError, match="different"):
        ops.write_context_kv_mx(kv, idx, idx, torch.ones(2, 64), rope, [caches[0], halves], 1e-6)
    assert launched == []
    ops.write_context_kv_mx(kv, idx, idx, torch.ones(2, 64), rope, caches, 1e-6)
    ops.write_context_kv_mx(kv, idx, idx, torch.ones(2, 64), rope, ops.mx_cache(4, 2, 8, 64, "cpu", 2), 1e-6)
    assert launched == ["fm_write_context_kv_mx"] * 2


def test_out_beside_and_over_operands(launched):
    """An output between the query's own values is taken; one over anything that the call reads is refused."""
    cache, wide = ops.mx_cache(4, 2, 8, 64, "cpu"), torch.zeros(6, 4, 160, dtype=BF)
    lens, table = torch.tensor([8, 8], dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    cu, query = torch.tensor([0, 3, 6], dtype=torch.int32), torch.zeros(6, 4, 64, dtype=BF)
    rope, weight = ops.rope_from_table(torch.zeros(8, 32, 2)), torch.ones(64)

    def attend(query=query, cache=cache, cu=cu, lens=lens, table=table, pro=None, **more):
        return ops.block_attention_paged_mx(query, cache, cu, lens, table, 3, 32, 0.1, prologue=pro, **more)

    for q, out in ((wide[:, :, :64], wide[:, :, 64:128]), (wide[:, :, 64:128], wide[:, :, :64]),
                   (wide[:, :2, :64], wide[:, 2:, :64]), (wide[:3, :, 64:128], wide[3:, :, 64:128]),
                   (wide[1:, :, 64:128], wide[:5, :, :64])):
        n = q.shape[0]
        own = torch.tensor([0, n // 2, n], dtype=torch.int32)
        assert attend(query=q, cu=own, out=out) is out
    assert launched == ["fm_block_attn_paged_mx"] * 5
    for q, out in ((wide[:, :, :64], wide[:, :, 32:96]), (wide[:, :, 32:96], wide[:, :, :64]),
                   (wide[:5, :, :64], wide[1:, :, :64]), (wide[:, :2, :64], wide[:, 1:3, :64]),
                   (wide[:3, :2, :64], wide[1:4, 1:3, 32:96])):
        with pytest.raises(ValueError, match="overlaps the query"):
            attend(query=q, cu=None, lens=lens[:1], table=table[:1], out=out)

    # `size` values of out's memory as an operand
    memory = torch.zeros(6 * 4 * 64, dtype=BF)
    out = memory.view(6, 4, 64)

    def held(dtype, *shape):
        size = torch.Size(shape).numel() * dtype.itemsize // 2
        return memory[64:64 + size].view(dtype).view(shape)

    for more in (dict(cu=held(torch.int32, 3)), dict(lens=held(torch.int32, 2)), dict(lens=held(torch.int64, 2)),
                 dict(table=held(torch.int32, 2, 4)), dict(pro=ops.Prologue(held(torch.float32, 64), rope, None, 1e-6)),
                 dict(pro=ops.Prologue(weight, ops.rope_from_table(held(torch.float32, 8, 32, 2)), None, 1e-6)),
                 dict(pro=ops.Prologue(weight, ops.rope_from_split(torch.zeros(8, 32), held(torch.float32, 8, 32)), None,
                                       1e-6)),
                 dict(pro=ops.Prologue(weight, rope, held(torch.int64, 6), 1e-6))):
        with pytest.raises(ValueError, match="overlaps what the call reads"):
            attend(out=out, **more)
    with pytest.raises(ValueError, match="overlaps the cache"):
        attend(cache=ops.MX(cache.codes, held(torch.uint8, 64, 4), 4, cache.shape), out=out)
    assert attend(query=out, out=out) is out and attend(out=out) is out


def test_rotary_halves_on_one_device():
    with pytest.raises(ValueError, match="device"):
        ops.rope_from_split(torch.zeros(8, 32), torch.zeros(8, 32, device="meta"))


def test_rows_of_a_write():
    """What a launch can count threads for: a call of more rows is refused before any is written."""
    pointers = (ctypes.c_void_p * 2)(256, 256)

    def write(tokens):
        return _native.lib().fm_write_context_kv_mx(X, tokens, 2, 16, 64, X, X, X, X, X, 64, 1, 8,
                                                    pointers, pointers, 64, 4, 4, 8, ctypes.c_float(1e-6), None)

    assert write(1 << 25) == _native.FM_ERR_INVALID and "too many" in _native.last_error()
    assert write((1 << 25) - 1) == _native.FM_ERR_INVALID and "too many" in _native.last_error()
