"""Contexts in microscaled 4 bits and log probabilities without a GPU: what the wrappers and the C entries
refuse before anything is launched, and the sizes of what they allocate."""

import ctypes
import math

import pytest
import torch

from flashmap_amd import _native, ops

BF = torch.bfloat16


@pytest.fixture
def host(monkeypatch):
    """The wrappers' own checks on CPU tensors; a launch fails the test."""
    monkeypatch.setattr(ops, "_check_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(ops, "call", lambda name, *a: pytest.fail(f"{name} was launched"))


def _cache(*lead, d=64):
    rows = math.prod(lead)
    codes, scales = torch.zeros(rows, d, dtype=torch.uint8), torch.zeros(rows, d // 16, dtype=torch.uint8)
    return ops.MX(codes, scales, 4, (*lead, 2 * d))


def _rope(d=64):
    return ops.rope_from_table(torch.zeros(8, d // 2, 2))


def test_cache_shapes():
    c = ops.mx_cache(3, 2, 16, 128, "cpu", layers=4)
    assert c.shape == (4, 3, 2, 16, 256) and c.codes.shape == (384, 128) and c.scales.shape == (384, 8)
    part = c[-1]
    assert part.shape == (3, 2, 16, 256) and part.codes.data_ptr() == c.codes[288:].data_ptr()
    assert part.scales.data_ptr() == c.scales[288:].data_ptr() and part.codes.shape == (96, 128)
    assert ops.mx_cache(3, 2, 1, 64, "cpu").codes.shape == (6, 64)
    for i in (4, -5):
        with pytest.raises(IndexError):
            c[i]
    with pytest.raises(IndexError):
        ops.MX(c.codes, c.scales, 4, (384, 256))[0]
    for bad in ((3, 2, 16, 80), (0, 2, 16, 64), (3, 2, 0, 64)):
        with pytest.raises(ValueError):
            ops.mx_cache(*bad, "cpu")


def test_cpu_tensors_are_refused():
    kv, idx, c = torch.zeros(2, 1, 2, 2, 64, dtype=BF), torch.zeros(2, dtype=torch.int64), _cache(4, 2, 8)
    table = torch.zeros(2, 4, dtype=torch.int32)
    for f in (lambda: ops.write_context_kv_mx(kv, idx, idx, torch.ones(64), _rope(), [c], 1e-6),
              lambda: ops.block_attention_paged_mx(kv[:, 0, 0], c, None, idx, table, 1, 8, 1.0),
              lambda: ops.log_probs_rows(torch.zeros(2, 8))):
        with pytest.raises(ValueError, match="GPU"):
            f()


def test_write_refuses(host):
    kv, idx, c = torch.zeros(2, 1, 2, 2, 64, dtype=BF), torch.zeros(2, dtype=torch.int64), _cache(4, 2, 8)

    def write(kv=kv, positions=idx, slots=idx, k_norm=torch.ones(64), rope=_rope(), caches=(c,)):
        ops.write_context_kv_mx(kv, positions, slots, k_norm, rope, caches, 1e-6)

    with pytest.raises(ValueError, match="tokens, layers, 2"):
        write(kv=kv[:, 0])
    with pytest.raises(TypeError, match="bfloat16"):
        write(kv=kv.float())
    with pytest.raises(ValueError, match="1 layers, the caches 2"):
        write(caches=[c, c])
    with pytest.raises(ValueError, match="1 layers, the caches 0"):
        write(caches=[])
    with pytest.raises(ValueError, match="1 layers, the caches 3"):
        write(caches=_cache(3, 4, 2, 8))
    with pytest.raises(ValueError, match="blocks, heads, page"):
        write(caches=[_cache(1, 4, 2, 8)])
    with pytest.raises(ValueError, match="2 heads x 64"):
        write(caches=[_cache(4, 3, 8)])
    with pytest.raises(ValueError, match="2 heads x 64"):
        write(caches=[_cache(4, 2, 8, d=128)])
    with pytest.raises(TypeError, match="4 bits"):
        write(caches=[ops.MX(c.codes, c.scales, 8, c.shape)])
    with pytest.raises(TypeError, match="4 bits"):
        write(caches=[ops.MX(c.codes.float(), c.scales, 4, c.shape)])
    with pytest.raises(ValueError, match="holds codes"):
        write(caches=[ops.MX(c.codes[1:], c.scales, 4, c.shape)])
    wide = torch.zeros(64, 72, dtype=torch.uint8)[:, :64]  # rows that are not 16-byte aligned
    with pytest.raises(ValueError, match="aligned"):
        write(caches=[ops.MX(wide, c.scales, 4, c.shape)])
    with pytest.raises(ValueError, match="aligned"):
        write(caches=[ops.MX(c.codes, c.scales[:1].expand(64, 4), 4, c.shape)])
    with pytest.raises(ValueError, match="share one shape"):
        write(kv=kv.expand(2, 2, 2, 2, 64), k_norm=torch.ones(128), caches=[c, _cache(5, 2, 8)])
    with pytest.raises(ValueError, match="k_norm"):
        write(k_norm=torch.ones(63))
    with pytest.raises(ValueError, match="rotary"):
        write(rope=_rope(128))
    with pytest.raises(ValueError, match="positions and slots"):
        write(slots=idx[:1])
    with pytest.raises(ValueError, match="positions and slots"):
        write(positions=idx[:, None])
    with pytest.raises(RuntimeError, match="no gradient"):
        write(kv=kv.clone().requires_grad_())
    write(kv=kv[:0], positions=idx[:0], slots=idx[:0])  # nothing to write


def test_attention_refuses(host):
    c, q = _cache(4, 2, 8), torch.zeros(6, 4, 64, dtype=BF)
    lens, table = torch.tensor([8, 8], dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)

    def attend(query=q, cache=c, cu=None, lens=lens, table=table, q_len=3, max_k=32, scale=0.1, **more):
        return ops.block_attention_paged_mx(query, cache, cu, lens, table, q_len, max_k, scale, **more)

    with pytest.raises(ValueError, match="tokens, heads"):
        attend(query=q[0])
    with pytest.raises(TypeError, match="bfloat16"):
        attend(query=q.float())
    with pytest.raises(ValueError, match="128 values"):
        attend(query=torch.zeros(6, 4, 128, dtype=BF))
    with pytest.raises(ValueError, match="divide"):
        attend(query=q[:, :3])
    with pytest.raises(ValueError, match="blocks, heads, page"):
        attend(cache=_cache(1, 4, 2, 8))
    with pytest.raises(TypeError, match="4 bits"):
        attend(cache=ops.MX(c.codes, c.scales, 8, c.shape))
    with pytest.raises(ValueError, match="batch x max_seqlen_q"):
        attend(q_len=4)
    with pytest.raises(ValueError, match="cu_seqlens_q"):
        attend(cu=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="block_table"):
        attend(table=table[:1])
    with pytest.raises(ValueError, match="seqused_k"):
        attend(lens=lens[:, None])
    for scale in (-0.1, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="not negative"):
            attend(scale=scale)
    with pytest.raises(ValueError, match="not negative"):
        attend(max_k=-1)
    with pytest.raises(RuntimeError, match="no gradient"):
        attend(query=q.clone().requires_grad_())
    with pytest.raises(ValueError, match="weight"):
        attend(prologue=ops.Prologue(torch.ones(32), _rope(), None, 1e-6))
    with pytest.raises(ValueError, match="positions"):
        attend(prologue=ops.Prologue(torch.ones(64), _rope(), torch.zeros(5, dtype=torch.int64), 1e-6))
    for out in (torch.zeros(6, 4, 64), torch.zeros(5, 4, 64, dtype=BF)):
        with pytest.raises(ValueError, match="out must be bfloat16"):
            attend(out=out)
    for out in (torch.zeros(6, 4, 68, dtype=BF)[:, :, :64], torch.zeros(1, 4, 64, dtype=BF).expand(6, 4, 64),
                torch.zeros(6, 64, 4, dtype=BF).transpose(1, 2)):
        with pytest.raises(ValueError, match="out must hold"):
            attend(out=out)
    buffer = torch.zeros(7, 4, 64, dtype=BF)
    with pytest.raises(ValueError, match="overlaps the query"):
        attend(query=buffer[:6], out=buffer[1:])
    memory = torch.zeros(64 * 64 // 2, dtype=BF)
    held = ops.MX(memory.view(torch.uint8).view(64, 64), c.scales, 4, c.shape)
    with pytest.raises(ValueError, match="overlaps the cache"):
        attend(cache=held, out=memory[:6 * 256].view(6, 4, 64))
    big = ops.MX(c.codes[:1].expand(1 << 32, 64), c.scales[:1].expand(1 << 32, 4), 4, (1 << 29, 2, 4, 128))
    with pytest.raises(ValueError):
        attend(cache=big)
    # nothing to do: no launch
    assert attend(query=q[:0], lens=lens[:0], table=table[:0]).shape == (0, 4, 64)
    assert attend(q_len=0).shape == q.shape


def test_log_probs_refuses(host):
    x = torch.zeros(3, 10)
    with pytest.raises(ValueError, match="rows, vocab"):
        ops.log_probs_rows(x[0])
    with pytest.raises(TypeError, match="float32"):
        ops.log_probs_rows(x.double())
    for top in (-1, 11, 33):
        with pytest.raises(ValueError, match="top"):
            ops.log_probs_rows(x, top=top)
    with pytest.raises(ValueError, match="top"):
        ops.log_probs_rows(torch.zeros(1, 100), top=33)
    for tokens in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, 1, dtype=torch.int64), torch.zeros(3)):
        with pytest.raises(ValueError, match="tokens"):
            ops.log_probs_rows(x, tokens)
    for temps in (torch.ones(2), torch.ones(3, 1), torch.ones(3, dtype=torch.int64)):
        with pytest.raises(ValueError, match="temperatures"):
            ops.log_probs_rows(x, temperatures=temps)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.log_probs_rows(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="empty vocabulary"):
        ops.log_probs_rows(torch.zeros(3, 0))
    got = ops.log_probs_rows(torch.zeros(0, 10), torch.zeros(0, dtype=torch.int64), 4)
    assert got.token.shape == (0,) and got.top_ids.shape == (0, 4)


def _err():
    return _native.last_error()


def test_entries_refuse():
    """The C entries' own checks: nothing is dereferenced before they return."""
    lib, n = _native.lib(), _native
    x, f = ctypes.c_void_p(256), ctypes.c_float
    rope = [x, x, 64, 1, 8]
    pointers = (ctypes.c_void_p * 2)(256, 256)
    odd = (ctypes.c_void_p * 2)(256, 264)

    def write(tokens=4, layers=2, heads=2, d=64, kv=x, codes=pointers, scales=pointers, rs=64, ss=4, blocks=4, page=8):
        return lib.fm_write_context_kv_mx(kv, tokens, layers, heads, d, x, x, x, *rope, codes, scales, rs, ss, blocks,
                                          page, f(1e-6), None)

    assert write(tokens=0) == n.FM_OK
    assert write(tokens=-1) == n.FM_ERR_INVALID and write(layers=0) == n.FM_ERR_INVALID
    assert write(d=96) == n.FM_ERR_UNSUPPORTED and "head_dim 96" in _err()
    assert write(kv=None) == n.FM_ERR_INVALID and "NULL" in _err()
    assert write(kv=ctypes.c_void_p(260)) == n.FM_ERR_INVALID and "aligned" in _err()
    assert write(codes=odd) == n.FM_ERR_INVALID and "layer 1" in _err()
    for bad in (dict(rs=72), dict(rs=48), dict(ss=6), dict(ss=0)):
        assert write(**bad) == n.FM_ERR_INVALID and "stride" in _err()
    assert write(page=0) == n.FM_ERR_INVALID and "geometry" in _err()
    assert write(tokens=1 << 40) == n.FM_ERR_INVALID and "too many" in _err()
    assert write(tokens=2 ** 63 - 1) == n.FM_ERR_INVALID and "too many" in _err()

    def attend(q=x, q_tokens=8, qst=256, qsh=64, rs=64, ss=4, blocks=4, page=8, width=4, batch=2, q_len=4, max_k=32,
               hq=4, hkv=2, d=64, scale=0.1, norm=None, table=None, ws=x, ws_bytes=1 << 40, cu=None):
        return lib.fm_block_attn_paged_mx(q, q_tokens, qst, qsh, x, 256, 64, cu, x, rs, x, ss, blocks, page, x, 4,
                                          width, x, batch, q_len, max_k, hq, hkv, d, f(scale), norm, table, table, 64, 1, 8,
                                          None, f(1e-6), ws, ws_bytes, None)

    assert attend(batch=0) == n.FM_OK and attend(q_len=0) == n.FM_OK
    assert attend(batch=-1) == n.FM_ERR_INVALID and attend(max_k=-1) == n.FM_ERR_INVALID
    assert attend(d=80) == n.FM_ERR_UNSUPPORTED
    assert attend(hq=5) == n.FM_ERR_INVALID and "divide" in _err()
    assert attend(hkv=0) == n.FM_ERR_INVALID
    assert attend(q=None) == n.FM_ERR_INVALID and "NULL" in _err()
    assert attend(ws=None) == n.FM_ERR_INVALID and "NULL" in _err()
    assert attend(q=ctypes.c_void_p(264)) == n.FM_ERR_INVALID and "aligned" in _err()
    assert attend(qst=250) == n.FM_ERR_INVALID and "multiples of 8" in _err()
    for bad in (dict(rs=72), dict(ss=2)):
        assert attend(**bad) == n.FM_ERR_INVALID and "cache rows" in _err()
    for bad in (dict(blocks=0), dict(page=0), dict(blocks=1 << 40), dict(page=1 << 30), dict(blocks=1 << 28, page=8)):
        assert attend(**bad) == n.FM_ERR_INVALID and "cache of 1 to" in _err()
    assert attend(scale=-1.0) == n.FM_ERR_INVALID and attend(scale=float("nan")) == n.FM_ERR_INVALID
    assert attend(norm=x) == n.FM_ERR_INVALID and "rotary" in _err()
    assert attend(q_tokens=7) == n.FM_ERR_INVALID and "batch x max_seqlen_q" in _err()
    assert attend(q_len=1 << 20, q_tokens=1 << 40) == n.FM_ERR_INVALID and "2^20" in _err()
    assert attend(width=1 << 30, max_k=2 ** 31 - 1) == n.FM_ERR_INVALID and "2^24" in _err()
    assert attend(ws_bytes=64) == n.FM_ERR_WORKSPACE

    def judge(dtype=0, rows=2, vocab=100, stride=100, top=4, logits=x, out=x, ws=x, ws_bytes=1 << 30, tokens=x):
        return lib.fm_log_probs_rows(logits, dtype, rows, vocab, stride, tokens, None, top, out, out, x, out, out, ws,
                                     ws_bytes, None)

    assert judge(rows=0) == n.FM_OK
    assert judge(dtype=3) == n.FM_ERR_INVALID and judge(rows=-1) == n.FM_ERR_INVALID
    for bad in (dict(top=33), dict(top=-1), dict(top=5, vocab=4)):
        assert judge(**bad) == n.FM_ERR_INVALID and "top" in _err()
    assert judge(vocab=0, top=0) == n.FM_ERR_INVALID and judge(vocab=1 << 31, stride=1 << 31) == n.FM_ERR_INVALID
    assert judge(stride=99) == n.FM_ERR_INVALID and "stride" in _err()
    assert judge(logits=ctypes.c_void_p(257)) == n.FM_ERR_INVALID and "aligned" in _err()
    assert judge(ws=ctypes.c_void_p(8)) == n.FM_ERR_INVALID and "16 bytes" in _err()
    assert judge(out=None) == n.FM_ERR_INVALID and judge(ws=None) == n.FM_ERR_INVALID
    assert judge(vocab=10_000, stride=10_000, ws_bytes=16) == n.FM_ERR_WORKSPACE


def test_workspace_sizes():
    lib = _native.lib()
    assert lib.fm_log_probs_workspace_bytes(0, 100, 4) == 0 and lib.fm_log_probs_workspace_bytes(3, 100, 33) == 0
    small, large = (lib.fm_log_probs_workspace_bytes(r, 151936, 20) for r in (1, 32))
    assert 75 * (16 + 8 * 20) == small < large
    # rows that fill the chip are a part each and leave no records
    for rows, vocab in ((1 << 20, 1000), (1024, 151936)):
        assert lib.fm_log_probs_workspace_bytes(rows, vocab, 32) == 16
    assert lib.fm_block_attn_paged_mx_workspace_bytes(0, 4, 2, 64) == 0
    assert lib.fm_block_attn_paged_mx_workspace_bytes(1 << 30, 4, 2, 64) == 0
