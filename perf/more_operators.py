"""Operators around a context held in 4 bits, whose speed is followed, with their plain forms.

A drafter's context (every layer's keys and values of every position) is what its attention
reads and what fills a server's memory. Its drafts are verified, so that the context's
precision costs acceptance and never correctness: it can be held in 4 bits. Three operators
make that up:

- ``write_context_kv_mx``: appending: a position's keys normed, rotated to the position and,
  with its values, stored in microscaled 4 bits in a paged cache;
- ``block_attention_paged_mx``: the attention of a block of queries (one token, a drafted
  block, several candidate blocks) over such a cache, the queries' norm and rotation on the way;
- ``log_probs_rows``: what a draft or its verification is judged by: the log probability of
  given tokens, their ranks, the entropy of the distribution and its most likely tokens.

The cache (OCP microscaling): a row holds a position's D keys and then its D values for one
head; a block of 32 values v has the scale 2^e, e = floor(log2 max |v|) - 2, not below -127; an
element is v / 2^e rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives (ties
to the even code, saturated at 6), the element of even index in the low half of its byte, and
the scale is stored as the byte e + 127. Rows lie as (blocks, heads, page, 2 D): with pages of
one position the cache is a pool of single positions.

``own`` false computes the operators from elementary torch operations in 32 bits (the row sum
of the keys' norm and what decides a code's rounding in 64 where it matters), ``own`` true
calls the package's. ``exact`` gives the same results in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 1e6
BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed() -> list[dict]:
    return [
        # The next token of one user: a single query row per head over a short context. Latency.
        {"name": "attend_token", "kind": "attend", "batch": 1, "q": 1, "hq": 32, "hkv": 8, "d": 128, "page": 16,
         "lo": 2048, "hi": 2048, "prologue": False, "ragged": False},
        # One user's drafted block of 16 slots on the 8B drafter's own heads, an odd context.
        {"name": "attend_block_b1", "kind": "attend", "batch": 1, "q": 16, "hq": 16, "hkv": 16, "d": 128, "page": 16,
         "lo": 4097, "hi": 4097, "prologue": True, "ragged": False},
        # A handful of requests: pages of 8, narrow heads, query blocks of different lengths, one
        # context still empty.
        {"name": "attend_ragged_b5", "kind": "attend", "batch": 5, "q": 13, "hq": 12, "hkv": 4, "d": 64, "page": 8,
         "lo": 0, "hi": 3001, "prologue": True, "ragged": True},
        # A full batch, contexts of 256 to 8192, four query heads per key head.
        {"name": "attend_b64", "kind": "attend", "batch": 64, "q": 16, "hq": 32, "hkv": 8, "d": 128, "page": 16,
         "lo": 256, "hi": 8192, "prologue": True, "ragged": False},
        # Few requests with long contexts.
        {"name": "attend_b8_32k", "kind": "attend", "batch": 8, "q": 16, "hq": 32, "hkv": 8, "d": 128, "page": 16,
         "lo": 32768, "hi": 32768, "prologue": True, "ragged": False},
        # Tree drafting: 8 candidate blocks a request over a pool of single positions.
        {"name": "attend_tree_pool", "kind": "attend", "batch": 4, "q": 128, "hq": 16, "hkv": 16, "d": 128, "page": 1,
         "lo": 1024, "hi": 8192, "prologue": True, "ragged": False},
        # The anchors of one user's next draft: one position into six layers.
        {"name": "append_token", "kind": "append", "tokens": 1, "layers": 6, "heads": 16, "d": 128, "page": 16,
         "skipped": 0.0},
        # The positions a full batch accepted, a quarter of them padding that is not stored.
        {"name": "append_accepted", "kind": "append", "tokens": 777, "layers": 6, "heads": 16, "d": 128, "page": 16,
         "skipped": 0.25},
        # A prompt's context rows into every layer.
        {"name": "append_prompt", "kind": "append", "tokens": 8192, "layers": 6, "heads": 16, "d": 128, "page": 16,
         "skipped": 0.0},
        # One user's sampled token and its 20 likeliest alternatives.
        {"name": "log_probs_token", "kind": "log_probs", "rows": 1, "vocab": 151936, "dtype": "bf16", "top": 20,
         "temps": False, "masked": 0.0},
        # A batch of requests with temperatures, float32 logits, most tokens ruled out by a grammar.
        {"name": "log_probs_b61_grammar", "kind": "log_probs", "rows": 61, "vocab": 128256, "dtype": "fp32", "top": 5,
         "temps": True, "masked": 0.9},
        # Every slot of a full batch's drafts.
        {"name": "log_probs_b64x16", "kind": "log_probs", "rows": 1024, "vocab": 151936, "dtype": "bf16", "top": 8,
         "temps": True, "masked": 0.0},
    ]


def _between(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["attend", "attend", "append", "log_probs"])
    if kind == "attend":
        d = rng.choice([128, 128, 128, 64])
        hkv, group = rng.choice([(16, 1), (8, 4), (8, 5), (4, 8), (2, 6), (5, 1), (1, 16)])
        q = rng.choice([1, 16, _between(rng, 1, 40), _between(rng, 1, 256)])
        hi = _between(rng, 1, 40000)
        # contexts in all, and scores: no more than the largest listed cases'
        q = max(1, min(q, 130_000_000 // (hi * hkv * group)))
        most = min(256, 260_000 * 8 // (hi * hkv), 130_000_000 // (hkv * group * q * hi))
        return {"kind": kind, "batch": _between(rng, 1, max(1, most)), "q": q, "hq": hkv * group, "hkv": hkv, "d": d,
                "page": rng.choice([1, 8, 16, 16, 24, 64]), "lo": rng.choice([0, 1, hi // 4, hi]), "hi": hi,
                "prologue": rng.random() < 0.6, "ragged": rng.random() < 0.4}
    if kind == "append":
        d, layers, heads = rng.choice([128, 128, 64]), rng.choice([1, 2, 5, 6]), rng.choice([1, 4, 8, 16, 20])
        most = min(60_000, 100_000_000 // (layers * heads * d))
        return {"kind": kind, "tokens": _between(rng, 1, most), "layers": layers, "heads": heads, "d": d,
                "page": rng.choice([1, 8, 16, 16, 24]), "skipped": rng.choice([0.0, 0.0, 0.3])}
    vocab = rng.choice([_between(rng, 2, 262144), rng.choice([32000, 50257, 128256, 151936])])
    return {"kind": kind, "rows": _between(rng, 1, max(1, min(20_000, 75_000_000 // vocab))), "vocab": vocab,
            "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "top": min(vocab, rng.choice([0, 1, 5, 20, 32])),
            "temps": rng.random() < 0.5, "masked": rng.choice([0.0, 0.0, 0.5, 0.98]) if vocab >= 1000 else 0.0}


def _lens_q(c: dict) -> list[int]:
    """Query tokens of each request."""
    return [c["q"] - 5 * b % c["q"] if c["ragged"] else c["q"] for b in range(c["batch"])]


def _held(values: float) -> float:
    """Bytes of so many values in 4 bits with a scale byte for every 32."""
    return values * (0.5 + 1 / BLOCK)


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "attend":
        contexts = c["batch"] * (c["lo"] + c["hi"]) / 2  # the mean of what is drawn
        rows = sum(_lens_q(c)) * c["hq"]
        return {"bytes": _held(contexts * c["hkv"] * 2 * c["d"]) + rows * c["d"] * 2 * 2 + 4 * contexts / c["page"],
                "flops": 4.0 * contexts / c["batch"] * rows * c["d"]}
    if c["kind"] == "append":
        # the cache comes back as values: written, read again and written as bf16
        n = c["tokens"] * c["layers"] * c["heads"] * 2.0 * c["d"]
        kept = n * (1 - c["skipped"])
        return {"bytes": 2 * kept + _held(kept) + _held(n) + 2 * n, "flops": 8.0 * n}
    size = DTYPES[c["dtype"]].itemsize
    return {"bytes": float(c["rows"]) * (c["vocab"] * size + 28 + 12 * c["top"]), "flops": 5.0 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------------------- inputs


def _table(positions: int, d: int) -> torch.Tensor:
    """Rotary table (positions, D / 2, [cos, sin]) in float32, its angles from 64 bits."""
    pair = torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d
    angles = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * THETA ** -pair
    return torch.stack([angles.cos(), angles.sin()], -1).float().contiguous()


def _prepare_attend(c: dict, g) -> dict:
    batch, page, d, hkv = c["batch"], c["page"], c["d"], c["hkv"]
    lens = torch.randint(c["lo"], c["hi"] + 1, (batch,), generator=g, device=DEV)
    if c["lo"] == 0:
        lens[0] = 0
    pages = (lens + page - 1) // page
    width = max(1, -(-c["hi"] // page))
    total = int(pages.sum())
    blocks = total + 3  # a few pages of others
    order = torch.randperm(blocks, generator=g, device=DEV)[:total]
    ids = torch.arange(width, device=DEV) + (pages.cumsum(0) - pages)[:, None]
    used = torch.arange(width, device=DEV) < pages[:, None]
    table = torch.where(used, torch.cat([order, order.new_zeros(1)])[ids.clamp(max=total)], 0).int()
    rows = blocks * hkv * page
    codes = torch.empty(rows, d, dtype=torch.uint8, device=DEV)
    scales = torch.empty(rows, 2 * d // BLOCK, dtype=torch.uint8, device=DEV)
    # keys after their norm, values of channels of different sizes
    channel = torch.cat([torch.ones(d, device=DEV), torch.exp(0.6 * torch.randn(d, generator=g, device=DEV))])
    for first in range(0, rows, 1 << 18):  # the float32 copies stay small
        part = slice(first, min(rows, first + (1 << 18)))
        v = torch.randn(part.stop - first, 2 * d, generator=g, device=DEV) * channel
        codes[part], scales[part] = _stored(*_blocks(v))
    lens_q = torch.tensor(_lens_q(c), device=DEV)
    cu = torch.cat([lens_q.new_zeros(1), lens_q.cumsum(0)])
    tokens = int(cu[-1])
    state = {"codes": codes, "scales": scales, "shape": (blocks, hkv, page, 2 * d), "table": table,
             "lens": lens.int(), "cu": cu.int(), "weight": None, "rope": None, "positions": None}
    query = torch.randn(tokens, c["hq"], d, generator=g, device=DEV)
    if c["prologue"]:
        state["weight"] = 0.8 + 0.8 * torch.rand(d, generator=g, device=DEV)
        state["rope"] = _table(c["hi"] + c["q"] + 1, d)
        request = torch.repeat_interleave(torch.arange(batch, device=DEV), lens_q)
        state["positions"] = lens[request] + torch.arange(tokens, device=DEV) - cu[request]
    state["query"] = (query * (3.0 if c["prologue"] else 1.2)).bfloat16()
    return state


def _prepare_append(c: dict, g) -> dict:
    tokens, layers, heads, d, page = c["tokens"], c["layers"], c["heads"], c["d"], c["page"]
    blocks = -(-tokens // page) + 1
    channel = torch.exp(0.4 * torch.randn(layers, 2, heads, d, generator=g, device=DEV))
    kv = torch.empty(tokens, layers, 2, heads, d, dtype=torch.bfloat16, device=DEV)
    for first in range(0, tokens, 1024):
        part = slice(first, min(tokens, first + 1024))
        kv[part] = torch.randn(part.stop - first, layers, 2, heads, d, generator=g, device=DEV) * channel
    slots = torch.randperm(blocks * page, generator=g, device=DEV)[:tokens]
    slots[torch.rand(tokens, generator=g, device=DEV) < c["skipped"]] = -1
    rows = layers * blocks * heads * page
    return {"kv": kv, "slots": slots, "positions": torch.arange(tokens, device=DEV) + 5, "rope": _table(tokens + 5, d),
            "weight": 0.75 + 0.5 * torch.rand(layers, d, generator=g, device=DEV),
            "codes": torch.zeros(rows, d, dtype=torch.uint8, device=DEV),
            "scales": torch.zeros(rows, 2 * d // BLOCK, dtype=torch.uint8, device=DEV),
            "shape": (layers, blocks, heads, page, 2 * d)}


def _prepare_log_probs(c: dict, g) -> dict:
    rows, vocab = c["rows"], c["vocab"]
    logits = torch.empty(rows, vocab, dtype=DTYPES[c["dtype"]], device=DEV)
    tokens = torch.empty(rows, dtype=torch.int64, device=DEV)
    for first in range(0, rows, 128):
        part = slice(first, min(rows, first + 128))
        n = part.stop - first
        x = 2.0 * torch.randn(n, vocab, generator=g, device=DEV)
        few = min(vocab, 24)
        first_one = torch.randint(vocab, (n, 1), generator=g, device=DEV)
        likely = (first_one + torch.arange(few, device=DEV) * (vocab // few)) % vocab  # all different
        x.scatter_(1, likely, 8.0 + 3.0 * torch.randn(likely.shape, generator=g, device=DEV))
        out = torch.rand(n, vocab, generator=g, device=DEV) < c["masked"]
        out.scatter_(1, likely[:, :1], False)  # a grammar leaves one token at least
        logits[part] = x.masked_fill_(out, -math.inf)
        pick = torch.randint(likely.shape[1], (n, 1), generator=g, device=DEV)
        tokens[part] = likely.gather(1, pick)[:, 0]
    temps = 0.5 + torch.rand(rows, generator=g, device=DEV) if c["temps"] else None
    return {"logits": logits, "tokens": tokens, "temps": temps}


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = {"attend": _prepare_attend, "append": _prepare_append, "log_probs": _prepare_log_probs}[case["kind"]]
    return make(case, g) | {"case": dict(case)}


# --------------------------------------------------------------------------- plain form


def _blocks(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Float32 rows as 4-bit elements (rows, blocks, 32) and the blocks' exponents."""
    v = v.view(v.shape[0], -1, BLOCK)
    top = v.abs().amax(-1)
    exponent = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(min=-127)
    y = v * torch.exp2(-exponent.float())[..., None]
    a = y.abs()  # past a midpoint, or on it towards the even code
    a = (0.5 * (a > 0.25) + 0.5 * (a >= 0.75) + 0.5 * (a > 1.25) + 0.5 * (a >= 1.75) + 1.0 * (a > 2.5)
         + 1.0 * (a >= 3.5) + 2.0 * (a > 5.0))
    return torch.copysign(a.float(), y), exponent


def _stored(elements: torch.Tensor, exponent: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Elements and exponents as the bytes that they are stored in."""
    a = elements.abs()
    code = ((a > 0).to(torch.uint8) + (a > 0.5) + (a > 1) + (a > 1.5) + (a > 2) + (a > 3) + (a > 4)).to(torch.uint8)
    code = (code + 8 * torch.signbit(elements).to(torch.uint8)).view(code.shape[0], -1)
    return code[:, 0::2] + 16 * code[:, 1::2], (exponent + 127).to(torch.uint8)


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Stored rows (..., bytes) as float32 values (..., 2 bytes)."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    y = table[torch.stack([codes & 15, codes >> 4], -1).int()].view(*scales.shape, BLOCK)
    return (y * torch.exp2(scales.float() - 127)[..., None]).view(*codes.shape[:-1], -1)


def _rotated(x: torch.Tensor, rope: torch.Tensor) -> torch.Tensor:
    """Pairs of neighbouring channels of x (tokens, ..., D) turned by their angles (tokens, D / 2, 2)."""
    rope = rope.view(rope.shape[0], *(1,) * (x.dim() - 2), -1, 2)
    e, o, cos, sin = x[..., 0::2], x[..., 1::2], rope[..., 0], rope[..., 1]
    return torch.stack([e * cos - o * sin, o * cos + e * sin], -1).flatten(-2)


def _plain_attend(s: dict) -> dict:
    c = s["case"]
    batch, hkv, d, page, q = c["batch"], c["hkv"], c["d"], c["page"], c["q"]
    group = c["hq"] // hkv
    x = s["query"].float()
    if s["weight"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"]
        x = _rotated(x, s["rope"][s["positions"]])
    # the queries' rows padded to (batch, q), and the contexts to the longest
    at = s["cu"][:-1, None].long() + torch.arange(q, device=DEV)
    live = at < s["cu"][1:, None]
    x = x[at.clamp(max=x.shape[0] - 1)].view(batch, q, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(batch * hkv, -1, d)
    ids = s["table"].long()
    length = ids.shape[1] * page
    held = [t.view(*s["shape"][:3], -1)[ids].transpose(1, 2).reshape(batch * hkv, length, -1)
            for t in (s["codes"], s["scales"])]
    kv = _values(*held)
    keys, values = kv[..., :d].transpose(1, 2).contiguous(), kv[..., d:].contiguous()
    scores = torch.bmm(x, keys) * d ** -0.5
    masked = (torch.arange(length, device=DEV) >= s["lens"][:, None]).repeat_interleave(hkv, 0)[:, None]
    scores = scores.masked_fill(masked, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.bmm(p, values) / total.masked_fill(total == 0, 1.0)  # an empty context: zeros
    out = out.view(batch, hkv, group, q, d).permute(0, 3, 1, 2, 4).reshape(batch, q, c["hq"], d)
    return {"out": out[live].bfloat16()}


def _plain_append(s: dict) -> dict:
    layers, blocks, heads, page, d2 = s["shape"]
    d = d2 // 2
    kv = s["kv"].float()
    keys, values = kv[:, :, 0], kv[:, :, 1]
    square = keys.double().square().sum(-1, keepdim=True).float()
    keys = keys * (1 / torch.sqrt(square / d + EPS)) * s["weight"][:, None]
    rows = torch.cat([_rotated(keys, s["rope"][s["positions"]]), values], -1)  # (tokens, layers, heads, 2 D)
    codes, scales = _stored(*_blocks(rows.view(-1, d2)))
    kept = (s["slots"] >= 0).nonzero()[:, 0]
    block, place = s["slots"][kept] // page, s["slots"][kept] % page
    for held, new in ((s["codes"], codes), (s["scales"], scales)):
        held.view(*s["shape"][:4], -1)[:, block, :, place] = new.view(-1, layers, heads, new.shape[-1])[kept]
    return {"cache": _values(s["codes"], s["scales"]).view(s["shape"]).bfloat16()}


def _plain_log_probs(s: dict) -> dict:
    c = s["case"]
    x = s["logits"].float()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["top"]] if c["top"] else None
    mine = x.gather(1, s["tokens"][:, None])
    rank = (x > mine).sum(-1) + 1
    if s["temps"] is not None:
        x = x / s["temps"][:, None]
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    out = {"token": (x.gather(1, s["tokens"][:, None]) - log_total)[:, 0], "rank": rank,
           "entropy": (log_total - (e * x.clamp(min=-1e4)).sum(-1, keepdim=True) / total)[:, 0]}
    return out | ({"top_ids": order, "top": x.gather(1, order) - log_total} if c["top"] else {})


# ---------------------------------------------------------------------------- the calls


def _own(s: dict) -> dict:
    from flashmap_amd import ops

    c = s["case"]
    if c["kind"] == "attend":
        prologue = None
        if s["weight"] is not None:
            prologue = ops.Prologue(s["weight"], ops.rope_from_table(s["rope"]), s["positions"], EPS)
        return {"out": ops.block_attention_paged_mx(s["query"], ops.MX(s["codes"], s["scales"], 4, s["shape"]), s["cu"],
                                                    s["lens"], s["table"], c["q"], c["hi"], c["d"] ** -0.5,
                                                    prologue=prologue)}
    if c["kind"] == "append":
        cache = ops.MX(s["codes"], s["scales"], 4, s["shape"])
        ops.write_context_kv_mx(s["kv"], s["positions"], s["slots"], s["weight"], ops.rope_from_table(s["rope"]), cache,
                                EPS)
        return {"cache": ops.mx_dequantize(cache)}
    r = ops.log_probs_rows(s["logits"], s["tokens"], top=c["top"], temperatures=s["temps"])
    out = {"token": r.token, "rank": r.rank, "entropy": r.entropy}
    return out | ({"top_ids": r.top_ids, "top": r.top} if c["top"] else {})


def run(state: dict) -> dict:
    if own:
        return _own(state)
    plain = {"attend": _plain_attend, "append": _plain_append, "log_probs": _plain_log_probs}[state["case"]["kind"]]
    return plain(state)


# ------------------------------------------------------------------- the same in 64 bits


def _exact_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Stored rows as float64, from the codes' sign, exponent and fraction bits."""
    code = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.int16, device=codes.device)
    code[:, 0::2], code[:, 1::2] = codes.short() % 16, codes.short() // 16
    sign, exponent, part = code // 8, code // 2 % 4, (code % 2).double() / 2
    y = torch.where(exponent > 0, (1 + part) * torch.exp2(exponent.double() - 1), part)
    y = torch.where(sign > 0, -y, y).view(codes.shape[0], -1, BLOCK)
    return (y * torch.exp2(scales.double() - 127)[..., None]).view(codes.shape[0], -1)


def _exact_rounded(v: torch.Tensor) -> torch.Tensor:
    """Float64 rows as the 4-bit values nearest to them, a value's last place taken from its own exponent."""
    blocks = v.view(v.shape[0], -1, BLOCK)
    top = blocks.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=1e-300)))
    e = e - (torch.exp2(e) > top).double() + (torch.exp2(e + 1) <= top).double()
    scale = torch.exp2(torch.where(top > 0, e - 2, -127.0).clamp(min=-127.0))
    y = blocks / scale
    place = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)
    return ((torch.round(y / place) * place).clamp(-6, 6) * scale).view(v.shape)


def _exact_turned(x: torch.Tensor, weight: torch.Tensor, rope: torch.Tensor) -> torch.Tensor:
    """Norm and rotation of float64 heads (tokens, heads, D) as complex numbers, rope (tokens, D / 2, 2)."""
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous())
    return torch.view_as_real(z * torch.view_as_complex(rope.double().contiguous())[:, None]).flatten(-2)


def _exact_attend(s: dict, c: dict) -> dict:
    page, d, hkv = c["page"], c["d"], c["hkv"]
    group = c["hq"] // hkv
    x = s["query"].double()
    if s["weight"] is not None:
        x = _exact_turned(x, s["weight"], s["rope"][s["positions"]])
    out = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    codes, scales = (t.view(*s["shape"][:3], -1) for t in (s["codes"], s["scales"]))
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    for b, n in enumerate(lens):
        if n == 0:
            continue
        at = torch.arange(n, device=DEV)
        block = s["table"][b].long()[at // page]
        for h in range(hkv):
            kv = _exact_values(codes[block, h, at % page], scales[block, h, at % page])
            rows = x[cu[b]:cu[b + 1], h * group:(h + 1) * group].reshape(-1, d)
            w = torch.softmax(rows @ kv[:, :d].T / math.sqrt(d), -1)
            out[cu[b]:cu[b + 1], h * group:(h + 1) * group] = (w @ kv[:, d:]).view(-1, group, d)
    return {"out": out}


def _exact_append(s: dict) -> dict:
    layers, blocks, heads, page, d2 = s["shape"]
    cache = torch.zeros(s["shape"], dtype=torch.float64, device=DEV)
    kept = s["slots"] >= 0
    for layer in range(layers):
        for part in torch.nonzero(kept)[:, 0].split(4096):
            kv = s["kv"][part, layer].double()
            keys = _exact_turned(kv[:, 0], s["weight"][layer], s["rope"][s["positions"][part]])
            rows = _exact_rounded(torch.cat([keys, kv[:, 1]], -1).reshape(-1, d2)).view(-1, heads, d2)
            cache[layer, s["slots"][part] // page, :, s["slots"][part] % page] = rows
    return {"cache": cache}


def _exact_log_probs(s: dict, c: dict) -> dict:
    rows = s["logits"].shape[0]
    out = {"token": torch.empty(rows, dtype=torch.float64, device=DEV), "rank": None,
           "entropy": torch.empty(rows, dtype=torch.float64, device=DEV)}
    if c["top"]:
        out |= {"top_ids": None, "top": torch.empty(rows, c["top"], dtype=torch.float64, device=DEV)}
    for first in range(0, rows, 64):
        part = slice(first, first + 64)
        x = s["logits"][part].double()
        if s["temps"] is not None:
            x = x / s["temps"][part].double()[:, None]
        x = x - torch.logsumexp(x, -1, keepdim=True)
        out["token"][part] = x.gather(1, s["tokens"][part][:, None])[:, 0]
        out["entropy"][part] = torch.special.entr(x.exp()).sum(-1)
        if c["top"]:
            out["top"][part] = x.topk(c["top"], -1).values
    return out


def exact(case: dict, seed: int) -> dict | None:
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return None if case["batch"] * case["hkv"] > 4096 else _exact_attend(s, case)
    return _exact_append(s) if case["kind"] == "append" else _exact_log_probs(s, case)
