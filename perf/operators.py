"""The microscaled operators whose speed is followed, with their plain forms.

A drafter's weights can be held in 4 bits: its drafts are verified, so that their precision
costs acceptance and never correctness, and a lightly loaded step does little else than
read weights. Four operators make that up:

- ``mx_quantize``: rows to 4 or 8 bits, one power-of-two scale per block of 32 values (with
  an MLP's activation applied on the way);
- ``mx_linear``: the product of such rows with 4-bit weights;
- ``rms_norm_mx``: a root-mean-square norm, the residual's addition in front of it, with
  8-bit output;
- ``adaln_residual_mx``: the DiT's gated residual and modulated norm with 8-bit output.

The format (OCP microscaling): a block of 32 values v has the scale 2^e, e = floor(log2 max
|v|) - 8 for e4m3 elements and - 2 for e2m1 elements, not below -127; an element is v / 2^e
rounded to nearest (ties to even) and saturated at 448 or 6. Rows are stored padded with
zeros to a multiple of 128 values: ``codes`` (rows, padded) bytes, or (rows, padded / 2) with
the element of even index in the low half of its byte, and ``scales`` (rows, padded / 32)
with the byte e + 127.

``own`` false computes the operators from elementary torch operations in 32 bits, ``own``
true calls the package's. ``exact`` gives the same results in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
BLOCK = 32
PAD = 128  # values that stored rows are padded to a multiple of
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed() -> list[dict]:
    return [
        # A single token's projection: nothing but latency.
        {"name": "linear_token", "kind": "linear", "rows": 1, "k": 2048, "n": 2048, "x": "bf16", "bias": False},
        # One user's block of 16 slots through the first half of an MLP.
        {"name": "linear_block", "kind": "linear", "rows": 16, "k": 2048, "n": 8192, "x": "bf16", "bias": True},
        # One user's block through the folded head: the largest weight of a draft step.
        {"name": "linear_head_b1", "kind": "linear", "rows": 16, "k": 2048, "n": 151936, "x": "bf16", "bias": False},
        # A full batch of 64 blocks through the second half of an MLP, quantized before.
        {"name": "linear_fc2_b64", "kind": "linear", "rows": 1024, "k": 8192, "n": 2048, "x": "mx8", "bias": True},
        # A full batch through the folded head.
        {"name": "linear_head_b64", "kind": "linear", "rows": 1024, "k": 2048, "n": 151936, "x": "mx8", "bias": False},
        # A long prompt's context rows, held in 4 bits, through the keys and values of six layers.
        {"name": "linear_context", "kind": "linear", "rows": 8192, "k": 2048, "n": 24576, "x": "mx4", "bias": False},
        # Weights brought to 4 bits when a drafter is loaded, and read back as values.
        {"name": "quantize_weight", "kind": "quantize", "rows": 24576, "k": 2048, "bits": 4, "dtype": "bf16",
         "activation": ""},
        # Between the halves of an MLP for a full batch: the activation and its 8 bits.
        {"name": "quantize_gelu_b64", "kind": "quantize", "rows": 1024, "k": 8192, "bits": 8, "dtype": "bf16",
         "activation": "gelu"},
        # The anchors' context rows of a small batch, odd row count.
        {"name": "rms_norm_b5", "kind": "rms_norm", "rows": 5, "k": 2048, "residual": False, "strided": False},
        # A long prompt's hidden states with the residual in front, rows of a wider buffer.
        {"name": "rms_norm_prompt", "kind": "rms_norm", "rows": 8192, "k": 4096, "residual": True, "strided": True},
        # The DiT's sublayer boundary for one user.
        {"name": "adaln_b1", "kind": "adaln", "rows": 16, "k": 2048, "residual": True},
        # The DiT's sublayer boundary for a full batch.
        {"name": "adaln_b64", "kind": "adaln", "rows": 1024, "k": 2048, "residual": True},
    ]


def _between(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cols(rng, lo: int, hi: int) -> int:
    """A row length: mostly whole blocks, some that end inside a block or a 16-byte group."""
    k = _between(rng, lo, hi)
    unit = rng.choice([128, 32, 32, 8, 1])
    return max(lo, k // unit * unit)


def draw(rng) -> dict:
    kind = rng.choice(["linear", "linear", "linear", "quantize", "rms_norm", "adaln"])
    if kind == "linear":
        rows = rng.choice([_between(rng, 1, 64), _between(rng, 1, 8192)])
        k = _cols(rng, 64, 20480)
        most = min(151936, 300_000_000 // k, 150_000_000 // rows, 300_000_000_000 // (rows * k))
        n = _between(rng, 64, max(64, most))
        return {"kind": kind, "rows": rows, "k": k, "n": n, "x": rng.choice(["bf16", "bf16", "mx8", "mx4"]),
                "bias": rng.random() < 0.5}
    if kind == "quantize":
        bits, activation = rng.choice([(4, ""), (4, ""), (8, ""), (8, "gelu"), (8, "swiglu")])
        k = _cols(rng, 64, 20480)
        return {"kind": kind, "rows": _between(rng, 1, max(1, min(30000, 60_000_000 // k))), "k": k, "bits": bits,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "activation": activation}
    k = _cols(rng, 64, 8192)
    rows = _between(rng, 1, max(1, min(16384, 40_000_000 // k)))
    if kind == "rms_norm":
        return {"kind": kind, "rows": rows, "k": k, "residual": rng.random() < 0.6, "strided": rng.random() < 0.4}
    return {"kind": kind, "rows": rows, "k": k, "residual": rng.random() < 0.8}


def _padded(k: int) -> int:
    return -(-k // PAD) * PAD


def work(case: dict) -> dict:
    rows, k = case["rows"], case["k"]
    held = {4: k / 2 + k / BLOCK, 8: k + k / BLOCK}  # bytes of a quantized row
    if case["kind"] == "linear":
        n = case["n"]
        x = {"bf16": 2.0 * k, "mx8": held[8], "mx4": held[4]}[case["x"]]
        return {"bytes": rows * x + n * held[4] + 2 * rows * n + (2 * n if case["bias"] else 0),
                "flops": 2.0 * rows * n * k}
    if case["kind"] == "quantize":
        size = DTYPES[case["dtype"]].itemsize
        into = rows * (2 if case["activation"] == "swiglu" else 1) * k * size
        # 4 bits come back as values: written, read again and written as bf16
        return {"bytes": into + rows * held[8] if case["bits"] == 8 else into + rows * (2 * held[4] + 2.0 * k),
                "flops": 4.0 * rows * k}
    streams = 3 if case["residual"] else 1  # bf16 rows: in, added, out
    return {"bytes": rows * (2.0 * k * streams + held[8]), "flops": 10.0 * rows * k}


# ------------------------------------------------------------------------------- inputs


def _activations(g, rows: int, k: int, dtype=torch.bfloat16) -> torch.Tensor:
    """Hidden states: normal rows, some channels far larger than others."""
    channel = torch.exp(0.6 * torch.randn(k, generator=g, device=DEV))
    return (torch.randn(rows, k, generator=g, device=DEV) * channel).to(dtype)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, k, kind = case["rows"], case["k"], case["kind"]
    state = {"case": dict(case)}
    if kind == "linear":
        n = case["n"]
        x = _activations(g, rows, k)
        state["x"] = x if case["x"] == "bf16" else _stored(*_blocks(x, 8 if case["x"] == "mx8" else 4))
        parts = []
        for first in range(0, n, 16384):  # the weight's float32 copies stay small
            w = torch.randn(min(16384, n - first), k, generator=g, device=DEV) / math.sqrt(k)
            parts.append(_stored(*_blocks(w, 4)))
        state["w"] = tuple(torch.cat(p) for p in zip(*parts))
        state["bias"] = torch.randn(n, generator=g, device=DEV).bfloat16() if case["bias"] else None
    elif kind == "quantize":
        wide = 2 * k if case["activation"] == "swiglu" else k
        state["x"] = _activations(g, rows, wide, DTYPES[case["dtype"]])
    elif kind == "rms_norm":
        x = _activations(g, rows, k + 64 if case["strided"] else k)
        state["x"] = x[:, :k]
        state["residual"] = torch.randn(rows, k, generator=g, device=DEV).bfloat16() if case["residual"] else None
        state["weight"] = 0.75 + 0.5 * torch.rand(k, generator=g, device=DEV)
    else:
        state["x"] = _activations(g, rows, k)
        state["y"] = torch.randn(rows, k, generator=g, device=DEV).bfloat16() if case["residual"] else None
        vectors = (0.3 * torch.randn(3, k, generator=g, device=DEV)).bfloat16()
        state["gate"], state["scale"], state["shift"] = (v.clone() for v in vectors)
    return state


# --------------------------------------------------------------------------- plain form


def _blocks(v: torch.Tensor, bits: int) -> tuple[torch.Tensor, torch.Tensor, int]:
    """``v`` (rows, k) as elements (rows, padded), the values before scaling, and the blocks'
    exponents (rows, padded / 32)."""
    v = v.float()
    v = torch.nn.functional.pad(v, (0, _padded(v.shape[1]) - v.shape[1])).view(v.shape[0], -1, BLOCK)
    top = v.abs().amax(-1)
    exponent = torch.where(top > 0, torch.frexp(top).exponent - 1 - (8 if bits == 8 else 2), -127).clamp(min=-127)
    y = v * torch.exp2(-exponent.float())[..., None]
    if bits == 8:
        y = y.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    else:  # the eight magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6: past a midpoint, or on it towards the even code
        a = y.abs()
        a = (0.5 * (a > 0.25) + 0.5 * (a >= 0.75) + 0.5 * (a > 1.25) + 0.5 * (a >= 1.75) + 1.0 * (a > 2.5)
             + 1.0 * (a >= 3.5) + 2.0 * (a > 5.0))
        y = torch.copysign(a.float(), y)
    return y.view(v.shape[0], -1), exponent, bits


def _stored(elements: torch.Tensor, exponent: torch.Tensor, bits: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Elements and exponents as the bytes that they are stored in."""
    scales = (exponent + 127).to(torch.uint8)
    if bits == 8:
        return elements.to(torch.float8_e4m3fn).view(torch.uint8), scales
    a = elements.abs()
    code = ((a > 0).to(torch.uint8) + (a > 0.5) + (a > 1) + (a > 1.5) + (a > 2) + (a > 3) + (a > 4)).to(torch.uint8)
    code = code + 8 * torch.signbit(elements).to(torch.uint8)
    return code[:, 0::2] + 16 * code[:, 1::2], scales


def _values(codes: torch.Tensor, scales: torch.Tensor, bits: int, k: int) -> torch.Tensor:
    """Stored rows as float32 values (rows, k)."""
    if bits == 8:
        y = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
        y = table[torch.stack([codes & 15, codes >> 4], -1).int()]
    y = y.view(codes.shape[0], -1, BLOCK) * torch.exp2(scales.float() - 127)[..., None]
    return y.view(codes.shape[0], -1)[:, :k]


def _plain_linear(s: dict, c: dict) -> torch.Tensor:
    k = c["k"]
    if c["x"] == "bf16":
        elements, exponent, _ = _blocks(s["x"], 8)
        x = (elements.view(c["rows"], -1, BLOCK) * torch.exp2(exponent.float())[..., None]).view(c["rows"], -1)[:, :k]
    else:
        x = _values(*s["x"], 8 if c["x"] == "mx8" else 4, k)
    out = x @ _values(*s["w"], 4, k).T
    return (out if s["bias"] is None else out + s["bias"].float()).bfloat16()


def _activated(x: torch.Tensor, name: str) -> torch.Tensor:
    if name == "gelu":
        return 0.5 * x * torch.special.erfc(x * -math.sqrt(0.5))
    if name == "swiglu":
        gate, up = x.chunk(2, dim=-1)
        return gate / (1 + torch.exp(-gate)) * up
    return x


def _eight_bits(v: torch.Tensor) -> dict:
    codes, scales = _stored(*_blocks(v, 8))
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


def _plain(s: dict) -> dict:
    c = s["case"]
    if c["kind"] == "linear":
        return {"out": _plain_linear(s, c)}
    x = s["x"].float()
    if c["kind"] == "quantize":
        v = _activated(x, c["activation"])
        if c["bits"] == 8:
            return _eight_bits(v)
        return {"values": _values(*_stored(*_blocks(v, 4)), 4, c["k"]).bfloat16()}
    if c["kind"] == "rms_norm":
        v = x if s["residual"] is None else x + s["residual"].float()
        out = _eight_bits(v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * s["weight"])
    else:
        v = x if s["y"] is None else x + s["gate"].float() * s["y"].float()
        mean = v.mean(-1, keepdim=True)
        norm = (v - mean) * torch.rsqrt((v - mean).square().mean(-1, keepdim=True) + EPS)
        out = _eight_bits(norm * (1 + s["scale"].float()) + s["shift"].float())
    return out if not c["residual"] else out | {"stream": v.bfloat16()}


# ---------------------------------------------------------------------------- the calls


def _own(s: dict) -> dict:
    from flashmap_amd import ops

    c = s["case"]
    if c["kind"] == "linear":
        x = s["x"] if c["x"] == "bf16" else ops.MX(*s["x"], 8 if c["x"] == "mx8" else 4, (c["rows"], c["k"]))
        return {"out": ops.mx_linear(x, ops.MX(*s["w"], 4, (c["n"], c["k"])), s["bias"])}
    if c["kind"] == "quantize":
        q = ops.mx_quantize(s["x"], bits=c["bits"], activation=c["activation"] or None)
        if c["bits"] == 4:
            return {"values": ops.mx_dequantize(q)}
        stream = None
    elif c["kind"] == "rms_norm":
        stream, q = ops.rms_norm_mx(s["x"], s["weight"], EPS, residual=s["residual"])
    else:
        stream, q = ops.adaln_residual_mx(s["x"], s["y"], s["gate"], (s["scale"], s["shift"]), EPS)
    out = {"codes": q.codes.view(torch.float8_e4m3fn), "scales": q.scales.view(torch.float8_e8m0fnu)}
    return out if stream is None else out | {"stream": stream}


def run(state: dict) -> dict:
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------- the same in 64 bits


def _exact_round(v: torch.Tensor, bits: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Elements and scales of float64 rows (rows, padded), a value's last place taken from its
    own exponent: 3 and 1 bits after the point, down to the smallest normal's."""
    top_exponent, last, least, most = (8, 3, -6, 448.0) if bits == 8 else (2, 1, 0, 6.0)
    blocks = v.view(v.shape[0], -1, BLOCK)
    top = blocks.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=1e-300)))
    e = e - (torch.exp2(e) > top).double() + (torch.exp2(e + 1) <= top).double()
    scale = torch.exp2(torch.where(top > 0, e - top_exponent, -127.0).clamp(min=-127.0))
    y = blocks / scale
    place = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** least))) - last)
    y = (torch.round(y / place) * place).clamp(-most, most)
    return y.view(v.shape), scale.squeeze(-1)


def _exact_values(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    """Stored rows as float64 (rows, padded), from the codes' sign, exponent and fraction bits."""
    if bits == 4:
        code = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.int16, device=codes.device)
        code[:, 0::2], code[:, 1::2] = codes.short() % 16, codes.short() // 16
        sign, exponent, part = code // 8, code // 2 % 4, (code % 2).double() / 2
        bias = 1
    else:
        code = codes.short()
        sign, exponent, part = code // 128, code // 8 % 16, (code % 8).double() / 8
        bias = 7
    y = torch.where(exponent > 0, (1 + part) * torch.exp2(exponent.double() - bias), part * 2.0 ** (1 - bias))
    y = torch.where(sign > 0, -y, y).view(codes.shape[0], -1, BLOCK)
    return (y * torch.exp2(scales.double() - 127)[..., None]).view(codes.shape[0], -1)


def _exact_eight(v: torch.Tensor) -> dict:
    out = torch.zeros(v.shape[0], _padded(v.shape[1]), dtype=torch.float64, device=v.device)
    out[:, :v.shape[1]] = v
    elements, scale = _exact_round(out, 8)
    return {"codes": elements, "scales": scale}


def exact(case: dict, seed: int) -> dict | None:
    s = prepare(case, seed)
    rows, k, kind = case["rows"], case["k"], case["kind"]
    if kind == "linear":
        if case["x"] == "bf16":
            wide = torch.zeros(rows, _padded(k), dtype=torch.float64, device=DEV)
            wide[:, :k] = s["x"].double()
            elements, scale = _exact_round(wide, 8)
            x = (elements.view(rows, -1, BLOCK) * scale[..., None]).view(rows, -1)
        else:
            x = _exact_values(*s["x"], 8 if case["x"] == "mx8" else 4)
        out = torch.empty(rows, case["n"], dtype=torch.float64, device=DEV)
        for first in range(0, case["n"], 8192):  # the weight's float64 copies stay small
            part = slice(first, first + 8192)
            out[:, part] = x @ _exact_values(s["w"][0][part], s["w"][1][part], 4).T
        return {"out": out if s["bias"] is None else out + s["bias"].double()}
    x = s["x"].double()
    if kind == "quantize":
        if case["activation"] == "gelu":
            x = (x * torch.special.ndtr(x)).float().double()  # the activation's value is a float32
        elif case["activation"] == "swiglu":
            x = x[:, :k] * torch.sigmoid(x[:, :k]) * x[:, k:]
        if case["bits"] == 8:
            return _exact_eight(x)
        wide = torch.zeros(rows, _padded(k), dtype=torch.float64, device=DEV)
        wide[:, :k] = x
        elements, scale = _exact_round(wide, 4)
        return {"values": (elements.view(rows, -1, BLOCK) * scale[..., None]).view(rows, -1)[:, :k]}
    if kind == "rms_norm":
        v = x if s["residual"] is None else x + s["residual"].double()
        out = _exact_eight(v / torch.sqrt((v * v).sum(-1, keepdim=True) / k + EPS) * s["weight"].double())
    else:
        v = x if s["y"] is None else s["y"].double() * s["gate"].double() + x
        centred = v - v.sum(-1, keepdim=True) / k
        norm = centred / torch.sqrt((centred * centred).sum(-1, keepdim=True) / k + EPS)
        out = _exact_eight(norm + norm * s["scale"].double() + s["shift"].double())
    return out if not case["residual"] else out | {"stream": v}
