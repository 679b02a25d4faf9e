"""Benchmark of the drafter cross-attention call on one MI355X.

Workload (the metric's configuration): one Qwen3-8B-shaped drafter layer's
cross-attention for a serving batch: 32 query / 8 KV heads (GQA 4), head_dim 128,
K = 16 draft rows per sequence, batch 64, context lengths drawn uniform in
[256, 8192] from seed 0, KV paged in 16-token blocks behind a randomly permuted block
table (vLLM's FlashAttention cache layout), bf16.

One call (one "step") = two launches: the split-KV block attention, whose consumer
wavefronts read the caller's query rows and apply the QK-RMSNorm + RoPE prologue
themselves at each segment start, and the log-sum-exp combine that writes the output
rows. The step's plan (computed once per step and shared by every layer, like
FlashAttention's scheduler metadata) is prepared before the timed region. Inputs are
resident in HBM when timing starts.

Timing: W warm-up calls and K timed calls right after set-up are reported as
`cold_us_per_call`; then the call runs back to back for `--settle-ms` while the GPU's
power controller settles (a load this heavy starting from idle first has its clocks cut
for some milliseconds), then W warm-up calls and exactly K timed calls give `value`.

Prints one JSON line. `value` is microseconds per call (lower is better); the line
also carries the achieved HBM bandwidth, a roofline record for the main attention
kernel (its own algorithmic bytes -- the call's minus the output rows the combine
writes -- over its average duration from HIP events recorded around each launch on its
stream; `call_bytes` = the whole call's; `traffic` = the measured HBM bytes per launch from the
calibrated FETCH_SIZE / WRITE_SIZE counters committed under profiles/, when present for
the workload) and the CPU baseline (the oracle on the host cores, on a bounded sample
of the same workload).
"""

from __future__ import annotations

import argparse
import json
import math
import os
import sys
import time
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent
sys.path.insert(0, str(ROOT))

METRIC = "drafter attn µs/call + achieved HBM TB/s, K=16, batch 64, ctx 256–8k, 1 GPU"
HBM_PEAK_GBS = 8000.0
MFMA_BF16_PEAK_TFLOPS = 2500.0

WORKLOADS = {
    # name: (batch, hq, hkv, head_dim, K, lo, hi, page)
    "c3-qwen3-8b-paged-b64": (64, 32, 8, 128, 16, 256, 8192, 16),
    "c4-qwen3-8b-long-b8": (8, 32, 8, 128, 16, 32768, 32768, 16),
    "c5-27b-gqa5-b32": (32, 40, 8, 128, 16, 1024, 8192, 16),
    "r8b-mha-b64": (64, 16, 16, 128, 16, 256, 8192, 16),
}


def build_inputs(name: str, seed: int = 0):
    """Seeded CPU draw in a fixed order: lengths, block-table permutation, query
    pre-norm rows, context K (pre-norm) and V. The cache is filled on the GPU by the
    context-KV writer (k-norm + RoPE at each context position)."""
    batch, hq, hkv, d, k_rows, lo, hi, page = WORKLOADS[name]
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(lo, hi + 1, (batch,), generator=g)
    pages = [math.ceil(int(n) / page) for n in lens]
    total = sum(pages)
    perm = torch.randperm(total, generator=g)
    bt = torch.zeros(batch, max(pages), dtype=torch.int32)
    o = 0
    for b, n in enumerate(pages):
        bt[b, :n] = perm[o:o + n].int()
        o += n
    q_pre = torch.randn(batch * k_rows, hq, d, generator=g).bfloat16()
    ctx = int(lens.sum())
    kv_pre = torch.empty(ctx, 1, 2, hkv, d, dtype=torch.bfloat16)
    chunk = 1 << 15
    for s in range(0, ctx, chunk):  # bounded fp32 temporaries
        e = min(ctx, s + chunk)
        kv_pre[s:e] = torch.randn(e - s, 1, 2, hkv, d, generator=g).bfloat16()
    positions = torch.cat([torch.arange(int(n)) for n in lens])
    slots = torch.cat([bt[b, torch.arange(int(n)) // page].long() * page + torch.arange(int(n)) % page
                       for b, n in enumerate(lens)])
    return dict(batch=batch, hq=hq, hkv=hkv, d=d, k_rows=k_rows, page=page, lens=lens, bt=bt, total=total,
                q_pre=q_pre, kv_pre=kv_pre, positions=positions, slots=slots, lo=lo, hi=hi)


def kernel_source_hash() -> str:
    """sha256 (16 hex digits) of the attention kernels' sources: counters recorded under
    profiles/ carry it, and are reported only for the build they were collected on."""
    import hashlib

    h = hashlib.sha256()
    for name in ("block_attn.hip", "fm_device.h"):
        h.update((ROOT / "flashmap_amd" / "csrc" / name).read_bytes())
    return h.hexdigest()[:16]


def traffic_record(name: str, workload: str):
    """Calibrated HBM bytes per launch of the main kernel from profiles/``name`` (FETCH_SIZE
    + WRITE_SIZE counters), when recorded for this workload on the kernel sources being
    timed; None otherwise."""
    f = ROOT / "profiles" / name
    if not f.exists():
        return None
    rec = json.loads(f.read_text())
    if rec.get("workload") != workload or rec.get("source_sha") != kernel_source_hash():
        return None
    return rec["traffic_bytes"]


def mfma_record(workload: str, batch: int, flops: float, kernel_ms: float, fp8: bool) -> dict:
    """MFMA utilisation of the main kernel: from the rocprofv3 counters committed under
    profiles/ for this workload (SQ_VALU_MFMA_BUSY_CYCLES over the SIMD-cycles of the
    dispatch) when they were collected on the kernel sources being timed (else marked
    stale), beside the algorithmic FLOPs over the HIP-event duration."""
    rec = {"tflops_algorithmic": round(flops / (kernel_ms * 1e-3) / 1e12, 1),
           "peak_tflops": MFMA_BF16_PEAK_TFLOPS,
           "util_algorithmic": round(flops / (kernel_ms * 1e-3) / 1e12 / MFMA_BF16_PEAK_TFLOPS, 4)}
    name = f"attn_fwd_{workload.split('-', 1)[0]}_paged_b{batch}{'_fp8' if fp8 else ''}.mfma.json"
    f = ROOT / "profiles" / name
    if f.exists():
        c = json.loads(f.read_text())
        if c.get("workload") == workload:
            rec.update({"source": f"profiles/{name}", "counters": c["counters"]})
            if c.get("source_sha") == kernel_source_hash():
                rec["util"] = c["util"]
            else:
                rec.update({"util": None, "stale": True, "util_recorded": c["util"],
                            "note": "counters recorded on other kernel sources than the ones timed"})
    return rec


def prologue_label(fp8: bool) -> str:
    """Where the paged drafter workloads' QK-RMSNorm + RoPE runs. e4m3 calls quantize the
    rows per head in a query pass; bf16 calls of at most one unit per share (the batch-64
    workloads: 512 units over 512 shares) read the caller's rows in the attention kernel
    unless FLASHMAP_QUERY_PASS=1 forces the pass."""
    if fp8:
        return "QK-RMSNorm + RoPE and the per-head e4m3 quantization in the call's query pass (its own launch)"
    if os.environ.get("FLASHMAP_QUERY_PASS") == "1":
        return "QK-RMSNorm + RoPE applied by the call's query pass (its own launch; FLASHMAP_QUERY_PASS=1)"
    return "QK-RMSNorm + RoPE applied inside the attention kernel to the caller's rows (no query pass: two launches)"


def algorithmic_bytes(inp, kv_bytes: int = 2) -> dict:
    lens, d, hq, hkv, k_rows, batch, page = (inp[k] for k in ("lens", "d", "hq", "hkv", "k_rows", "batch", "page"))
    sum_l = int(lens.sum())
    kv = sum_l * hkv * d * 2 * kv_bytes
    qo = 2 * batch * k_rows * hq * d * 2
    table = 4 * sum(math.ceil(int(n) / page) for n in lens)
    meta = 8 * batch
    rope = batch * k_rows * d * 4
    flops = 4 * k_rows * hq * d * sum_l
    total = kv + qo + table + meta + rope
    # the main kernel's own share: everything but the output rows, which the combine writes;
    # e4m3 calls: its queries are the pass's e4m3 rows and their scales (the pass applied the
    # prologue: no rotary rows)
    kernel = total - qo // 2
    if kv_bytes == 1:
        kernel = kv + batch * k_rows * hq * (d + 4) + table + meta
    return dict(kv=kv, total=total, kernel=kernel, flops=flops, sum_l=sum_l)


def cpu_paged_cache(inp, table) -> torch.Tensor:
    """The bf16 paged cache on the host, as the GPU writer fills it (untimed set-up)."""
    from oracle import attention as ref

    d, hkv, page = inp["d"], inp["hkv"], inp["page"]
    cache = torch.zeros(inp["total"], hkv, page, 2 * d, dtype=torch.bfloat16)
    pos, slots, kv = inp["positions"], inp["slots"], inp["kv_pre"]
    w = torch.ones(d)
    for s in range(0, kv.shape[0], 1 << 15):
        e = min(kv.shape[0], s + (1 << 15))
        rows = table[pos[s:e]]
        k = ref.project_keys(kv[s:e, 0, 0], w, rows[..., 0][:, None], rows[..., 1][:, None], 1e-6)
        blk, tok = slots[s:e] // page, slots[s:e] % page
        cache[blk, :, tok, :d] = k
        cache[blk, :, tok, d:] = kv[s:e, 0, 1]
    return cache


def cpu_model() -> str:
    """The host CPU's model string (``/proc/cpuinfo``)."""
    try:
        with open("/proc/cpuinfo") as f:
            for line in f:
                if line.startswith("model name"):
                    return line.split(":", 1)[1].strip()
    except OSError:
        pass
    return "unknown"


def cpu_timed(run, weights: list, unit: str, what: str, budget_s: float, threads: int | None = None,
              warmups: int = 2, calls: int = 5) -> dict:
    """The CPU baseline's protocol: ``run(n)`` does the call's work for its first ``n``
    items (sequences, requests, rows), ``weights[i]`` is item i's share of the work (context
    positions, rows). One probe of the first item prices the work; the sample is the
    longest prefix whose call fits ``budget_s / (warmups + calls)``; then ``warmups``
    untimed calls of the sample and the median of ``calls`` timed ones, scaled to the
    whole call by weight."""
    cores = threads or len(os.sched_getaffinity(0))
    torch.set_num_threads(cores)
    t0 = time.perf_counter()
    run(1)
    per_weight = (time.perf_counter() - t0) / max(weights[0], 1)
    per_call = budget_s / (warmups + calls)
    n, acc = 0, 0.0
    while n < len(weights) and (n == 0 or (acc + weights[n]) * per_weight <= per_call):
        acc += weights[n]
        n += 1
    for _ in range(warmups):
        run(n)
    times = []
    for _ in range(calls):
        t0 = time.perf_counter()
        run(n)
        times.append(time.perf_counter() - t0)
    med = sorted(times)[len(times) // 2]
    total = sum(weights)
    return {"value": round(med * total / acc * 1e6, 1), "unit": unit, "cores": cores, "kind": "port",
            "cpu_model": cpu_model(),
            "sample": f"first {n} of {len(weights)} {what} ({int(acc)} of {int(total)} by weight): median of "
                      f"{calls} calls after {warmups} warm-ups, scaled to the whole call by weight"}


def cpu_baseline(inp, budget_s: float = 12.0) -> dict:
    """The oracle (fp32 torch on the host cores) on the call's work: per sequence, the
    Q prologue, the block-table gather of K/V from the paged cache, then attention
    (``cpu_timed``'s protocol, weighted by context positions)."""
    from oracle import attention as ref

    d, k_rows = inp["d"], inp["k_rows"]
    table = ref.rope_table(inp["hi"] + k_rows + 1, d, 1e6)
    w = torch.ones(d)
    lens, bt = inp["lens"], inp["bt"]
    cache = cpu_paged_cache(inp, table)

    def one(b):
        n = int(lens[b])
        k, v = ref.gather_vllm(cache, bt, n, b)
        q = inp["q_pre"][b * k_rows:(b + 1) * k_rows]
        qn = ref.rms_norm_rope_vllm(q, w, table, n + torch.arange(k_rows), 1e-6)
        return ref.attention(qn.transpose(0, 1), k, v)

    def run(count):
        for b in range(count):
            one(b)

    rec = cpu_timed(run, [int(n) for n in lens], "us/call", "sequences", budget_s)
    rec["sample"] += " (context positions); fp32 oracle Q prologue + block-table gather + attention"
    return rec


# The drafter workloads onto an e4m3 (fp8) paged cache: name -> the bf16 workload whose
# draw it shares. The cache is written by the fp8 context writer (scales 1); the queries
# are bf16, normed and rotated and quantized per (sequence, head) inside the call.
FP8_WORKLOADS = {
    "c3-qwen3-8b-paged-b64-fp8": "c3-qwen3-8b-paged-b64",
}

# Target verify attention (SplitKVVerify's call): name -> (batch, hq, hkv, head_dim,
# verify tokens, ctx lo, ctx hi, mask). Contexts as the drafter workloads draw them,
# held in an SGLang token pool at randomly permuted slots.
VERIFY_WORKLOADS = {
    "verify-qwen3-8b-chain-b64": (64, 32, 8, 128, 17, 256, 8192, "causal"),
    "verify-qwen3-8b-tree-b64": (64, 32, 8, 128, 17, 256, 8192, "qlen"),
}


# The drafter workload over vLLM's virtual context-cache layout: name -> (the bf16
# workload whose draw it shares, heads per cache, DiT layer timed). The context writer
# packs (layer + 1) DiT layers' heads into caches of that many heads (each layer's K/V
# the shared draw); the timed layer's KV heads then lie in several runs and one launch
# attends to them all.
VIRTUAL_WORKLOADS = {
    "c3-qwen3-8b-virtual-hpc3": ("c3-qwen3-8b-paged-b64", 3, 1),
}

# Tree drafting on SGLang's token pool: name -> (requests, hq, hkv, head_dim, candidates,
# ctx lo, ctx hi). A request's candidate blocks sit side by side in the query axis
# (n_cand * 16 rows) over its one context (the reference's MHA drafter shape, the
# candidate counts its default budget of 32 gives at batch 1 and 4).
TREE_WORKLOADS = {
    "tree-r8b-b1-n32": (1, 16, 16, 128, 32, 8192, 8192),
    "tree-r8b-b4-n8": (4, 16, 16, 128, 8, 1024, 8192),
    # One candidate per request: the SGLang drafter's own cross-attention call at C3's shape
    # (batch 64, 32/8 heads, contexts U[256, 8192]: C3's draw, pool slots permuted).
    "c3shape-sglang-pool-b64": (64, 32, 8, 128, 1, 256, 8192),
}
# The same calls onto e4m3 pools (flashmap_sglang::paged_cross_attention_fp8): name -> the
# bf16 workload whose shape and draw it takes (the pools' values rounded to e4m3).
TREE_FP8_WORKLOADS = {
    "c3shape-sglang-pool-b64-fp8": "c3shape-sglang-pool-b64",
}


# The draft step's token selection over bf16 logits: name -> (rows, vocabulary, mode).
# Rows = 64 requests x 16 draft rows; Qwen3's vocabulary. "argmax": split_argmax (vLLM's
# greedy draft); "sample": sample_rows with every row sampled (SGLang's fused sampler,
# Gumbel-max on the Philox stream).
SELECT_WORKLOADS = {
    "argmax-b64x16-v151936": (1024, 151936, "argmax"),
    "sample-b64x16-v151936": (1024, 151936, "sample"),
}


def run_select(args, dev) -> dict:
    """One call = one selection over the logits (tile pass + row pass)."""
    from flashmap_amd import ops

    rows, vocab, mode = SELECT_WORKLOADS[args.workload]
    g = torch.Generator(device=dev).manual_seed(0)
    logits = torch.randn(rows, vocab, generator=g, device=dev, dtype=torch.bfloat16)
    temps = torch.full((rows,), 0.8, device=dev)
    greedy = torch.zeros(rows, dtype=torch.bool, device=dev)
    seed = torch.tensor(1, dtype=torch.int64, device=dev)
    if mode == "argmax":
        def call():
            ops.argmax_rows(logits)
    else:
        def call():
            ops.sample_rows(logits, temps, greedy, seed)
    timing = _measure(call, args, kernel_events=False)
    ms = timing["ms"]
    total = rows * vocab * 2 + rows * 8
    gbs = total / (ms * 1e-3) / 1e9
    result = {
        "metric": f"draft-step token selection µs/call ({mode}), {rows} rows x {vocab} bf16 logits, 1 GPU",
        "value": round(ms * 1e3, 2), "unit": "us/call", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup,
        "ms_per_step": round(ms, 5), "higher_is_better": False, "scaling": "weak", "vs_baseline": None,
        "dtype": "bf16 logits, fp32 keys", "data": "synthetic: seeded GPU draw of the logits",
        "config": {"workload": args.workload, "rows": rows, "vocab": vocab, "mode": mode},
        "roofline": {"bound": "hbm", "achieved": round(gbs, 1), "peak": HBM_PEAK_GBS, "unit": "GB/s",
                     "frac": round(gbs / HBM_PEAK_GBS, 4), "traffic": None, "bytes_per_launch": total,
                     "note": "whole call (tile pass + row pass) from events around the calls"
                             + ("; the sampled path is ALU-bound: one Philox-4x32-10 and two logs per logit"
                                if mode == "sample" else "")},
        **_timing_fields(timing),
    }
    if not args.no_cpu_baseline:
        from oracle import sampling as S

        x = logits[:64].float().cpu().numpy()
        tc, gc = temps[:64].cpu().numpy(), greedy[:64].cpu().numpy()

        def run(n):
            if mode == "argmax":
                S.split_argmax(x[:n])
            else:
                S.sample_rows(x[:n], tc[:n], gc[:n], 1)

        weights = [1] * rows  # the sample is at most the 64 rows copied to the host
        rec = cpu_timed(lambda n: run(min(n, 64)), weights[:64], "us/call", "rows", args.cpu_budget, threads=1)
        rec["value"] = round(rec["value"] * rows / 64, 1)
        rec["sample"] += f", of the first 64 of {rows} rows (scaled by rows); numpy oracle, one thread"
        result["cpu_baseline"] = rec
    return result


# The K side and the block self-attention, each as one launch over a draft step's data:
# "kv-write-c3-vllm": the context writer over C3's draw (245380 positions, 8 KV heads of
# 128, one layer): each key k-normed and rotated at its position, key and value stored at
# the position's slot of a vLLM cache of 16-token pages behind a permuted block table;
# "kv-write-c3-pool": the same rows into SGLang token pools, one pool row per position at
# a permuted location; "self-attn-8b-b64x16": the 8B drafter layer's block self-attention,
# 64 blocks x 16 slots, 16 heads of 128, q/k RMSNorm + RoPE at the slots' positions inside;
# "norm-rope-c3-q": the standalone QK-RMSNorm + RoPE (the plugins' rms_norm_rope op) over
# C3's query rows, 64 x 16 draft tokens x 32 heads of 128, each at its position.
KERNEL_WORKLOADS = {
    "kv-write-c3-vllm": "vllm",
    "kv-write-c3-pool": "pool",
    "self-attn-8b-b64x16": "self",
    "norm-rope-c3-q": "norm",
}


def run_kernel(args, dev) -> dict:
    """One call = one launch of the writer or of the block self-attention."""
    from flashmap_amd import ops
    from oracle import attention as ref

    kind = KERNEL_WORKLOADS[args.workload]
    g = torch.Generator().manual_seed(0)
    if kind == "norm":
        inp = build_inputs("c3-qwen3-8b-paged-b64")
        x, d, k_rows = inp["q_pre"], inp["d"], inp["k_rows"]
        tokens, heads = x.shape[0], x.shape[1]
        w = 0.75 + 0.5 * torch.rand(d, generator=g)
        pos = torch.cat([int(n) + torch.arange(k_rows) for n in inp["lens"]])
        table = ref.rope_table(inp["hi"] + k_rows + 1, d, 1e6)
        x_d, w_d, pos_d = x.to(dev), w.to(dev), pos.to(dev)
        rope = ops.rope_from_table(table.to(dev))
        out_d = torch.empty_like(x_d)

        def call():
            ops.rms_norm_rope(x_d, w_d, rope, pos_d, 1e-6, out=out_d)

        total = tokens * heads * d * 2 * 2 + tokens * (8 + 4 * d)  # rows in and out, positions, rotary rows
        flops = None
        what = f"QK-RMSNorm + RoPE µs/call, {tokens} tokens x {heads} heads of {d}"
        config = {"workload": args.workload, "tokens": tokens, "heads": heads, "head_dim": d,
                  "rope": "vLLM table (positions, head_dim / 2, [cos, sin]) gathered at each token's position"}
    elif kind == "self":
        blocks, t, heads, d = 64, 16, 16, 128
        qkv = torch.randn(blocks, t, 3, heads, d, generator=g).bfloat16()
        qn, kn = 0.75 + 0.5 * torch.rand(d, generator=g), 0.75 + 0.5 * torch.rand(d, generator=g)
        anchors = torch.randint(256, 8192, (blocks,), generator=g)
        pos = (anchors[:, None] + 1 + torch.arange(t)).reshape(-1)
        table = ref.rope_table(8192 + t + 1, d, 1e6)
        qkv_d, qn_d, kn_d, pos_d = qkv.to(dev), qn.to(dev), kn.to(dev), pos.to(dev)
        rope = ops.rope_from_table(table.to(dev))

        def call():
            ops.block_self_attention(qkv_d, qn_d, kn_d, rope, pos_d, 1e-6)

        total = blocks * t * heads * d * 2 * 4 + blocks * t * (8 + 4 * d)  # qkv in, out, positions, rotary rows
        flops = blocks * heads * 4 * t * t * d
        what = f"block self-attention µs/call, {blocks} blocks x {t} slots, {heads} heads of {d}"
        config = {"workload": args.workload, "blocks": blocks, "block_size": t, "heads": heads, "head_dim": d,
                  "prologue": "q/k RMSNorm + RoPE inside the kernel"}
    else:
        inp = build_inputs("c3-qwen3-8b-paged-b64")
        hkv, d, page = inp["hkv"], inp["d"], inp["page"]
        kv, pos = inp["kv_pre"], inp["positions"]
        tokens = kv.shape[0]
        kn = 0.75 + 0.5 * torch.rand(1, d, generator=g)
        kv_d, pos_d, kn_d = kv.to(dev), pos.to(dev), kn.to(dev)
        if kind == "vllm":
            table = ref.rope_table(inp["hi"] + 1, d, 1e6)
            rope = ops.rope_from_table(table.to(dev))
            cache = torch.zeros(inp["total"], hkv, page, 2 * d, dtype=torch.bfloat16, device=dev)
            ptrs = torch.tensor([cache.data_ptr()], dtype=torch.int64, device=dev)
            slots_d = inp["slots"].to(dev)
            strides = (cache.stride(0), cache.stride(1), cache.stride(2), d)

            def call():
                ops.write_context_kv(kv_d, pos_d, slots_d, kn_d, rope, ptrs, strides, page, 1e-6)
        else:
            cat = ref.rope_cat_table(inp["hi"] + 1, d, 1e6)
            rope = ops.rope_from_cat(cat.to(dev))
            pool = tokens + 64
            locs = torch.randperm(pool, generator=g)[:tokens]
            kbuf = torch.zeros(pool, hkv, d, dtype=torch.bfloat16, device=dev)
            vbuf = torch.zeros_like(kbuf)
            meta = torch.tensor([[kbuf.data_ptr(), vbuf.data_ptr(), kbuf.stride(0), vbuf.stride(0)]],
                                dtype=torch.int64, device=dev)
            rows_d, locs_d = kv_d.view(tokens, 2 * hkv * d), locs.to(dev)

            def call():
                ops.write_context_kv_pool(rows_d, meta, kn_d, rope, pos_d, locs_d, 1, hkv * d, d, 1e-6)

        total = tokens * (2 * 2 * hkv * d * 2 + 16 + 4 * d)  # rows in and out, position and slot, rotary row
        flops = None
        what = f"context K/V write µs/call ({kind}), {tokens} positions x {hkv} KV heads of {d}"
        config = {"workload": args.workload, "positions": tokens, "kv_heads": hkv, "head_dim": d,
                  "layout": "vllm paged (blocks, kv_heads, 16, 2*head_dim)" if kind == "vllm"
                  else "sglang token pools (pool, kv_heads, head_dim), permuted rows",
                  "prologue": "k RMSNorm + RoPE of each key"}
    timing = _measure(call, args, kernel_events=False)
    ms = timing["ms"]
    gbs = total / (ms * 1e-3) / 1e9
    result = {
        "metric": what + ", 1 GPU",
        "value": round(ms * 1e3, 2), "unit": "us/call", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup,
        "ms_per_step": round(ms, 5), "higher_is_better": False, "scaling": "weak", "vs_baseline": None,
        "dtype": "bf16", "data": "synthetic: seeded CPU draw" + (" (C3's lengths and rows)" if kind != "self" else ""),
        "config": config,
        "roofline": {"bound": "hbm", "achieved": round(gbs, 1), "peak": HBM_PEAK_GBS, "unit": "GB/s",
                     "frac": round(gbs / HBM_PEAK_GBS, 4), "traffic": None, "bytes_per_launch": total,
                     "note": "one launch per call, timed by events around the calls"
                             + (f"; {flops / 1e6:.0f} MFLOP per call: latency-bound at this size" if flops else "")},
        **_timing_fields(timing),
    }
    if not args.no_cpu_baseline:
        if kind == "norm":
            def run(n):
                ref.rms_norm_rope_vllm(x[:n], w, table, pos[:n], 1e-6)

            rec = cpu_timed(run, [1] * tokens, "us/call", "tokens", args.cpu_budget)
        elif kind == "self":
            half = table[pos.long()]
            cos, sin = half[..., 0].view(blocks, t, d // 2), half[..., 1].view(blocks, t, d // 2)

            def run(n):
                ref.block_self_attention(qkv[:n].float(), qn, kn, cos[:n], sin[:n], 1e-6)

            rec = cpu_timed(run, [1] * blocks, "us/call", "blocks", args.cpu_budget)
        elif kind == "vllm":
            want = [torch.zeros(inp["total"], hkv, page, 2 * d, dtype=torch.bfloat16)]

            def run(n):
                ref.write_context_kv_vllm(kv[:n], pos[:n], inp["slots"][:n], kn, table, want, page, 1e-6)

            rec = cpu_timed(run, [1] * tokens, "us/call", "positions", args.cpu_budget)
        else:
            wk = [torch.zeros(pool, hkv, d, dtype=torch.bfloat16)]
            wv = [torch.zeros_like(wk[0])]
            rows = kv.view(tokens, 2 * hkv * d)

            def run(n):
                ref.write_context_kv_pool(rows[:n], wk, wv, kn, cat, pos[:n], locs[:n], 1, hkv * d, d, 1e-6)

            rec = cpu_timed(run, [1] * tokens, "us/call", "positions", args.cpu_budget)
        result["cpu_baseline"] = rec
    return result


def _flushed(call, args, dev, flush_mb: int = 512) -> dict:
    """Timing of a latency-bound call, its K/V read from HBM: each timed call is preceded
    by a write of ``flush_mb`` MB, which evicts the 4 MB L2s and the 256 MB Infinity
    Cache, and bracketed by its own events (the flush, about 100 us, covers the host's
    launch path, so the call's kernels run back to back).

    - ``ms``: the median over K such calls;
    - ``warm_ms``: K back-to-back calls (inputs resident in the caches);
    - ``graph_ms``: K back-to-back replays of the call captured in a HIP graph (the form
      an engine's captured draft step takes);
    - ``kernel_ms``: the main kernel's own HIP events over K calls, each after a flush."""
    import ctypes

    from flashmap_amd import _native

    flush = torch.empty(flush_mb << 20, dtype=torch.uint8, device=dev)
    for _ in range(args.warmup):
        call()
    torch.cuda.synchronize()
    warm_ms = _events_ms(call, args.steps)
    pairs = [(torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)) for _ in range(args.steps)]
    for i, (e0, e1) in enumerate(pairs):
        flush.fill_(i & 0xFF)
        e0.record()
        call()
        e1.record()
    torch.cuda.synchronize()
    each = sorted(e0.elapsed_time(e1) for e0, e1 in pairs)
    lib = _native.lib()
    lib.fm_profile_enable(1)
    for i in range(args.steps):
        flush.fill_(i & 0xFF)
        call()
    torch.cuda.synchronize()
    tot, cnt = ctypes.c_double(), ctypes.c_int64()
    _native.call("fm_profile_read", ctypes.byref(tot), ctypes.byref(cnt))
    lib.fm_profile_enable(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(args.warmup):
        graph.replay()
    graph_ms = _events_ms(graph.replay, args.steps)
    return {"ms": each[len(each) // 2], "warm_ms": warm_ms, "graph_ms": graph_ms,
            "kernel_ms": tot.value / max(cnt.value, 1)}


# The vLLM plugin's draft step (flashmap_amd.draft_step.DraftStep): name -> (requests,
# ctx lo, ctx hi, jumps, drafter config overrides). The released 8B drafter's shape
# (hidden 2048, 16 heads of 128, 6 layers, GELU MLP 8192) over a Qwen3-8B target (hidden
# 4096, vocabulary 151936); contexts drawn as C3's, paged in 16-token blocks. Two jumps
# (Algorithm 8) carry a state over the whole vocabulary between them and run the DiT, and
# so every layer's cross-attention, twice. b1 and b4: one user and four, 1024 positions each.
DRAFT_STEP_WORKLOADS = {
    "draft-step-8b-b1": (1, 1024, 1024, 1, {}),
    "draft-step-8b-b4": (4, 1024, 1024, 1, {}),
    "draft-step-8b-b64": (64, 256, 8192, 1, {}),
    "draft-step-8b-b64-2jump": (64, 256, 8192, 2, {}),
}


def run_draft_step(args, dev) -> dict:
    """One call = one draft step for the batch: the anchors' context rows written, then
    per jump the DiT input (one jump: the folded noise read-out; several: the state's
    embedding), 6 DiT layers (each with its cross-attention over its paged cache) and,
    between jumps, the state's update; then the folded head over the vocabulary and the
    greedy argmax. The plan is built per step inside the call."""
    from flashmap_amd import drafter as d
    from flashmap_amd.draft_step import DraftStep

    batch, lo, hi, jumps, over = DRAFT_STEP_WORKLOADS[args.workload]
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(lo, hi + 1, (batch,), generator=g)  # C3's draw: context positions incl. the anchor
    page = 16
    pages = [math.ceil(int(n) / page) for n in lens]
    total = sum(pages)
    perm = torch.randperm(total, generator=g)
    bt = torch.zeros(batch, max(pages), dtype=torch.int32)
    o = 0
    for b, n in enumerate(pages):
        bt[b, :n] = perm[o:o + n].int()
        o += n
    torch.manual_seed(0)
    model = d.FlashMapDraftModel(d.drafter_config(**over)).to(dev, torch.bfloat16)
    cfg = model.config
    gd = torch.Generator(device=dev).manual_seed(0)
    embed = torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=gd, device=dev).bfloat16()
    lm_head = (torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=gd, device=dev) / 64).bfloat16()
    step = DraftStep(model, embed, lm_head, max_model_len=hi + cfg.block_size + 1, num_steps=jumps, mx=args.mx)
    heads, hd = step.heads, step.head_dim
    caches = []
    for _ in model.layers:
        c = torch.empty(total, heads, page, 2 * hd, dtype=torch.bfloat16, device=dev)
        c.normal_(generator=gd)
        caches.append(c)
    layout = step.cache_layout(caches)
    anchors = torch.randint(0, cfg.vocab_size, (batch,), generator=g).to(dev)
    a_pos = (lens - 1).to(dev)
    a_slots = (bt[torch.arange(batch), (lens - 1) // page].long() * page + (lens - 1) % page).to(dev)
    z = torch.randn(batch * cfg.block_size, step.noise_columns, generator=gd, device=dev)
    bt_d = bt.to(dev)
    tokens = torch.empty(batch * cfg.block_size, dtype=torch.int64, device=dev)

    def call():
        tokens.copy_(step.greedy(step(anchors, a_pos, a_slots, z, caches, bt_d, layout)))

    timing = _measure(call, args)
    ms, kernel_ms = timing["ms"], timing["kernel_ms"]
    sum_l = int(lens.sum())
    k_rows, layers = cfg.block_size, len(model.layers)
    attn_bytes = sum_l * heads * hd * 2 * 2 + 2 * batch * k_rows * heads * hd * 2 + 4 * total + 8 * batch \
        + batch * k_rows * hd * 4
    attn_own = attn_bytes - batch * k_rows * heads * hd * 2  # the combine writes the output rows
    gbs = attn_own / (kernel_ms * 1e-3) / 1e9
    dim, inter, th, vocab = cfg.hidden_size, cfg.intermediate_size, cfg.target_hidden_size, cfg.vocab_size
    rows = batch * k_rows
    dit_flops = 2 * rows * layers * (6 * dim * dim + 2 * dim * inter)
    if jumps == 1:  # the folded noise read-out
        entry_flops = 2 * rows * th * dim
    else:  # per jump the state's two projections onto the embedding and x_embed; the jump head between
        entry_flops = jumps * (2 * 2 * rows * vocab * th + 2 * rows * th * dim) + (jumps - 1) * 2 * rows * dim * vocab
    gemm_flops = jumps * dit_flops + entry_flops + 2 * rows * vocab * dim + 2 * batch * (th * dim + 2 * layers * dim * dim)
    result = {
        "metric": f"{jumps}-jump draft step µs/step (anchor write, " + (
            "noise read-out" if jumps == 1 else "state embedding and update") + f", {jumps} x 6 DiT layers, "
                  f"folded head, argmax), 8B drafter, K=16, batch {batch}, ctx "
                  + ("256–8k" if (lo, hi) == (256, 8192) else f"{lo}") + _mx_words(args) + ", 1 GPU",
        "value": round(ms * 1e3, 2), "unit": "us/step", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup,
        "ms_per_step": round(ms, 5), "higher_is_better": False, "scaling": "weak", "vs_baseline": None,
        "dtype": _step_dtype(args),
        "data": "synthetic: random-init drafter and target embedding / LM head, random paged K/V, "
                                 "seeded draw of lengths and block table (C3's)",
        "config": {"workload": args.workload, "batch": batch, "jumps": jumps, "hidden": dim, "heads": heads,
                   "head_dim": hd, "layers": layers, "intermediate": inter, "mlp": cfg.mlp_type, "vocab": vocab,
                   "target_hidden": th, "block_queries": k_rows, "ctx_lo": lo, "ctx_hi": hi, "ctx_sum": sum_l,
                   "page": page},
        "roofline": {"bound": "hbm", "kernel": "attn_fwd_kernel (the step's cross-attention, one launch per layer)",
                     "achieved": round(gbs, 1), "peak": HBM_PEAK_GBS, "unit": "GB/s",
                     "frac": round(gbs / HBM_PEAK_GBS, 4), "traffic": None, "bytes_per_launch": attn_own,
                     "call_bytes": attn_bytes,
                     "kernel_us": round(kernel_ms * 1e3, 2)},
        "attention_share": round(jumps * layers * kernel_ms / ms, 4),
        "gemm_tflop_per_step": round(gemm_flops / 1e12, 4),
        **_timing_fields(timing),
    }
    if not args.no_cpu_baseline:
        result["cpu_baseline"] = draft_step_cpu_baseline(step, lm_head, lens, anchors.cpu(), z.cpu(), args.cpu_budget)
    return result


def _mx_words(args) -> str:
    return ", projections and head on microscaled 4-bit weights" if args.mx else ""


def _step_dtype(args) -> str:
    return "mxfp4 weights x mxfp8 rows, bf16 elsewhere" if args.mx else "bf16"


def draft_step_cpu_baseline(step, lm_head, lens, anchors, z, budget_s) -> dict:
    """The draft-step oracle (bf16/fp32 torch on the host cores, prepared from the
    drafter's raw weights) request by request, each over a CPU paged cache of its own
    context (random values: the time does not depend on them); ``cpu_timed``'s protocol,
    weighted by requests."""
    from oracle import draft_step as oracle

    model = step.model
    sd = {k: v.detach().cpu() for k, v in model.state_dict().items()}
    w = oracle.prepare(sd, dict(vars(model.config)), step.embed_weight.cpu(), lm_head.cpu(), None, step.num_steps,
                       int(lens.max()) + step.block + 1)
    k, page = step.block, 16
    g = torch.Generator().manual_seed(1)
    held = {}

    def request(b):
        if b not in held:  # set-up, outside the timed calls after the first
            n = int(lens[b])
            blocks = math.ceil(n / page)
            held[b] = ([torch.randn(blocks, step.heads, page, 2 * step.head_dim, generator=g).bfloat16()
                        for _ in model.layers], torch.arange(blocks, dtype=torch.int32)[None],
                       torch.tensor([n - 1]))
        return held[b]

    def run(count):
        for b in range(count):
            caches, bt, pos = request(b)
            oracle.write_anchors(w, anchors[b:b + 1], pos, pos.clone(), caches, page)
            if step.num_steps == 1:  # the noise through the embedding (its values do not change the time)
                oracle.draft(w, pos, caches, bt, noise_embeds=z[b * k:(b + 1) * k].bfloat16())[1].argmax(-1)
            else:
                oracle.draft(w, pos, caches, bt, state=z[b * k:(b + 1) * k])[1].argmax(-1)

    rec = cpu_timed(run, [1] * len(lens), "us/step", "requests", budget_s)
    rec["sample"] += "; the oracle's anchor write, DiT input, DiT per jump and head + LM head + argmax"
    return rec


# The SGLang plugin's one-jump draft step (flashmap_amd.sglang_step.SGLangDraftStep): name
# -> (requests, candidates per request, ctx lo, ctx hi). The 8B drafter over a Qwen3-8B
# target as for the vLLM step; each layer's context in an SGLang token pool at randomly
# permuted rows. With candidates (tree drafting) a request's blocks attend together to its
# one context.
SGLANG_STEP_WORKLOADS = {
    "sglang-draft-step-8b-b64": (64, 1, 256, 8192),
    "sglang-draft-step-8b-b4-n8": (4, 8, 1024, 8192),
}


def run_sglang_step(args, dev) -> dict:
    """One call = one SGLang draft step: the anchors' pool rows written, the folded noise
    read-out, 6 DiT layers (each with its token-paged cross-attention), the folded head
    and the sampler (every row greedy). The plan is built per step inside the call."""
    from flashmap_amd import drafter as d
    from flashmap_amd.sglang_step import SGLangDraftStep

    requests, n_cand, lo, hi = SGLANG_STEP_WORKLOADS[args.workload]
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(lo, hi + 1, (requests,), generator=g)  # context positions incl. the anchor
    ctx = int(lens.sum())
    slots = torch.randperm(ctx, generator=g).to(torch.int32)
    page_table = torch.zeros(requests, hi, dtype=torch.int32)
    o = 0
    for r in range(requests):
        page_table[r, :int(lens[r])] = slots[o:o + int(lens[r])]
        o += int(lens[r])
    torch.manual_seed(0)
    model = d.FlashMapDraftModel(d.drafter_config()).to(dev, torch.bfloat16)
    cfg = model.config
    gd = torch.Generator(device=dev).manual_seed(0)
    embed = torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=gd, device=dev).bfloat16()
    lm_head = (torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=gd, device=dev) / 64).bfloat16()
    step = SGLangDraftStep(model, embed, lm_head, max_positions=hi + cfg.block_size + 1, mx=args.mx)
    heads, hd, k = step.heads, step.head_dim, cfg.block_size
    k_bufs, v_bufs = [], []
    for _ in model.layers:
        for bufs in (k_bufs, v_bufs):
            b = torch.empty(ctx, heads, hd, dtype=torch.bfloat16, device=dev)
            b.normal_(generator=gd)
            bufs.append(b)
    meta = step.pool_meta(k_bufs, v_bufs)
    anchors = torch.randint(0, cfg.vocab_size, (requests,), generator=g).to(dev)
    a_pos = (lens - 1).to(dev)
    a_locs = page_table[torch.arange(requests), lens - 1].long().to(dev)
    rows = requests * n_cand * k
    z = torch.randn(rows, cfg.target_hidden_size, generator=gd, device=dev)
    pt = page_table.to(dev)
    temps = torch.ones(rows, device=dev)
    greedy = torch.ones(rows, dtype=torch.bool, device=dev)
    seed = torch.tensor(7, dtype=torch.int64, device=dev)
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)

    def call():
        hidden = step(anchors, a_pos, a_locs, z, k_bufs, v_bufs, pt, n_cand=n_cand, meta=meta)
        tokens.copy_(step.sample(hidden, temps, greedy, seed))

    timing = _measure(call, args)
    ms, kernel_ms = timing["ms"], timing["kernel_ms"]
    layers = len(model.layers)
    own = ctx * heads * hd * 2 * 2 + 4 * ctx + 4 * requests + rows * heads * hd * 2  # K/V, rows, lengths, Q
    gbs = own / (kernel_ms * 1e-3) / 1e9
    dim, inter, th, vocab = cfg.hidden_size, cfg.intermediate_size, cfg.target_hidden_size, cfg.vocab_size
    gemm_flops = 2 * rows * (layers * (6 * dim * dim + 2 * dim * inter) + th * dim + vocab * dim) \
        + 2 * requests * (th * dim + 2 * layers * dim * dim)
    result = {
        "metric": f"SGLang one-jump draft step µs/step ({n_cand} candidate(s) per request: anchor write, noise "
                  "read-out, 6 DiT layers, folded head, sampler), 8B drafter" + _mx_words(args) + ", 1 GPU",
        "value": round(ms * 1e3, 2), "unit": "us/step", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup,
        "ms_per_step": round(ms, 5), "higher_is_better": False, "scaling": "weak", "vs_baseline": None,
        "dtype": _step_dtype(args),
        "data": "synthetic: random-init drafter and target embedding / LM head, random pools, "
                                 "seeded draw of lengths and pool rows",
        "config": {"workload": args.workload, "requests": requests, "candidates": n_cand, "hidden": dim,
                   "heads": heads, "head_dim": hd, "layers": layers, "intermediate": inter, "mlp": cfg.mlp_type,
                   "vocab": vocab, "target_hidden": th, "block_queries": k, "ctx_lo": lo, "ctx_hi": hi,
                   "ctx_sum": ctx, "layout": "sglang token pools (pool, heads, head_dim), page table"},
        "roofline": {"bound": "hbm", "kernel": "attn_fwd_kernel (the step's cross-attention, one launch per layer)",
                     "achieved": round(gbs, 1), "peak": HBM_PEAK_GBS, "unit": "GB/s",
                     "frac": round(gbs / HBM_PEAK_GBS, 4), "traffic": None, "bytes_per_launch": own,
                     "kernel_us": round(kernel_ms * 1e3, 2)},
        "attention_share": round(layers * kernel_ms / ms, 4),
        "gemm_tflop_per_step": round(gemm_flops / 1e12, 4),
        **_timing_fields(timing),
    }
    if not args.no_cpu_baseline:
        result["cpu_baseline"] = sglang_step_cpu_baseline(step, lm_head, lens, anchors.cpu(), n_cand, args.cpu_budget)
    return result


def sglang_step_cpu_baseline(step, lm_head, lens, anchors, n_cand, budget_s) -> dict:
    """The SGLang step's oracle (bf16/fp32 torch on the host cores, prepared from the
    drafter's raw weights) request by request over a pool of its own context (random
    values); ``cpu_timed``'s protocol, weighted by requests."""
    from oracle import draft_step as oracle

    model = step.model
    sd = {key: v.detach().cpu() for key, v in model.state_dict().items()}
    w = oracle.prepare(sd, dict(vars(model.config)), step.embed_weight.cpu(), lm_head.cpu(), None, 1,
                       int(lens.max()) + step.block + 1)
    k = step.block
    g = torch.Generator().manual_seed(1)
    held = {}

    def request(r):
        if r not in held:
            n = int(lens[r])
            held[r] = ([torch.randn(n, step.heads, step.head_dim, generator=g).bfloat16() for _ in model.layers],
                       [torch.randn(n, step.heads, step.head_dim, generator=g).bfloat16() for _ in model.layers],
                       torch.arange(n, dtype=torch.int32)[None], torch.tensor([n - 1]),
                       torch.randn(n_cand * k, step.cfg.target_hidden_size, generator=g).bfloat16())
        return held[r]

    def run(count):
        for r in range(count):
            kb, vb, pt, pos, noise = request(r)
            oracle.pool_write_anchors(w, anchors[r:r + 1], pos, pos.clone(), kb, vb)
            oracle.pool_draft(w, pos, kb, vb, pt, noise, n_cand)[1].argmax(-1)

    rec = cpu_timed(run, [1] * len(lens), "us/step", "requests", budget_s)
    rec["sample"] += "; the oracle's anchor write, read-out, DiT over token pools and head + LM head + argmax"
    return rec


# The batch-1 contiguous case (FlashMapCache views): name -> (batch, hq, hkv, head_dim, K,
# context positions). Keys are drawn as already normed and rotated (the cache's state).
CONTIG_WORKLOADS = {
    "c2-qwen3-8b-contig-b1": (1, 32, 8, 128, 16, 2048),
}


def run_contig(args, dev) -> dict:
    """One call = the block attention with the query prologue applied in the kernel, on
    contiguous (batch, kv heads, positions, head_dim) keys and values (FlashMapCache
    views), the rotary angles as FlashMapAttention.forward passes them: one (cos, sin)
    row per draft token. Latency-bound at batch 1: timed call by call after an L2 /
    Infinity Cache flush (see _flushed)."""
    from flashmap_amd import ops
    from flashmap_amd.drafter import _token_rope, rope_tables
    from oracle import attention as ref

    batch, hq, hkv, d, k_rows, ctx = CONTIG_WORKLOADS[args.workload]
    g = torch.Generator().manual_seed(0)
    q = torch.randn(batch, k_rows, hq, d, generator=g).bfloat16()
    keys = torch.randn(batch, hkv, ctx, d, generator=g).bfloat16()
    values = torch.randn(batch, hkv, ctx, d, generator=g).bfloat16()
    table = ref.rope_table(ctx + k_rows + 1, d, 1e6)
    qpos = (ctx + torch.arange(k_rows)).repeat(batch)
    w = torch.ones(d)
    qd, kd, vd = q.to(dev), keys.to(dev), values.to(dev)
    rope = _token_rope(rope_tables(qpos.view(batch, k_rows).to(dev), d, 1e6), batch, k_rows)
    pro = ops.Prologue(w.to(dev), rope, None, 1e-6)
    out = torch.empty_like(qd)

    def call():
        ops.block_attention_contig(qd, kd, vd, d ** -0.5, prologue=pro, out=out)

    t = _flushed(call, args, dev)
    ms, kernel_ms = t["ms"], t["kernel_ms"]
    kv = batch * hkv * ctx * d * 2 * 2
    total = kv + 2 * batch * k_rows * hq * d * 2 + batch * k_rows * d * 4
    own = total - batch * k_rows * hq * d * 2  # the merge writes the output rows
    gbs = own / (kernel_ms * 1e-3) / 1e9
    result = {
        "metric": METRIC.replace("batch 64, ctx 256–8k", f"batch {batch}, ctx {ctx} contiguous"),
        "value": round(ms * 1e3, 2), "unit": "us/call", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup,
        "ms_per_step": round(ms, 5), "higher_is_better": False, "scaling": "weak", "vs_baseline": None,
        "dtype": "bf16", "data": "synthetic: seeded CPU draw (q, K, V)",
        "config": {"workload": args.workload, "batch": batch, "q_heads": hq, "kv_heads": hkv, "head_dim": d,
                   "block_queries": k_rows, "ctx": ctx, "layout": "contiguous (batch, kv_heads, ctx, head_dim)",
                   "prologue": "QK-RMSNorm + RoPE inside the attention kernel (no query pass), "
                               "one (cos, sin) row per draft token as FlashMapAttention passes them"},
        "roofline": {"bound": "hbm", "kernel": "attn_small_kernel", "achieved": round(gbs, 1), "peak": HBM_PEAK_GBS,
                     "unit": "GB/s", "frac": round(gbs / HBM_PEAK_GBS, 4), "traffic": None, "bytes_per_launch": own,
                     "call_bytes": total,
                     "kernel_us": round(kernel_ms * 1e3, 2)},
        "warm_us_per_call": round(t["warm_ms"] * 1e3, 2),
        "graph_us_per_call": round(t["graph_ms"] * 1e3, 2),
        "timing": "value: median of K calls, each after a 512 MB write that evicts L2 and the Infinity "
                  "Cache (K/V from HBM), between its own events; warm: K back-to-back calls; graph: K "
                  "back-to-back replays of the captured call; kernel_us: HIP events around the main "
                  "kernel, after a flush",
    }
    if not args.no_cpu_baseline:
        def run(count):
            for b in range(count):
                qn = ref.rms_norm_rope_vllm(q[b], w, table, qpos[b * k_rows:(b + 1) * k_rows], 1e-6)
                ref.attention(qn.transpose(0, 1), keys[b], values[b])

        rec = cpu_timed(run, [ctx] * batch, "us/call", "sequences", args.cpu_budget)
        rec["sample"] += "; fp32 oracle prologue + attention"
        result["cpu_baseline"] = rec
    return result


def _events_ms(call, steps: int) -> float:
    """ms per call over exactly ``steps`` back-to-back calls, bracketed by synchronizations."""
    torch.cuda.synchronize()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(steps):
        call()
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) / steps


def _measure(call, args, kernel_events: bool = True) -> dict:
    """The timing protocol of every workload.

    1. cold: W warm-up calls, then K timed calls, right after the set-up (the GPU has
       been idle): reported, not the value.
    2. settle: back-to-back calls for ``--settle-ms`` (default 100 ms). When a load this
       heavy starts, the GPU's power controller first cuts the clocks (measured: the main
       kernel goes from 165 us to about 205 us within 4 ms of the load's start and comes
       back over about 25 ms; a plain 1 GiB copy shows no such dip), so calls timed inside
       that window measure the controller's transient, not the sustained rate.
    3. the value: W warm-up calls, then exactly K timed calls.
    4. the main kernel alone: K calls with HIP events recorded around each of its
       launches on its stream (fm_profile_*).
    """
    import ctypes

    from flashmap_amd import _native

    for _ in range(args.warmup):
        call()
    cold = _events_ms(call, args.steps)
    settle_calls = 0
    t0 = time.perf_counter()
    while (time.perf_counter() - t0) * 1e3 < args.settle_ms:
        for _ in range(10):
            call()
        settle_calls += 10
        torch.cuda.synchronize()
    settle_ms = (time.perf_counter() - t0) * 1e3
    for _ in range(args.warmup):
        call()
    ms = _events_ms(call, args.steps)
    kernel_ms = None
    if kernel_events:
        lib = _native.lib()
        lib.fm_profile_enable(1)
        for _ in range(args.steps):
            call()
        torch.cuda.synchronize()
        tot, cnt = ctypes.c_double(), ctypes.c_int64()
        _native.call("fm_profile_read", ctypes.byref(tot), ctypes.byref(cnt))
        lib.fm_profile_enable(0)
        kernel_ms = tot.value / max(cnt.value, 1)
    return {"ms": ms, "kernel_ms": kernel_ms, "cold_ms": cold,
            "settle": {"ms": round(settle_ms, 1), "calls": settle_calls}}


def drift_series(call, calls: int, dev, copy_every: int = 250) -> dict:
    """The call back to back from an idle GPU: each call's duration (events around it), the
    shader clock right after it (fm_clock_probe: shader-clock ticks over 100 MHz real-time
    ticks across a 4000-tick spin), and a 1 GiB copy every ``copy_every`` calls as a
    bandwidth control. Summaries per 50 calls, the first 40 calls in full."""
    import ctypes

    from flashmap_amd import _native

    probes = torch.zeros(calls, 2, dtype=torch.int64, device=dev)
    src = torch.empty(1 << 30, dtype=torch.uint8, device=dev).fill_(1)
    dst = torch.empty_like(src)
    stream = torch.cuda.current_stream().cuda_stream
    call()
    dst.copy_(src)
    torch.cuda.synchronize()
    time.sleep(0.5)  # idle, as after set-up
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(2 * calls)]
    copies = []
    for i in range(calls):
        ev[2 * i].record()
        call()
        ev[2 * i + 1].record()
        _native.call("fm_clock_probe", ctypes.c_void_p(probes[i].data_ptr()), ctypes.c_uint64(4000),
                     ctypes.c_void_p(stream))
        if copy_every and (i + 1) % copy_every == 0:
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            dst.copy_(src)
            b.record()
            copies.append((i + 1, a, b))
    torch.cuda.synchronize()
    us = [ev[2 * i].elapsed_time(ev[2 * i + 1]) * 1e3 for i in range(calls)]
    p = probes.cpu().double()
    ghz = (p[:, 0] / (p[:, 1] / 100e6) / 1e9).tolist()
    start = [ev[0].elapsed_time(ev[2 * i]) for i in range(calls)]
    med = lambda xs: sorted(xs)[len(xs) // 2]  # noqa: E731
    return {
        "workload": "c3-qwen3-8b-paged-b64", "calls": calls,
        "first_40": [{"ms_since_start": round(start[i], 2), "us": round(us[i], 1), "sclk_ghz": round(ghz[i], 2)}
                     for i in range(min(40, calls))],
        "per_50": [{"calls": f"{s}-{min(calls, s + 50) - 1}", "median_us": round(med(us[s:s + 50]), 1),
                    "median_sclk_ghz": round(med(ghz[s:s + 50]), 2)} for s in range(0, calls, 50)],
        "copy_1gib": [{"after_call": i, "tbs": round(2 * (1 << 30) / (a.elapsed_time(b) * 1e-3) / 1e12, 3)}
                      for i, a, b in copies],
    }


def _timing_fields(t: dict) -> dict:
    """The extra keys every bench line carries about its timing protocol."""
    return {"cold_us_per_call": round(t["cold_ms"] * 1e3, 2), "settle": t["settle"],
            "timing": "value: K back-to-back calls after --settle-ms of calls and W warm-ups; "
                      "cold_us_per_call: the same K calls before the settling, right after set-up"}


def _time_call(call, args) -> tuple[float, float, dict]:
    """(ms per call, ms per main-kernel launch, the timing record)."""
    t = _measure(call, args)
    return t["ms"], t["kernel_ms"], t


def tree_inputs(workload: str):
    """Seeded CPU draw of a token-pool workload, in a fixed order: lengths, the pool slots
    (a permutation), the queries (requests, n_cand x 16, heads, head_dim) and the K and V
    pools (rounded to e4m3 for the fp8 workloads). Returns (lens, page table, q, k pool,
    v pool)."""
    fp8 = workload in TREE_FP8_WORKLOADS
    requests, hq, hkv, d, n_cand, lo, hi = TREE_WORKLOADS[TREE_FP8_WORKLOADS.get(workload, workload)]
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(lo, hi + 1, (requests,), generator=g)
    ctx = int(lens.sum())
    slots = torch.randperm(ctx, generator=g).to(torch.int32)
    pt = torch.zeros(requests, hi, dtype=torch.int32)
    o = 0
    for b in range(requests):
        pt[b, :int(lens[b])] = slots[o:o + int(lens[b])]
        o += int(lens[b])
    q = torch.randn(requests, n_cand * 16, hq, d, generator=g).bfloat16()
    kb = torch.randn(ctx, hkv, d, generator=g).bfloat16()
    vb = torch.randn(ctx, hkv, d, generator=g).bfloat16()
    if fp8:  # e4m3 pools (round to nearest even, saturating at 448)
        kb, vb = (x.float().clamp(-448.0, 448.0).to(torch.float8_e4m3fn) for x in (kb, vb))
    return lens, pt, q, kb, vb


def run_tree(args, dev) -> dict:
    """One call = flashmap_sglang::paged_cross_attention of every request's candidates
    side by side: query packing, the split-KV stream and the combine."""
    from flashmap_amd import ops

    fp8 = args.workload in TREE_FP8_WORKLOADS
    requests, hq, hkv, d, n_cand, lo, hi = TREE_WORKLOADS[TREE_FP8_WORKLOADS.get(args.workload, args.workload)]
    q_len = n_cand * 16
    lens, pt, q, kb, vb = tree_inputs(args.workload)
    ctx = int(lens.sum())
    q, kb, vb = q.to(dev), kb.to(dev), vb.to(dev)
    lens_d, pt_d = lens.to(dev, torch.int32), pt.to(dev)
    plan = ops.attention_plan(lens_d)
    out = torch.empty_like(q)

    def call():
        if fp8:
            ops.block_attention_token_paged_fp8(q, kb, vb, lens_d, pt_d, plan=plan, out=out)
        else:
            ops.block_attention_token_paged(q, kb, vb, lens_d, pt_d, plan=plan, out=out)

    ms, kernel_ms, timing = _time_call(call, args)
    kv = ctx * hkv * d * 2 * (1 if fp8 else 2)
    total = kv + 4 * ctx + 4 * requests + 2 * requests * q_len * hq * d * 2
    flops = 4 * q_len * hq * d * ctx
    own = total - requests * q_len * hq * d * 2  # the combine writes the output rows
    gbs = own / (kernel_ms * 1e-3) / 1e9
    tflops = flops / (kernel_ms * 1e-3) / 1e12
    hbm_frac, mfma_frac = gbs / HBM_PEAK_GBS, tflops / MFMA_BF16_PEAK_TFLOPS
    mfma_bound = flops / (MFMA_BF16_PEAK_TFLOPS * 1e12) > own / (HBM_PEAK_GBS * 1e9)
    result = {
        "metric": "tree-drafting cross-attn µs/call, n_cand x 16 rows per request, 1 GPU",
        "value": round(ms * 1e3, 2), "unit": "us/call", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup,
        "ms_per_step": round(ms, 5), "higher_is_better": False, "scaling": "weak", "vs_baseline": None,
        "dtype": "e4m3 K/V, bf16 q" if fp8 else "bf16",
        "data": "synthetic: seeded CPU draw (lengths, pool slots, q, K/V)",
        "config": {"workload": args.workload, "requests": requests, "q_heads": hq, "kv_heads": hkv, "head_dim": d,
                   "candidates": n_cand, "q_rows_per_request": q_len, "ctx_lo": lo, "ctx_hi": hi, "ctx_sum": ctx,
                   "layout": "sglang token pool (pool, kv_heads, head_dim), page table",
                   "kv_dtype": "e4m3" if fp8 else "bf16"},
        "roofline": ({"bound": "mfma", "achieved": round(tflops, 1), "peak": MFMA_BF16_PEAK_TFLOPS,
                      "unit": "TFLOP/s", "frac": round(mfma_frac, 4)} if mfma_bound else
                     {"bound": "hbm", "achieved": round(gbs, 1), "peak": HBM_PEAK_GBS, "unit": "GB/s",
                      "frac": round(hbm_frac, 4)}),
        "hbm_frac": round(hbm_frac, 4), "mfma_frac": round(mfma_frac, 4),
    }
    result["roofline"].update({"kernel": "attn_fwd_kernel", "traffic": None, "bytes_per_launch": own,
                               "call_bytes": total,
                               "flops_per_launch": flops, "kernel_us": round(kernel_ms * 1e3, 2)})
    result.update(_timing_fields(timing))
    if not args.no_cpu_baseline:
        result["cpu_baseline"] = tree_cpu_baseline(q, kb, vb, lens, pt, args.cpu_budget, fp8)
    return result


def tree_cpu_baseline(q, kb, vb, lens, pt, budget_s, fp8: bool = False) -> dict:
    """The token-paged oracle (the e4m3 one for e4m3 pools) on the host cores, request by
    request until the budget is spent, scaled to the whole call by context positions."""
    from oracle import attention as ref

    kc, vc, qc = kb.cpu(), vb.cpu(), q.cpu()
    if fp8:  # widened once (exact): the oracle would widen the whole pool for every request
        kc, vc = kc.float(), vc.float()

    def run(count):
        for b in range(count):
            if fp8:
                ref.block_attention_token_paged_fp8(qc[b:b + 1], kc, vc, lens[b:b + 1], pt[b:b + 1])
            else:
                ref.block_attention_token_paged(qc[b:b + 1], kc, vc, lens[b:b + 1], pt[b:b + 1])

    rec = cpu_timed(run, [int(n) for n in lens], "us/call", "requests", budget_s)
    rec["sample"] += (f" (context positions); fp32 oracle token-paged"
                      f"{' e4m3 (pools widened to fp32 once)' if fp8 else ''} attention")
    return rec


def verify_inputs(workload: str):
    """Seeded CPU draw of a verify workload, in a fixed order: lengths, the context's pool
    slots (a permutation), the queries, the verify tokens' keys and values, then the pools'
    rows (drawn in slot order, 32768 at a time). Returns (lens, q, k_ext, v_ext, key pool,
    value pool, kv_indptr, kv_indices, custom mask or None)."""
    batch, hq, hkv, d, length, lo, hi, mask = VERIFY_WORKLOADS[workload]
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(lo, hi + 1, (batch,), generator=g)
    ctx = int(lens.sum())
    slots = torch.randperm(ctx, generator=g).to(torch.int32)
    q = torch.randn(batch * length, hq, d, generator=g).bfloat16()
    k_ext = torch.randn(batch * length, hkv, d, generator=g).bfloat16()
    v_ext = torch.randn(batch * length, hkv, d, generator=g).bfloat16()
    kb = torch.empty(ctx, hkv, d, dtype=torch.bfloat16)
    vb = torch.empty_like(kb)
    chunk = 1 << 15
    for s in range(0, ctx, chunk):  # bounded fp32 temporaries
        e = min(ctx, s + chunk)
        kb[slots[s:e].long()] = torch.randn(e - s, hkv, d, generator=g).bfloat16()
        vb[slots[s:e].long()] = torch.randn(e - s, hkv, d, generator=g).bfloat16()
    indptr = torch.zeros(batch + 1, dtype=torch.int32)
    indptr[1:] = torch.cumsum(lens, 0).to(torch.int32)
    cmask = None
    if mask == "qlen":
        tril = torch.ones(length, length, dtype=torch.bool).tril()
        cmask = tril.reshape(-1).repeat(batch)
    return lens, q, k_ext, v_ext, kb, vb, indptr, slots, cmask


def run_verify(args, dev) -> dict:
    """One call = fm_verify_attention over the batch: plan, query packing, the split-KV
    stream of every request's context, and the combine that attends the verify tokens
    and merges."""
    import ctypes

    from flashmap_amd import _native, ops

    batch, hq, hkv, d, length, lo, hi, mask = VERIFY_WORKLOADS[args.workload]
    lens, q, k_ext, v_ext, kb, vb, indptr, indices, cmask = (
        x.to(dev) if isinstance(x, torch.Tensor) and i > 0 else x for i, x in enumerate(verify_inputs(args.workload)))
    ctx = int(lens.sum())
    out = torch.empty_like(q)

    def call():
        ops.verify_attention(q, k_ext, v_ext, kb, vb, indptr, indices, cmask, None, mask == "qlen", out=out,
                             max_context=hi)

    ms, kernel_ms, timing = _time_call(call, args)
    kv = ctx * hkv * d * 2 * 2
    total = kv + 4 * ctx + 4 * (batch + 1) + 2 * batch * length * hq * d * 2 + batch * length * hkv * d * 2 * 2
    # the main kernel's own share: the context and the query rows (the query pass reads the
    # verify tokens' K/V, the combine writes the output rows)
    own = kv + 4 * ctx + 4 * (batch + 1) + batch * length * hq * d * 2
    achieved = own / (kernel_ms * 1e-3) / 1e9
    traffic = traffic_record(f"attn_fwd_{args.workload.replace('-qwen3-8b-', '_').replace('-', '_')}.traffic.json",
                             args.workload)
    result = {
        "metric": "target verify attn µs/call + achieved HBM TB/s, 17 verify tokens, batch 64, ctx 256–8k, 1 GPU",
        "value": round(ms * 1e3, 2), "unit": "us/call", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup,
        "ms_per_step": round(ms, 5), "higher_is_better": False, "scaling": "weak", "vs_baseline": None,
        "dtype": "bf16", "data": "synthetic: seeded CPU draw (lengths, pool slots, q, K/V)",
        "config": {"workload": args.workload, "batch": batch, "q_heads": hq, "kv_heads": hkv, "head_dim": d,
                   "verify_tokens": length, "ctx_lo": lo, "ctx_hi": hi, "ctx_sum": ctx, "mask": mask,
                   "layout": "sglang token pool (pool, kv_heads, head_dim), kv_indptr/kv_indices"},
        "hbm_tbs": round(total / (ms * 1e-3) / 1e12, 3),
        "roofline": {"bound": "hbm", "kernel": "attn_fwd_kernel", "achieved": round(achieved, 1),
                     "peak": HBM_PEAK_GBS, "unit": "GB/s", "frac": round(achieved / HBM_PEAK_GBS, 4),
                     "traffic": traffic, "bytes_per_launch": own, "call_bytes": total,
                     "kernel_us": round(kernel_ms * 1e3, 2)},
        **_timing_fields(timing),
    }
    if not args.no_cpu_baseline:
        result["cpu_baseline"] = verify_cpu_baseline(q, k_ext, v_ext, kb, vb, indptr, indices, cmask, mask, lens,
                                                     length, args.cpu_budget)
    return result


def verify_cpu_baseline(q, k_ext, v_ext, kb, vb, indptr, indices, cmask, mask, lens, length, budget_s) -> dict:
    """The verify oracle on the host cores, request by request until the budget is
    spent, scaled to the whole call by context positions."""
    from oracle import attention as ref

    ip, idx = indptr.cpu(), indices.cpu()
    kh, vh, qh, keh, veh = kb.cpu(), vb.cpu(), q.cpu(), k_ext.cpu(), v_ext.cpu()
    mh = None if cmask is None else cmask.cpu()

    def run(count):
        for b in range(count):
            lo_, hi_ = int(ip[b]), int(ip[b + 1])
            rows = idx[lo_:hi_].long()
            sub_ip = torch.tensor([0, hi_ - lo_], dtype=torch.int32)
            tok = slice(b * length, (b + 1) * length)
            sub_mask = None if mh is None else mh[b * length * length:(b + 1) * length * length]
            ref.verify_attention(qh[tok], keh[tok], veh[tok], kh[rows], vh[rows], sub_ip, torch.arange(hi_ - lo_),
                                 sub_mask, None, mask == "qlen")

    rec = cpu_timed(run, [int(n) for n in lens], "us/call", "requests", budget_s)
    rec["sample"] += " (context positions); fp32 oracle verify attention (pool rows gathered on the host)"
    return rec


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--warmup", type=int, default=5)
    ap.add_argument("--workload", default="c3-qwen3-8b-paged-b64",
                    choices=sorted(WORKLOADS) + sorted(FP8_WORKLOADS) + sorted(VERIFY_WORKLOADS)
                    + sorted(VIRTUAL_WORKLOADS) + sorted(TREE_WORKLOADS) + sorted(TREE_FP8_WORKLOADS)
                    + sorted(SELECT_WORKLOADS) + sorted(KERNEL_WORKLOADS)
                    + sorted(CONTIG_WORKLOADS) + sorted(DRAFT_STEP_WORKLOADS) + sorted(SGLANG_STEP_WORKLOADS))
    ap.add_argument("--mx", action="store_true",
                    help="the draft steps' projections and head on microscaled 4-bit weights")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--cpu-budget", type=float, default=12.0)
    ap.add_argument("--settle-ms", type=float, default=100.0,
                    help="back-to-back calls before the timed ones (the GPU's clocks settle under the load)")
    ap.add_argument("--drift", type=int, default=0,
                    help="only print the per-call duration and shader-clock series of N calls of the C3 call "
                         "from an idle GPU")
    ap.add_argument("--calibrate-copy", type=int, default=0,
                    help="only run N copies of a 1 GiB buffer (HBM counter calibration)")
    args = ap.parse_args()
    if args.mx and args.workload not in DRAFT_STEP_WORKLOADS and args.workload not in SGLANG_STEP_WORKLOADS:
        ap.error(f"--mx: {args.workload} has no projections (the draft steps have)")
    if args.gpus != 1:
        print(json.dumps({"error": "this benchmark runs on one GPU; the hot path is measured per GPU "
                          "(multi-GPU sharding is a design note, not a measured configuration)"}))
        return 2
    dev = torch.device("cuda", 0)
    if args.calibrate_copy:
        src = torch.empty(1 << 30, dtype=torch.uint8, device=dev).fill_(1)
        dst = torch.empty_like(src)
        for _ in range(args.calibrate_copy):
            dst.copy_(src)
        torch.cuda.synchronize()
        print(json.dumps({"calibrate_copy_bytes": src.numel(), "copies": args.calibrate_copy}))
        return 0

    if args.workload in VERIFY_WORKLOADS:
        print(json.dumps(run_verify(args, dev)))
        return 0
    if args.workload in TREE_WORKLOADS or args.workload in TREE_FP8_WORKLOADS:
        print(json.dumps(run_tree(args, dev)))
        return 0
    if args.workload in SELECT_WORKLOADS:
        print(json.dumps(run_select(args, dev)))
        return 0
    if args.workload in KERNEL_WORKLOADS:
        print(json.dumps(run_kernel(args, dev)))
        return 0
    if args.workload in CONTIG_WORKLOADS:
        print(json.dumps(run_contig(args, dev)))
        return 0
    if args.workload in DRAFT_STEP_WORKLOADS:
        print(json.dumps(run_draft_step(args, dev)))
        return 0
    if args.workload in SGLANG_STEP_WORKLOADS:
        print(json.dumps(run_sglang_step(args, dev)))
        return 0

    from flashmap_amd import _native, ops
    from oracle import attention as ref

    fp8 = args.workload in FP8_WORKLOADS
    virtual = VIRTUAL_WORKLOADS.get(args.workload)
    inp = build_inputs(FP8_WORKLOADS.get(args.workload) or (virtual[0] if virtual else args.workload))
    batch, hq, hkv, d, k_rows, page = (inp[k] for k in ("batch", "hq", "hkv", "d", "k_rows", "page"))
    table = ref.rope_table(inp["hi"] + k_rows + 1, d, 1e6).to(dev)
    rope = ops.rope_from_table(table)
    w = torch.ones(d, device=dev)
    lens = inp["lens"].to(dev, torch.int32)
    bt = inp["bt"].to(dev)
    cache = torch.zeros(inp["total"], hkv, page, 2 * d, dtype=torch.uint8 if fp8 else torch.bfloat16, device=dev)
    ptrs = torch.tensor([cache.data_ptr()], dtype=torch.int64, device=dev)
    writer_args = (inp["kv_pre"].to(dev), inp["positions"].to(dev), inp["slots"].to(dev),
                   w[None].expand(1, d).contiguous(), rope, ptrs,
                   (cache.stride(0), cache.stride(1), cache.stride(2), d), page, 1e-6)
    runs = None
    if virtual:  # (layer + 1) DiT layers packed into caches of hpc heads
        from flashmap_amd import context_cache as cc

        _, hpc, layer = virtual
        vplan = cc.ContextCachePlan(layer + 1, hkv, -(-(layer + 1) * hkv // hpc), hpc, True, "")
        del cache
        caches = [torch.zeros(inp["total"], hpc, page, 2 * d, dtype=torch.bfloat16, device=dev)
                  for _ in range(vplan.num_caches)]
        c0 = caches[0]
        ops.write_context_kv(inp["kv_pre"].to(dev).repeat(1, layer + 1, 1, 1, 1), inp["positions"].to(dev),
                             inp["slots"].to(dev), w[None].expand(layer + 1, d).contiguous(), rope,
                             torch.tensor([c.data_ptr() for c in caches], dtype=torch.int64, device=dev),
                             (c0.stride(0), c0.stride(1), c0.stride(2), d), page, 1e-6, heads_per_cache=hpc)
        runs = vplan.segments[layer]
    elif fp8:
        ops.write_context_kv_fp8(*writer_args, torch.ones(1, 2, device=dev))
    else:
        ops.write_context_kv(*writer_args)
    q_pre = inp["q_pre"].to(dev)
    qpos = torch.cat([int(n) + torch.arange(k_rows) for n in inp["lens"]]).to(dev)
    cu = (torch.arange(batch + 1, dtype=torch.int32) * k_rows).to(dev)
    pro = ops.Prologue(w, rope, qpos, 1e-6)
    max_k = inp["hi"]
    plan = ops.attention_plan(lens)
    out = torch.empty_like(q_pre)

    def call():
        if runs is not None:
            ops.block_attention_paged_runs(q_pre, caches, runs, cu, lens, bt, k_rows, max_k, d ** -0.5,
                                           prologue=pro, plan=plan, out=out)
        elif fp8:
            ops.block_attention_paged_fp8(q_pre, cache, cu, lens, bt, k_rows, max_k, d ** -0.5,
                                          prologue=pro, plan=plan, out=out)
        else:
            ops.block_attention_paged(q_pre, cache, cu, lens, bt, k_rows, max_k, d ** -0.5,
                                      prologue=pro, plan=plan, out=out)

    if args.drift:
        print(json.dumps(drift_series(call, args.drift, dev)))
        return 0
    ms, kernel_ms, timing = _time_call(call, args)

    ab = algorithmic_bytes(inp, kv_bytes=1 if fp8 else 2)
    traffic = traffic_record(f"attn_fwd_{args.workload.split('-', 1)[0]}_paged_b{batch}{'_fp8' if fp8 else ''}"
                             ".traffic.json", args.workload)
    us = ms * 1e3
    achieved = ab["kernel"] / (kernel_ms * 1e-3) / 1e9  # GB/s of the main kernel on its own bytes
    result = {
        "metric": METRIC,
        "value": round(us, 2),
        "unit": "us/call",
        "n_gpus": 1,
        "steps": args.steps,
        "warmup": args.warmup,
        "ms_per_step": round(ms, 5),
        "higher_is_better": False,
        "scaling": "weak",
        "vs_baseline": None,
        "dtype": "e4m3 K/V, bf16 q" if fp8 else "bf16",
        "data": "synthetic: seeded CPU draw (lengths, permuted block table, q, K/V), K k-normed and "
                "rotated on the GPU by the context writer",
        "config": {
            "workload": args.workload,
            "batch": batch, "q_heads": hq, "kv_heads": hkv, "head_dim": d, "block_queries": k_rows,
            "ctx_lo": inp["lo"], "ctx_hi": inp["hi"], "ctx_sum": ab["sum_l"], "page": page,
            "layout": "vllm paged (blocks, kv_heads, page, 2*head_dim)" + (
                f", virtual context-cache layout: caches of {virtual[1]} heads, runs {runs}" if virtual else ""),
            "prologue": prologue_label(fp8),
            "kv_dtype": "e4m3" if fp8 else "bf16",
        },
        "hbm_tbs": round(ab["total"] / (ms * 1e-3) / 1e12, 3),
        "kv_tbs": round(ab["kv"] / (ms * 1e-3) / 1e12, 3),
        "roofline": {
            "bound": "hbm",
            "kernel": "attn_fwd_kernel",
            "achieved": round(achieved, 1),
            "peak": HBM_PEAK_GBS,
            "unit": "GB/s",
            "frac": round(achieved / HBM_PEAK_GBS, 4),
            "traffic": traffic,
            "bytes_per_launch": ab["kernel"],
            "call_bytes": ab["total"],
            "kernel_us": round(kernel_ms * 1e3, 2),
        },
        "mfma": mfma_record(args.workload, batch, ab["flops"], kernel_ms, fp8),
        **_timing_fields(timing),
    }
    if not args.no_cpu_baseline:
        result["cpu_baseline"] = cpu_baseline(inp, args.cpu_budget)
    print(json.dumps(result))
    return 0


if __name__ == "__main__":
    sys.exit(main())
