"""The draft steps with their projections in microscaled 4 bits (``mx=True``), as a serving
program calls them: every operator call of the step, on the inputs that the step gave it, against
float64 within _mx_checks.py's bounds; the step as a whole against the bf16 step on the weights
that the 4 bits stand for, which has everything but the 8-bit operands' rounding; replays of a
captured step."""

import pytest
import torch

from _inputs import gen
from _mx_checks import check_activation, check_adaln, check_product, check_rms_norm, codes_of
from flashmap_amd import ops
from flashmap_amd.draft_step import DraftStep
from flashmap_amd.sglang_step import SGLangDraftStep
from oracle import mx
from test_gpu_draft_step import CASES, _model, _paged_context

pytestmark = pytest.mark.gpu


@pytest.fixture
def calls(monkeypatch):
    """The microscaled calls made: (name, arguments, result), tensors as they were then."""
    made = []

    def copy(v):
        if isinstance(v, ops.MX):
            return ops.MX(v.codes.clone(), v.scales.clone(), v.bits, v.shape)
        if isinstance(v, (tuple, list)):
            return tuple(copy(u) for u in v)
        return v.clone() if isinstance(v, torch.Tensor) else v

    def record(name):
        call = getattr(ops, name)

        def recorded(*args, **kwargs):
            held = copy(args), {k: copy(v) for k, v in kwargs.items()}
            out = call(*args, **kwargs)
            made.append((name, *held, copy(out)))
            return out

        monkeypatch.setattr(ops, name, recorded)

    for name in ("mx_linear", "mx_quantize", "rms_norm_mx", "adaln_residual_mx"):
        record(name)
    return made


def _check(calls) -> dict:
    """Every call against float64; how many there were of each."""
    count = {}
    for name, args, kwargs, out in calls:
        count[name] = count.get(name, 0) + 1
        host = [a.cpu() if isinstance(a, torch.Tensor) else a for a in args]
        if name == "mx_linear":
            bias = args[2] if len(args) > 2 else None
            x = args[0] if isinstance(args[0], ops.MX) else args[0].reshape(-1, args[0].shape[-1])
            xv = (mx.values(*codes_of(x), x.bits) if isinstance(x, ops.MX) else mx.values(*mx.quantize(x.cpu(), 8), 8))
            check_product(out.reshape(-1, out.shape[-1]), xv, mx.values(*codes_of(args[1]), 4), bias)
        elif name == "mx_quantize" and len(args) == 3:
            check_activation(out, host[0], args[2])
        elif name == "rms_norm_mx":
            check_rms_norm(out[0], out[1], host[0], None, host[1].float(), args[2])
        elif name == "adaln_residual_mx":
            x, y, gate, (scale, shift), eps = host[0], host[1], host[2], args[3], args[4]
            if kwargs.get("gate_per_row"):
                gate = gate.view(-1, 1)
            check_adaln(out[0], out[1], x if y is None else x.expand_as(y), y, gate, scale.cpu(), shift.cpu(), eps)
    return count


def _stood_for(w: torch.Tensor) -> torch.Tensor:
    return ops.mx_dequantize(ops.mx_quantize(w, 4))


def _as_stored(step, joined) -> None:
    """A bf16 step on the values that the 4-bit weights stand for (bf16 holds them exactly)."""
    model = step.model
    for layer in model.layers:
        held = [layer.self_attn.o_proj, layer.cross_attn.q_proj, layer.cross_attn.o_proj]
        held += ([layer.mlp.gate_up_proj, layer.mlp.down_proj] if layer.mlp.mlp_type == "swiglu"
                 else [layer.mlp.fc1, layer.mlp.fc2])
        for module in held:
            module.weight.data = _stood_for(module.weight.data)
    for module in (model.fc, model.anchor_proj):
        module.weight.data = _stood_for(module.weight.data)
    step.self_qkv = [_stood_for(w) for w in step.self_qkv]
    for name in joined:
        setattr(step, name, _stood_for(getattr(step, name)))


# A step's wiring: the 8-bit operands' rounding is at most 2^-4 of a value, 2^-5.5 of a row's norm
# (uniform in the step: 2^-4 / sqrt 3 at the top of a binade, half that at its bottom); the models'
# two layers have 15 such operands behind each other, independent: sqrt(15) 2^-5.5 = 0.09. A wrong
# weight or a lost bias gives errors of a row's own size.
WIRING = 0.25


def _close(got, want, what):
    g, w = got.double().cpu().flatten(0, -2), want.double().cpu().flatten(0, -2)
    rel = (g - w).norm(dim=-1) / w.norm(dim=-1).clamp_min(1e-30)
    print(f"  {what}: worst row {rel.max():.4f}, mean {rel.mean():.5f}", flush=True)
    assert rel.max() <= WIRING, what


def _vllm(name, dev, steps):
    model = _model(dict(CASES[name]), dev, 11)
    cfg = model.config
    g = gen(5)
    embed = torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g).bfloat16().to(dev)
    lm_head = (torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g) / 8).bfloat16().to(dev)
    hot = torch.arange(0, 2 * cfg.state_vocab_size, 2).to(dev) if cfg.state_vocab_size else None

    def make(held):
        return DraftStep(model, embed, lm_head, max_model_len=512, hot_ids=hot, num_steps=steps, mx=held)

    step = make(True)
    lens = torch.tensor([37, 100, 0, 64])
    states = torch.randn(int(lens.sum()), len(cfg.target_layer_ids) * cfg.target_hidden_size, generator=g).bfloat16()
    anchors = torch.randint(0, cfg.vocab_size, (len(lens),), generator=g).to(dev)
    z = torch.randn(len(lens) * cfg.block_size, step.noise_columns, generator=g).to(dev)

    def run(step=step):
        caches, layout, bt, _, _, a_slots = _paged_context(step, states, lens, dev, gen(6))
        hidden = step(anchors, lens.to(dev), a_slots.to(dev), z, caches, bt.to(dev), layout)
        return caches, hidden, step.logits(hidden)

    return step, run, make


@pytest.mark.parametrize("steps", [1, 2])
@pytest.mark.parametrize("name", sorted(CASES))
def test_vllm_step(dev, calls, name, steps):
    print(f"mx draft step {name}, {steps} jump(s)", flush=True)
    step, run, make = _vllm(name, dev, steps)
    layers = len(step.model.layers)
    assert all(q.bits == 4 for layer in step.mx_layers for q in (layer.qkv, layer.self_o, layer.up, layer.down))
    assert isinstance(step.head_weight, ops.MX) and isinstance(step.noise_embed, ops.MX)
    calls.clear()
    caches, hidden, logits = run()
    assert hidden.dtype == logits.dtype == torch.bfloat16 and torch.isfinite(logits).all()
    count = _check(calls)
    # per jump: three norms, an activation and six projections a layer, x_embed or the noise's
    # read-out; between jumps the head; the context's and anchors' two products each; the head
    assert count["adaln_residual_mx"] == 3 * layers * steps and count["rms_norm_mx"] == 2
    assert sum(name == "mx_quantize" and len(args) == 3 for name, args, *_ in calls) == layers * steps
    assert count["mx_linear"] == (6 * layers + 1) * steps + (steps - 1) + 4 + 1
    if steps == 1:
        plain = make(False)
        _as_stored(plain, ("context_kv_weight", "noise_embed", "head_weight"))
        ref_caches, ref_hidden, ref_logits = run(plain)
        for i, (c, r) in enumerate(zip(caches, ref_caches)):
            _close(c.view(*c.shape[:-1], 2, -1), r.view(*r.shape[:-1], 2, -1), f"cache {i}")
        _close(hidden, ref_hidden, "hidden")
        _close(logits, ref_logits, "logits")


def test_vllm_step_captured(dev):
    """A captured step with microscaled projections, replayed with eager steps in between."""
    step, run, _ = _vllm("gelu_full_vocab", dev, 1)
    want = run()[2]
    graph = torch.cuda.CUDAGraph()
    caches, layout, bt, _, _, a_slots = _paged_context(
        step, torch.randn(5, step.mx_fc.cols, generator=gen(1)).bfloat16(), torch.tensor([5]), dev, gen(2))
    args = (torch.tensor([7], device=dev), torch.tensor([5], device=dev), a_slots.to(dev),
            torch.randn(step.block, step.noise_columns, generator=gen(3)).to(dev), caches, bt.to(dev), layout)
    eager = step.logits(step(*args))
    with torch.cuda.graph(graph):
        out = step.logits(step(*args))
    for _ in range(3):
        out.zero_()
        graph.replay()
        again = run()[2]
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(again, want)


@pytest.mark.parametrize("n_cand", [1, 3])
def test_sglang_step(dev, calls, n_cand):
    model = _model(dict(CASES["gelu_full_vocab"]), dev, 17)
    cfg = model.config
    g = gen(21)
    embed = torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g).bfloat16().to(dev)
    lm_head = (torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g) / 8).bfloat16().to(dev)
    step = SGLangDraftStep(model, embed, lm_head, max_positions=400, mx=True)
    lens = torch.tensor([45, 0, 77])
    requests, pool = len(lens), int(lens.sum()) + len(lens) + 4
    perm = torch.randperm(pool, generator=g)
    table = torch.zeros(requests, int(lens.max()) + 1, dtype=torch.int32)
    o = 0
    for r, n in enumerate(lens.tolist()):
        table[r, :n + 1] = perm[o:o + n + 1].int()
        o += n + 1
    pos = torch.cat([torch.arange(n) for n in lens.tolist()])
    req = torch.cat([torch.full((n,), r) for r, n in enumerate(lens.tolist())])
    feats = torch.randn(len(pos), len(cfg.target_layer_ids) * cfg.target_hidden_size, generator=g).bfloat16().to(dev)
    anchors = torch.randint(0, cfg.vocab_size, (requests,), generator=g).to(dev)
    a_locs = table[torch.arange(requests), lens].long().to(dev)
    z = torch.randn(requests * n_cand * step.block, cfg.target_hidden_size, generator=g).to(dev)

    def run(step=step):
        k_bufs = [torch.zeros(pool, step.heads, step.head_dim, dtype=torch.bfloat16, device=dev) for _ in model.layers]
        v_bufs = [torch.zeros_like(b) for b in k_bufs]
        meta = step.pool_meta(k_bufs, v_bufs)
        step.write_context(feats, pos.to(dev), table[req, pos].long().to(dev), meta)
        hidden = step(anchors, lens.to(dev), a_locs, z, k_bufs, v_bufs, table.to(dev), n_cand=n_cand, meta=meta)
        return v_bufs, hidden, step.logits(hidden)

    calls.clear()
    v_bufs, hidden, logits = run()
    assert _check(calls)["mx_linear"] == 6 * len(model.layers) + 1 + 4 + 1
    greedy = torch.ones(hidden.shape[0], dtype=torch.bool, device=dev)
    tokens = step.sample(hidden, torch.ones(hidden.shape[0], device=dev), greedy, torch.tensor(5, device=dev))
    assert torch.equal(tokens, logits.float().argmax(-1))
    made = [name for name, *_ in calls]
    layers = len(model.layers)
    assert made.count("adaln_residual_mx") == 3 * layers and made.count("rms_norm_mx") == 2
    plain = SGLangDraftStep(model, embed, lm_head, max_positions=400)
    _as_stored(plain, ("ctx_kv_weight", "noise_embed", "head_weight"))
    ref_v, ref_hidden, ref_logits = run(plain)
    for i, (c, r) in enumerate(zip(v_bufs, ref_v)):
        _close(c, r, f"values {i}")
    _close(hidden, ref_hidden, "hidden")
    _close(logits, ref_logits, "logits")
