"""Which weight of a draft step with ``mx=True`` goes where: restricted draft vocabularies (a head of
their own between jumps), two jumps, SGLang's step with both activations, each against the bf16
step on the values that the 4-bit weights stand for."""

import pytest
import torch

from _inputs import gen
from flashmap_amd import ops
from flashmap_amd.draft_step import DraftStep
from flashmap_amd.sglang_step import SGLangDraftStep
from test_gpu_draft_step import CASES, _model, _paged_context
from test_gpu_mx_steps import _as_stored, _check, _stood_for, calls  # noqa: F401  (calls: a fixture)

pytestmark = pytest.mark.gpu


def _off(got, want, what):
    """The 8-bit operands' rounding is 2^-5.5 of a row's norm at most (uniform in a code's step: 2^-4 /
    sqrt 3 at the top of a binade, half that at its bottom); a jump has 15 such operands behind each
    other at most, each read once and independent: sqrt(15) 2^-5.5, and as many bf16 roundings of
    2^-9. A weight in another's place, a lost bias or gain gives errors of a row's own size."""
    g, w = got.double().cpu().flatten(0, -2), want.double().cpu().flatten(0, -2)
    rel = (g - w).norm(dim=-1) / w.norm(dim=-1).clamp_min(1e-30)
    print(f"  {what}: worst row {rel.max():.4f}, mean {rel.mean():.5f}", flush=True)
    assert rel.max() <= 15 ** 0.5 * (2.0 ** -5.5 + 2.0 ** -9), what


def _watch(step, monkeypatch, states=None):
    """The jumps' final rows and, between jumps, (the state before, the head's logits, the state after).
    ``states`` take the updated ones' place: the posterior of a second jump sharpens what the first
    one's roundings moved, so that only jumps from one state can be compared."""
    rows, updates = [], []
    dit, update = step._dit, ops.state_update

    def watched(*args):
        rows.append(dit(*args))
        return rows[-1]

    def updated(state, logits, *times):
        before = state.clone()
        out = update(state, logits, *times)
        updates.append((before, logits.clone(), state.clone()))
        if states is not None:
            state.copy_(states[len(updates) - 1])
        return out

    monkeypatch.setattr(step, "_dit", watched)
    monkeypatch.setattr(ops, "state_update", updated)
    return rows, updates


@pytest.mark.parametrize("steps", [1, 2])
@pytest.mark.parametrize("name", sorted(CASES))
def test_vllm_step(dev, calls, monkeypatch, name, steps):  # noqa: F811
    print(f"mx draft step {name}, {steps} jump(s)", flush=True)
    model = _model(dict(CASES[name]), dev, 11)
    cfg, g = model.config, gen(5)
    embed = torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g).bfloat16().to(dev)
    lm_head = (torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g) / 8).bfloat16().to(dev)
    hot = torch.arange(0, 2 * cfg.state_vocab_size, 2).to(dev) if cfg.state_vocab_size else None
    if name == "gelu_hot_ids":
        hot = torch.arange(3, cfg.vocab_size, 3).to(dev)

    def make(mx):
        return DraftStep(model, embed, lm_head, max_model_len=512, hot_ids=hot, num_steps=steps, mx=mx)

    step, plain = make(True), make(False)
    states_vocab = cfg.state_vocab_size or cfg.vocab_size
    assert step.head_weight.shape[0] == (cfg.vocab_size if hot is None else len(hot))
    if steps == 2:
        head = step.jump_head[0]
        assert head.bits == 4 and head.shape[0] == states_vocab
        assert (head is step.head_weight) == (name != "gelu_hot_ids")
    lens = torch.tensor([37, 100, 0, 64])
    states = torch.randn(int(lens.sum()), len(cfg.target_layer_ids) * cfg.target_hidden_size, generator=g).bfloat16()
    anchors = torch.randint(0, cfg.vocab_size, (len(lens),), generator=g).to(dev)
    z = torch.randn(len(lens) * cfg.block_size, step.noise_columns, generator=g).to(dev)

    def run(step, after=None):
        caches, layout, bt, _, _, a_slots = _paged_context(step, states, lens, dev, gen(6))
        with monkeypatch.context() as m:
            rows, updates = _watch(step, m, after)
            hidden = step(anchors, lens.to(dev), a_slots.to(dev), z, caches, bt.to(dev), layout)
        return caches, rows, updates, hidden, step.logits(hidden), step.greedy(hidden)

    calls.clear()
    caches, rows, updates, hidden, logits, tokens = run(step)
    _check(calls)
    assert len(rows) == steps and len(updates) == steps - 1 and torch.equal(rows[-1], hidden)
    best = logits.float().argmax(-1)
    assert torch.equal(tokens, best if hot is None else hot[best])

    _as_stored(plain, ("context_kv_weight", "noise_embed"))
    plain.head_weight = _stood_for(plain.head_weight)
    if steps == 2:
        model.x_embed.weight.data = _stood_for(model.x_embed.weight.data)
        plain.jump_head = _stood_for(plain.jump_head[0]) if name == "gelu_hot_ids" else plain.head_weight, plain.jump_head[1]
    want_caches, want_rows, want_updates, want_hidden, want_logits, _ = run(plain, [after for _, _, after in updates])
    for i, (c, r) in enumerate(zip(caches, want_caches)):
        _off(c.view(*c.shape[:-1], 2, -1), r.view(*r.shape[:-1], 2, -1), f"cache {i}")
    _off(rows[0], want_rows[0], "rows of the first jump")
    if steps == 2:
        (before, between, after), (want_before, want_between, _) = updates[0], want_updates[0]
        assert torch.equal(before, want_before) and torch.equal(before, z)
        assert between.shape == want_between.shape == (len(z), states_vocab)
        _off(between, want_between, "logits between the jumps")
        same = before.clone()
        ops.state_update(same, between, *(step.jumps[0][i] for i in (0, 2)))
        assert torch.equal(same, after)
    _off(hidden, want_hidden, "hidden")
    _off(logits, want_logits, "logits")


@pytest.mark.parametrize("n_cand", [1, 3])
@pytest.mark.parametrize("name", ["gelu_full_vocab", "swiglu_state_vocab"])
def test_sglang_step(dev, calls, name, n_cand):  # noqa: F811
    print(f"mx SGLang draft step {name}, {n_cand} candidate(s)", flush=True)
    model = _model(dict(CASES[name]), dev, 17)
    cfg, g = model.config, gen(21)
    embed = torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g).bfloat16().to(dev)
    lm_head = (torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g) / 8).bfloat16().to(dev)
    hot = torch.arange(1, 2 * cfg.state_vocab_size, 2).to(dev) if cfg.state_vocab_size else None
    step, plain = (SGLangDraftStep(model, embed, lm_head, max_positions=400, hot_ids=hot, mx=mx) for mx in (True, False))
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

    def run(step):
        k_bufs = [torch.zeros(pool, step.heads, step.head_dim, dtype=torch.bfloat16, device=dev) for _ in model.layers]
        v_bufs = [torch.zeros_like(b) for b in k_bufs]
        meta = step.pool_meta(k_bufs, v_bufs)
        step.write_context(feats, pos.to(dev), table[req, pos].long().to(dev), meta)
        hidden = step(anchors, lens.to(dev), a_locs, z, k_bufs, v_bufs, table.to(dev), n_cand=n_cand, meta=meta)
        return k_bufs, v_bufs, hidden, step.logits(hidden)

    calls.clear()
    k_bufs, v_bufs, hidden, logits = run(step)
    _check(calls)
    made = [kind for kind, args, *_ in calls if kind == "mx_quantize" and len(args) == 3]
    assert len(made) == len(model.layers) and logits.shape[1] == (cfg.vocab_size if hot is None else len(hot))
    greedy = torch.ones(hidden.shape[0], dtype=torch.bool, device=dev)
    tokens = step.sample(hidden, torch.ones(hidden.shape[0], device=dev), greedy, torch.tensor(5, device=dev))
    best = logits.float().argmax(-1)
    assert torch.equal(tokens, best if hot is None else hot[best])
    _as_stored(plain, ("ctx_kv_weight", "noise_embed", "head_weight"))
    want_k, want_v, want_hidden, want_logits = run(plain)
    for i in range(len(model.layers)):
        _off(k_bufs[i], want_k[i], f"keys {i}")
        _off(v_bufs[i], want_v[i], f"values {i}")
    _off(hidden, want_hidden, "hidden")
    _off(logits, want_logits, "logits")
