"""Draft steps over 4-bit contexts as a server runs them: captured once and replayed over growing contexts, with a
padded request, the caches one a layer or one of all layers, with bf16 and with 4-bit weights."""

import pytest
import torch

from _context_mx_checks import BF
from _inputs import gen, paged_layout
from flashmap_amd import ops
from flashmap_amd.draft_step import DraftStep
from test_gpu_draft_step import CASES, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps,mx", [(1, False), (1, True), (2, False)])
def test_captured(dev, steps, mx):
    model = _model(CASES["gelu_full_vocab"], dev, 31)
    cfg, g = model.config, gen(32)
    embed = torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g).bfloat16().to(dev)
    lm_head = (torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g) / 8).bfloat16().to(dev)
    step = DraftStep(model, embed, lm_head, max_model_len=512, num_steps=steps, mx=mx)
    lens, page, grown = torch.tensor([37, 130, 5]), 16, 3
    batch, k = len(lens), cfg.block_size
    bt, total = paged_layout((lens + 1 + grown).tolist(), page, g)
    states = torch.randn(int(lens.sum()), len(cfg.target_layer_ids) * cfg.target_hidden_size, generator=g).bfloat16()
    pos = torch.cat([torch.arange(int(n)) for n in lens])
    req = torch.cat([torch.full((int(n),), b) for b, n in enumerate(lens)])
    slots = bt[req, pos // page].long() * page + pos % page

    def caches(joined):
        if joined:
            return ops.mx_cache(total, step.heads, page, step.head_dim, dev, len(model.layers))
        return [ops.mx_cache(total, step.heads, page, step.head_dim, dev) for _ in model.layers]

    held = [caches(False), caches(True), caches(False)]
    for c in held:
        step.write_context(states.to(dev), pos.to(dev), slots.to(dev), step.cache_layout(c))
    args = [torch.zeros(batch, dtype=torch.int64, device=dev) for _ in range(3)]  # anchors, positions, slots
    z = torch.zeros(batch * k, step.noise_columns, device=dev)

    def fill(i):
        at = lens + i
        a_slots = bt[torch.arange(batch), at // page].long() * page + at % page
        if i == 1:  # the last request is padding: nothing of it is kept
            a_slots[2] = -1
        h = gen(40 + i)
        for t, v in zip((*args, z), (torch.randint(0, cfg.vocab_size, (batch,), generator=h), at, a_slots,
                                     torch.randn(z.shape, generator=h))):
            t.copy_(v)

    def run(c):
        hidden = step(*args, z, c, bt.to(dev), step.cache_layout(c))
        logits = step.logits(hidden)
        said = ops.log_probs_rows(logits, logits.argmax(-1), 2)
        return [hidden, logits, said.token, said.rank, said.top_ids]

    table = bt.to(dev)
    fill(0)
    run(held[2])  # loads what is loaded at first use
    torch.cuda.synchronize()
    layout = step.cache_layout(held[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hidden = step(*args, z, held[0], table, layout)
        logits = step.logits(hidden)
        said = ops.log_probs_rows(logits, step.greedy(hidden), 2)
    for i in range(grown):
        fill(i)
        want = run(held[1])
        for t in (hidden, logits, said.token):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, one in zip((hidden, logits, said.token, said.rank, said.top_ids), want):
            assert torch.isfinite(one.float()).all() and torch.equal(got, one)
        for layer, part in zip(held[0], held[1]):
            assert torch.equal(layer.codes, part.codes) and torch.equal(layer.scales, part.scales)
    assert hidden.dtype is BF
