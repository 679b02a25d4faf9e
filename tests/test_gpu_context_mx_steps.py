"""The draft step over contexts in microscaled 4 bits, and its operators as a server runs them: in
captured graphs, on streams of their own, one after the other.

The step is held to the oracle's step over bf16 caches that hold the 4-bit caches' values (which bf16
holds exactly), with the bars of the step over bf16 caches: the attention differs from it by the rounding
of probabilities and queries to 8 bits, which bf16 attention has as well."""

import pytest
import torch

from _context_mx_checks import BF, cache_values, check, make
from _inputs import gen, paged_layout
from flashmap_amd import fold, ops
from flashmap_amd.draft_step import DraftStep, _rope_table
from oracle import draft_step as oracle
from test_gpu_draft_step import CASES, PAGE, _check_logits, _close_rows, _model, _oracle_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps", [1, 2])
@pytest.mark.parametrize("page", [1, 16])
def test_draft_step(dev, steps, page):
    """Context and anchors written, drafted over, sampled and judged."""
    name = "gelu_full_vocab"
    model = _model(CASES[name], dev, 11)
    cfg, g = model.config, gen(5)
    embed = torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g).bfloat16().to(dev)
    lm_head = (torch.randn(cfg.vocab_size, cfg.target_hidden_size, generator=g) / 8).bfloat16().to(dev)
    step = DraftStep(model, embed, lm_head, max_model_len=512, num_steps=steps)
    lens = torch.tensor([37, 100, 0, 64])
    batch, k = len(lens), cfg.block_size
    states = torch.randn(int(lens.sum()), len(cfg.target_layer_ids) * cfg.target_hidden_size, generator=g).bfloat16()
    bt, total = paged_layout((lens + 1).tolist(), page, g)
    caches = [ops.mx_cache(total, step.heads, page, step.head_dim, dev) for _ in model.layers]
    pos = torch.cat([torch.arange(int(n)) for n in lens])
    req = torch.cat([torch.full((int(n),), b) for b, n in enumerate(lens)])
    slots = bt[req, pos // page].long() * page + pos % page
    step.write_context(states.to(dev), pos.to(dev), slots.to(dev), step.cache_layout(caches))
    a_slots = bt[torch.arange(batch), lens // page].long() * page + lens % page
    anchors = torch.randint(0, cfg.vocab_size, (batch,), generator=g)
    z = torch.randn(batch * k, step.noise_columns, generator=g)
    hidden = step(anchors.to(dev), lens.to(dev), a_slots.to(dev), z.to(dev), caches, bt.to(dev))
    logits = step.logits(hidden)
    tokens = step.greedy(hidden)
    said = ops.log_probs_rows(logits, tokens, 3)
    torch.cuda.synchronize()

    # A block's scale 2^e puts its largest magnitude to [4, 8): the widest step, 4 to 6, is off by 1 of at
    # least 4, and what passes 6 by less than 2 of 8: 1/4 of the largest; and the bf16 rows' own bar, 2 ulps
    # and an ulp of the row.
    w = _oracle_weights(model, embed, lm_head, None, steps, 512 + k + 1)
    held = [cache_values(c).to(BF) for c in caches]
    plain = [torch.zeros(total, step.heads, page, 2 * step.head_dim, dtype=BF) for _ in caches]
    oracle.write_context(w, states, pos, slots, plain, page)
    oracle.write_anchors(w, anchors, lens, a_slots, plain, page)
    for got, want in zip(held, plain):
        got, want = (t.double().reshape(-1, step.head_dim // 32, 32) for t in (got, want))
        top = want.abs().amax(-1, keepdim=True)
        rms = want.pow(2).mean((1, 2), keepdim=True).sqrt()  # of a head's keys, or values
        assert ((got - want).abs() <= 0.25 * top + 2.0 ** -6 * top + 2.0 ** -7 * rms).all()
    if steps == 1:
        noise = (z.to(dev).double() @ fold.noise_factor(embed)[0]).bfloat16().cpu()
        want_h, want = oracle.draft(w, lens, held, bt, noise_embeds=noise)
    else:
        want_h, want = oracle.draft(w, lens, held, bt, state=z)
    _close_rows(hidden, want_h, "hidden", ulps=4, rel=2e-2 * steps, row_rel=1e-2 * steps)
    _check_logits(logits, want, None, f"{name} x{steps}")

    # A greedy token is the likeliest one, ties aside.
    exact = torch.log_softmax(logits.double(), -1)
    lp = exact.gather(1, tokens.reshape(-1, 1))[:, 0]
    tol = 2.0 ** -20 * (1 + exact.abs().amax(-1))
    assert ((said.token.double() - lp).abs() <= tol).all()
    assert ((said.top[:, 0].double() - exact.amax(-1)).abs() <= tol).all() and (said.rank >= 1).all()


def test_step_refuses_mixed_caches(dev):
    cache = ops.mx_cache(2, 2, 16, 128, dev)
    with pytest.raises(TypeError, match="all be microscaled"):
        DraftStep.cache_layout([cache, torch.zeros(2, 2, 16, 256, dtype=BF, device=dev)])


def _work(dev, seed, lens, hq, hkv, d, page):
    """A server's step over fixed buffers: append, attend, judge; and a way to set new inputs."""
    g = torch.Generator().manual_seed(seed)
    cache, table, _ = make(lens, hkv, d, page, seed, dev)
    cache = ops.MX(cache.codes, cache.scales, 4, (1, *cache.shape))
    batch, vocab = len(lens), 3000
    rope = ops.rope_from_table(_rope_table(600, d, 1e4, torch.device(dev)))
    weight = (0.5 + torch.rand(1, d, generator=g)).to(dev)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
    last = torch.tensor(lens) - 1
    positions = last.to(dev)
    slots = (table.cpu()[torch.arange(batch), last // page].long() * page + last % page).to(dev)
    kv = torch.empty(batch, 1, 2, hkv, d, dtype=BF, device=dev)
    query = torch.empty(batch * 4, hq, d, dtype=BF, device=dev)
    logits = torch.empty(batch, vocab, dtype=BF, device=dev)
    tokens = torch.arange(batch, device=dev)

    def fill(i):
        h = torch.Generator().manual_seed(1000 * seed + i)
        for t in (kv, query, logits):
            t.copy_(torch.randn(t.shape, generator=h).to(BF))

    def run():
        ops.write_context_kv_mx(kv, positions, slots, weight, rope, cache, 1e-6)
        out = ops.block_attention_paged_mx(query, cache[0], None, lens_t, table, 4, max(lens), d ** -0.5)
        said = ops.log_probs_rows(logits, tokens, 5)
        return [out, said.token, said.rank, said.entropy, said.top_ids, said.top]

    return fill, run


SHAPES = [dict(lens=[70, 5, 513], hq=4, hkv=2, d=128, page=16), dict(lens=[1, 300], hq=16, hkv=1, d=64, page=1)]


def test_graphs_and_streams(dev):
    """Two captured graphs side by side, replayed with new inputs and eager work between, and both
    shapes at once on two streams: always what a call alone gives."""
    works = [_work(dev, i + 1, **s) for i, s in enumerate(SHAPES)]
    for fill, run in works:
        fill(0)
        run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for fill, run in works:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    for i in range(4):
        want = []
        for fill, run in works:
            fill(i)
            want.append([t.clone() for t in run()])
        for out in outs:
            for t in out:
                t.zero_()
        for graph in (graphs if i % 2 else graphs[::-1]):
            graph.replay()
        torch.cuda.synchronize()
        for got, one in zip(outs, want):
            for a, b in zip(got, one):
                assert torch.equal(a, b)
    streams = [torch.cuda.Stream() for _ in works]
    torch.cuda.synchronize()
    for i in range(3):
        got = []
        for (fill, run), s in zip(works, streams):
            with torch.cuda.stream(s):
                got.append([run() for _ in range(4)])
        torch.cuda.synchronize()
        for several, (fill, run) in zip(got, works):
            for a in several:
                for x, y in zip(a, run()):
                    assert torch.equal(x, y)


def test_same_inputs_twice(dev):
    """One call's result does not depend on what ran before it: equal bits, call after call."""
    lens = [2000, 17, 0, 640]
    cache, table, _ = make(lens, 4, 128, 16, 3, dev)
    query = torch.randn(64, 16, 128, generator=gen(4)).to(BF).to(dev)
    lens_t = torch.tensor(lens, device=dev)
    outs = [ops.block_attention_paged_mx(query, cache, None, lens_t, table, 16, 2000, 0.1) for _ in range(5)]
    x = torch.randn(7, 50_000, generator=gen(5)).to(dev)
    said = [ops.log_probs_rows(x, torch.arange(7, device=dev), 32) for _ in range(5)]
    for o, s in zip(outs[1:], said[1:]):
        assert torch.equal(o, outs[0])
        assert all(torch.equal(a, b) for a, b in zip(vars(s).values(), vars(said[0]).values()))


@pytest.mark.parametrize("rows_per_head", [17, 33, 49, 65, 100, 128, 200])
def test_row_groups(dev, rows_per_head):
    """Every count of row blocks and row groups, the last block not full."""
    lens, d = [40, 333], 128
    cache, table, rows = make(lens, 1, d, 8, 7, dev)
    query = torch.randn(2 * rows_per_head, 1, d, generator=gen(8)).to(BF).to(dev)
    n = rows_per_head
    out = ops.block_attention_paged_mx(query, cache, None, torch.tensor(lens, device=dev), table, n, 333, 0.1)
    check(out, query, rows, [n] * 2, 0.1)


def test_padded_batch(dev):
    """A captured batch's padding: requests of no context and tokens of no slot leave no trace."""
    lens, d, heads = [50, 0, 129, 0], 128, 2
    cache, table, rows = make(lens, heads, d, 16, 9, dev)
    cu = torch.tensor([0, 16, 16, 32, 32], dtype=torch.int32, device=dev)
    query = torch.randn(48, 8, d, generator=gen(10)).to(BF).to(dev)
    out = torch.full_like(query, 7.0)
    got = ops.block_attention_paged_mx(query, cache, cu, torch.tensor(lens, device=dev), table, 16, 129, 0.1, out=out)
    check(got[:32], query[:32], [rows[0], rows[2]], [16, 16], 0.1)
    assert (out[32:] == 7.0).all()
    before = cache.codes.clone(), cache.scales.clone()
    joined = ops.MX(cache.codes, cache.scales, 4, (1, *cache.shape))
    kv = torch.randn(3, 1, 2, heads, d, generator=gen(11)).to(BF).to(dev)
    none = torch.full((3,), -1, device=dev)
    ops.write_context_kv_mx(kv, torch.zeros(3, dtype=torch.int64, device=dev), none, torch.ones(1, d, device=dev),
                            ops.rope_from_table(_rope_table(8, d, 1e4, torch.device(dev))), joined, 1e-6)
    assert torch.equal(cache.codes, before[0]) and torch.equal(cache.scales, before[1])
