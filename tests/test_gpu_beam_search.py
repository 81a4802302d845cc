"""A beam search over the paged cache: selection, forked tables, split blocks, written tokens and
attention together, with ends, a compaction in the middle, eager and as a replayed graph."""

import math

import pytest
import torch

from kvserve_amd import paged

from _paged_ref import attention
from _shared_ref import consistent, score_bound, select

pytestmark = pytest.mark.gpu

REQUESTS, BEAMS, VOCAB, H, G, D, S, LAYERS = 3, 4, 300, 2, 2, 64, 4, 2
ROWS = REQUESTS * BEAMS


class Model:
    """Keys and values that are known from a token and its place alone."""

    def __init__(self, dev, blocks):
        gen = torch.Generator(device=dev).manual_seed(0)
        rand = lambda *s: torch.randn(s, generator=gen, device=dev).to(torch.bfloat16)
        self.kv, self.place = rand(LAYERS, 2, VOCAB, H, D), rand(64, H, D)
        self.query, self.out = rand(VOCAB, H * G, D), rand(H * G * D, VOCAB) * 0.3
        self.caches = [torch.zeros((2, blocks, S, H, D), dtype=torch.bfloat16, device=dev) for _ in range(LAYERS)]
        self.layers = paged.LayerCaches(self.caches)

    def rows(self, layer, part, tokens, places):
        return self.kv[layer, part][tokens] + self.place[places]


def run(model, tables, tokens, places, order, slots, starts, err=None):
    """One step for tokens of live rows (`order`: the live rows first); returns logits [ROWS, VOCAB] and
    each layer's (query, attention)."""
    tok = tokens.long().clamp(min=0)[order]
    pos = places.long().clamp(min=0, max=63)[order]
    x, seen = 0.0, []
    for layer, cache in enumerate(model.caches):
        paged.write_kv(model.rows(layer, 0, tok, pos), model.rows(layer, 1, tok, pos), cache, slots, check=False, err=err)
        query = model.query[tok]
        out = torch.zeros_like(query)
        paged.tree_attention(query, cache, tables.tables, tables.lengths, starts, max_query=1, out=out, check=False, err=err)
        seen.append((query, out))
        x = x + out.flatten(1).float()
    logits = torch.zeros((ROWS, VOCAB), device=tok.device)
    logits[order] = (x @ model.out.float())
    return logits, seen


def test_a_search_keeps_every_hypothesis(cuda):
    model, end = Model(cuda, 200), 7
    tables = paged.SharedBlockTables(200, S, ROWS, 16, cuda, free_blocks=range(3, 200))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    # prompts of 9, 12 and 1 tokens in each request's first row, then in all its beams
    prompts = [[(17 * i + 5 * r) % VOCAB for i in range(n)] for r, n in enumerate((9, 12, 1))]
    first = [0] * ROWS
    for r, p in enumerate(prompts):
        first[r * BEAMS] = len(p)
    slots, _ = tables.update(i32(first), sum(first))
    tok = torch.tensor(sum(prompts, []), device=cuda)
    pos = torch.tensor([i for p in prompts for i in range(len(p))], device=cuda)
    for layer, cache in enumerate(model.caches):
        paged.write_kv(model.rows(layer, 0, tok, pos), model.rows(layer, 1, tok, pos), cache, slots)
    history = {r * BEAMS: list(p) for r, p in enumerate(prompts)}
    gen = torch.Generator(device=cuda).manual_seed(1)
    logits = torch.randn((ROWS, VOCAB), generator=gen, device=cuda) * 2
    scores = torch.full((ROWS,), -math.inf, device=cuda)
    scores[::BEAMS] = 0.0  # one hypothesis a request to begin with
    ended = 0
    for step in range(14):
        if step == 9:
            scores[BEAMS:2 * BEAMS] = -math.inf  # the second request is done: its rows give their blocks back
        best = paged.select_beams(logits, scores, BEAMS, 2 * BEAMS, end_token=end)
        want = select(logits, scores, BEAMS, 2 * BEAMS, end)
        assert all(torch.equal(best[k].cpu(), want[k]) for k in (0, 1, 3, 4))
        fine = torch.isfinite(want[2])
        assert bool(((best.scores.cpu().double() - want[2]).abs() <= score_bound(want[2]))[fine].all())
        ended += int((best.all_tokens == end).sum())
        slots, starts = tables.fork(best.parents, 1, ROWS)
        paged.copy_blocks(model.layers, tables.copies)
        if step == 6:
            paged.copy_blocks(model.layers, tables.compact())
            assert int(tables.tables.max()) < 3 + 197 - int(tables.state[1])
            # (the slots were given out under the old names)
            live = torch.nonzero(best.parents >= 0).flatten()
            last = tables.lengths[live].long() - 1
            slots[:live.numel()] = tables.tables[live, last // S].long() * S + last % S
        scores = best.scores
        history = {i: history[p] + [t] for i, (p, t) in enumerate(zip(best.parents.tolist(), best.tokens.tolist()))
                   if p >= 0}
        order = torch.argsort((best.parents < 0).int(), stable=True)
        logits, seen = run(model, tables, best.tokens, tables.lengths - 1, order, slots, starts)
        # every row's table leads to its own tokens
        lengths, rows = tables.lengths.tolist(), tables.tables.tolist()
        assert {i: len(h) for i, h in history.items()} == {i: n for i, n in enumerate(lengths) if n}
        for i, h in history.items():
            t, p = torch.tensor(h, device=cuda), torch.arange(len(h), device=cuda)
            block = torch.tensor(rows[i], device=cuda)[p // S]
            for layer, cache in enumerate(model.caches):
                for part in (0, 1):
                    assert torch.equal(cache[part, block, p % S], model.rows(layer, part, t, p)), (step, i, layer)
        for cache, (query, out) in zip(model.caches, seen):
            ref, _, bound = attention(query, cache, tables.tables, tables.lengths, starts)
            n = int(starts[-1])
            assert bool(((out.double() - ref).abs() <= bound)[:n].all())
        consistent(rows, lengths, tables.shares.tolist(), tables.free.tolist(), tables.state.tolist(), S, (0, 1, 2))
    assert ended and len(history) == 2 * BEAMS
    tables.fork(torch.full((ROWS,), -1, dtype=torch.int32, device=cuda), 0, 0)
    assert tables.state.tolist()[1] == 197 and int(tables.shares.abs().sum()) == 0


def test_a_step_as_a_graph(cuda):
    """Selection, fork, copies, writes and attention in one graph, replayed with eager steps between, against the
    same steps eager."""
    def begin():
        model = Model(cuda, 120)
        tables = paged.SharedBlockTables(120, S, ROWS, 14, cuda)
        first = torch.zeros(ROWS, dtype=torch.int32, device=cuda)
        first[::BEAMS] = 6
        tables.update(first, 18)
        gen = torch.Generator(device=cuda).manual_seed(5)
        for cache in model.caches:
            cache.copy_(torch.randn(cache.shape, generator=gen, device=cuda))
        logits = torch.randn((ROWS, VOCAB), generator=gen, device=cuda)
        scores = torch.full((ROWS,), -math.inf, device=cuda)
        scores[::BEAMS] = 0.0
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=cuda)
        best = paged.BeamChoice(i32(ROWS), i32(ROWS), scores, i32(REQUESTS, 8), i32(REQUESTS, 8),
                                torch.zeros((REQUESTS, 8), device=cuda))
        return dict(model=model, tables=tables, logits=logits, best=best, err=i32(1),
                    slots=torch.zeros(ROWS, dtype=torch.int64, device=cuda), starts=i32(ROWS + 1))

    def step(s, check):
        paged.select_beams(s["logits"], s["best"].scores, BEAMS, 8, end_token=3, out=s["best"], err=s["err"], check=check)
        s["tables"].fork(s["best"].parents, 1, ROWS, slots=s["slots"], starts=s["starts"], err=s["err"], check=check)
        paged.copy_blocks(s["model"].layers, s["tables"].copies, err=s["err"], check=check)
        order = torch.argsort((s["best"].parents < 0).int(), stable=True)
        logits, _ = run(s["model"], s["tables"], s["best"].tokens, s["tables"].lengths - 1, order, s["slots"],
                        s["starts"], s["err"])
        s["logits"].copy_(logits)

    eager, captured = begin(), begin()
    for s in (eager, captured):
        step(s, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(captured, False)
    torch.cuda.current_stream().wait_stream(side)
    step(eager, False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured, None)
    for i in range(10):
        step(eager, False)
        if i % 4 == 3:
            step(captured, False)
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert int(eager["err"]) == 0 and int(captured["err"]) == 0
        for k in ("tables", "lengths", "shares", "free", "state", "copies"):
            assert torch.equal(getattr(eager["tables"], k), getattr(captured["tables"], k)), (i, k)
        for a, b in zip(eager["best"], captured["best"]):
            assert torch.equal(a, b), i
        for a, b in zip(eager["model"].caches, captured["model"].caches):
            assert torch.equal(a, b), i
