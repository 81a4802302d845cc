"""What the operators of sequences that share blocks are measured on: beam search's selection over
beams and vocabulary, block tables forked, reordered and freed with counted blocks, blocks copied
in every layer, and the pool compacted.

A case is one call that a serving program makes; `draw` gives more of the same ranges.

  select_one      one request's beams: nothing but latency
  select_batch    64 requests' beams over a large vocabulary, with an end token
  select_fp32     logits in 32 bits, most of the vocabulary banned, requests that are done
  select_odd      an odd vocabulary in padded rows, fp16, 5 beams
  fork_one        one request's beams reordered and grown by a token
  fork_step       a step of 64 requests' beams: reordered, grown by a token, what nobody holds freed
  fork_mixed      requests of all sorts in one update: forks, joins, ends, prefixes taken over
  copy_step       the partly filled blocks that a step's forks split, every layer
  copy_blocks     whole blocks, as a compaction moves them, every layer
  copy_odd        12 tokens a block, 5 KV heads of 80 channels, K and V adjacent
  compact_small   a small pool
  compact_pool    a pool of 65536 blocks, shared prefixes, a third free
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the least there is to select from
        dict(name="select_one", kind="select", requests=1, beams=4, vocab=32000, count=8, dtype="bf16", pad=0, end=True,
             banned=0.0, lowest=False, done=0.0),
        # 64 requests of 8 beams; with the whole blocks the largest case
        dict(name="select_batch", kind="select", requests=64, beams=8, vocab=131072, count=16, dtype="bf16", pad=0,
             end=True, banned=0.0, lowest=False, done=0.0),
        # constrained decoding: banned tokens hold the type's lowest value
        dict(name="select_fp32", kind="select", requests=16, beams=4, vocab=152064, count=4, dtype="fp32", pad=0,
             end=False, banned=0.9, lowest=True, done=0.2),
        # nothing aligned
        dict(name="select_odd", kind="select", requests=13, beams=5, vocab=50021, count=11, dtype="fp16", pad=3, end=True,
             banned=0.1, lowest=False, done=0.0),
        # one request of 512 tokens and 4 beams
        dict(name="fork_one", kind="fork", requests=1, beams=4, block=16, columns=64, lo=512, hi=512, grow=1,
             mixed=False, lens_seed=1),
        # 64 ragged requests of 4 beams
        dict(name="fork_step", kind="fork", requests=64, beams=4, block=16, columns=768, lo=1024, hi=12000, grow=1,
             mixed=False, lens_seed=2),
        # 256 groups of 4 rows, everything at once
        dict(name="fork_mixed", kind="fork", requests=256, beams=4, block=16, columns=512, lo=1, hi=8000, grow=33,
             mixed=True, lens_seed=3),
        # 28 layers of 4 KV heads: a step's split blocks
        dict(name="copy_step", kind="copy", layers=28, kv_heads=4, head_dim=128, block=16, rows=64, pairs=24, part=True,
             dtype="bf16", layout="flash", lens_seed=4),
        # 32 layers of 8 KV heads: a compaction's moves
        dict(name="copy_blocks", kind="copy", layers=32, kv_heads=8, head_dim=128, block=16, rows=200, pairs=200,
             part=False, dtype="bf16", layout="flash", lens_seed=5),
        dict(name="copy_odd", kind="copy", layers=3, kv_heads=5, head_dim=80, block=12, rows=77, pairs=50, part=True,
             dtype="fp16", layout="kv_adjacent", lens_seed=6),
        dict(name="compact_small", kind="compact", blocks=1024, requests=8, beams=2, block=16, columns=128, held=0.5,
             lens_seed=7),
        dict(name="compact_pool", kind="compact", blocks=65536, requests=128, beams=4, block=16, columns=768, held=0.66,
             lens_seed=8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["select", "select", "fork", "fork", "copy", "compact"])
    lens_seed = rng.randrange(1 << 30)
    if kind == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = _log_int(rng, 1000, 152064)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 64 * 8 * 131072 * 2 // (4 if dtype == "fp32" else 2) // (beams * vocab)
        end = rng.random() < 0.7
        return dict(kind="select", requests=_log_int(rng, 1, max(1, min(64, most))), beams=beams, vocab=vocab,
                    count=2 * beams + rng.choice([0, 0, 1]) if end else beams + rng.choice([0, 0, 3]), dtype=dtype,
                    pad=rng.choice([0, 0, 1, 8]), end=end, banned=rng.choice([0.0, 0.0, 0.1, 0.9]),
                    lowest=rng.random() < 0.5, done=rng.choice([0.0, 0.0, 0.3]))
    if kind == "fork":
        block, columns = rng.choice([1, 12, 16, 16, 32, 64, 128]), _log_int(rng, 16, 768)
        return dict(kind="fork", requests=_log_int(rng, 1, 256), beams=rng.choice([1, 2, 3, 4]), block=block,
                    columns=columns, lo=1, hi=max(1, min(block * columns - 40, 8000)), grow=rng.choice([0, 1, 1, 8]),
                    mixed=rng.random() < 0.5, lens_seed=lens_seed)
    if kind == "copy":
        pairs = rng.randint(1, 100)
        return dict(kind="copy", layers=rng.choice([1, 16, 28, 32]), kv_heads=rng.choice([1, 2, 4, 5, 8]),
                    head_dim=rng.choice([64, 80, 96, 128]), block=rng.choice([1, 12, 16, 16, 32]), pairs=pairs,
                    rows=pairs + rng.choice([0, 7, 100]), part=rng.random() < 0.6, dtype=rng.choice(["bf16", "fp16"]),
                    layout=rng.choice(["flash", "kv_adjacent"]), lens_seed=lens_seed)
    blocks = _log_int(rng, 16, 65536)
    return dict(kind="compact", blocks=blocks, requests=_log_int(rng, 1, 128), beams=rng.choice([1, 2, 4]),
                block=rng.choice([1, 12, 16, 128]), columns=_log_int(rng, 8, 768), held=rng.choice([0.1, 0.5, 0.66, 0.9]),
                lens_seed=lens_seed)


# ------------------------------------------------------------------ shapes (from the case alone)
def _blocks(tokens, block):
    return (tokens + block - 1) // block


def _groups(case, r, budget=None):
    """Rows of requests whose beams share blocks: [(tokens, blocks shared with the whole group, blocks
    shared with the group's first half)], beams rows a request.  `budget`: the most blocks in all."""
    S, B, rows = case["block"], case["beams"], []
    lo, hi = case.get("lo", 1), case.get("hi", case["block"] * case["columns"])
    for _ in range(case["requests"]):
        n = r.randint(lo, hi)
        if budget is not None:
            n = min(n, max(budget - B, 0) * S // 2)
        whole = _blocks(n, S)
        shared = r.randint(whole * 3 // 4, n // S) if n // S >= whole * 3 // 4 else n // S
        half = r.randint(shared, n // S)
        for b in range(B):
            rows.append((n, shared, half if b < B // 2 else shared))
        if budget is not None:
            budget -= 2 * whole + B
    return rows


def _rows_of(case, rows):
    """Block numbers 0 .. n - 1 in the order in which rows first hold them: (list a row, holders a block)."""
    S, B, tables, holders = case["block"], case["beams"], [], []
    for i, (n, shared, half) in enumerate(rows):
        b, have = i % B, _blocks(n, S)
        first = tables[i - b] if b else None
        row = []
        for k in range(have):
            if b and (k < shared or (k < half and b < B // 2)):
                row.append(first[k])
                holders[first[k]] += 1
            else:
                row.append(len(holders))
                holders.append(1)
        tables.append(row)
    return tables, holders


def _fork_plan(case):
    """(rows, parents, new lengths, blocks taken at most)."""
    r, B, S = random.Random(case["lens_seed"]), case["beams"], case["block"]
    rows = _groups(case, r)
    top, parents, new = S * case["columns"], [], []
    for i, (n, _, _) in enumerate(rows):
        first, u = i - i % B, r.random()
        parent = first + r.randrange(B)
        if not case["mixed"]:
            if u < 0.02:  # a beam that has ended
                parent, length = -1, 0
            else:
                length = rows[parent][0] + case["grow"]
        elif u < 0.1:
            parent, length = -1, 0
        elif u < 0.2:
            parent, length = -1, r.randint(1, case["hi"])
        elif u < 0.3:  # a new request over a running one's prefix
            parent = r.randrange(len(rows))
            length = r.randint(0, rows[parent][0])
        elif u < 0.5:
            parent, length = i, max(0, n - r.randint(0, case["grow"]))
        else:
            length = rows[parent][0] + r.randint(0, case["grow"])
        parents.append(parent)
        new.append(min(length, top))
    return rows, parents, new


def _copy_plan(case):
    """[tokens of a pair, or -1 for a row that copies nothing]."""
    r = random.Random(case["lens_seed"])
    used = set(r.sample(range(case["rows"]), case["pairs"])) if case["part"] else set(range(case["pairs"]))
    S = case["block"]
    return [(r.randint(1, max(1, S - 1)) if case["part"] else S) if i in used else -1 for i in range(case["rows"])]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    return {"select": _prepare_select, "fork": _prepare_fork, "copy": _prepare_copy,
            "compact": _prepare_compact}[case["kind"]](case, gen, seed, dev)


def _int32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _prepare_select(case, gen, seed, dev):
    R, B, V, n = case["requests"], case["beams"], case["vocab"], case["count"]
    dtype = DTYPES[case["dtype"]]
    rows = torch.empty((R * B, V + case["pad"]), dtype=dtype, device=dev)
    rows.normal_(0.0, 2.5, generator=gen)
    # a few tokens that stand out, as a model's answers have them
    strong = torch.randint(0, V, (R * B, 6), generator=gen, device=dev)
    rows.scatter_(1, strong, (torch.randn((R * B, 6), generator=gen, device=dev) * 2 + 9).to(dtype))
    logits = rows[:, :V]
    if case["banned"]:
        out = torch.rand(V, generator=gen, device=dev) < case["banned"]
        out[torch.randint(0, V, (1 + V // 100,), generator=gen, device=dev)] = False
        logits.masked_fill_(out, torch.finfo(dtype).min if case["lowest"] else -math.inf)
    scores = -30.0 * torch.rand((R, B), generator=gen, device=dev)
    scores.masked_fill_(torch.rand((R, 1), generator=gen, device=dev) < case["done"], -math.inf)
    i32, f32 = dict(dtype=torch.int32, device=dev), dict(dtype=torch.float32, device=dev)
    return dict(kind="select", logits=logits, scores=scores.flatten(), beams=B, count=n,
                end=seed % V if case["end"] else None,
                out=(torch.empty(R * B, **i32), torch.empty(R * B, **i32), torch.empty(R * B, **f32),
                     torch.empty((R, n), **i32), torch.empty((R, n), **i32), torch.empty((R, n), **f32)),
                err=torch.zeros(1, **i32))


def _place(rows, columns, ids):
    """Tables int32 [rows, columns] of the rows' block numbers under other names, -1 behind them."""
    flat = torch.tensor([k for row in rows for k in row], dtype=torch.long, device=ids.device)
    counts = torch.tensor([len(row) for row in rows], device=ids.device).unsqueeze(1)
    at = torch.cumsum(counts, 0) - counts
    col = torch.arange(columns, device=ids.device).unsqueeze(0)
    if not flat.numel():
        return torch.full((len(rows), columns), -1, dtype=torch.int32, device=ids.device)
    got = ids[flat[(at + col).clamp(max=flat.numel() - 1)]].to(torch.int32)
    return torch.where(col < counts, got, torch.full_like(got, -1))


def _prepare_fork(case, gen, seed, dev):
    plan, parents, new = _fork_plan(case)
    rows, holders = _rows_of(case, plan)
    S, C, R = case["block"], case["columns"], len(rows)
    spare = sum(_blocks(n, S) for n in new) - sum(min(len(rows[p]), n // S) for p, n in zip(parents, new) if p >= 0) + 9
    held, N = len(holders), len(holders) + spare
    ids = torch.randperm(N, generator=gen, device=dev)
    shares = torch.zeros(N, dtype=torch.int32, device=dev)
    shares[ids[:held]] = _int32(holders, dev) - 1
    head = random.Random(seed).randrange(N)
    ring = torch.full((N,), -1, dtype=torch.int32, device=dev)
    ring[(head + torch.arange(spare, device=dev)) % N] = ids[held:].to(torch.int32)
    grown = sum(max(0, n - (plan[p][0] if p >= 0 else 0)) for p, n in zip(parents, new)) + 5
    i32 = dict(dtype=torch.int32, device=dev)
    lengths, tables = _int32([n for n, _, _ in plan], dev), _place(rows, C, ids)
    state = dict(kind="fork", lengths=lengths, tables=tables, shares=shares, free=ring, state=_int32([head, spare], dev),
                 parents=_int32(parents, dev), new=_int32(new, dev) if case["mixed"] else case["grow"], block=S,
                 max_tokens=grown, err=torch.zeros(1, **i32),
                 out=(torch.empty_like(tables), torch.empty_like(lengths), torch.empty_like(shares),
                      torch.empty(2, **i32), torch.empty(grown, dtype=torch.int64, device=dev),
                      torch.empty(R + 1, **i32), torch.empty((R, 3), **i32)))
    if own:
        from kvserve_amd import paged
        state["workspace"] = paged.fork_workspace(N, R, C, dev)
    return state


def _prepare_copy(case, gen, seed, dev):
    S, H, D = case["block"], case["kv_heads"], case["head_dim"]
    tokens, blocks = _copy_plan(case), 2 * case["rows"] + 5
    shape = (2, blocks, S, H, D) if case["layout"] == "flash" else (blocks, 2, S, H, D)
    caches = []
    for _ in range(case["layers"]):
        cache = torch.empty(shape, device=dev, dtype=DTYPES[case["dtype"]])
        cache.normal_(generator=gen)
        caches.append(cache)
    ids = torch.randperm(blocks, generator=gen, device=dev).tolist()
    rows = [[ids[2 * i], ids[2 * i + 1], t] if t > 0 else [-1, -1, -1] for i, t in enumerate(tokens)]
    state = dict(kind="copy", caches=caches, copies=_int32(rows, dev), layout=case["layout"], block=S,
                 err=torch.zeros(1, dtype=torch.int32, device=dev))
    if own:
        from kvserve_amd import paged
        state["layers"] = paged.LayerCaches(caches)
    return state


def _prepare_compact(case, gen, seed, dev):
    r, N, C = random.Random(case["lens_seed"]), case["blocks"], case["columns"]
    plan = _groups(case, r, budget=int(N * case["held"]))
    rows, holders = _rows_of(case, plan)
    held = len(holders)
    ids = torch.randperm(N, generator=gen, device=dev)
    shares = torch.zeros(N, dtype=torch.int32, device=dev)
    shares[ids[:held]] = _int32(holders, dev) - 1
    away = min(3, N - held)  # blocks that are not the tables' to hand out
    head, count = random.Random(seed).randrange(N), N - held - away
    ring = torch.full((N,), -1, dtype=torch.int32, device=dev)
    ring[(head + torch.arange(count, device=dev)) % N] = ids[held:held + count].to(torch.int32)
    i32 = dict(dtype=torch.int32, device=dev)
    tables = _place(rows, C, ids)
    state = dict(kind="compact", lengths=_int32([n for n, _, _ in plan], dev), tables=tables, shares=shares, free=ring,
                 state=_int32([head, count], dev), block=case["block"], err=torch.zeros(1, **i32),
                 out=(torch.empty_like(tables), torch.empty_like(shares), torch.empty_like(ring), torch.empty(2, **i32),
                      torch.empty((N // 2, 3), **i32)))
    if own:
        from kvserve_amd import paged
        state["workspace"] = paged.compact_workspace(N, dev)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    return {"select": _plain_select, "fork": _plain_fork, "copy": _plain_copy,
            "compact": _plain_compact}[state["kind"]](state)


def _run_own(s):
    from kvserve_amd import paged

    if s["kind"] == "select":
        return tuple(paged.select_beams(s["logits"], s["scores"], s["beams"], s["count"], end_token=s["end"],
                                        out=s["out"], err=s["err"], check=False))
    if s["kind"] == "fork":
        got = paged.fork_block_tables(s["lengths"], s["parents"], s["new"], s["tables"], s["shares"], s["free"],
                                      s["state"], s["block"], s["max_tokens"], out=s["out"],
                                      workspace=s["workspace"], err=s["err"], check=False)
        return tuple(got) + (s["free"],)
    if s["kind"] == "copy":
        paged.copy_blocks(s["layers"], s["copies"], err=s["err"], check=False)
        return s["caches"]
    return tuple(paged.compact_block_tables(s["lengths"], s["tables"], s["shares"], s["free"], s["state"], s["block"],
                                            out=s["out"], workspace=s["workspace"], err=s["err"], check=False))


def _plain_select(s):
    B, n = s["beams"], s["count"]
    rows, V = s["logits"].shape
    R, dev = rows // B, s["logits"].device
    # the order of two beams' candidates hangs on the difference of two long sums: 64 bits
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    lse = (torch.exp(x - top).sum(1, keepdim=True).log() + top)
    # a row's best tokens, the lowest first among equals: keys in which both stand
    bits = (s["logits"].float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits)
    key = torch.topk((order << 32) | (0x7fffffff - torch.arange(V, device=dev)), min(n, V), 1).values
    token = 0x7fffffff - (key & 0xffffffff)
    score = s["scores"].double().unsqueeze(1)
    v = score + (x.gather(1, token) - lse)
    fine = torch.isfinite(lse) & torch.isfinite(score) & (v.float() > -math.inf)
    v = torch.where(fine, v, torch.full_like(v, -math.inf)).reshape(R, -1)
    v, at = torch.sort(v, dim=1, descending=True, stable=True)
    k = min(n, v.shape[1])
    v, at = v[:, :k], at[:, :k]
    there = v > -math.inf
    none = torch.full_like(at, -1)
    row = torch.arange(R, device=dev).unsqueeze(1) * B + at // min(n, V)
    all_parents = torch.nn.functional.pad(torch.where(there, row, none), (0, n - k), value=-1)
    all_tokens = torch.nn.functional.pad(torch.where(there, token.reshape(R, -1).gather(1, at), none), (0, n - k), value=-1)
    all_scores = torch.nn.functional.pad(v.float(), (0, n - k), value=-math.inf)
    go = all_parents >= 0
    if s["end"] is not None:
        go &= all_tokens != s["end"]
    rank = torch.cumsum(go, 1) - 1
    to = torch.where(go & (rank < B), rank, torch.full_like(rank, B))
    put = lambda v, none: torch.full((R, B + 1), none, dtype=v.dtype, device=dev).scatter_(1, to, v)[:, :B].flatten()
    return (put(all_parents, -1).int(), put(all_tokens, -1).int(), put(all_scores, -math.inf), all_parents.int(),
            all_tokens.int(), all_scores)


def _plain_fork(s):
    S, tables, ring = s["block"], s["tables"], s["free"]
    (R, C), N, dev = tables.shape, ring.numel(), tables.device
    length, parents = s["lengths"].long(), s["parents"].long()
    head, count = s["state"][0].long(), s["state"][1].long()
    me, col = torch.arange(R, device=dev), torch.arange(C, device=dev).unsqueeze(0)
    has, p = parents >= 0, parents.clamp(min=0)
    zero = torch.zeros_like(length)
    base = torch.where(has, length[p], zero)
    new = torch.where(has, base + s["new"], zero) if isinstance(s["new"], int) else s["new"].long()
    kept = torch.minimum(base, new)
    full, rest, want, have = kept // S, kept % S, (new + S - 1) // S, (length + S - 1) // S
    # one child takes a partly kept block over where nobody else holds it
    to = torch.where(has, p, torch.full_like(p, R))
    most = torch.zeros(R + 1, dtype=torch.long, device=dev).scatter_reduce_(0, to, kept, "amax")[p]
    block = tables[p, full.clamp(max=C - 1)].long().clamp(0, N - 1)
    alone = (rest > 0) & (full == most // S) & (s["shares"][block] == 0)
    to = torch.where(alone, p, torch.full_like(p, R))
    first = torch.full((R + 1,), R, dtype=torch.long, device=dev).scatter_reduce_(0, to, me, "amin")[p]
    keeps = alone & (first == me)
    copies_it = (rest > 0) & ~keeps
    stay = full + keeps
    take = want - stay
    before = torch.cumsum(take, 0) - take
    m = stay.unsqueeze(1)
    fresh = ring[(head + before.unsqueeze(1) + (col - m).clamp(min=0)) % N]
    mine = tables[p]
    out = torch.where(col < m, mine, torch.where(col < want.unsqueeze(1), fresh, torch.full_like(fresh, -1)))
    # holders of every block, before and after
    spare = torch.full_like(tables, N)
    tally = lambda ids: torch.zeros(N + 1, dtype=torch.long, device=dev).scatter_add_(
        0, ids.flatten().long(), torch.ones(R * C, dtype=torch.long, device=dev))[:N]
    was = tally(torch.where(col < have.unsqueeze(1), tables, spare))
    now = tally(torch.where(out >= 0, out, spare))
    shares = (now - 1).clamp(min=0).int()
    gone = (was > 0) & (now == 0)
    place = torch.where(gone, (head + count + torch.cumsum(gone, 0) - 1) % N, torch.full_like(now, N))
    longer = torch.cat([ring, ring[:1]])
    longer[place] = torch.arange(N, dtype=torch.int32, device=dev)
    ring.copy_(longer[:N])
    state = torch.stack([(head + take.sum()) % N, count - take.sum() + gone.sum()]).int()
    # the blocks to be copied, in the order of their rows
    to = torch.where(copies_it, torch.cumsum(copies_it, 0) - 1, torch.full_like(me, R))
    copies = torch.full((R + 1, 3), -1, dtype=torch.int32, device=dev)
    copies[to] = torch.stack([block, out.long().gather(1, full.clamp(max=C - 1).unsqueeze(1)).squeeze(1), rest], 1).int()
    # the slots of the new tokens, row after row
    tokens = new - kept
    starts = torch.cat([zero[:1], torch.cumsum(tokens, 0)])
    i = torch.arange(s["max_tokens"], device=dev)
    r = torch.searchsorted(starts, i, right=True) - 1
    inside = r < R
    r = r.clamp(max=R - 1)
    pos = kept[r] + i - starts[r]
    slots = torch.where(inside, out[r, (pos // S).clamp(max=C - 1)].long() * S + pos % S, torch.full_like(pos, -1))
    return out, new.int(), shares, state, slots, starts.int(), copies[:R], ring


def _parts(cache, layout):
    return (cache[0], cache[1]) if layout == "flash" else (cache[:, 0], cache[:, 1])


def _plain_copy(s):
    c = s["copies"].long()
    t = torch.arange(s["block"], device=c.device).unsqueeze(0)
    used = t < c[:, 2:]
    src, dst = c[:, :1].expand_as(used)[used], c[:, 1:2].expand_as(used)[used]
    place = t.expand_as(used)[used]
    for cache in s["caches"]:
        for part in _parts(cache, s["layout"]):
            part[dst, place] = part[src, place]
    return s["caches"]


def _plain_compact(s):
    tables, ring, S = s["tables"], s["free"], s["block"]
    (R, C), N, dev = tables.shape, ring.numel(), tables.device
    head, count = s["state"][0].long(), s["state"][1].long()
    col, ids = torch.arange(C, device=dev).unsqueeze(0), torch.arange(N, device=dev)
    inside = col < ((s["lengths"].long() + S - 1) // S).unsqueeze(1)
    spare = torch.full_like(ids, N)
    mark = lambda at: torch.zeros(N + 1, dtype=torch.bool, device=dev).scatter_(
        0, at.flatten(), torch.ones(at.numel(), dtype=torch.bool, device=dev))[:N]
    held = mark(torch.where(inside, tables.long(), spare[0]))
    free = mark(torch.where(ids < count, ring[(head + ids) % N].long(), spare))
    pool = held | free
    rank, n = torch.cumsum(pool, 0) - pool.long(), held.sum()
    low = pool & (rank < n)
    src, dst = held & ~low, free & low
    number = lambda which: torch.cumsum(which, 0) - 1
    to = torch.full((N + 1,), N, dtype=torch.long, device=dev).scatter_(0, torch.where(dst, number(dst), spare), ids)
    moved = torch.where(src, to[number(src).clamp(min=0)], ids)
    name = torch.cat([moved, spare[:1]])
    out = torch.where(inside, name[tables.long().clamp(min=0)].int(), torch.full_like(tables, -1))
    shares = torch.zeros(N + 1, dtype=torch.int32, device=dev).scatter_(0, torch.where(held, moved, spare), s["shares"])[:N]
    new_ring = torch.full((N + 1,), -1, dtype=torch.int32, device=dev).scatter_(
        0, torch.where(pool & ~low, rank - n, spare), ids.int())[:N]
    moves = torch.full((N + 1, 3), -1, dtype=torch.int32, device=dev)
    moves[torch.where(src, number(src), spare)] = torch.stack([ids, moved, torch.full_like(ids, S)], 1).int()
    moves[N:] = -1
    return out, shares, new_ring, torch.stack([torch.zeros_like(n), pool.sum() - n]).int(), moves[:N // 2]


# ------------------------------------------------------------------ work
def work(case):
    if case["kind"] == "select":
        n = case["requests"] * case["beams"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * case["vocab"] * size + 16 * n + 12 * case["requests"] * case["count"],
                "flops": 3 * n * case["vocab"]}
    if case["kind"] == "copy":
        moved = sum(t for t in _copy_plan(case) if t > 0)
        return {"bytes": 2 * moved * case["layers"] * 2 * case["kv_heads"] * case["head_dim"] * 2, "flops": 0}
    S = case["block"]
    if case["kind"] == "fork":
        plan, parents, new = _fork_plan(case)
        rows, holders = _rows_of(case, plan)
        # lengths, parents, new ones; the rows looked at; whole new tables, shares, slots, copies
        ints = 4 * len(rows) + sum(map(len, rows)) + len(rows) * case["columns"] + 2 * len(holders) + 3 * len(rows)
        tokens = sum(max(0, n - (plan[p][0] if p >= 0 else 0)) for p, n in zip(parents, new))
        return {"bytes": 4 * ints + 8 * tokens, "flops": 0}
    rows = _groups(case, random.Random(case["lens_seed"]), budget=int(case["blocks"] * case["held"]))
    ints = len(rows) + sum(_blocks(n, S) for n, _, _ in rows) + len(rows) * case["columns"] + 5 * case["blocks"]
    return {"bytes": 4 * ints, "flops": 0}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"select": _exact_select, "fork": _exact_fork, "copy": _exact_copy,
            "compact": _exact_compact}[case["kind"]](case, s)


def _exact_select(case, s):
    """Request after request: every candidate of every beam in one list, sorted."""
    B, n, V, dev = case["beams"], case["count"], case["vocab"], s["logits"].device
    lists = [[], [], [], [], [], []]
    for r in range(case["requests"]):
        beam = s["logits"][r * B:(r + 1) * B].to(torch.float64)
        value = torch.log_softmax(beam, -1) + s["scores"][r * B:(r + 1) * B, None].to(torch.float64)
        value = torch.nan_to_num(value, nan=-math.inf).flatten()
        best, at = torch.sort(-value, stable=True)
        found = [(-b, i) for b, i in zip(best[:n].tolist(), at[:n].tolist()) if -b > -3.4e38]
        every = [(r * B + i // V, i % V, b) for b, i in found]
        every += [(-1, -1, -math.inf)] * (n - len(every))
        on = [c for c in every if c[0] >= 0 and c[1] != s["end"]][:B]
        on += [(-1, -1, -math.inf)] * (B - len(on))
        for k in range(3):
            lists[k] += [c[k] for c in on]
            lists[3 + k].append([c[k] for c in every])
    types = [torch.int32, torch.int32, torch.float64] * 2
    return tuple(torch.tensor(v, dtype=t, device=dev) for v, t in zip(lists, types))


def _put(dev, *values):
    return tuple(torch.tensor(v, dtype=t, device=dev) for v, t in values)


def _exact_fork(case, s):
    """The update as a program on the host makes it, one row after the other."""
    S, dev, I = case["block"], s["tables"].device, torch.int32
    tables, ring, length = s["tables"].tolist(), s["free"].tolist(), s["lengths"].tolist()
    parents, (head, count) = s["parents"].tolist(), s["state"].tolist()
    N, C, R = len(ring), len(tables[0]), len(tables)
    new = s["new"].tolist() if case["mixed"] else [length[p] + s["new"] if p >= 0 else 0 for p in parents]
    kept = [min(length[p], n) if p >= 0 else 0 for p, n in zip(parents, new)]
    holders = {}
    for row, n in zip(tables, length):
        for b in row[:_blocks(n, S)]:
            holders[b] = holders.get(b, 0) + 1
    owner = {}  # who goes on in a parent's block
    longest = {}
    for p, k in zip(parents, kept):
        longest[p] = max(longest.get(p, 0), k)
    for r, (p, k) in enumerate(zip(parents, kept)):
        if p >= 0 and k % S and longest[p] < (k // S + 1) * S and longest[p] >= k // S * S \
                and holders[tables[p][k // S]] == 1:
            owner.setdefault(p, r)
    out, copies, slots, starts, taken = [], [], [], [0], 0
    after = {}
    for r, (p, k, n) in enumerate(zip(parents, kept, new)):
        row = tables[p][:k // S] if p >= 0 else []
        if k % S and owner.get(p) == r:
            row = row + [tables[p][k // S]]
        for b in row:
            after[b] = after.get(b, 0) + 1
        if k % S and owner.get(p) != r:
            copies.append([tables[p][k // S], ring[(head + taken) % N], k % S])
        while len(row) < _blocks(n, S):
            row.append(ring[(head + taken) % N])
            taken += 1
        slots += [row[i // S] * S + i % S for i in range(k, n)]
        starts.append(len(slots))
        out.append(row + [-1] * (C - len(row)))
    gone = sorted(b for b in holders if b not in after)
    for i, b in enumerate(gone):
        ring[(head + count + i) % N] = b
    shares = [max(0, after.get(b, 0) - 1) for b in range(N)]
    slots += [-1] * (s["max_tokens"] - len(slots))
    copies += [[-1, -1, -1]] * (R - len(copies))
    return _put(dev, (out, I), (new, I), (shares, I), ([(head + taken) % N, count - taken + len(gone)], I),
                (slots, torch.int64), (starts, I), (copies, I), (ring, I))


def _exact_copy(case, s):
    moves = [m for m in s["copies"].tolist() if m[0] >= 0]
    caches = []
    for cache in s["caches"]:
        whole = cache.double()
        for a, b, t in moves:
            if case["layout"] == "flash":
                whole[:, b, :t] = cache[:, a, :t].double()
            else:
                whole[b, :, :t] = cache[a, :, :t].double()
        caches.append(whole)
    return caches


def _exact_compact(case, s):
    S, dev, I = case["block"], s["tables"].device, torch.int32
    tables, ring, length, shares = s["tables"].tolist(), s["free"].tolist(), s["lengths"].tolist(), s["shares"].tolist()
    head, count = s["state"].tolist()
    N = len(ring)
    held = sorted({b for row, n in zip(tables, length) for b in row[:_blocks(n, S)]})
    free = sorted(ring[(head + i) % N] for i in range(count))
    pool = sorted(held + free)
    low, name = set(pool[:len(held)]), {b: b for b in held}
    away = [b for b in held if b not in low]
    room = [b for b in free if b in low]
    name.update(zip(away, room))
    out = [[name[b] for b in row[:_blocks(n, S)]] + [-1] * (len(row) - _blocks(n, S)) for row, n in zip(tables, length)]
    new_shares = [0] * N
    for b in held:
        new_shares[name[b]] = shares[b]
    rest = pool[len(held):]
    moves = [[a, b, S] for a, b in zip(away, room)]
    moves += [[-1, -1, -1]] * (N // 2 - len(moves))
    return _put(dev, (out, I), (new_shares, I), (rest + [-1] * (N - len(rest)), I), ([0, len(rest)], I),
                (torch.tensor(moves, dtype=I).reshape(N // 2, 3).tolist(), I))
