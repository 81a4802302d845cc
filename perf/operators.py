"""What the operators of a decode instance are measured on: block tables built from request
lengths, keys and values written by slot, attention of drafted tokens over the paged cache,
and the accepted drafts kept.

A case is one call that a serving program makes; `draw` gives more of the same ranges.

  tables_decode     a decode step of a full batch: every request grows by its drafts
  tables_mixed      prompts come in, requests end, drafts are taken back: one update of all
  write_step        one step's keys and values, rows of a fused projection
  write_prompt      a chunk of prompts, rows of a fused projection
  attend_one        one request, one token: nothing but latency
  attend_decode     one token for each of many ragged requests
  attend_tree       a 26-node tree over a batch of short contexts, fp16, head_dim 64
  attend_long_tree  a 64-node tree over long contexts, 8 query heads a KV head
  attend_prompt     a whole causal prompt over its own cache
  attend_odd        chunks of 1 to 300 tokens, head_dim 80, 3 query heads a KV head, K and V adjacent
  keep_one          one request's accepted path, every layer
  keep_batch        a batch's accepted paths, every layer
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # 256 running requests, a draft of 8 tokens each, tables of 12288 tokens (ragged batch lengths)
        dict(name="tables_decode", kind="tables", requests=256, block=16, columns=768, lo=1024, hi=12000,
             grow=8, joins=0.0, ends=0.0, shrinks=0.0, short=False, lens_seed=1),
        # 1024 requests of all sorts in one update
        dict(name="tables_mixed", kind="tables", requests=1024, block=16, columns=1024, lo=1, hi=8192, grow=33,
             joins=0.1, ends=0.1, shrinks=0.3, short=False, lens_seed=2),
        # 96 requests' next tokens, some rows padding
        dict(name="write_step", kind="write", tokens=96, kv_heads=8, group=4, head_dim=128, block=16, pad=0.1,
             dtype="bf16", layout="flash"),
        # a chunk of 16384 prompt tokens
        dict(name="write_prompt", kind="write", tokens=16384, kv_heads=8, group=4, head_dim=128, block=16, pad=0.0,
             dtype="bf16", layout="flash"),
        # the shortest answer there is: 512 cached tokens (config 1), one query token
        dict(name="attend_one", kind="attend", requests=1, kv_heads=8, group=4, head_dim=128, block=16,
             prefix_lo=511, prefix_hi=511, new_lo=1, new_hi=1, tree=False, dtype="bf16", layout="flash", empty=False,
             lens_seed=3),
        # config 3's ragged lengths, decoded one token at a time
        dict(name="attend_decode", kind="attend", requests=64, kv_heads=8, group=4, head_dim=128, block=16,
             prefix_lo=1024, prefix_hi=12288, new_lo=1, new_hi=1, tree=False, dtype="bf16", layout="flash",
             empty=False, lens_seed=4),
        # drafted trees over many short requests (config 5's head size)
        dict(name="attend_tree", kind="attend", requests=96, kv_heads=4, group=7, head_dim=64, block=16,
             prefix_lo=200, prefix_hi=2000, new_lo=26, new_hi=26, tree=True, dtype="fp16", layout="flash",
             empty=False, lens_seed=5),
        # config 4's length with the widest trees; with the prompt the largest case
        dict(name="attend_long_tree", kind="attend", requests=8, kv_heads=8, group=8, head_dim=128, block=16,
             prefix_lo=24576, prefix_hi=32768, new_lo=64, new_hi=64, tree=True, dtype="bf16", layout="flash",
             empty=False, lens_seed=6),
        # config 2's request attended as a prompt
        dict(name="attend_prompt", kind="attend", requests=1, kv_heads=8, group=4, head_dim=128, block=16,
             prefix_lo=0, prefix_hi=0, new_lo=8192, new_hi=8192, tree=False, dtype="bf16", layout="flash",
             empty=False, lens_seed=7),
        # prompts in chunks mixed with decodes, odd everything, requests without a block among them
        dict(name="attend_odd", kind="attend", requests=13, kv_heads=5, group=3, head_dim=80, block=12,
             prefix_lo=0, prefix_hi=3001, new_lo=1, new_hi=300, tree=False, dtype="bf16", layout="kv_adjacent",
             empty=True, lens_seed=8),
        # 28 layers x 4 KV heads (the runtime's dispatch benchmark)
        dict(name="keep_one", kind="keep", requests=1, layers=28, kv_heads=4, head_dim=128, block=16, drafts=26,
             path=5, lo=100, hi=100, dtype="bf16", layout="flash", lens_seed=9),
        # 32 layers x 8 KV heads, paths of up to 8 tokens
        dict(name="keep_batch", kind="keep", requests=32, layers=32, kv_heads=8, head_dim=128, block=16, drafts=32,
             path=8, lo=1, hi=48, dtype="bf16", layout="flash", lens_seed=10),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _fit(case):
    """Fewer requests, heads or queries until a drawn case costs no more than the largest listed ones."""
    while True:
        cost = work(case)
        if cost["bytes"] <= 1.5e9 and cost["flops"] <= 4e11:
            return case
        name = next(k for k in ("requests", "group", "kv_heads", "new_hi", "prefix_hi") if case[k] > 1)
        case[name] //= 2
        case["new_lo"] = min(case["new_lo"], case["new_hi"])
        case["prefix_lo"] = min(case["prefix_lo"], case["prefix_hi"])


def draw(rng):
    kind = rng.choice(["tables", "write", "decode", "tree", "tree", "prompt", "chunks", "keep"])
    lens_seed = rng.randrange(1 << 30)
    shape = dict(kv_heads=rng.choice([1, 2, 4, 5, 8]), group=rng.choice([1, 2, 3, 4, 5, 7, 8, 16]),
                 head_dim=rng.choice([64, 64, 80, 96, 112, 120, 128, 128, 128, 160, 192, 256]),
                 block=rng.choice([1, 12, 16, 16, 16, 32, 64, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                 layout=rng.choice(["flash", "flash", "kv_adjacent"]))
    if kind == "tables":
        block = rng.choice([1, 12, 16, 16, 32, 64, 128])
        columns = _log_int(rng, 8, 1024)
        hi = block * columns - 64 if block * columns > 128 else block * columns // 2
        return dict(kind="tables", requests=_log_int(rng, 1, 1024), block=block, columns=columns, lo=1,
                    hi=min(hi, 8192), grow=rng.choice([1, 1, 8, 33]), joins=rng.choice([0.0, 0.1, 0.5]),
                    ends=rng.choice([0.0, 0.1, 0.4]), shrinks=rng.choice([0.0, 0.3]),
                    short=rng.random() < 0.25, lens_seed=lens_seed)
    if kind == "write":
        return dict(shape, kind="write", tokens=_log_int(rng, 1, 12000), kv_heads=rng.choice([1, 2, 4, 8]),
                    group=rng.choice([1, 4, 7]), pad=rng.choice([0.0, 0.1]))
    if kind == "keep":
        layers = rng.choice([16, 28, 32])
        del shape["group"]
        drafts = rng.randint(17, 64)
        return dict(shape, kind="keep", requests=_log_int(rng, 1, 24), layers=layers,
                    kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 80, 128]),
                    block=rng.choice([1, 12, 16, 32]), drafts=drafts, path=rng.randint(1, 8), lo=0,
                    hi=48, lens_seed=lens_seed)
    base = dict(shape, kind="attend", tree=False, empty=rng.random() < 0.2, lens_seed=lens_seed)
    if kind == "decode":
        hi = _log_int(rng, 16, 8192)
        return _fit(dict(base, requests=_log_int(rng, 1, 64), prefix_lo=rng.choice([0, hi // 4, hi]), prefix_hi=hi,
                         new_lo=1, new_hi=rng.choice([1, 1, 2, 5])))
    if kind == "tree":
        nodes = rng.choice([2, 5, 8, 13, 26, 32, 61, 64, 100])
        hi = _log_int(rng, 16, 16384)
        return _fit(dict(base, requests=_log_int(rng, 1, 64), prefix_lo=hi // 4, prefix_hi=hi,
                         new_lo=rng.choice([1, nodes, nodes]), new_hi=nodes, tree=True))
    if kind == "prompt":
        new = _log_int(rng, 64, 4096)
        return _fit(dict(base, requests=1, prefix_lo=0, prefix_hi=rng.choice([0, 0, 1000]), new_lo=new, new_hi=new,
                         kv_heads=rng.choice([1, 2, 4, 8]), group=rng.choice([1, 4, 7]),
                         head_dim=rng.choice([64, 80, 128, 128, 192, 256])))
    new = _log_int(rng, 2, 400)
    return _fit(dict(base, requests=rng.randint(2, 12), prefix_lo=0, prefix_hi=_log_int(rng, 1, 4000), new_lo=1,
                     new_hi=new))


# ------------------------------------------------------------------ lengths (from the case alone)
def _attend_lens(case):
    """[(cache length with the queries, queries)] a request."""
    r = random.Random(case["lens_seed"])
    out = []
    for _ in range(case["requests"]):
        t = r.randint(case["new_lo"], case["new_hi"])
        out.append((r.randint(case["prefix_lo"], case["prefix_hi"]) + t, t))
    if case["empty"]:
        out[0] = (0, 1)  # a request that got no block: its query sees nothing
        if len(out) > 1:
            out[-1] = (out[-1][0], 0)  # a request that sits this step out
    return out


def _tables_lens(case):
    """[(tokens before, tokens after)] a request."""
    r = random.Random(case["lens_seed"])
    top = case["block"] * case["columns"]
    out = []
    for _ in range(case["requests"]):
        now, u = r.randint(case["lo"], case["hi"]), r.random()
        if u < case["joins"]:
            now, new = 0, now
        elif u < case["joins"] + case["ends"]:
            new = 0
        elif u < case["joins"] + case["ends"] + case["shrinks"]:
            new = max(0, now - r.randint(0, case["grow"]))
        else:
            new = now + case["grow"]
        out.append((now, min(new, top)))
    return out


def _blocks(tokens, block):
    return (tokens + block - 1) // block


def _tree_words(r, nodes, words):
    """Visibility of a random tree in breadth: node i sees itself and its ancestors.  Node 0
    is the last token of the answer, all others descend from it."""
    seen = []
    rows = []
    for i in range(nodes):
        bits = (seen[r.randrange(max(0, i - 12), i)] if i else 0) | (1 << i)
        seen.append(bits)
        row = [(bits >> (64 * w)) & ((1 << 64) - 1) for w in range(words)]
        rows.append([v - (1 << 64) if v >> 63 else v for v in row])
    return rows


# ------------------------------------------------------------------ inputs
def _cache(case, blocks, gen, dev):
    S, H, D = case["block"], case["kv_heads"], case["head_dim"]
    shape = (2, blocks, S, H, D) if case["layout"] == "flash" else (blocks, 2, S, H, D)
    cache = torch.empty(shape, device=dev, dtype=DTYPES[case["dtype"]])
    cache.normal_(generator=gen)
    # a few strong key channels a head, as the engine's workloads have them
    keys = cache[0] if case["layout"] == "flash" else cache[:, 0]
    strong = torch.ones((H, D), device=dev, dtype=cache.dtype)
    for h in range(H):
        strong[h, torch.randperm(D, generator=gen, device=dev)[:4]] = 4.0
    keys *= strong
    return cache


def _tables(counts, columns, blocks, gen, dev):
    """Block tables [requests, columns]: each request's blocks scattered over the pool, -1 behind."""
    ids = torch.randperm(blocks, generator=gen, device=dev).to(torch.int32)
    col = torch.arange(columns, device=dev).unsqueeze(0)
    n = torch.tensor(counts, device=dev).unsqueeze(1)
    first = torch.cumsum(n, 0) - n
    where = (first + col).clamp(max=blocks - 1)
    return torch.where(col < n, ids[where], torch.full_like(ids[where], -1)), ids


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    return {"tables": _prepare_tables, "write": _prepare_write, "attend": _prepare_attend,
            "keep": _prepare_keep}[case["kind"]](case, gen, seed, dev)


def _int32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _prepare_tables(case, gen, seed, dev):
    lens = _tables_lens(case)
    S, R, C = case["block"], case["requests"], case["columns"]
    have = [_blocks(a, S) for a, _ in lens]
    take = sum(max(0, _blocks(b, S) - _blocks(a, S)) for a, b in lens)
    free = take // 2 if case["short"] else take + 7
    pool = sum(have) + free
    pool = max(pool, 1)
    tables, ids = _tables(have, C, pool, gen, dev)
    # the free blocks lie in a ring that has been turned
    head = random.Random(seed).randrange(pool)
    ring = torch.full((pool,), -1, dtype=torch.int32, device=dev)
    ring[(head + torch.arange(free, device=dev)) % pool] = ids[sum(have):sum(have) + free]
    tokens = sum(max(0, b - a) for a, b in lens)
    state = dict(kind="tables", block=S, max_tokens=tokens + 5, tables=tables, free=ring,
                 lengths=_int32([a for a, _ in lens], dev), new_lengths=_int32([b for _, b in lens], dev),
                 state=_int32([head, free], dev), err=torch.zeros(1, dtype=torch.int32, device=dev))
    state["out"] = (torch.empty_like(tables), torch.empty(R, dtype=torch.int32, device=dev),
                    torch.empty(2, dtype=torch.int32, device=dev),
                    torch.empty(tokens + 5, dtype=torch.int64, device=dev),
                    torch.empty(R + 1, dtype=torch.int32, device=dev))
    return state


def _prepare_write(case, gen, seed, dev):
    T, H, D, S = case["tokens"], case["kv_heads"], case["head_dim"], case["block"]
    blocks = _blocks(T, S) + 3
    cache = _cache(case, blocks, gen, dev)
    # one projection gives the rows of queries, keys and values
    qkv = torch.empty((T, case["kv_heads"] * (case["group"] + 2), D), device=dev, dtype=cache.dtype)
    qkv.normal_(generator=gen)
    first = H * case["group"]
    slots = torch.randperm(blocks * S, generator=gen, device=dev)[:T]
    slots = torch.where(torch.rand(T, generator=gen, device=dev) < case["pad"], torch.full_like(slots, -1), slots)
    return dict(kind="write", key=qkv[:, first:first + H], value=qkv[:, first + H:], cache=cache, slots=slots,
                layout=case["layout"], block=S, err=torch.zeros(1, dtype=torch.int32, device=dev))


def _prepare_attend(case, gen, seed, dev):
    lens = _attend_lens(case)
    S, H, G, D = case["block"], case["kv_heads"], case["group"], case["head_dim"]
    counts = [_blocks(n, S) for n, _ in lens]
    blocks = max(sum(counts), 1) + 3
    cache = _cache(case, blocks, gen, dev)
    tables, _ = _tables(counts, max(counts + [1]) + 1, blocks, gen, dev)
    total = sum(t for _, t in lens)
    query = torch.empty((total, H * G, D), device=dev, dtype=cache.dtype)
    query.normal_(generator=gen)
    starts = [0]
    for _, t in lens:
        starts.append(starts[-1] + t)
    max_query = max(max(t for _, t in lens), 1)
    mask = None
    if case["tree"]:
        words, r = _blocks(max_query, 64), random.Random(seed)
        rows = []
        for _, t in lens:
            rows += _tree_words(r, t, words)
        mask = torch.tensor(rows, dtype=torch.int64, device=dev).reshape(total, words)
    return dict(kind="attend", query=query, cache=cache, tables=tables, lengths=_int32([n for n, _ in lens], dev),
                starts=_int32(starts, dev), mask=mask, max_query=max_query,
                max_length=max(max(n for n, _ in lens), 1), scale=1.0 / math.sqrt(D), layout=case["layout"], block=S,
                host_lens=lens, out=torch.empty_like(query), err=torch.zeros(1, dtype=torch.int32, device=dev))


def _prepare_keep(case, gen, seed, dev):
    r, R, S = random.Random(case["lens_seed"]), case["requests"], case["block"]
    base = [r.randint(case["lo"], case["hi"]) for _ in range(R)]
    counts = [_blocks(n + case["drafts"], S) for n in base]
    blocks = sum(counts) + 2
    tables, _ = _tables(counts, max(counts), blocks, gen, dev)
    caches = [_cache(case, blocks, gen, dev) for _ in range(case["layers"])]
    # the root is kept where it is; the nodes behind it come from deeper in the tree
    r, paths = random.Random(seed), []
    for _ in range(R):
        n = r.randint(1, case["path"])
        paths.append([0] + sorted(r.sample(range(case["path"], case["drafts"]), n - 1)) + [-1] * (case["path"] - n))
    state = dict(kind="keep", caches=caches, tables=tables, lengths=_int32(base, dev), accepted=_int32(paths, dev),
                 layout=case["layout"], block=S, out=torch.empty(R, dtype=torch.int32, device=dev),
                 err=torch.zeros(1, dtype=torch.int32, device=dev))
    if own:
        from kvserve_amd import paged
        state["layers"] = paged.LayerCaches(caches)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    return {"tables": _plain_tables, "write": _plain_write, "attend": _plain_attend,
            "keep": _plain_keep}[state["kind"]](state)


def _run_own(s):
    from kvserve_amd import paged

    if s["kind"] == "tables":
        got = paged.build_block_tables(s["lengths"], s["new_lengths"], s["tables"], s["free"], s["state"], s["block"],
                                       s["max_tokens"], out=s["out"], err=s["err"], check=False)
        return tuple(got) + (s["free"],)
    if s["kind"] == "write":
        paged.write_kv(s["key"], s["value"], s["cache"], s["slots"], err=s["err"], check=False)
        return s["cache"]
    if s["kind"] == "attend":
        return paged.tree_attention(s["query"], s["cache"], s["tables"], s["lengths"], s["starts"],
                                    max_query=s["max_query"], max_length=s["max_length"], tree_mask=s["mask"],
                                    scale=s["scale"], out=s["out"], err=s["err"], check=False)
    lengths = paged.keep_drafts(s["layers"], s["tables"], s["lengths"], s["accepted"], out=s["out"], err=s["err"],
                                check=False)
    return [lengths] + s["caches"]


def _plain_tables(s):
    S, tables, ring = s["block"], s["tables"], s["free"]
    N, C, dev = ring.numel(), tables.shape[1], tables.device
    now, new = s["lengths"].long(), s["new_lengths"].long()
    head, count = s["state"][0].long(), s["state"][1].long()
    have, want = (now + S - 1) // S, (new + S - 1) // S
    take, give = (want - have).clamp(min=0), (have - want).clamp(min=0)
    upto = torch.cumsum(take, 0)
    fits = upto <= count
    granted = fits | (take == 0)
    after = torch.where(granted, new, now)
    keep = torch.where(granted, want, have)
    taken = torch.where(fits, upto, torch.zeros_like(upto)).max()
    col = torch.arange(C, device=dev).unsqueeze(0)
    h, k = have.unsqueeze(1), keep.unsqueeze(1)
    fresh = ring[(head + (upto - take).unsqueeze(1) + (col - h).clamp(min=0)) % N]
    out = torch.where(col < torch.minimum(h, k), tables, torch.where(col < k, fresh, torch.full_like(tables, -1)))
    back = (col >= k) & (col < h)
    before = (torch.cumsum(give, 0) - give).unsqueeze(1)
    ring[((head + count + before + col - k) % N)[back]] = tables[back]
    state = torch.stack([(head + taken) % N, count - taken + give.sum()]).int()
    # the slots of the new tokens, request after request
    tokens = (new - now).clamp(min=0)
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), torch.cumsum(tokens, 0)])
    i = torch.arange(s["max_tokens"], device=dev)
    r = torch.searchsorted(starts, i, right=True) - 1
    inside = r < now.numel()
    r = r.clamp(max=now.numel() - 1)
    pos = now[r] + i - starts[r]
    block = out[r, (pos // S).clamp(max=C - 1)].long()
    slots = torch.where(inside & granted[r], block * S + pos % S, torch.full_like(pos, -1))
    return out, after.int(), state, slots, starts.int(), ring


def _parts(cache, layout):
    return (cache[0], cache[1]) if layout == "flash" else (cache[:, 0], cache[:, 1])


def _plain_write(s):
    k, v = _parts(s["cache"], s["layout"])
    used = s["slots"] >= 0
    slots = s["slots"][used]
    block, place = slots // s["block"], slots % s["block"]
    k[block, place] = s["key"][used]
    v[block, place] = s["value"][used]
    return s["cache"]


def _plain_attend(s):
    keys, values = _parts(s["cache"], s["layout"])
    H, D = keys.shape[-2:]
    G = s["query"].shape[1] // H
    out, at = s["out"], 0
    for r, (n, t) in enumerate(s["host_lens"]):
        if t == 0:
            continue
        q = s["query"][at:at + t].float().reshape(t, H, G, D)
        blocks = s["tables"][r, :(n + s["block"] - 1) // s["block"]].long()
        pos = torch.arange(n, device=q.device) - (n - t)  # place among the queries; before them negative
        if s["mask"] is None:
            seen = pos.unsqueeze(0) <= torch.arange(t, device=q.device).unsqueeze(1)
        else:
            j = pos.clamp(min=0)
            bits = (s["mask"][at:at + t][:, j // 64] >> (j % 64)) & 1
            seen = (pos < 0) | (bits == 1)
        seen = seen.repeat_interleave(G, 0)
        for h in range(H):
            if n == 0:
                out[at:at + t, h * G:(h + 1) * G] = 0
                continue
            k = keys[blocks, :, h].reshape(-1, D)[:n].float()
            v = values[blocks, :, h].reshape(-1, D)[:n].float()
            x = (q[:, h].reshape(t * G, D) @ k.t()) * s["scale"]
            x = torch.where(seen, x, torch.full_like(x, -math.inf))
            top = x.max(1, keepdim=True).values
            x = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = x.sum(1, keepdim=True)
            o = (x @ v) / torch.where(total == 0, torch.ones_like(total), total)
            out[at:at + t, h * G:(h + 1) * G] = o.reshape(t, G, D).to(out.dtype)
        at += t
    return out


def _plain_keep(s):
    S, R, A = s["block"], s["accepted"].shape[0], s["accepted"].shape[1]
    dev = s["tables"].device
    kept = s["accepted"] >= 0
    base = s["lengths"].long().unsqueeze(1)
    r = torch.arange(R, device=dev).unsqueeze(1).expand(R, A)[kept]
    src = (base + s["accepted"].long())[kept]
    dst = (base + torch.arange(A, device=dev).unsqueeze(0))[kept]
    src_block, dst_block = s["tables"][r, src // S].long(), s["tables"][r, dst // S].long()
    for cache in s["caches"]:
        for part in _parts(cache, s["layout"]):
            part[dst_block, dst % S] = part[src_block, src % S]
    s["out"].copy_(s["lengths"] + kept.sum(1).int())
    return [s["out"]] + s["caches"]


# ------------------------------------------------------------------ work
def work(case):
    S = case["block"]
    if case["kind"] == "tables":
        lens = _tables_lens(case)
        tokens = sum(max(0, b - a) for a, b in lens)
        held = sum(_blocks(a, S) for a, _ in lens)
        moved = sum(abs(_blocks(b, S) - _blocks(a, S)) for a, b in lens)
        # lengths in (2) and out, the blocks held and moved, the whole new tables, slots and starts
        ints = 4 * case["requests"] + held + 2 * moved + case["requests"] * case["columns"]
        return {"bytes": 4 * ints + 8 * tokens, "flops": 0}
    H, D = case["kv_heads"], case["head_dim"]
    if case["kind"] == "write":
        return {"bytes": case["tokens"] * (8 + 2 * 2 * H * D * 2) * (1 - case["pad"]), "flops": 0}
    if case["kind"] == "keep":
        mean = (case["path"] + 1) / 2 - 1  # the root stays
        return {"bytes": max(1, case["requests"] * mean * case["layers"] * 2 * 2 * H * D * 2), "flops": 0}
    G, nbytes, pairs = case["group"], 0, 0
    for n, t in _attend_lens(case):
        if t == 0:
            continue
        nbytes += 2 * 2 * H * D * n + 4 * _blocks(n, S) + 2 * 2 * t * H * G * D
        nbytes += 8 * t * _blocks(t, 64) if case["tree"] else 0
        if n:
            pairs += t * (n - t) + t * (t + 1) // 2
    return {"bytes": max(nbytes, 1), "flops": 4 * D * H * G * pairs}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, s)
    if case["kind"] == "write":
        return _exact_write(case, s)
    if case["kind"] == "keep":
        return _exact_keep(case, s)
    return _exact_tables(case, s)


def _exact_attend(case, s):
    """Softmax over the visible keys, key positions in pieces with a shared maximum."""
    S, H, G, D = case["block"], case["kv_heads"], case["group"], case["head_dim"]
    flash = case["layout"] == "flash"
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=s["query"].device)
    at = 0
    for r, (n, t) in enumerate(_attend_lens(case)):
        if n and t:
            p = torch.arange(n, device=out.device)
            block, place = s["tables"][r][p // S].long(), p % S
            first = n - t
            for h in range(H):
                if flash:
                    k, v = s["cache"][0, block, place, h].double(), s["cache"][1, block, place, h].double()
                else:
                    k, v = s["cache"][block, 0, place, h].double(), s["cache"][block, 1, place, h].double()
                for a in range(0, t, 1024):
                    b = min(t, a + 1024)
                    q = s["query"][at + a:at + b, h * G:(h + 1) * G].double()  # [queries, G, D]
                    x = torch.matmul(q.reshape(-1, D), k.t()).reshape(b - a, G, n) * s["scale"]
                    hidden = torch.zeros((b - a, n), dtype=torch.bool, device=out.device)
                    if s["mask"] is None:
                        i = torch.arange(a, b, device=out.device)
                        hidden = p.unsqueeze(0) > first + i.unsqueeze(1)
                    else:
                        for j in range(t):
                            word = s["mask"][at + a:at + b, j // 64]
                            hidden[:, first + j] = torch.bitwise_and(torch.bitwise_right_shift(word, j % 64), 1) == 0
                    x.masked_fill_(hidden.unsqueeze(1), -math.inf)
                    w = torch.softmax(x, -1)
                    w.masked_fill_(hidden.unsqueeze(1), 0.0)
                    out[at + a:at + b, h * G:(h + 1) * G] = torch.matmul(w.reshape(-1, n), v).reshape(b - a, G, D)
        at += t
    return out


def _exact_write(case, s):
    S = case["block"]
    rows = s["cache"].double()
    for part, new in ((0, s["key"]), (1, s["value"])):
        plane = (rows[part] if case["layout"] == "flash" else rows[:, part])
        flat = plane.reshape(-1, *plane.shape[2:]).clone()
        for_rows = torch.nonzero(s["slots"] >= 0).flatten()
        flat.index_copy_(0, s["slots"][for_rows], new[for_rows].double())
        plane.copy_(flat.reshape(plane.shape))
    assert S * plane.shape[0] == flat.shape[0]
    return rows


def _exact_keep(case, s):
    S = case["block"]
    tables, base, paths = s["tables"].tolist(), s["lengths"].tolist(), s["accepted"].tolist()
    moves, after = [], []
    for table, first, path in zip(tables, base, paths):
        path = [j for j in path if j >= 0]
        after.append(first + len(path))
        for i, j in enumerate(path):
            src, dst = first + j, first + i
            moves.append((table[src // S], src % S, table[dst // S], dst % S))
    m = torch.tensor(moves, device=s["tables"].device)
    caches = []
    for cache in s["caches"]:
        whole = cache.double()
        if case["layout"] == "flash":
            whole[:, m[:, 2], m[:, 3]] = cache[:, m[:, 0], m[:, 1]].double()
        else:
            whole[m[:, 2], :, m[:, 3]] = cache[m[:, 0], :, m[:, 1]].double()
        caches.append(whole)
    return [torch.tensor(after, dtype=torch.int32, device=s["tables"].device)] + caches


def _exact_tables(case, s):
    """The update as a program on the host makes it, one request after the other."""
    S, dev = case["block"], s["tables"].device
    tables, ring = s["tables"].tolist(), s["free"].tolist()
    now, new = s["lengths"].tolist(), s["new_lengths"].tolist()
    head, count = s["state"].tolist()
    N, asked, taken, returned = len(ring), 0, 0, []
    after, slots, starts = [], [], [0]
    for row, a, b in zip(tables, now, new):
        have, want = -(-a // S), -(-b // S)
        old = row[:have]
        asked += max(0, want - have)
        if want > have and asked > count:
            after.append(a)
            slots += [-1] * (b - a)
        else:
            for i in range(have, want):
                row[i] = ring[(head + asked - want + i) % N]
            taken = asked if asked <= count else taken
            returned += old[want:]
            for i in range(want, have):
                row[i] = -1
            after.append(b)
            slots += [row[p // S] * S + p % S for p in range(a, b)]
        starts.append(len(slots))
    for i, block in enumerate(returned):
        ring[(head + count + i) % N] = block
    slots += [-1] * (s["max_tokens"] - len(slots))
    put = lambda v, t: torch.tensor(v, dtype=t, device=dev)
    return (put(tables, torch.int32), put(after, torch.int32),
            put([(head + taken) % N, count - taken + len(returned)], torch.int32), put(slots, torch.int64),
            put(starts, torch.int32), put(ring, torch.int32))
