"""A beam search on a decode instance: compressed requests come in, answers grow by several beams.

    python examples/beam_search.py [--requests 4] [--beams 4] [--layers 4] [--steps 24] [--prompt 2000]

A sender compresses the paged KV of its requests; the instance decompresses each into one row's
blocks and forks it: the beams share the prompt's blocks.  Each step selects the best continuations
of every request, reorders the rows, splits the partly filled blocks that two beams go on in, writes
the new tokens' keys and values and attends over prompt and answer; halfway the pool is compacted.  The
model is a stand-in (random projections); the cache, its tables, the attention and the search are the
real ones.
"""

from __future__ import annotations

import argparse
import math
import random
import sys
import time
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from kvserve_amd import paged  # noqa: E402
from kvserve_amd.engine import FusedKVCodec  # noqa: E402
from kvserve_amd.workloads import SEED_HADAMARD, kv_blocks, llama_row_profiles  # noqa: E402

VOCAB, END = 4096, 2


class BeamInstance:
    """Caches and shared block tables of a batch of requests, `beams` rows each."""

    def __init__(self, layers: int, kv_heads: int, group: int, head_dim: int, block: int, blocks: int, requests: int,
                 beams: int, columns: int, device="cuda", seed: int = 0):
        self.caches = [torch.zeros((2, blocks, block, kv_heads, head_dim), dtype=torch.bfloat16, device=device)
                       for _ in range(layers)]
        self.layers = paged.LayerCaches(self.caches)
        self.requests, self.beams, rows = requests, beams, requests * beams
        self.tables = paged.SharedBlockTables(blocks, block, rows, columns, device)
        self.kv_heads, self.group, self.head_dim = kv_heads, group, head_dim
        hidden = kv_heads * group * head_dim
        gen = torch.Generator(device=device).manual_seed(seed)
        weight = lambda *s: (torch.randn(s, generator=gen, device=device) * s[0]**-0.5).to(torch.bfloat16)
        self.embed = weight(VOCAB, hidden) * 16
        self.qkv = [weight(hidden, hidden + 2 * kv_heads * head_dim) for _ in range(layers)]
        self.out = [weight(hidden, hidden) for _ in range(layers)]
        self.head = weight(hidden, VOCAB)
        self.logits = torch.randn((rows, VOCAB), generator=gen, device=device).to(torch.bfloat16)
        self.scores = torch.full((rows,), -math.inf, device=device)
        self.best = [-math.inf] * requests  # score of the best answer that has ended

    def receive(self, codec: FusedKVCodec, packets, lengths) -> None:
        """Take blocks for prompts of `lengths` tokens in each request's first row and decompress
        them there; one hypothesis a request to begin with."""
        new = torch.zeros_like(self.tables.lengths)
        new[::self.beams] = torch.tensor(lengths, dtype=torch.int32, device=new.device)
        self.tables.update(new, sum(lengths))
        for packet, row, n in zip(packets, self.tables.tables[::self.beams].tolist(), lengths):
            codec.decompress(packet, self.caches, row[:-(-n // self.tables.block_size)])
        self.scores[::self.beams] = 0.0

    def step(self, max_length: int, check=None) -> paged.BeamChoice:
        """Select, reorder and run the model on every beam's new token."""
        rows = self.requests * self.beams
        best = paged.select_beams(self.logits, self.scores, self.beams, 2 * self.beams, end_token=END, check=check)
        slots, starts = self.tables.fork(best.parents, 1, rows, check=check)
        paged.copy_blocks(self.layers, self.tables.copies, check=check)
        # rows without a hypothesis have no token: the others' come first, as their slots do
        order = torch.argsort((best.parents < 0).int(), stable=True)
        x, heads, kv = self.embed[best.tokens.clamp(min=0).long()[order]], self.kv_heads * self.group, self.kv_heads
        for cache, w_in, w_out in zip(self.caches, self.qkv, self.out):
            qkv = (x @ w_in).view(rows, heads + 2 * kv, self.head_dim)
            paged.write_kv(qkv[:, heads:heads + kv], qkv[:, heads + kv:], cache, slots, check=check)
            seen = torch.zeros((rows, heads, self.head_dim), dtype=x.dtype, device=x.device)
            paged.tree_attention(qkv[:, :heads], cache, self.tables.tables, self.tables.lengths, starts, max_query=1,
                                 max_length=max_length, out=seen, check=check)
            x = x + seen.flatten(1) @ w_out
        self.logits[order] = x @ self.head
        self.scores = best.scores
        return best

    def compact(self, check=None) -> None:
        """Bring the held blocks to the front of the pool (between two steps)."""
        paged.copy_blocks(self.layers, self.tables.compact(check=check), check=check)


def main(argv=None) -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("requests", 4), ("beams", 4), ("layers", 4), ("steps", 24), ("prompt", 2000)):
        parser.add_argument(f"--{name}", type=int, default=value)
    args = parser.parse_args(argv)
    if min(args.requests, args.beams, args.layers, args.steps) < 1 or args.prompt < 2 or args.beams > 32:
        parser.error("at least one request, beam (and at most 32), layer and step, and prompts of two tokens")
    dev, heads, dim, block, rng = torch.device("cuda", 0), 8, 128, 16, random.Random(0)
    lengths = [rng.randint(args.prompt // 2, args.prompt) for _ in range(args.requests)]
    counts = [-(-n // block) for n in lengths]

    # the sender: each request's blocks in its pools, compressed
    gen = torch.Generator(device=dev).manual_seed(1)
    codec = FusedKVCodec(heads, dim, block, 4, SEED_HADAMARD)
    profiles = llama_row_profiles(args.layers, heads)
    packets = []
    for n in counts:
        pools = [kv_blocks(gen, n, block, heads, dim, device=dev) for _ in range(args.layers)]
        packets.append(codec.compress(pools, list(range(n)), profiles))

    answer = -(-(args.steps + 1) // block) + 2  # blocks of a beam besides its prompt's
    room = max(counts) + answer
    blocks = sum(counts) + args.requests * args.beams * answer
    inst = BeamInstance(args.layers, heads, 4, dim, block, blocks, args.requests, args.beams, room, dev)
    inst.receive(codec, packets, lengths)
    begin = None
    for i in range(args.steps + 1):
        if i == 1:  # the first step loads the projections' kernels
            torch.cuda.synchronize()
            begin = time.perf_counter()
        best = inst.step(room * block, check=False)
        if i == args.steps // 2:
            inst.compact(check=False)
        ended = torch.where(best.all_tokens == END, best.all_scores, torch.full_like(best.all_scores, -math.inf)).amax(1)
        inst.best = ended if i == 0 else torch.maximum(inst.best, ended)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - begin
    tables = inst.tables
    held, alone = blocks - int(tables.state[1]), int(-(-tables.lengths // block).sum())
    print(f"{args.requests} requests of {min(lengths)} to {max(lengths)} tokens, {args.beams} beams, {args.steps + 1} "
          f"steps, {seconds / args.steps * 1e3:.2f} ms a step; {held} blocks held where rows of their own would hold "
          f"{alone}; best scores {[round(v, 2) for v in inst.scores.view(args.requests, -1)[:, 0].tolist()]}")


if __name__ == "__main__":
    main()
