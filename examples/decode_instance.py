"""A decode instance end to end: compressed requests come in, answers grow by drafted trees.

    python examples/decode_instance.py [--requests 8] [--layers 4] [--steps 6] [--prompt 2000]

A sender compresses the paged KV of its requests; the instance takes blocks for them, decompresses
into its own caches, and then decodes: each step gives every request blocks for a tree of drafts,
writes the drafts' keys and values, attends over prompt, answer and tree, keeps the accepted path
and gives the other drafts' blocks back.  The model is a stand-in (random projections, and a
random choice for the sampler); the cache, its tables and the attention are the real ones.
"""

from __future__ import annotations

import argparse
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

PARENTS = [-1, 0, 0, 0, 1, 1, 2, 4, 4, 7]  # a tree of 10 drafts, 4 deep behind its root


class DecodeInstance:
    """Caches, block tables and the step of a batch of requests."""

    def __init__(self, layers: int, kv_heads: int, group: int, head_dim: int, block: int, blocks: int, requests: int,
                 columns: int, device="cuda", seed: int = 0):
        self.caches = [torch.zeros((2, blocks, block, kv_heads, head_dim), dtype=torch.bfloat16, device=device)
                       for _ in range(layers)]
        self.layers = paged.LayerCaches(self.caches)
        self.tables = paged.BlockTables(blocks, block, requests, columns, device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)  # tokens without drafts
        self.kv_heads, self.group, self.head_dim = kv_heads, group, head_dim
        hidden = kv_heads * group * head_dim
        gen = torch.Generator(device=device).manual_seed(seed)
        weight = lambda *s: (torch.randn(s, generator=gen, device=device) * s[0]**-0.5).to(torch.bfloat16)
        self.embed = weight(256, hidden) * 16
        self.qkv = [weight(hidden, hidden + 2 * kv_heads * head_dim) for _ in range(layers)]
        self.out = [weight(hidden, hidden) for _ in range(layers)]

    def receive(self, codec: FusedKVCodec, packets, lengths) -> None:
        """Take blocks for requests of `lengths` tokens and decompress them there."""
        new = torch.tensor(lengths, dtype=torch.int32, device=self.lengths.device)
        self.tables.update(new, sum(lengths))
        for packet, row, n in zip(packets, self.tables.tables.tolist(), lengths):
            codec.decompress(packet, self.caches, row[:-(-n // self.tables.block_size)])
        self.lengths = new

    def step(self, tokens: torch.Tensor, mask: torch.Tensor, path: torch.Tensor, max_length: int, check=None):
        """One step: `tokens` [requests, drafts], `mask` their visibility words [drafts, words],
        `path` int32 [requests, width] the drafts that turn out accepted.  Returns each layer's
        (queries, attention)."""
        requests, drafts = tokens.shape
        slots, starts = self.tables.update(self.lengths + drafts, requests * drafts, check=check)
        mask = mask.repeat(requests, 1)
        x, seen = self.embed[tokens.flatten()], []
        heads, kv = self.kv_heads * self.group, self.kv_heads
        for cache, w_in, w_out in zip(self.caches, self.qkv, self.out):
            rows = (x @ w_in).view(-1, heads + 2 * kv, self.head_dim)
            query, key, value = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
            paged.write_kv(key, value, cache, slots, check=check)
            got = paged.tree_attention(query, cache, self.tables.tables, self.tables.lengths, starts, max_query=drafts,
                                       max_length=max_length, tree_mask=mask, check=check)
            x = x + got.flatten(1) @ w_out
            seen.append((query, got))
        kept = torch.empty_like(self.lengths)
        paged.keep_drafts(self.layers, self.tables.tables, self.lengths, path, out=kept, check=check)
        self.tables.update(kept, 0, check=check)
        self.lengths = kept
        return seen


def accepted_paths(rng: random.Random, parents, requests: int):
    """A walk down from the root for each request, -1 behind its end: what a sampler accepted."""
    paths = []
    for _ in range(requests):
        path = [0]
        while True:
            children = [i for i, p in enumerate(parents) if p == path[-1]]
            if not children or rng.random() < 0.3:
                break
            path.append(rng.choice(children))
        paths.append(path)
    width = max(map(len, paths))
    return [p + [-1] * (width - len(p)) for p in paths]


def main(argv=None) -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("requests", 8), ("layers", 4), ("steps", 6), ("prompt", 2000)):
        parser.add_argument(f"--{name}", type=int, default=value)
    args = parser.parse_args(argv)
    if min(args.requests, args.layers, args.steps) < 1 or args.prompt < 2:
        parser.error("at least one request, layer and step, and prompts of two tokens")
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

    room = -(-(args.prompt + (args.steps + 1) * len(PARENTS)) // block) + 1
    inst = DecodeInstance(args.layers, heads, 4, dim, block, args.requests * room, args.requests, room, dev)
    inst.receive(codec, packets, lengths)
    mask = paged.tree_mask(PARENTS, device=dev)
    first = int(inst.lengths.sum())
    for i in range(args.steps + 1):
        if i == 1:  # the first step loads the projections' kernels
            torch.cuda.synchronize()
            begin = time.perf_counter()
        tokens = torch.randint(0, 256, (args.requests, len(PARENTS)), generator=gen, device=dev)
        path = torch.tensor(accepted_paths(rng, PARENTS, args.requests), dtype=torch.int32, device=dev)
        inst.step(tokens, mask, path, room * block, check=False)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - begin
    grown = int(inst.lengths.sum()) - first
    print(f"{args.requests} requests of {min(lengths)} to {max(lengths)} tokens received in "
          f"{sum(p.compressed_bytes() for p in packets) / 2**20:.1f} MiB; {grown} tokens in {args.steps + 1} steps, "
          f"{seconds / args.steps * 1e3:.2f} ms a step; {int(inst.tables.state[1])} of {inst.tables.num_blocks} "
          "blocks free")


if __name__ == "__main__":
    main()
