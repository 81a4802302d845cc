"""The decode-instance example: received requests and several drafted steps against a mirror of
every token's keys and values kept outside the blocks."""

import random
import sys
from pathlib import Path

import pytest
import torch

from kvserve_amd import paged
from kvserve_amd.engine import FusedKVCodec
from kvserve_amd.workloads import SEED_HADAMARD, kv_blocks, llama_row_profiles

from _paged_ref import attention

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
import decode_instance as example  # noqa: E402

pytestmark = pytest.mark.gpu


def test_accepted_paths_are_walks():
    rng = random.Random(0)
    for path in example.accepted_paths(rng, example.PARENTS, 50):
        nodes = [p for p in path if p >= 0]
        assert nodes[0] == 0 and all(example.PARENTS[b] == a for a, b in zip(nodes, nodes[1:]))
        assert path == nodes + [-1] * (len(path) - len(nodes))


def dense(inst, layer, r, n):
    """Request r's first n tokens' keys and values out of the blocks: [2, n, H, D]."""
    S = inst.tables.block_size
    p = torch.arange(n, device=inst.lengths.device)
    return inst.caches[layer][:, inst.tables.tables[r].long()[p // S], p % S]


def test_steps_keep_every_token(cuda):
    L, H, G, D, S, lengths = 2, 4, 2, 64, 16, [70, 33, 1, 160]
    R, room = len(lengths), 20
    gen = torch.Generator(device=cuda).manual_seed(5)
    codec = FusedKVCodec(H, D, S, 4, SEED_HADAMARD)
    profiles = llama_row_profiles(L, H)
    pools, packets = [], []
    for n in lengths:
        blocks = -(-n // S)
        pools.append([kv_blocks(gen, blocks, S, H, D, device=cuda) for _ in range(L)])
        packets.append(codec.compress(pools[-1], list(range(blocks)), profiles))
    inst = example.DecodeInstance(L, H, G, D, S, R * room, R, room, cuda)
    inst.receive(codec, packets, lengths)
    mirror = []
    for r, n in enumerate(lengths):
        straight = [torch.zeros_like(p) for p in pools[r]]  # the same packet into blocks in order
        codec.decompress(packets[r], straight, list(range(straight[0].shape[1])))
        mirror.append([p.flatten(1, 2)[:, :n] for p in straight])
        for layer in range(L):
            assert torch.equal(dense(inst, layer, r, n), mirror[r][layer])
    mask, rng, drafts = paged.tree_mask(example.PARENTS, device=cuda), random.Random(1), len(example.PARENTS)
    for _ in range(5):
        tokens = torch.randint(0, 256, (R, drafts), generator=gen, device=cuda)
        paths = example.accepted_paths(rng, example.PARENTS, R)
        before = inst.lengths.tolist()
        x = inst.embed[tokens.flatten()]
        seen = inst.step(tokens, mask, torch.tensor(paths, dtype=torch.int32, device=cuda), room * S, check=True)
        for layer, (query, got) in enumerate(seen):
            rows = (x @ inst.qkv[layer]).view(R, drafts, -1, D)[:, :, H * G:]
            key, value = rows[:, :, :H], rows[:, :, H:]
            for r in range(R):
                # a cache of one request, its tokens and drafts in one block
                whole = torch.cat([mirror[r][layer], torch.stack([key[r], value[r]])], 1)
                n = whole.shape[1]
                i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
                want, _, bound = attention(query[r * drafts:(r + 1) * drafts], whole.unsqueeze(1), i32([[0]]), i32([n]),
                                           i32([0, drafts]), mask)
                assert ((got[r * drafts:(r + 1) * drafts].double() - want).abs() <= bound).all()
                kept = [j for j in paths[r] if j >= 0]
                mirror[r][layer] = torch.cat([mirror[r][layer], torch.stack([key[r][kept], value[r][kept]])], 1)
            x = x + got.flatten(1) @ inst.out[layer]
        after = inst.lengths.tolist()
        assert after == [b + sum(j >= 0 for j in p) for b, p in zip(before, paths)]
        assert inst.tables.lengths.tolist() == after
        held = [b for row in inst.tables.tables.tolist() for b in row if b >= 0]
        assert len(set(held)) == len(held) == sum(-(-n // S) for n in after)
        assert int(inst.tables.state[1]) == R * room - len(held)
        for r in range(R):
            for layer in range(L):
                assert torch.equal(dense(inst, layer, r, after[r]), mirror[r][layer])


def test_the_example_runs(cuda, capsys):
    example.main(["--requests", "3", "--layers", "2", "--steps", "3", "--prompt", "200"])
    assert "3 requests" in capsys.readouterr().out
