"""The module behind the unchecked calls, for the operators of rows that share blocks: what it takes gives
the same as the checked way, and what it does not take is left to the wrappers' checks."""

import ctypes

import pytest
import torch

from kvserve_amd import paged

BF16 = torch.bfloat16


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def arguments(dev):
    """Right arguments of each function of the module (right on a GPU)."""
    cache = torch.arange(2 * 6 * 16 * 128, device=dev).view(2, 6, 16, 2, 64).to(BF16)
    layers = paged._lib.Cache(cache.data_ptr(), 6 * 16 * 128, 16 * 128, 6, 16, 2, 64)
    lengths, tables, shares = i32([20, 17], dev), i32([[0, 1], [0, 3]], dev), i32([1, 0, 0, 0, 0, 0], dev)
    ring, state = i32([2, 4, 5, -1, -1, -1], dev), i32([0, 3], dev)
    fork = paged.ForkUpdate(i32([[0] * 2] * 2, dev), i32([0, 0], dev), i32([0] * 6, dev), i32([0, 0], dev),
                            torch.zeros(6, dtype=torch.int64, device=dev), i32([0] * 3, dev), i32([[0] * 3] * 2, dev))
    packed = paged.Compaction(i32([[0] * 2] * 2, dev), i32([0] * 6, dev), i32([0] * 6, dev), i32([0, 0], dev),
                              i32([[0] * 3] * 3, dev))
    best = paged.BeamChoice(i32([0] * 4, dev), i32([0] * 4, dev), torch.zeros(4, device=dev), i32([[0] * 4] * 2, dev),
                            i32([[0] * 4] * 2, dev), torch.zeros((2, 4), device=dev))
    return {
        "fork_block_tables": [lengths, i32([1, 1], dev), i32([18, 17], dev), tables, shares, ring, state, 16, 6, fork,
                              paged.fork_workspace(6, 2, 2, dev), None],
        "copy_blocks": [ctypes.addressof(layers), torch.tensor([cache.data_ptr()], device=dev),
                        i32([[0, 4, 16], [1, 5, 3]], dev), None],
        "compact_block_tables": [lengths, tables, shares, ring, state, 16, packed, paged.compact_workspace(6, dev), None],
        "select_beams": [torch.arange(36, device=dev).view(4, 9).to(BF16), torch.zeros(4, device=dev), 2, 4, 8, best, None],
    }, (layers, cache)


def test_host_tensors_and_junk_are_not_taken():
    args, _keep = arguments("cpu")
    for name, good in args.items():
        call = getattr(paged._calls, name)
        assert call(*good) is False
        assert call() is False and call(*good, None) is False
        for i in range(len(good)):
            for junk in (None, 3, -1, 1 << 70, "x", 1.5, (), torch.zeros(2)):
                if name == "copy_blocks" and i == 0 and isinstance(junk, int):
                    continue  # an address is the caller's word
                assert call(*good[:i], junk, *good[i + 1:]) is False, (name, i, junk)


def outputs(args, keep):
    return {"fork_block_tables": list(args["fork_block_tables"][9]) + [args["fork_block_tables"][5]],
            "copy_blocks": [keep[1]], "compact_block_tables": list(args["compact_block_tables"][6]),
            "select_beams": list(args["select_beams"][5])}


@pytest.mark.gpu
def test_taken_calls_give_the_checked_ways_results(cuda):
    got, keep_a = arguments(cuda)
    want, keep_b = arguments(cuda)
    for name in got:
        assert getattr(paged._calls, name)(*got[name]) is True, name
    a = want["fork_block_tables"]
    paged.fork_block_tables(*a[:9], out=a[9], check=True)
    a = want["compact_block_tables"]
    paged.compact_block_tables(*a[:6], out=a[6], check=True)
    paged.copy_blocks([keep_b[1]], want["copy_blocks"][2], check=True)
    a = want["select_beams"]
    paged.select_beams(*a[:4], end_token=a[4], out=a[5], check=True)
    torch.cuda.synchronize()
    for name, made in outputs(got, keep_a).items():
        for x, y in zip(made, outputs(want, keep_b)[name]):
            assert torch.equal(x, y), name


WRONG = [("fork_block_tables", i, f) for i in (0, 1, 2, 3, 4, 5, 6, 10) for f in (lambda t: t.long(), lambda t: t.cpu())]
WRONG += [("fork_block_tables", i, f) for i in (0, 1, 2, 4, 5, 6) for f in (lambda t: t[:1], lambda t: t.repeat(2)[::2])]
WRONG += [("fork_block_tables", 7, lambda v: 0), ("fork_block_tables", 8, lambda v: 5),
          ("fork_block_tables", 9, lambda o: o[:6]), ("fork_block_tables", 9, lambda o: (o[0].long(),) + tuple(o[1:])),
          ("fork_block_tables", 10, lambda t: t[:paged.fork_workspace(6, 2, 2, "cpu").numel() - 1]), ("fork_block_tables", 10, lambda t: t[1:]),
          ("fork_block_tables", 2, lambda t: -1), ("fork_block_tables", 2, lambda t: None)]
WRONG += [("compact_block_tables", i, f) for i in (0, 1, 2, 3, 4, 7) for f in (lambda t: t.long(), lambda t: t.cpu())]
WRONG += [("compact_block_tables", 5, lambda v: 0), ("compact_block_tables", 6, lambda o: o[:4]),
          ("compact_block_tables", 6, lambda o: tuple(o[:4]) + (o[4][:2],)), ("compact_block_tables", 7, lambda t: t[:9]),
          ("compact_block_tables", 7, lambda t: torch.cat([t, t]))]
WRONG += [("copy_blocks", 2, lambda t: t.long()), ("copy_blocks", 2, lambda t: t[:, :2]), ("copy_blocks", 2, lambda t: t[0]),
          ("copy_blocks", 1, lambda t: t.int()), ("copy_blocks", 3, lambda e: 0)]
WRONG += [("select_beams", 0, lambda t: t.double()), ("select_beams", 0, lambda t: t[:3]), ("select_beams", 0, lambda t: t.t()),
          ("select_beams", 0, lambda t: t[0]), ("select_beams", 1, lambda t: t.half()), ("select_beams", 1, lambda t: t[:2]),
          ("select_beams", 2, lambda v: 0), ("select_beams", 3, lambda v: 1), ("select_beams", 3, lambda v: 65),
          ("select_beams", 4, lambda v: -1), ("select_beams", 5, lambda o: o[:5]),
          ("select_beams", 5, lambda o: tuple(o[:5]) + (o[5].double(),))]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(WRONG)))
def test_wrong_arguments_come_back_and_are_named(cuda, case):
    name, i, change = WRONG[case]
    args, keep = arguments(cuda)
    good = args[name]
    bad = good[:i] + [change(good[i])] + good[i + 1:]
    before = [t.clone() for t in outputs(args, keep)[name]]
    assert getattr(paged._calls, name)(*bad) is False
    with pytest.raises((TypeError, ValueError)):
        if name == "fork_block_tables":
            paged.fork_block_tables(*bad[:9], out=bad[9], workspace=bad[10], check=False)
        elif name == "compact_block_tables":
            paged.compact_block_tables(*bad[:6], out=bad[6], workspace=bad[7], check=False)
        elif name == "select_beams":
            paged.select_beams(*bad[:4], end_token=bad[4], out=bad[5], check=False)
        elif i == 2:
            paged.copy_blocks([keep[1]], bad[2], check=False)
        else:
            raise TypeError("the wrapper makes these itself")
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, outputs(args, keep)[name]))
