"""Operators of a decode instance over its paged KV caches: block tables built on the GPU from
request lengths, keys and values written by slot, attention of drafted tokens over the cache,
and the accepted drafts kept; and, for requests with several answers, rows that share blocks,
blocks copied, the pool compacted and beam search's selection.

A received request is written into its blocks by `FusedKVCodec.decompress`; from there on a
step with drafts is

    slots, starts = tables.update(lengths + drafts, max_tokens)          # blocks for the drafts
    write_kv(key, value, cache, slots)                                   # each layer
    out = tree_attention(query, cache, tables.tables, tables.lengths, starts,
                         max_query=drafts, tree_mask=mask)               # each layer
    lengths = keep_drafts(layers, tables.tables, lengths, accepted)      # all layers at once
    tables.update(lengths, 0)                                            # blocks given back

and one of a beam search, over `SharedBlockTables`,

    best = select_beams(logits, scores, beams, 2 * beams, end_token=end)
    slots, starts = tables.fork(best.parents, 1, rows)                   # reordered, grown by a token
    copy_blocks(layers, tables.copies)                                   # partly filled blocks split

Everything is enqueued on the current stream of the tensors' device and reads lengths, tables
and slots on the GPU.  Errors found there (a block id outside the cache, too few free blocks, a
length out of range) are bits of a device word.  As in `kvserve_amd.ops`, a call synchronizes
and raises by default; `check=False` (or KVSERVE_AMD_CHECK_ERRORS=0) keeps it asynchronous,
and the bits are then OR-ed into the caller's int32 word `err`, if one is given.  While a stream
is being captured nothing is checked.
"""

from __future__ import annotations

import ctypes
import math
from typing import Iterable, NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib
from .engine import raise_device_error
from .ops import _check_default

# A call that is not checked goes through this module at once (4 us instead of 13); what it does
# not take comes back, to the checks and errors here, and so does everything where the module is
# not built.
_calls = _lib.calls()

_INT32_MAX = 2**31 - 1  # sizes are 32-bit words in the library's structs
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}


# ------------------------------------------------------------------ shared checks
def _unchecked(check: Optional[bool]) -> bool:
    """Whether the call may go through `_calls`."""
    if check or (check is None and _check_default()):
        return False
    if isinstance(_calls, _lib._NoCalls):
        _calls.tell()
        return False
    return True


def _tensor(t, name: str, dtype: torch.dtype, shape, device=None) -> int:
    """Address of a contiguous CUDA tensor of this type and shape (None: any size)."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{name} must be a {dtype} tensor")
    if t.dim() != len(shape) or any(w is not None and n != w for n, w in zip(t.shape, shape)):
        raise ValueError(f"{name} must have shape {tuple('any' if w is None else w for w in shape)}, "
                         f"not {tuple(t.shape)}")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} must be a CUDA tensor on {device or 'the GPU'}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _cache_struct(cache: torch.Tensor) -> _lib.Cache:
    """C description of a cache [2, P, S, H, D] or [P, 2, S, H, D] (the first is tested first)."""
    if not isinstance(cache, torch.Tensor) or cache.element_size() != 2 or cache.dtype.is_complex:
        raise TypeError("the KV cache must be a 16-bit tensor")
    if cache.dim() != 5 or 2 not in cache.shape[:2]:
        raise ValueError(f"Unsupported KV layout shape: {tuple(cache.shape)}")
    if max(cache.shape) > _INT32_MAX:
        raise ValueError(f"the KV cache's sizes must be in 31 bits, not {tuple(cache.shape)}")
    if not cache.is_cuda or not cache.is_contiguous() or not cache.numel():
        raise ValueError("the KV cache must be a contiguous, non-empty CUDA tensor")
    S, H, D = cache.shape[2:]
    if cache.shape[0] == 2:
        return _lib.Cache(cache.data_ptr(), cache.shape[1] * S * H * D, S * H * D, cache.shape[1], S, H, D)
    return _lib.Cache(cache.data_ptr(), S * H * D, 2 * S * H * D, cache.shape[0], S, H, D)


class _Call:
    """The device, stream and error word of one call."""

    def __init__(self, device: torch.device, check: Optional[bool], err: Optional[torch.Tensor]):
        self.device = device
        self.check = (_check_default() if check is None else check) and not torch.cuda.is_current_stream_capturing()
        if err is not None:
            _tensor(err, "err", torch.int32, (1,), device)
        elif self.check:
            err = torch.zeros(1, dtype=torch.int32, device=device)
        self.err = err
        self.err_ptr = None if err is None else err.data_ptr()

    def run(self, name: str, *args) -> None:
        fn = getattr(_lib.load(), name)
        if torch.cuda.current_device() == self.device.index:
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
        else:
            with torch.cuda.device(self.device):
                rc = fn(*args, torch.cuda.current_stream().cuda_stream)
        _lib.check(rc, name)
        if self.check:
            raise_device_error(int(self.err.item()))


# ------------------------------------------------------------------ block tables
class TablesUpdate(NamedTuple):
    """What `build_block_tables` gives back."""

    tables: torch.Tensor   # int32 [R, columns]
    lengths: torch.Tensor  # int32 [R], the old length where a request was refused
    state: torch.Tensor    # int32 [2]: head and count of the free ring
    slots: torch.Tensor    # int64 [max_tokens], -1 where there is none
    starts: torch.Tensor   # int32 [R + 1]: each request's first new token in `slots`


def build_block_tables(lengths: torch.Tensor, new_lengths: torch.Tensor, tables: torch.Tensor, free: torch.Tensor,
                       state: torch.Tensor, block_size: int, max_tokens: int, *, out: Optional[Sequence] = None,
                       ticket: Optional[torch.Tensor] = None, check: Optional[bool] = None,
                       err: Optional[torch.Tensor] = None) -> TablesUpdate:
    """Block tables, free blocks and slot map for requests that go from `lengths` to
    `new_lengths` tokens (int32 [R]); a request of n tokens holds ceil(n / block_size) blocks.

    `tables` int32 [R, columns] holds the present blocks, `free` int32 [blocks] a ring of the
    free ones beginning at state[0], state[1] of them.  A growing request takes blocks at the
    ring's head, a shrinking one's go behind its last (`free` is changed in place; they can be
    taken by the next call); the ring needs room for every block of the pool.  Blocks given back
    past its room are dropped, and the call raises ValueError where it checks.  Requests are served in order; one whose blocks, with those asked
    for before it, exceed the free ones is refused: it keeps its length, its tokens get slot -1,
    and the call raises RuntimeError where it checks.  More than `max_tokens` new tokens raise
    ValueError there; tables and lengths have then moved on, and the slots past `max_tokens` are
    lost, so the bound has to hold.

    `out`: the tensors of a `TablesUpdate` to write into.  Tables may be `tables` itself;
    lengths and state may both be `lengths` and `state` themselves, with `ticket`, an int32 word
    of zero."""
    if type(out) is tuple:
        out = TablesUpdate(*out)
    if type(out) is TablesUpdate and _unchecked(check) and _calls.build_block_tables(
            lengths, new_lengths, tables, free, state, block_size, max_tokens, out, ticket, err):
        return out
    if type(block_size) is not int or not 1 <= block_size <= _INT32_MAX or type(max_tokens) is not int \
            or not 0 <= max_tokens <= _INT32_MAX:
        raise ValueError("block_size must be a positive integer and max_tokens a nonnegative one, in 31 bits")
    now = _tensor(lengths, "lengths", torch.int32, (None,))
    dev, R = lengths.device, lengths.numel()
    new = _tensor(new_lengths, "new_lengths", torch.int32, (R,), dev)
    tab = _tensor(tables, "tables", torch.int32, (R, None), dev)
    ring = _tensor(free, "free", torch.int32, (None,), dev)
    st = _tensor(state, "state", torch.int32, (2,), dev)
    C = tables.shape[1]
    if out is None:
        made = torch.empty(2 * R + 3, dtype=torch.int32, device=dev)
        out = TablesUpdate(torch.empty_like(tables), made[:R], made[R:R + 2],
                           torch.empty(max_tokens, dtype=torch.int64, device=dev), made[R + 2:])
    else:
        out = TablesUpdate(*out)
        for name, t, like in (("out.tables", out.tables, (R, C)), ("out.lengths", out.lengths, (R,)),
                              ("out.state", out.state, (2,)), ("out.starts", out.starts, (R + 1,))):
            _tensor(t, name, torch.int32, like, dev)
        _tensor(out.slots, "out.slots", torch.int64, (max_tokens,), dev)
    if (out.lengths.data_ptr() == now and R > 0) != (out.state.data_ptr() == st and R > 0):
        raise ValueError("lengths and state are written over together or not at all")
    if R and out.lengths.data_ptr() == now and ticket is None:
        raise ValueError("lengths written over need a ticket word")
    if R and new == out.lengths.data_ptr():
        raise ValueError("out.lengths must not be new_lengths")
    if ticket is not None:
        _tensor(ticket, "ticket", torch.int32, (1,), dev)
    call = _Call(dev, check, err)
    if R == 0:
        out.state.copy_(state)
        out.slots.fill_(-1)
        out.starts.zero_()
        return out
    args = _lib.TablesArgs(now, new, tab, ring, st, out.tables.data_ptr(), out.lengths.data_ptr(),
                           out.state.data_ptr(), out.slots.data_ptr(), out.starts.data_ptr(),
                           None if ticket is None else ticket.data_ptr(), call.err_ptr, R, C, free.numel(), block_size,
                           max_tokens, 0)
    call.run("kvmi_build_tables", args)
    return out


class BlockTables:
    """The block tables of a decode instance's requests and the free blocks of its caches, kept
    on the GPU.  All layers share them.

      tables   int32 [requests, columns]: each request's blocks, -1 behind them
      lengths  int32 [requests]: tokens each request holds (0: none, no blocks)

    `free_blocks`: the blocks it may hand out (default: all `num_blocks`).  Rewritten in place by
    `update`, so the tensors can be captured in a graph once and for all."""

    def __init__(self, num_blocks: int, block_size: int, requests: int, columns: int, device="cuda",
                 free_blocks: Optional[Iterable[int]] = None):
        for name, v in (("num_blocks", num_blocks), ("block_size", block_size), ("requests", requests),
                        ("columns", columns)):
            if type(v) is not int or not 1 <= v <= _INT32_MAX:
                raise ValueError(f"{name} must be a positive integer in 31 bits")
        ids = list(range(num_blocks)) if free_blocks is None else [int(b) for b in free_blocks]
        if len(set(ids)) != len(ids) or (ids and (min(ids) < 0 or max(ids) >= num_blocks)):
            raise ValueError("free_blocks must be distinct block ids of the cache")
        self.num_blocks, self.block_size = num_blocks, block_size
        i32 = dict(dtype=torch.int32, device=device)
        self.free = torch.tensor(ids + [-1] * (num_blocks - len(ids)), **i32)
        self.state = torch.tensor([0, len(ids)], **i32)
        self.tables = torch.full((requests, columns), -1, **i32)
        self.lengths = torch.zeros(requests, **i32)
        self._ticket = torch.zeros(1, **i32)

    def update(self, new_lengths: torch.Tensor, max_tokens: int, *, slots: Optional[torch.Tensor] = None,
               starts: Optional[torch.Tensor] = None, check: Optional[bool] = None,
               err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Bring every request to `new_lengths` (int32 [requests], on the GPU): blocks are taken
        and given back, `tables` and `lengths` rewritten.  Returns (slots, starts) of the new
        tokens, at most `max_tokens`; see `build_block_tables`."""
        dev = self.tables.device
        if slots is None:
            slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
        if starts is None:
            starts = torch.empty(self.lengths.numel() + 1, dtype=torch.int32, device=dev)
        build_block_tables(self.lengths, new_lengths, self.tables, self.free, self.state, self.block_size, max_tokens,
                           out=(self.tables, self.lengths, self.state, slots, starts), ticket=self._ticket,
                           check=check, err=err)
        return slots, starts


# ------------------------------------------------------------------ slot writes
def write_kv(key: torch.Tensor, value: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, *,
             check: Optional[bool] = None, err: Optional[torch.Tensor] = None) -> None:
    """Write rows of new keys and values ([tokens, H, D] of the cache's type; any strides with
    adjacent channels, so slices of one projection will do) into the paged cache: token i's to
    block slots[i] // S, place slots[i] % S.  `slots` is int64 [tokens]; -1 skips a token.  No
    two tokens may share a slot."""
    if _unchecked(check) and _calls.write_kv(key, value, cache, slots, err):
        return
    c = _cache_struct(cache)
    for name, t in (("key", key), ("value", value)):
        if not isinstance(t, torch.Tensor) or t.dtype != cache.dtype:
            raise TypeError(f"{name} must be a {cache.dtype} tensor, as the cache is")
        if t.dim() != 3 or t.shape[1] != c.num_heads or t.shape[2] != c.head_dim or t.shape[0] != key.shape[0]:
            raise ValueError(f"{name} must have shape (tokens, {c.num_heads}, {c.head_dim}), not {tuple(t.shape)}")
        if t.device != cache.device or (t.stride(2) != 1 and c.head_dim > 1):
            raise ValueError(f"{name} must be on {cache.device} with adjacent channels")
    n = key.shape[0]
    where = _tensor(slots, "slots", torch.int64, (n,), cache.device)
    call = _Call(cache.device, check, err)
    if n:
        call.run("kvmi_write_kv", c, key.data_ptr(), value.data_ptr(), key.stride(0), key.stride(1), value.stride(0),
                 value.stride(1), where, n, call.err_ptr)


# ------------------------------------------------------------------ attention
def tree_mask(parents: Sequence[int], words: Optional[int] = None, device="cuda") -> torch.Tensor:
    """Visibility words of one drafted tree for `tree_attention`: int64 [nodes, words], bit j of
    row i set where draft i sees draft j, i.e. j is i itself or one of its ancestors.
    parents[i] < i is the draft that i follows, or -1."""
    nodes = len(parents)
    least = max(1, (nodes + 63) // 64)
    words = least if words is None else words
    if words < least:
        raise ValueError(f"{nodes} drafts need {least} mask words")
    bits = []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError("a draft's parent comes before it, or is -1")
        bits.append((bits[p] if p >= 0 else 0) | (1 << i))
    rows = [[(b >> (64 * w)) & ((1 << 64) - 1) for w in range(words)] for b in bits]
    rows = [[v - (1 << 64) if v >> 63 else v for v in row] for row in rows]
    return torch.tensor(rows, dtype=torch.int64, device=device).reshape(nodes, words)


def _attention_args(query, cache, tables, lengths, starts, max_query, max_length, mask, scale, out, lse):
    c = _cache_struct(cache)
    dev = cache.device
    if cache.dtype not in _DTYPES:
        raise TypeError("attention takes a bfloat16 or float16 cache")
    if c.head_dim % 8 or c.head_dim > 256:
        raise ValueError("attention takes head sizes that are multiples of 8 up to 256")
    if not isinstance(query, torch.Tensor) or query.dtype != cache.dtype:
        raise TypeError(f"query must be a {cache.dtype} tensor, as the cache is")
    if query.dim() != 3 or query.shape[2] != c.head_dim or not query.shape[1] or query.shape[1] % c.num_heads:
        raise ValueError(f"query must have shape (tokens, a multiple of {c.num_heads}, {c.head_dim}), "
                         f"not {tuple(query.shape)}")
    if query.device != dev:
        raise ValueError(f"query must be on {dev}")
    if query.stride(2) != 1 or query.stride(0) % 8 or query.stride(1) % 8 or query.data_ptr() % 16:
        query = query.clone(memory_format=torch.contiguous_format)  # the kernels read 16-byte rows
    R = lengths.numel() if isinstance(lengths, torch.Tensor) else 0
    n, heads = query.shape[0], query.shape[1]
    ptrs = (_tensor(tables, "tables", torch.int32, (R, None), dev), _tensor(lengths, "lengths", torch.int32, (R,), dev),
            _tensor(starts, "starts", torch.int32, (R + 1,), dev))
    if max_length is None:
        max_length = tables.shape[1] * c.block_size
    if type(max_length) is int:
        max_length = min(max_length, _INT32_MAX)
    for name, v in (("max_query", max_query), ("max_length", max_length)):
        if type(v) is not int or v < 0:
            raise ValueError(f"{name} must be a nonnegative integer")
    words = 0
    if mask is not None:
        _tensor(mask, "tree_mask", torch.int64, (n, None), dev)
        words = mask.shape[1]
        if words * 64 < min(max_query, n):
            raise ValueError("tree_mask has fewer bits than max_query")
    scale = 1.0 / math.sqrt(c.head_dim) if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError("scale must be positive and finite")
    _tensor(out, "out", cache.dtype, (n, heads, c.head_dim), dev)
    args = _lib.AttentionArgs(c, query.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), *ptrs,
                              None if mask is None else mask.data_ptr(), None, 0, None, query.stride(0),
                              query.stride(1), scale, _DTYPES[cache.dtype], R, tables.shape[1], n, heads,
                              min(max_query, n), max_length, words, 0)
    return args, query


def tree_attention(query: torch.Tensor, cache: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
                   starts: torch.Tensor, *, max_query: int, max_length: Optional[int] = None,
                   tree_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, return_lse: bool = False, check: Optional[bool] = None,
                   err: Optional[torch.Tensor] = None):
    """Attention of each request's last tokens over its paged cache.

    query      [tokens, query heads, D], bfloat16 or float16 as the cache; query head h reads KV
               head h // (query heads / KV heads)
    cache      [2, P, S, H, D] or [P, 2, S, H, D]; the queries' own keys and values are in it
    tables     int32 [R, columns] block tables of at most 65535 requests; lengths int32 [R] tokens in
               the cache, queries included
    starts     int32 [R + 1]: request r's queries are rows starts[r] .. starts[r + 1] - 1
    max_query  the most queries of a request; max_length the longest length (default: what the
               tables hold; a tighter bound gives better launches)
    tree_mask  int64 [tokens, words]: bit j % 64 of word j // 64 says that a query sees draft j of
               its request (`tree_mask()` makes them).  Without it the queries are a causal chain:
               one token, a chunk or a whole prompt.
    Every query sees all tokens before its request's first query.  A query that sees nothing
    gives zeros.  Rows of no request are left as they are in `out`.  No gradient flows back.

    The requests with the most queries choose the kernel for all: a prompt's chunk beside single
    tokens over long contexts is much faster as a call for the chunk and one for the tokens.

    Returns `out`, or (out, lse) with the fp32 natural log of each row's sum [tokens, query heads].
    """
    if not isinstance(query, torch.Tensor) or not query.is_cuda:
        raise TypeError("query must be a CUDA tensor")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if not return_lse and _unchecked(check) and _calls.tree_attention(
            query, cache, tables, lengths, starts, max_query, max_length, tree_mask, scale, out, err):
        return out
    lse = torch.full(query.shape[:2], -math.inf, dtype=torch.float32, device=query.device) if return_lse else None
    if isinstance(out, torch.Tensor) and out.data_ptr() % 16 and out.is_contiguous():
        # the kernels write 8 and 16 bytes at a time
        whole = tree_attention(query, cache, tables, lengths, starts, max_query=max_query, max_length=max_length,
                               tree_mask=tree_mask, scale=scale, out=out.clone(), return_lse=return_lse, check=check,
                               err=err)
        out.copy_(whole[0] if return_lse else whole)
        return (out, whole[1]) if return_lse else out
    args, query = _attention_args(query, cache, tables, lengths, starts, max_query, max_length, tree_mask, scale, out,
                                  lse)
    call = _Call(cache.device, check, err)
    args.err = call.err_ptr
    size = _lib.load().kvmi_attention_workspace_bytes(args)
    if size < 0:
        raise ValueError("kvmi_tree_attention: invalid arguments (KVMI_EINVAL)")
    if size:
        space = torch.empty(size, dtype=torch.uint8, device=cache.device)
        args.workspace, args.workspace_bytes = space.data_ptr(), size
    call.run("kvmi_tree_attention", args)
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------ kept drafts
class LayerCaches:
    """The caches of a model's layers (same type, shape and device, each a memory of its own: layers
    that share one are given once), with their addresses on the GPU: made once, for `keep_drafts`."""

    def __init__(self, caches: Sequence[torch.Tensor]):
        self.caches = list(caches)
        if not self.caches:
            raise ValueError("at least one layer's cache is needed")
        first = self.caches[0]
        self.struct = _cache_struct(first)
        for c in self.caches:
            _cache_struct(c)
            if c.shape != first.shape or c.dtype != first.dtype or c.device != first.device:
                raise ValueError("the layers' caches must have one type, shape and device")
        bases = [c.data_ptr() for c in self.caches]
        # two layers in one memory would move the same rows twice, each in the other's way
        ordered, size = sorted(bases), first.numel() * first.element_size()
        if any(b - a < size for a, b in zip(ordered, ordered[1:])):
            raise ValueError("the layers' caches must not share memory")
        either = 0
        for b in bases:
            either |= b
        self.struct.base = either
        self.device = first.device
        self.bases = torch.tensor(bases, dtype=torch.int64, device=self.device)
        self._struct_at = ctypes.addressof(self.struct)


def keep_drafts(caches, tables: torch.Tensor, lengths: torch.Tensor, accepted: torch.Tensor, *,
                out: Optional[torch.Tensor] = None, check: Optional[bool] = None,
                err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keep the accepted path of each request's drafts: in every layer (`LayerCaches`, or a
    sequence of caches) row lengths[r] + accepted[r, i] moves to lengths[r] + i.

    lengths   int32 [R]: tokens before the drafts
    accepted  int32 [R, width <= 1024]: numbers of the accepted drafts, strictly increasing, -1
              behind the last
    Returns the lengths with the kept drafts, int32 [R] (`out`, not `lengths` itself).  A request
    whose path is not increasing or leaves its blocks is left as it is."""
    layers = caches if isinstance(caches, LayerCaches) else LayerCaches(caches)
    if out is not None and _unchecked(check) and _calls.keep_drafts(
            layers._struct_at, layers.bases, tables, lengths, accepted, out, err):
        return out
    R = lengths.numel() if isinstance(lengths, torch.Tensor) else 0
    now = _tensor(lengths, "lengths", torch.int32, (R,), layers.device)
    tab = _tensor(tables, "tables", torch.int32, (R, None), layers.device)
    path = _tensor(accepted, "accepted", torch.int32, (R, None), layers.device)
    if accepted.shape[1] > 1024:
        raise ValueError("accepted holds at most 1024 drafts a request")
    if out is None:
        out = torch.empty_like(lengths)
    res = _tensor(out, "out", torch.int32, (R,), layers.device)
    if R and res == now:
        raise ValueError("out must not be lengths")
    call = _Call(layers.device, check, err)
    if R:
        call.run("kvmi_keep_drafts", layers.struct, layers.bases.data_ptr(), len(layers.caches), tab, tables.shape[1],
                 now, path, R, accepted.shape[1], res, call.err_ptr)
    return out


# ------------------------------------------------------------------ rows that share blocks
class ForkUpdate(NamedTuple):
    """What `fork_block_tables` gives back."""

    tables: torch.Tensor   # int32 [R, columns]
    lengths: torch.Tensor  # int32 [R]
    shares: torch.Tensor   # int32 [blocks]
    state: torch.Tensor    # int32 [2]: head and count of the free ring
    slots: torch.Tensor    # int64 [max_tokens], -1 where there is none
    starts: torch.Tensor   # int32 [R + 1]: each row's first new token in `slots`
    copies: torch.Tensor   # int32 [R, 3]: blocks to be copied, for `copy_blocks`


def _words(size: int, device) -> torch.Tensor:
    if size < 0:
        raise ValueError("the sizes of a pool and its rows must be positive, and the pool's at most 2**24 blocks")
    return torch.zeros((size + 3) // 4, dtype=torch.int32, device=device)


def _sizes(**sizes) -> None:
    for name, v in sizes.items():
        if type(v) is not int or not 1 <= v <= _INT32_MAX:
            raise ValueError(f"{name} must be a positive integer in 31 bits")


def fork_workspace(blocks: int, rows: int, columns: int, device="cuda") -> torch.Tensor:
    """Workspace of `fork_block_tables` for a pool of `blocks` and `rows` rows of `columns` entries.
    A call leaves it ready for the next one of the same sizes; no two calls may use it at a time, nor
    two captured graphs that may run at a time."""
    _sizes(blocks=blocks, rows=rows, columns=columns)
    return _words(_lib.load().kvmi_fork_workspace_bytes(blocks, rows, columns), device)


def compact_workspace(blocks: int, device="cuda") -> torch.Tensor:
    """Workspace of `compact_block_tables` for a pool of `blocks`; as that of `fork_workspace`."""
    _sizes(blocks=blocks)
    return _words(_lib.load().kvmi_compact_workspace_bytes(blocks), device)


def _space(workspace: Optional[torch.Tensor], size: int, device) -> torch.Tensor:
    if size < 0:
        raise ValueError("the sizes of a pool and its rows must be positive, and the pool's at most 2**24 blocks")
    if workspace is None:
        return _words(size, device)
    _tensor(workspace, "workspace", torch.int32, (None,), device)
    if workspace.numel() != (size + 3) // 4 or workspace.data_ptr() % 16:
        raise ValueError(f"workspace must be one made for these sizes: {(size + 3) // 4} words, 16-byte aligned")
    return workspace


def _in_place(pairs) -> bool:
    """Whether the outputs are the inputs themselves: all of them, or none."""
    same = [a.data_ptr() == b.data_ptr() and a.numel() > 0 for a, b in pairs if a.numel()]
    if any(same) and not all(same):
        raise ValueError("the outputs are the inputs themselves, all of them or none")
    return any(same)


def fork_block_tables(lengths: torch.Tensor, parents: Optional[torch.Tensor], new_lengths, tables: torch.Tensor,
                      shares: torch.Tensor, free: torch.Tensor, state: torch.Tensor, block_size: int, max_tokens: int,
                      *, out: Optional[Sequence] = None, workspace: Optional[torch.Tensor] = None,
                      check: Optional[bool] = None, err: Optional[torch.Tensor] = None) -> ForkUpdate:
    """Block tables whose rows may share blocks: row r becomes the first tokens of row parents[r]
    and grows from there, all rows at once.  This forks a request (several rows of one parent),
    reorders beams, takes over a prefix, lets rows join and end, and frees what no row holds any more.

    lengths      int32 [R <= 4096]: tokens of each row, in ceil(n / block_size) blocks
    parents      int32 [R]: the row that each goes on from, -1 for one that starts empty; None:
                 every row itself
    new_lengths  int32 [R]: tokens after the call; min(new, the parent's) of them are the
                 parent's.  Or an integer: that many more than the parent has, and no tokens where there
                 is no parent
    tables       int32 [R, columns]; rows that share a block have it in the same column, and a row's last
                 block is its own while it is partly filled (every call leaves them so)
    shares       int32 [blocks <= 2**24]: how many rows hold a block besides the first
    free, state  the ring of free blocks, int32 [blocks], and its head and count, as in
                 `build_block_tables`; `free` is changed in place

    Whole blocks of kept tokens are shared.  A partly kept one goes on with a single row, where no
    other holds it; the other rows take a block for these tokens, and `copies` lists (from, to,
    tokens): `copy_blocks` has to run on them before the new tokens are written, and before the next
    call, which may hand out the blocks copied from.  Blocks that no row holds any more go behind the
    ring's last free one, in the order of their ids.

    All or nothing: with too few free blocks the call raises RuntimeError where it checks, with more
    than `max_tokens` new tokens or a length or parent out of range ValueError; rows and ring are
    then as they were, slots and copies -1.

    `out`: the tensors of a `ForkUpdate` to write into; tables, lengths, shares and state may be the
    inputs themselves, all four.  `workspace`: of `fork_workspace` (made here if not given)."""
    if type(out) is tuple:
        out = ForkUpdate(*out)
    if type(out) is ForkUpdate and workspace is not None and _unchecked(check) and _calls.fork_block_tables(
            lengths, parents, new_lengths, tables, shares, free, state, block_size, max_tokens, out, workspace, err):
        return out
    _sizes(block_size=block_size)
    if type(max_tokens) is not int or not 0 <= max_tokens <= _INT32_MAX:
        raise ValueError("max_tokens must be a nonnegative integer in 31 bits")
    now = _tensor(lengths, "lengths", torch.int32, (None,))
    dev, R = lengths.device, lengths.numel()
    from_rows = None if parents is None else _tensor(parents, "parents", torch.int32, (R,), dev)
    new, grow = None, 0
    if type(new_lengths) is int:
        grow = new_lengths
        if not 0 <= grow <= _INT32_MAX:
            raise ValueError("new_lengths must be a tensor, or a nonnegative integer in 31 bits")
    else:
        new = _tensor(new_lengths, "new_lengths", torch.int32, (R,), dev)
    tab = _tensor(tables, "tables", torch.int32, (R, None), dev)
    counts = _tensor(shares, "shares", torch.int32, (None,), dev)
    N, C = shares.numel(), tables.shape[1]
    ring = _tensor(free, "free", torch.int32, (N,), dev)
    st = _tensor(state, "state", torch.int32, (2,), dev)
    if R > 4096:
        raise ValueError("fork_block_tables takes up to 4096 rows")
    if out is None:
        made = torch.empty(5 * R + 3 + N, dtype=torch.int32, device=dev)
        out = ForkUpdate(torch.empty_like(tables), made[:R], made[5 * R + 3:], made[R:R + 2],
                         torch.empty(max_tokens, dtype=torch.int64, device=dev), made[R + 2:2 * R + 3],
                         made[2 * R + 3:5 * R + 3].view(R, 3))
    else:
        out = ForkUpdate(*out)
        for name, t, like in (("out.tables", out.tables, (R, C)), ("out.lengths", out.lengths, (R,)),
                              ("out.shares", out.shares, (N,)), ("out.state", out.state, (2,)),
                              ("out.starts", out.starts, (R + 1,)), ("out.copies", out.copies, (R, 3))):
            _tensor(t, name, torch.int32, like, dev)
        _tensor(out.slots, "out.slots", torch.int64, (max_tokens,), dev)
    in_place = _in_place(((out.tables, tables), (out.lengths, lengths), (out.shares, shares), (out.state, state)))
    if R and out.lengths.data_ptr() in (new, from_rows):
        raise ValueError("out.lengths must be neither new_lengths nor parents")
    call = _Call(dev, check, err)
    if R == 0:
        if not in_place:
            out.shares.copy_(shares)
            out.state.copy_(state)
        out.slots.fill_(-1)
        out.starts.zero_()
        return out
    if N == 0 or C == 0:
        raise ValueError("the pool and the rows of the tables must not be empty")
    space = _space(workspace, _lib.load().kvmi_fork_workspace_bytes(N, R, C), dev)
    args = _lib.ForkArgs(now, from_rows, new, tab, counts, ring, st, out.tables.data_ptr(), out.lengths.data_ptr(),
                         out.shares.data_ptr(), out.state.data_ptr(), out.slots.data_ptr(), out.starts.data_ptr(),
                         out.copies.data_ptr(), space.data_ptr(), space.numel() * 4, call.err_ptr, R, C, N, block_size,
                         max_tokens, grow)
    call.run("kvmi_fork_tables", args)
    return out


def copy_blocks(caches, copies: torch.Tensor, *, check: Optional[bool] = None,
                err: Optional[torch.Tensor] = None) -> None:
    """Copy blocks in every layer (`LayerCaches`, or a sequence of caches): for each row (from, to,
    tokens) of `copies`, int32 [n, 3], the first `tokens` tokens of block `from`, keys and values, go to
    block `to`.  Rows with a negative `from` are skipped.  No block may be written by two rows, nor
    read by one and written by another.  A row with a block outside the cache, or more tokens than a
    block has, copies nothing."""
    layers = caches if isinstance(caches, LayerCaches) else LayerCaches(caches)
    if _unchecked(check) and _calls.copy_blocks(layers._struct_at, layers.bases, copies, err):
        return
    rows = _tensor(copies, "copies", torch.int32, (None, 3), layers.device)
    call = _Call(layers.device, check, err)
    if copies.shape[0]:
        call.run("kvmi_copy_blocks", layers.struct, layers.bases.data_ptr(), len(layers.caches), rows,
                 copies.shape[0], call.err_ptr)


class Compaction(NamedTuple):
    """What `compact_block_tables` gives back."""

    tables: torch.Tensor  # int32 [R, columns]
    shares: torch.Tensor  # int32 [blocks]
    free: torch.Tensor    # int32 [blocks]: the ring, from 0 on, -1 behind its last
    state: torch.Tensor   # int32 [2]: 0 and the ring's count
    copies: torch.Tensor  # int32 [blocks // 2, 3]: the moves, for `copy_blocks`


def compact_block_tables(lengths: torch.Tensor, tables: torch.Tensor, shares: torch.Tensor, free: torch.Tensor,
                         state: torch.Tensor, block_size: int, *, out: Optional[Sequence] = None,
                         workspace: Optional[torch.Tensor] = None, check: Optional[bool] = None,
                         err: Optional[torch.Tensor] = None) -> Compaction:
    """Move the blocks that rows hold to the front of the pool.  Arguments as in
    `fork_block_tables`.  The pool is what the rows hold and what the ring has free (a block in
    neither stays out of it); of n held blocks those among the pool's n lowest ids stay, and the others
    move, in order, to the free ids among these n.  Tables and shares come back under the new names, the
    ring with the rest of the pool in order, and `copies` with the moves: `copy_blocks` has to run on
    them before the blocks are read or handed out.

    `out`: the tensors of a `Compaction` to write into; tables, shares, free and state may be the
    inputs themselves, all four.  `workspace`: of `compact_workspace` (made here if not given)."""
    if type(out) is tuple:
        out = Compaction(*out)
    if type(out) is Compaction and workspace is not None and _unchecked(check) and _calls.compact_block_tables(
            lengths, tables, shares, free, state, block_size, out, workspace, err):
        return out
    _sizes(block_size=block_size)
    now = _tensor(lengths, "lengths", torch.int32, (None,))
    dev, R = lengths.device, lengths.numel()
    tab = _tensor(tables, "tables", torch.int32, (R, None), dev)
    counts = _tensor(shares, "shares", torch.int32, (None,), dev)
    N, C = shares.numel(), tables.shape[1]
    ring = _tensor(free, "free", torch.int32, (N,), dev)
    st = _tensor(state, "state", torch.int32, (2,), dev)
    if out is None:
        out = Compaction(torch.empty_like(tables), torch.empty_like(shares), torch.empty_like(free),
                         torch.empty_like(state), torch.empty((N // 2, 3), dtype=torch.int32, device=dev))
    else:
        out = Compaction(*out)
        for name, t, like in (("out.tables", out.tables, (R, C)), ("out.shares", out.shares, (N,)),
                              ("out.free", out.free, (N,)), ("out.state", out.state, (2,)),
                              ("out.copies", out.copies, (N // 2, 3))):
            _tensor(t, name, torch.int32, like, dev)
    _in_place(((out.tables, tables), (out.shares, shares), (out.free, free), (out.state, state)))
    if N == 0 or C == 0:
        raise ValueError("the pool and the rows of the tables must not be empty")
    space = _space(workspace, _lib.load().kvmi_compact_workspace_bytes(N), dev)
    call = _Call(dev, check, err)
    args = _lib.CompactArgs(now, tab, counts, ring, st, out.tables.data_ptr(), out.shares.data_ptr(),
                            out.free.data_ptr(), out.state.data_ptr(), out.copies.data_ptr(), space.data_ptr(),
                            space.numel() * 4, call.err_ptr, R, C, N, block_size)
    call.run("kvmi_compact_tables", args)
    return out


class SharedBlockTables(BlockTables):
    """`BlockTables` whose rows may share blocks: up to 4096 rows, several of which may belong to one
    request.

      shares  int32 [num_blocks]: how many rows hold a block besides the first
      copies  int32 [requests, 3]: the blocks that the last `fork` or `update` split; `copy_blocks` on
              them comes before the new tokens are written, and before the next call of these or `compact`

    Rewritten in place like the others."""

    def __init__(self, num_blocks: int, block_size: int, requests: int, columns: int, device="cuda",
                 free_blocks: Optional[Iterable[int]] = None):
        super().__init__(num_blocks, block_size, requests, columns, device, free_blocks)
        if requests > 4096:
            raise ValueError("SharedBlockTables takes up to 4096 rows")
        i32 = dict(dtype=torch.int32, device=self.tables.device)
        self.shares = torch.zeros(num_blocks, **i32)
        self.copies = torch.full((requests, 3), -1, **i32)
        self._moves = torch.full((num_blocks // 2, 3), -1, **i32)
        self._fork_space = fork_workspace(num_blocks, requests, columns, self.tables.device)
        self._compact_space = compact_workspace(num_blocks, self.tables.device)

    def fork(self, parents: Optional[torch.Tensor], new_lengths, max_tokens: int, *,
             slots: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
             check: Optional[bool] = None, err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Row r becomes the first tokens of row parents[r] (int32 [requests]; -1: it starts empty)
        and grows to new_lengths[r] tokens, or, where that is an integer, by so many.  Returns (slots,
        starts) of the new tokens, at most `max_tokens`, and leaves in `copies` what `copy_blocks` has
        to copy before they are written; see `fork_block_tables`."""
        dev = self.tables.device
        if slots is None:
            slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
        if starts is None:
            starts = torch.empty(self.lengths.numel() + 1, dtype=torch.int32, device=dev)
        fork_block_tables(self.lengths, parents, new_lengths, self.tables, self.shares, self.free, self.state,
                          self.block_size, max_tokens, out=(self.tables, self.lengths, self.shares, self.state, slots,
                                                            starts, self.copies),
                          workspace=self._fork_space, check=check, err=err)
        return slots, starts

    def update(self, new_lengths: torch.Tensor, max_tokens: int, *, slots: Optional[torch.Tensor] = None,
               starts: Optional[torch.Tensor] = None, check: Optional[bool] = None,
               err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """`fork` with every row as its own parent.  A row that shrinks into a block that others
        hold gets one of its own (`copies`)."""
        return self.fork(None, new_lengths, max_tokens, slots=slots, starts=starts, check=check, err=err)

    def compact(self, *, check: Optional[bool] = None, err: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Bring the held blocks to the front of the pool; returns the moves, int32
        [num_blocks // 2, 3], on which `copy_blocks` has to run next (rewritten by the next call).  See
        `compact_block_tables`."""
        compact_block_tables(self.lengths, self.tables, self.shares, self.free, self.state, self.block_size,
                             out=(self.tables, self.shares, self.free, self.state, self._moves),
                             workspace=self._compact_space, check=check, err=err)
        return self._moves


# ------------------------------------------------------------------ beam search's selection
_LOGITS = {**_DTYPES, torch.float32: _lib.DTYPE_FP32}


class BeamChoice(NamedTuple):
    """What `select_beams` gives back."""

    parents: torch.Tensor      # int32 [requests * beams]: the row that each beam goes on from, -1: none
    tokens: torch.Tensor       # int32 [requests * beams]
    scores: torch.Tensor       # float32 [requests * beams]
    all_parents: torch.Tensor  # int32 [requests, count]: the candidates, best first
    all_tokens: torch.Tensor   # int32 [requests, count]
    all_scores: torch.Tensor   # float32 [requests, count]


def select_beams(logits: torch.Tensor, scores: torch.Tensor, beams: int, count: Optional[int] = None, *,
                 end_token: Optional[int] = None, out: Optional[Sequence] = None, check: Optional[bool] = None,
                 err: Optional[torch.Tensor] = None) -> BeamChoice:
    """Beam search's step over the vocabulary: of each request's candidates (beam, token), with the value
    scores[beam] + log_softmax(logits[beam])[token], the `count` best, and of these the `beams` best
    that do not end.

    logits     [requests * beams, vocabulary], bfloat16, float16 or float32, a request's beams one
               after the other; any row stride, tokens adjacent
    scores     float32 [requests * beams]: sums of log-probabilities so far; -inf for a beam that is not
               in use (its logits do not matter)
    count      beams <= count <= 64 candidates a request; default: beams, or with an end token twice that,
               at most 64 (so that with more than 32 beams fewer than `beams` may go on: 64 less those
               that end)
    end_token  candidates with this token are listed, but do not go on; where several tokens end an
               answer, choose those that go on from the `all_...` outputs

    Values are in 64 bits until their last rounding; among equal ones the lower beam comes first, then
    the larger logit, then the lower token (a row's sum is right to 1e-10 of it: beams whose values are closer
    than that may stand in either order, unless their logits are the same).  A value of -inf is no
    candidate: behind the last stand parent and token -1 and score -inf.  So `parents` is what
    `fork_block_tables` takes: a row without one gives its blocks back.  A beam with NaN or +inf in its
    score or logits has no candidates, and the call raises ValueError where it checks.  No gradient
    flows back.

    Banned tokens may hold -inf or the type's lowest value.  A beam with no token left is given a score of
    -inf, or -inf throughout: a log-sum in 64 bits is right to 2^-53 of the row's largest logit, so a row of
    bfloat16's or float32's lowest value throughout would give each token the beam's own score.

    `out`: the tensors of a `BeamChoice` to write into."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise TypeError("logits must be a CUDA tensor")
    if type(beams) is not int or not 1 <= beams <= 64:
        raise ValueError("beams must be an integer in [1, 64]")
    if count is None:
        count = min(2 * beams, 64) if end_token is not None else beams
    if type(out) is tuple:
        out = BeamChoice(*out)
    if type(out) is BeamChoice and _unchecked(check) and _calls.select_beams(logits, scores, beams, count, end_token,
                                                                            out, err):
        return out
    if type(count) is not int or not beams <= count <= 64:
        raise ValueError("count must be an integer in [beams, 64]")
    if logits.dtype not in _LOGITS:
        raise TypeError("logits must be a bfloat16, float16 or float32 tensor")
    if logits.dim() != 2 or logits.shape[0] % beams or not 1 <= logits.shape[1] <= _INT32_MAX:
        raise ValueError(f"logits must have shape (a multiple of {beams}, vocabulary), not {tuple(logits.shape)}")
    n, V = logits.shape
    if n > 65535:
        raise ValueError("select_beams takes up to 65535 rows")
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("a row's logits must be adjacent")
    if end_token is None:
        end = -1
    elif type(end_token) is int and 0 <= end_token <= _INT32_MAX:
        end = end_token
    else:
        raise ValueError("end_token must be a nonnegative integer, or None")
    dev, R = logits.device, n // beams
    before = _tensor(scores, "scores", torch.float32, (n,), dev)
    if out is None:
        whole = torch.empty(2 * n + 2 * R * count, dtype=torch.int32, device=dev)
        real = torch.empty(n + R * count, dtype=torch.float32, device=dev)
        out = BeamChoice(whole[:n], whole[n:2 * n], real[:n], whole[2 * n:2 * n + R * count].view(R, count),
                         whole[2 * n + R * count:].view(R, count), real[n:].view(R, count))
    else:
        out = BeamChoice(*out)
        for name, t, dtype, like in (("out.parents", out.parents, torch.int32, (n,)),
                                     ("out.tokens", out.tokens, torch.int32, (n,)),
                                     ("out.scores", out.scores, torch.float32, (n,)),
                                     ("out.all_parents", out.all_parents, torch.int32, (R, count)),
                                     ("out.all_tokens", out.all_tokens, torch.int32, (R, count)),
                                     ("out.all_scores", out.all_scores, torch.float32, (R, count))):
            _tensor(t, name, dtype, like, dev)
    call = _Call(dev, check, err)
    if n == 0:
        return out
    args = _lib.SelectArgs(logits.data_ptr(), before, *(t.data_ptr() for t in out), None, 0, call.err_ptr,
                           logits.stride(0), _LOGITS[logits.dtype], R, beams, V, count, end)
    size = _lib.load().kvmi_select_workspace_bytes(args)
    if size < 0:
        raise ValueError("kvmi_select_beams: invalid arguments (KVMI_EINVAL)")
    space = torch.empty(size, dtype=torch.uint8, device=dev)
    args.workspace, args.workspace_bytes = space.data_ptr(), size
    call.run("kvmi_select_beams", args)
    return out
