// Rows that share blocks of the paged cache: block tables forked with counted blocks, blocks
// copied in every layer, the pool compacted.
#include "kvmi_paged.hpp"

#include <algorithm>
#include <climits>

namespace kvmi {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kRange = 1024;        // block ids of a workgroup that goes through the pool, 4 a thread
constexpr int kMostForkRows = 4096;  // 20 bytes of LDS each

inline int ranges_of(int blocks) { return (blocks + kRange - 1) / kRange; }

// Sums over the workgroup, given to every thread.
template <int N>
__device__ __forceinline__ void block_sums(uint32_t (&v)[N], uint32_t (*lds)[kWaves]) {
#pragma unroll
  for (int d = 32; d; d >>= 1)
#pragma unroll
    for (int x = 0; x < N; ++x) v[x] = add_sat(v[x], __shfl_xor(v[x], d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int x = 0; x < N; ++x) lds[x][threadIdx.x >> 6] = v[x];
  __syncthreads();
#pragma unroll
  for (int x = 0; x < N; ++x) v[x] = add_sat(add_sat(lds[x][0], lds[x][1]), add_sat(lds[x][2], lds[x][3]));
}

// Sum of the threads before this one; `lds` has a word a wave.
__device__ __forceinline__ uint32_t before_in_block(uint32_t v, uint32_t* lds) {
  uint32_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t t = __shfl_up(s, d, 64);
    if ((threadIdx.x & 63) >= d) s += t;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  uint32_t carry = 0;
  for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) carry += lds[w];
  return s - v + carry;
}

// ---------------------------------------------------------------- forked tables
// Workspace, in 32-bit words.  `words` counts what happens to a block's holders: rows that go on
// without it in the upper half, rows that come to it besides one in the lower (at most
// kMostForkRows of either, so the halves do not meet).
struct ForkSpace {
  int64_t words, counts, ticket, taken, lengths, tables, size;
};
__host__ __device__ inline ForkSpace fork_space(int blocks, int rows, int columns) {
  ForkSpace s;
  s.words = 0;
  s.counts = blocks;  // freed blocks of each range of ids
  s.ticket = s.counts + (blocks + kRange - 1) / kRange;
  s.taken = s.ticket + 1;  // blocks taken out of the ring, -1 where the call changes nothing
  s.lengths = s.taken + 1;
  s.tables = (s.lengths + rows + 3) / 4 * 4;
  s.size = s.tables + (int64_t)rows * columns;
  return s;
}

// Workgroup (r, y) makes part y of row r, and counts what becomes of the blocks that row r held.
// Every workgroup goes through all rows for itself, as the tables of unshared blocks are made: who
// goes on in a partly kept block, and what the rows before take, so nobody waits.  Counts are sums of
// integers, so the order of the atomics does not matter: a block is free when all that held it
// have let go, which the last of them sees.
__global__ __launch_bounds__(kThreads) void fork_rows_kernel(kvmi_fork_args a, BlockOf div, bool in_place) {
  extern __shared__ int lds[];
  __shared__ uint32_t sums[6][kWaves];
  __shared__ int children, shortest;
  const int R = a.rows, C = a.columns, N = a.blocks, S = a.block_size, tid = threadIdx.x, r = blockIdx.x;
  int *const most = lds, *const owner = most + R, *const parent = owner + R, *const kept = parent + R,
            *const next = kept + R;
  const int top = C * S;
  const int head = (int)((uint32_t)a.state[0] % (uint32_t)N), count = a.state[1];
  int bad = count < 0 || count > N;
  for (int i = tid; i < R; i += kThreads) {
    most[i] = -1;
    owner[i] = INT_MAX;
  }
  if (tid == 0) {
    children = 0;
    shortest = INT_MAX;
  }
  __syncthreads();
  for (int i = tid; i < R; i += kThreads) {
    int p = a.parents ? gld(a.parents + i) : i;
    const int mine = gld(a.lengths + i);
    if (p < -1 || p >= R || (uint32_t)mine > (uint32_t)top) {
      bad = 1;
      p = -1;
    }
    int base = p >= 0 ? gld(a.lengths + p) : 0;
    int64_t n = a.new_lengths ? (int64_t)gld(a.new_lengths + i) : p >= 0 ? (int64_t)base + a.grow : 0;
    if ((uint32_t)base > (uint32_t)top || n < 0 || n > top) {
      bad = 1;
      base = 0;
      n = 0;
    }
    parent[i] = p;
    kept[i] = min(base, (int)n);
    next[i] = (int)n;
    if (p >= 0) atomicMax(&most[p], kept[i]);
  }
  __syncthreads();
  for (int i = tid; i < R; i += kThreads) {
    const int p = parent[i], full = div(kept[i]);
    if (p < 0 || kept[i] == full * S || div(most[p]) != full) continue;
    const int b = gld(a.tables + (int64_t)p * C + full);
    if ((uint32_t)b < (uint32_t)N && gld(a.shares + b) == 0) atomicMin(&owner[p], i);
  }
  __syncthreads();

  // blocks taken, new tokens and copies of all rows, and of those before this one
  uint32_t sum[6] = {0, 0, 0, 0, 0, 0};
  for (int i = tid; i < R; i += kThreads) {
    const int p = parent[i], full = div(kept[i]), want = next[i] ? div(next[i] - 1) + 1 : 0;
    const bool rest = kept[i] != full * S, goes_on = rest && owner[p] == i;
    const uint32_t v[3] = {(uint32_t)(want - full - goes_on), (uint32_t)(next[i] - kept[i]), rest && !goes_on};
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      sum[x] = add_sat(sum[x], v[x]);
      if (i < r) sum[3 + x] = add_sat(sum[3 + x], v[x]);
    }
  }
  block_sums(sum, sums);
  bad = __syncthreads_or(bad);
  const bool fits = sum[0] <= (uint32_t)max(count, 0), ok = !bad && fits && sum[1] <= (uint32_t)a.max_tokens;
  const ForkSpace at = fork_space(N, R, C);
  const int step = kThreads * gridDim.y, lane = blockIdx.y * kThreads + tid;
  if (r == 0 && lane == 0) {
    flag_error(a.err, bad || sum[1] > (uint32_t)a.max_tokens ? KVMI_ERR_LENGTH : fits ? 0 : KVMI_ERR_NO_BLOCKS);
    a.workspace[at.taken] = ok ? (int)sum[0] : -1;
    a.starts[0] = 0;
  }
  const int32_t* const old = a.tables + (int64_t)r * C;
  int32_t* const out = (in_place ? a.workspace + at.tables : a.out_tables) + (int64_t)r * C;
  int32_t* const copy = a.copies + 3 * (int64_t)r;
  if (!ok) {
    if (!in_place)
      for (int k = lane; k < C; k += step) gst(out + k, gld(old + k));
    for (int64_t k = (int64_t)r * step + lane; k < a.max_tokens; k += (int64_t)R * step) gst(a.slots + k, (int64_t)-1);
    if (lane == 0) {
      if (!in_place) a.out_lengths[r] = a.lengths[r];
      a.starts[r + 1] = 0;
      copy[0] = copy[1] = copy[2] = -1;
    }
    return;
  }

  // the new row
  const int p = parent[r], from_kept = kept[r], n = next[r];
  const int full = div(from_kept), rest = from_kept - full * S, want = n ? div(n - 1) + 1 : 0;
  const int stay = full + (rest && owner[p] == r);
  const uint32_t from = ring_at(head, sum[3], N);
  const int32_t* const source = a.tables + (int64_t)max(p, 0) * C;
  auto entry = [&](int k) -> int32_t {
    return k >= want ? -1 : gld(k < stay ? source + k : a.free_blocks + ring_at(from, k - stay, N));
  };
  if ((C & 3) == 0 && (((uintptr_t)a.tables | (uintptr_t)out) & 15) == 0) {
    for (int k = 4 * lane; k < C; k += 4 * step) {
      uint4 v = make_uint4(~0u, ~0u, ~0u, ~0u);
      if (k + 4 <= stay) {
        v = gld((const uint4*)(source + k));
      } else if (k < want) {
        v.x = entry(k);
        v.y = entry(k + 1);
        v.z = entry(k + 2);
        v.w = entry(k + 3);
      }
      gst((uint4*)(out + k), v);
    }
  } else {
    for (int k = lane; k < C; k += step) gst(out + k, entry(k));
  }
  int64_t* const slots = a.slots + sum[4];
  for (int i = lane; i < n - from_kept; i += step) {
    const int pos = from_kept + i, k = div(pos);
    gst(slots + i, (int64_t)entry(k) * S + (pos - k * S));
  }
  if (r == R - 1)
    for (int64_t k = (int64_t)sum[1] + lane; k < a.max_tokens; k += step) gst(a.slots + k, (int64_t)-1);
  if (lane == 0) {
    (in_place ? a.workspace + at.lengths : a.out_lengths)[r] = n;
    a.starts[r + 1] = (int)sum[4] + (n - from_kept);
    // copies first, in the order of their rows
    const bool copies = rest && stay == full;
    int32_t* const to = a.copies + 3 * (int64_t)(copies ? sum[5] : sum[2] + (r - sum[5]));
    to[0] = copies ? gld(source + full) : -1;
    to[1] = copies ? entry(full) : -1;
    to[2] = copies ? rest : -1;
  }

  // what becomes of the blocks that row r held: its children's whole blocks, and the block in
  // which one of them goes on
  const int mine = a.lengths[r], have = mine ? div(mine - 1) + 1 : 0;
  const int own_column = owner[r] == INT_MAX ? -1 : div(most[r]);
  __syncthreads();  // `most` becomes the list of this row's children
  for (int i = tid; i < R; i += kThreads)
    if (parent[i] == r) {
      const int whole = div(kept[i]);
      most[atomicAdd(&children, 1)] = whole;
      atomicMin(&shortest, whole);
    }
  __syncthreads();
  const int kids = children, all_below = shortest;
  bool foreign = false;
  for (int k = lane; k < have; k += step) {
    int holders = k == own_column;
    if (k < all_below)
      holders += kids;
    else
      for (int c = 0; c < kids; ++c) holders += most[c] > k;
    if (holders == 1) continue;
    const int b = gld(old + k);
    if ((uint32_t)b >= (uint32_t)N) {
      foreign = true;
    } else if (holders == 0) {
      const uint32_t before = atomicAdd((uint32_t*)a.workspace + at.words + b, 0x10000u);
      if ((int)(before >> 16) == gld(a.shares + b)) atomicAdd(a.workspace + at.counts + b / kRange, 1);
    } else {
      atomicAdd((uint32_t*)a.workspace + at.words + b, (uint32_t)(holders - 1));
    }
  }
  if (foreign) flag_error(a.err, KVMI_ERR_BLOCK_ID);
}

// Workgroup g < ranges goes through 1024 block ids: their new shares, and the free ones behind the
// ring's last, after those of the ranges before.  The last to arrive writes the state and clears
// the counts, when nobody reads them any more.  The other workgroups bring rows that are made in
// place from the workspace to their table.
__global__ __launch_bounds__(kThreads) void fork_blocks_kernel(kvmi_fork_args a, int ranges, bool in_place) {
  __shared__ uint32_t sums[2][kWaves], scan[kWaves];
  __shared__ int last;
  const int N = a.blocks, tid = threadIdx.x, g = blockIdx.x;
  const ForkSpace at = fork_space(N, a.rows, a.columns);
  const int taken = a.workspace[at.taken];
  if (g >= ranges) {
    if (taken < 0) return;
    const int64_t all = (int64_t)a.rows * a.columns, step = (int64_t)(gridDim.x - ranges) * kThreads;
    const int64_t first = (int64_t)(g - ranges) * kThreads + tid;
    const int32_t* const rows = a.workspace + at.tables;
    if ((all & 3) == 0 && (((uintptr_t)rows | (uintptr_t)a.out_tables) & 15) == 0) {
      for (int64_t i = first; i < all / 4; i += step) gst((uint4*)a.out_tables + i, gld((const uint4*)rows + i));
    } else {
      for (int64_t i = first; i < all; i += step) gst(a.out_tables + i, gld(rows + i));
    }
    for (int64_t i = first; i < a.rows; i += step) a.out_lengths[i] = a.workspace[at.lengths + i];
    return;
  }
  const int head = (int)((uint32_t)a.state[0] % (uint32_t)N), given = a.state[1];
  const int count = given < 0 ? 0 : given > N ? N : given;
  int32_t* const counts = a.workspace + at.counts;
  uint32_t sum[2] = {0, 0};  // freed before this range, and in all
  for (int i = tid; i < ranges; i += kThreads) {
    const uint32_t v = gld(counts + i);
    sum[1] += v;
    if (i < g) sum[0] += v;
  }
  block_sums(sum, sums);
  uint32_t word[4];
  int shares[4];
  const int first = g * kRange + 4 * tid;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const bool in = first + x < N;
    word[x] = in ? gld((const uint32_t*)a.workspace + at.words + first + x) : 0;
    shares[x] = in ? gld(a.shares + first + x) : 0;
  }
  uint32_t free = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) free += word[x] >> 16 && (int)(word[x] >> 16) > shares[x];
  uint32_t place = sum[0] + before_in_block(free, scan);
  bool lost = false;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if (first + x >= N) break;
    const int gone = (int)(word[x] >> 16), b = first + x;
    const int now = max(0, shares[x] + (int)(word[x] & 0xffffu) - gone);
    if (!in_place || now != shares[x]) a.out_shares[b] = now;
    if (word[x]) a.workspace[at.words + b] = 0;
    if (gone && gone > shares[x]) {
      if (place < (uint32_t)(N - count))
        a.free_blocks[((int64_t)head + count + place) % N] = b;
      else
        lost = true;
      ++place;
    }
  }
  if (lost) flag_error(a.err, KVMI_ERR_LENGTH);
  __syncthreads();
  if (tid == 0) last = atomicAdd(a.workspace + at.ticket, 1) == ranges - 1;
  __syncthreads();
  if (!last) return;
  for (int i = tid; i < ranges; i += kThreads) counts[i] = 0;
  if (tid == 0) {
    a.workspace[at.ticket] = 0;
    const int out = max(taken, 0), back = min((int)sum[1], N - count);
    a.out_state[0] = taken < 0 ? a.state[0] : (head + out) % N;
    a.out_state[1] = taken < 0 ? given : count - out + back;
  }
}

// ---------------------------------------------------------------- copied blocks
struct CopyArgs {
  kvmi_cache cache;
  void* const* bases;
  const int32_t* copies;
  int32_t* err;
  int n;
};

// Workgroups (x, layer and part): each looks at every gridDim.x-th row, 64 at a time, a row a lane,
// and copies those that are to be copied in units of V (16 bytes, or 2 where something is not
// aligned), eight loads of a thread before its stores.
template <class V>
__global__ __launch_bounds__(kThreads) void copy_kernel(CopyArgs a) {
  constexpr int U = sizeof(V) / 2, kAtOnce = 8;
  const int tid = threadIdx.x, lane = tid & 63, part = blockIdx.y & 1, layer = blockIdx.y >> 1;
  const int S = a.cache.block_size;
  const int64_t row = (int64_t)a.cache.num_heads * a.cache.head_dim / U;
  uint16_t* const base = (uint16_t*)(uintptr_t)gld((const int64_t*)a.bases + layer) + part * a.cache.part_stride;
  for (int64_t first = blockIdx.x; first < a.n; first += 64 * (int64_t)gridDim.x) {
    const int64_t mine = first + lane * (int64_t)gridDim.x;
    int from = -1, to = 0, tokens = 0;
    if (mine < a.n) {
      from = gld(a.copies + 3 * mine);
      to = gld(a.copies + 3 * mine + 1);
      tokens = gld(a.copies + 3 * mine + 2);
    }
    if (from >= 0) {
      const int bad = (from >= a.cache.num_blocks || (uint32_t)to >= (uint32_t)a.cache.num_blocks ? KVMI_ERR_BLOCK_ID
                                                                                                  : 0) |
                      ((uint32_t)tokens > (uint32_t)S ? KVMI_ERR_LENGTH : 0);
      if (bad && blockIdx.y == 0 && tid < 64) flag_error(a.err, bad);
      if (bad || from == to) from = -1;
    }
    for (uint64_t left = __ballot(from >= 0); left; left &= left - 1) {
      const int i = __builtin_ctzll(left);
      const V* const src = (const V*)(base + __builtin_amdgcn_readlane(from, i) * a.cache.block_stride);
      V* const dst = (V*)(base + __builtin_amdgcn_readlane(to, i) * a.cache.block_stride);
      const int64_t units = __builtin_amdgcn_readlane(tokens, i) * row;
      for (int64_t u0 = tid; u0 < units; u0 += kAtOnce * kThreads) {
        V held[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x)
          if (u0 + x * kThreads < units) held[x] = gld(src + u0 + x * kThreads);
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x)
          if (u0 + x * kThreads < units) gst(dst + u0 + x * kThreads, held[x]);
      }
    }
  }
}

// ---------------------------------------------------------------- a compacted pool
struct CompactSpace {  // in bytes; the two marks are zero between the calls
  int64_t held, free, counts, moves, names, from, to, shares, size;
};
__host__ __device__ inline CompactSpace compact_space(int blocks) {
  CompactSpace s;
  const int64_t bytes = ((int64_t)blocks + 15) / 16 * 16;
  s.held = 0;
  s.free = bytes;
  s.counts = 2 * bytes;  // held blocks, and the pool's, of each range
  s.moves = s.counts + 8 * (((int64_t)blocks + kRange - 1) / kRange);
  s.names = s.moves + 8;
  s.from = s.names + 4 * (int64_t)blocks;
  s.to = s.from + 4 * (int64_t)(blocks / 2);
  s.shares = s.to + 4 * (int64_t)(blocks / 2);
  s.size = s.shares + 4 * (int64_t)(blocks / 2);
  return s;
}
__device__ __forceinline__ int row_blocks(const kvmi_compact_args& a, const BlockOf& div, int r, bool* bad) {
  const int n = a.lengths[r], top = a.columns * a.block_size;
  *bad = (uint32_t)n > (uint32_t)top;
  const int cut = n < 0 ? 0 : n > top ? top : n;
  return cut ? div(cut - 1) + 1 : 0;
}

// Marks what the rows hold (workgroups of `parts` a row) and what the ring has free.
__global__ __launch_bounds__(kThreads) void compact_mark_kernel(kvmi_compact_args a, BlockOf div, int parts) {
  const int N = a.blocks, tid = threadIdx.x;
  const CompactSpace at = compact_space(N);
  uint8_t* const space = (uint8_t*)a.workspace;
  const int64_t rows = (int64_t)a.rows * parts;
  int bits = 0;
  if ((int64_t)blockIdx.x < rows) {
    const int r = blockIdx.x / parts, y = blockIdx.x % parts;
    bool bad;
    const int have = row_blocks(a, div, r, &bad);
    if (bad && y == 0 && tid == 0) bits |= KVMI_ERR_LENGTH;
    for (int k = y * kThreads + tid; k < have; k += parts * kThreads) {
      const int b = gld(a.tables + (int64_t)r * a.columns + k);
      if ((uint32_t)b < (uint32_t)N)
        gst(space + at.held + b, (uint8_t)1);
      else
        bits |= KVMI_ERR_BLOCK_ID;
    }
  } else {
    const int head = (int)((uint32_t)a.state[0] % (uint32_t)N), given = a.state[1];
    const int count = given < 0 ? 0 : given > N ? N : given;
    if (given != count && (int64_t)blockIdx.x == rows && tid == 0) bits |= KVMI_ERR_LENGTH;
    const int first = (int)(blockIdx.x - rows) * kRange;
    for (int i = first + tid; i < min(count, first + kRange); i += kThreads) {
      const int b = gld(a.free_blocks + ring_at(head, i, N));
      if ((uint32_t)b < (uint32_t)N)
        gst(space + at.free + b, (uint8_t)1);
      else
        bits |= KVMI_ERR_BLOCK_ID;
    }
  }
  flag_error(a.err, bits);
}

// The marks of four ids: bit 0 held, bit 1 in the pool, in bytes.
__device__ __forceinline__ uint32_t marks_of(const uint8_t* space, const CompactSpace& at, int N, int first,
                                             uint32_t* free) {
  uint32_t held = 0;
  *free = 0;
  if (first < N) {  // (the marks reach to a multiple of 16 and are zero there)
    held = gld((const uint32_t*)(space + at.held + first));
    *free = gld((const uint32_t*)(space + at.free + first));
  }
  return held;
}

__global__ __launch_bounds__(kThreads) void compact_count_kernel(kvmi_compact_args a) {
  __shared__ uint32_t sums[2][kWaves];
  const CompactSpace at = compact_space(a.blocks);
  const uint8_t* const space = (const uint8_t*)a.workspace;
  uint32_t free;
  const uint32_t held = marks_of(space, at, a.blocks, blockIdx.x * kRange + 4 * threadIdx.x, &free);
  uint32_t sum[2] = {(uint32_t)__popc(held), (uint32_t)__popc(held | free)};
  block_sums(sum, sums);
  if (threadIdx.x == 0) {
    uint32_t* const counts = (uint32_t*)(space + at.counts);
    gst(counts + 2 * blockIdx.x, sum[0]);
    gst(counts + 2 * blockIdx.x + 1, sum[1]);
  }
}

// Workgroup g: the places of 1024 ids among the held blocks and in the pool.  The pool's first n ids
// stay or are taken (n: held blocks), so the number of moves is that of the free ones among them:
// those of the ranges below the one where n falls, and some in it, which each looks up for itself.
__global__ __launch_bounds__(kThreads) void compact_rank_kernel(kvmi_compact_args a, int ranges) {
  __shared__ uint32_t sums[4][kWaves], scan[kWaves], cut[3];
  const int N = a.blocks, tid = threadIdx.x, g = blockIdx.x;
  const CompactSpace at = compact_space(N);
  uint8_t* const space = (uint8_t*)a.workspace;
  const uint32_t* const counts = (const uint32_t*)(space + at.counts);
  uint32_t sum[4] = {0, 0, 0, 0};  // held and pool before this range, and in all
  for (int i = tid; i < ranges; i += kThreads) {
    const uint32_t h = gld(counts + 2 * i), u = gld(counts + 2 * i + 1);
    sum[2] += h;
    sum[3] += u;
    if (i < g) {
      sum[0] += h;
      sum[1] += u;
    }
  }
  block_sums(sum, sums);
  const uint32_t n = sum[2];
  // the range in which the pool's n-th id falls, and what is held and in the pool before it
  uint32_t held_before = 0, pool_before = 0;
  if (tid == 0) cut[0] = 0x7fffffff;
  for (int i0 = 0; i0 < ranges; i0 += kThreads) {
    const int i = i0 + tid;
    const uint32_t h = i < ranges ? gld(counts + 2 * i) : 0, u = i < ranges ? gld(counts + 2 * i + 1) : 0;
    const uint32_t hb = held_before + before_in_block(h, scan);
    const uint32_t ub = pool_before + before_in_block(u, scan);
    if (ub < n && ub + u >= n) {
      cut[0] = i;
      cut[1] = hb;
      cut[2] = ub;
    }
    uint32_t all[2] = {h, u};
    block_sums(all, sums);
    held_before += all[0];
    pool_before += all[1];
  }
  __syncthreads();
  uint32_t moves = 0;
  if (cut[0] != 0x7fffffff) {
    uint32_t free;
    const uint32_t held = marks_of(space, at, N, cut[0] * kRange + 4 * tid, &free), pool = held | free;
    uint32_t u = cut[2] + before_in_block(__popc(pool), scan);
    uint32_t low[1] = {0};  // held in the range below the cut
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (!(pool >> (8 * x) & 1)) continue;
      low[0] += u < n && (held >> (8 * x) & 1);
      ++u;
    }
    block_sums(low, sums);
    moves = n - cut[1] - low[0];
  }
  // this range
  const int first = g * kRange + 4 * tid;
  uint32_t free;
  const uint32_t held = marks_of(space, at, N, first, &free), pool = held | free;
  uint32_t h = sum[0] + before_in_block(__popc(held), scan), u = sum[1] + before_in_block(__popc(pool), scan);
  int32_t* const names = (int32_t*)(space + at.names);
  const uint32_t left = sum[3] - n;  // free blocks afterwards
  int bits = 0;
  for (int x = 0; x < 4 && first + x < N; ++x) {
    const int b = first + x;
    const bool is_held = held >> (8 * x) & 1, in_pool = pool >> (8 * x) & 1;
    if (is_held && (free >> (8 * x) & 1)) bits |= KVMI_ERR_BLOCK_ID;
    int shares = is_held ? gld(a.shares + b) : 0, name = b;
    bool write = true;
    if (in_pool && u >= n) {
      gst(a.out_free + (u - n), b);
      if (is_held) {
        const uint32_t i = h - (n - moves);
        gst((int32_t*)(space + at.from) + i, b);
        gst((int32_t*)(space + at.shares) + i, shares);
        name = -1 - (int)i;
        shares = 0;
      }
    } else if (in_pool && !is_held) {
      gst((int32_t*)(space + at.to) + (u - h), b);
      write = false;  // comes from the block that moves here
    }
    gst(names + b, name);
    if (write) gst(a.out_shares + b, shares);
    if ((uint32_t)b >= left) gst(a.out_free + b, -1);
    h += is_held;
    u += in_pool;
  }
  if (first < N) {  // the marks are left zero for the next call; no other workgroup but at the cut reads them
    if (cut[0] != (uint32_t)g) {
      gst((uint32_t*)(space + at.held + first), 0u);
      gst((uint32_t*)(space + at.free + first), 0u);
    }
  }
  flag_error(a.err, bits);
  if (g == 0 && tid == 0) {
    ((uint32_t*)(space + at.moves))[0] = moves;
    ((uint32_t*)(space + at.moves))[1] = cut[0];
    a.out_state[0] = 0;
    a.out_state[1] = (int)left;
  }
}

// The rows under the new names, and the list of moves.
__global__ __launch_bounds__(kThreads) void compact_name_kernel(kvmi_compact_args a, BlockOf div, int parts) {
  const int N = a.blocks, tid = threadIdx.x;
  const CompactSpace at = compact_space(N);
  uint8_t* const space = (uint8_t*)a.workspace;
  const int32_t* const to = (const int32_t*)(space + at.to);
  const int64_t rows = (int64_t)a.rows * parts;
  if ((int64_t)blockIdx.x < rows) {
    const int r = blockIdx.x / parts, y = blockIdx.x % parts;
    bool bad;
    const int have = row_blocks(a, div, r, &bad);
    const int32_t* const names = (const int32_t*)(space + at.names);
    for (int k = y * kThreads + tid; k < a.columns; k += parts * kThreads) {
      int b = -1;
      if (k < have) {
        b = gld(a.tables + (int64_t)r * a.columns + k);
        if ((uint32_t)b < (uint32_t)N) {
          const int name = gld(names + b);
          b = name >= 0 ? name : gld(to + (-1 - name));
        }
      }
      gst(a.out_tables + (int64_t)r * a.columns + k, b);
    }
    return;
  }
  const int moves = gld((const int32_t*)(space + at.moves)), range = gld((const int32_t*)(space + at.moves) + 1);
  const int first = (int)(blockIdx.x - rows) * kRange;
  for (int i = first + tid; i < min(N / 2, first + kRange); i += kThreads) {
    const bool moved = i < moves;
    const int b = moved ? gld(to + i) : -1;
    gst(a.copies + 3 * (int64_t)i, moved ? gld((const int32_t*)(space + at.from) + i) : -1);
    gst(a.copies + 3 * (int64_t)i + 1, b);
    gst(a.copies + 3 * (int64_t)i + 2, moved ? a.block_size : -1);
    if (moved) gst(a.out_shares + b, gld((const int32_t*)(space + at.shares) + i));
  }
  // the marks that all workgroups looked at before
  const int id = range * kRange + 4 * tid;
  if ((int64_t)blockIdx.x == rows && range != 0x7fffffff && id < N) {
    gst((uint32_t*)(space + at.held + id), 0u);
    gst((uint32_t*)(space + at.free + id), 0u);
  }
}

}  // namespace
}  // namespace kvmi

extern "C" int64_t kvmi_fork_workspace_bytes(int32_t blocks, int32_t rows, int32_t columns) {
  if (blocks < 1 || rows < 0 || columns < 1) return KVMI_EINVAL;
  return 4 * kvmi::fork_space(blocks, rows, columns).size;
}

extern "C" int kvmi_fork_tables(const kvmi_fork_args* args, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!args) return KVMI_EINVAL;
  const kvmi_fork_args& a = *args;
  if (a.rows < 0 || a.rows > kMostForkRows || a.columns < 1 || a.blocks < 1 || a.block_size < 1 || a.max_tokens < 0 ||
      a.grow < 0)
    return KVMI_EINVAL;
  if ((int64_t)a.columns * a.block_size > kMostPlaces || (int64_t)a.blocks * a.block_size > 0x7fffffffLL ||
      (int64_t)a.columns * a.rows > 0x7fffffffLL)
    return KVMI_EINVAL;
  if (a.rows == 0) return KVMI_OK;
  if (!a.lengths || !a.tables || !a.shares || !a.free_blocks || !a.state || !a.out_tables || !a.out_lengths ||
      !a.out_shares || !a.out_state || !a.starts || !a.copies || !a.workspace || (a.max_tokens && !a.slots))
    return KVMI_EINVAL;
  const bool in_place = a.out_tables == a.tables;
  if (in_place != (a.out_lengths == a.lengths) || in_place != (a.out_shares == a.shares) ||
      in_place != (a.out_state == a.state))
    return KVMI_EINVAL;
  if (a.new_lengths == a.out_lengths || a.parents == a.out_lengths || (uintptr_t)a.workspace % 8 ||
      a.workspace_bytes < kvmi_fork_workspace_bytes(a.blocks, a.rows, a.columns))
    return KVMI_EINVAL;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t most = std::max<int64_t>((a.columns + 1023) / 1024, ((int64_t)a.max_tokens + 4095) / 4096);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(most, std::min(64, 2048 / a.rows)));
  hipLaunchKernelGGL(fork_rows_kernel, dim3((unsigned)a.rows, (unsigned)parts), dim3(kThreads), 20 * (size_t)a.rows,
                     st, a, block_of(a.block_size), in_place);
  const int ranges = ranges_of(a.blocks);
  const int64_t copies = in_place ? std::min<int64_t>(1024, ((int64_t)a.rows * a.columns + 4095) / 4096) : 0;
  hipLaunchKernelGGL(fork_blocks_kernel, dim3((unsigned)(ranges + copies)), dim3(kThreads), 0, st, a, ranges,
                     in_place);
  return launched();
}

extern "C" int kvmi_copy_blocks(const kvmi_cache* cache, void* const* bases, int32_t layers, const int32_t* copies,
                                int32_t n, int32_t* err, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!cache_ok(cache, false) || layers < 1 || layers > 32767 || n < 0) return KVMI_EINVAL;
  if (n == 0) return KVMI_OK;
  if (!bases || !copies) return KVMI_EINVAL;
  const CopyArgs a{*cache, bases, copies, err, n};
  const int x = std::min(n, std::max(1, 16384 / (2 * layers)));
  const dim3 grid((unsigned)x, 2u * (unsigned)layers);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (strides16(cache) && aligned16(cache->base))
    hipLaunchKernelGGL((copy_kernel<uint4>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((copy_kernel<uint16_t>), grid, dim3(kThreads), 0, st, a);
  return launched();
}

extern "C" int64_t kvmi_compact_workspace_bytes(int32_t blocks) {
  if (blocks < 1) return KVMI_EINVAL;
  return kvmi::compact_space(blocks).size;
}

extern "C" int kvmi_compact_tables(const kvmi_compact_args* args, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!args) return KVMI_EINVAL;
  const kvmi_compact_args& a = *args;
  if (a.rows < 0 || a.columns < 1 || a.blocks < 1 || a.block_size < 1) return KVMI_EINVAL;
  if ((int64_t)a.columns * a.block_size > kMostPlaces || (int64_t)a.blocks * a.block_size > 0x7fffffffLL ||
      (int64_t)a.columns * a.rows > 0x7fffffffLL)
    return KVMI_EINVAL;
  if ((a.rows && (!a.lengths || !a.tables || !a.out_tables)) || !a.shares || !a.free_blocks || !a.state ||
      !a.out_shares || !a.out_free || !a.out_state || (a.blocks > 1 && !a.copies) || !a.workspace)
    return KVMI_EINVAL;
  const bool in_place = a.out_shares == a.shares;
  if ((a.rows && in_place != (a.out_tables == a.tables)) || in_place != (a.out_free == a.free_blocks) ||
      in_place != (a.out_state == a.state) || (uintptr_t)a.workspace % 8 ||
      a.workspace_bytes < kvmi_compact_workspace_bytes(a.blocks))
    return KVMI_EINVAL;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int ranges = ranges_of(a.blocks), parts = std::min(64, (a.columns + 1023) / 1024);
  const int64_t rows = (int64_t)a.rows * parts;
  if (rows + ranges > 0x7fffffffLL) return KVMI_EINVAL;
  const BlockOf div = block_of(a.block_size);
  hipLaunchKernelGGL(compact_mark_kernel, dim3((unsigned)(rows + ranges)), dim3(kThreads), 0, st, a, div, parts);
  hipLaunchKernelGGL(compact_count_kernel, dim3((unsigned)ranges), dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(compact_rank_kernel, dim3((unsigned)ranges), dim3(kThreads), 0, st, a, ranges);
  hipLaunchKernelGGL(compact_name_kernel, dim3((unsigned)(rows + ranges)), dim3(kThreads), 0, st, a, div, parts);
  return launched();
}
