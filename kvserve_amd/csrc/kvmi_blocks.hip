// Rows that share blocks of the paged cache: block tables forked with counted blocks, blocks
// copied in every layer, the pool compacted.
#include "kvmi_paged.hpp"

#include <algorithm>
#include <climits>

namespace kvmi {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kRange = 1024;        // block ids of a workgroup that goes through the pool, 4 a thread
constexpr int kCounted = 64;        // block ids of a count
constexpr int kMostForkRows = 4096;  // 32 bytes of LDS each
// Every workgroup of kRange ids adds up the counts of the whole pool, work that goes with its square: a fork
// of 8 rows takes 13 us in a pool of 2^18 blocks, 27 of 2^20, 106 of 2^22 and 1060 of 2^24, a compaction 15, 25,
// 84 and 760, nearly all of it these sums in the largest two.
constexpr int kMostBlocks = 1 << 24;

inline int ranges_of(int blocks) { return (blocks + kRange - 1) / kRange; }

// The wave's sums go from row to row of 16 lanes in registers.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t sum_with(uint32_t x) {
  return add_sat(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false));
}
// Sum of the lanes up to this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x = sum_with<0x111, 0xf>(x);  // the lane 1, 2, 4, 8 before in the row
  x = sum_with<0x112, 0xf>(x);
  x = sum_with<0x114, 0xf>(x);
  x = sum_with<0x118, 0xf>(x);
  x = sum_with<0x142, 0xa>(x);  // the last lane of the row before, of the half before
  return sum_with<0x143, 0xc>(x);
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(x), 63);
}
// Sums over the workgroup, given to every thread.
template <int N>
__device__ __forceinline__ void block_sums(uint32_t (&v)[N], uint32_t (*lds)[kWaves]) {
#pragma unroll
  for (int x = 0; x < N; ++x) v[x] = wave_sum(v[x]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int x = 0; x < N; ++x) lds[x][threadIdx.x >> 6] = v[x];
  __syncthreads();
#pragma unroll
  for (int x = 0; x < N; ++x) v[x] = add_sat(add_sat(lds[x][0], lds[x][1]), add_sat(lds[x][2], lds[x][3]));
}

// Sums of the threads before this one.
template <int N>
__device__ __forceinline__ void before_in_block(uint32_t (&v)[N], uint32_t (*lds)[kWaves]) {
  uint32_t s[N];
#pragma unroll
  for (int x = 0; x < N; ++x) s[x] = wave_scan(v[x]);
  __syncthreads();
  if ((threadIdx.x & 63) == 63)
#pragma unroll
    for (int x = 0; x < N; ++x) lds[x][threadIdx.x >> 6] = s[x];
  __syncthreads();
#pragma unroll
  for (int x = 0; x < N; ++x) {
    v[x] = s[x] - v[x];
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) v[x] += lds[x][w];
  }
}

// ---------------------------------------------------------------- forked tables
// What one row becomes, and what the rows before it take.
struct ForkRow {
  int parent, kept, next;
  int stay;                         // blocks that it has from its parent
  uint32_t takes, tokens, copies;   // of the rows before it
  int kids, shortest, longest;      // its children, and the whole blocks that they keep of it
  int own_column;                   // the block in which one of them goes on, or -1
  int length;                       // before the call
};
struct ForkSum {
  int taken;  // blocks out of the ring; -1 where the call changes nothing
  uint32_t tokens, copies;
  int head, count;  // of the ring, as given (the head inside it)
  int turn;         // which of the two counts this call uses
  int unused;
};
// Workspace, in 32-bit words.  `words` counts what happens to a block's holders: rows that go on
// without it in the upper half, rows that come to it besides one in the lower (at most
// kMostForkRows of either, so the halves do not meet).  Of the two sets of `counts`, freed blocks of each
// 64 ids, a call uses the one that `turn` names and clears the other, which nobody reads then.  (Counted
// by 1024 ids, thousands of atomics met at one address: 1024 rows 44 us a call, 27 by 64.)
struct ForkSpace {
  int64_t words, counts, turn, sum, rows, lengths, tables, size;
  int counted;  // counts of a set
};
__host__ __device__ inline ForkSpace fork_space(int blocks, int rows, int columns) {
  ForkSpace s;
  s.words = 0;
  s.counts = blocks;
  s.counted = (blocks + kCounted - 1) / kCounted;
  s.turn = s.counts + 2 * (int64_t)s.counted;
  s.sum = (s.turn + 4) / 4 * 4;
  s.rows = s.sum + 8;
  s.lengths = s.rows + 12 * (int64_t)rows;
  s.tables = (s.lengths + rows + 3) / 4 * 4;
  s.size = s.tables + (int64_t)rows * columns;
  return s;
}

// The plan of all rows, made by one workgroup in its LDS, 32 bytes a row: one trip to memory, and one more
// only where a row is cut inside a block, which others may hold (a row's own last block is held by
// nobody else while it is partly filled).
struct ForkPlan {
  int *length, *parent, *kept, *next, *most, *owner, *kids, *shortest;
  int* bad;  // one word
};
template <int THREADS>
__device__ __forceinline__ ForkPlan plan_rows(const kvmi_fork_args& a, const BlockOf& div, int* lds) {
  const int R = a.rows, C = a.columns, N = a.blocks, S = a.block_size, top = C * S, tid = threadIdx.x;
  ForkPlan f{lds, lds + R, lds + 2 * R, lds + 3 * R, lds + 4 * R, lds + 5 * R, lds + 6 * R, lds + 7 * R, lds + 8 * R};
  int bad = 0;
  auto unshared = [&](int row, int column) -> int {
    const int b = gld(a.tables + (int64_t)row * C + column);
    return (uint32_t)b < (uint32_t)N && gld(a.shares + b) == 0;
  };
  for (int i = tid; i < R; i += THREADS) {
    int p = a.parents ? gld(a.parents + i) : i, n = a.new_lengths ? gld(a.new_lengths + i) : 0;
    int length = gld(a.lengths + i);
    if (p < -1 || p >= R || (uint32_t)length > (uint32_t)top || (uint32_t)n > (uint32_t)top) {
      bad = 1;
      p = -1;
      length = n = 0;
    }
    f.length[i] = length;
    f.parent[i] = p;
    f.next[i] = n;
    f.most[i] = -1;
    f.owner[i] = f.shortest[i] = INT_MAX;
    f.kids[i] = 0;
  }
  if (tid == 0) *f.bad = 0;
  __syncthreads();
  for (int i = tid; i < R; i += THREADS) {
    const int p = f.parent[i], base = p >= 0 ? f.length[p] : 0;
    if (!a.new_lengths) {
      const int64_t n = p >= 0 ? (int64_t)base + a.grow : 0;
      if (n > top) bad = 1;
      f.next[i] = (int)min(n, (int64_t)top);
    }
    const int kept = min(base, f.next[i]), whole = div(kept);
    f.kept[i] = kept;
    if (p >= 0) {
      atomicMax(&f.most[p], kept);
      atomicMin(&f.shortest[p], whole);
      atomicAdd(&f.kids[p], 1);
    }
  }
  if (bad) *f.bad = 1;
  __syncthreads();
  for (int i = tid; i < R; i += THREADS) {
    const int p = f.parent[i], kept = f.kept[i], whole = div(kept);
    if (p < 0 || kept == whole * S || div(f.most[p]) != whole) continue;
    if (kept == f.length[p] || unshared(p, whole)) atomicMin(&f.owner[p], i);
  }
  __syncthreads();
  return f;
}
// What row i adds to the sums: blocks taken, new tokens, copies.
__device__ __forceinline__ int stays(const ForkPlan& f, const BlockOf& div, int S, int i) {
  const int whole = div(f.kept[i]);
  return whole + (f.kept[i] != whole * S && f.owner[f.parent[i]] == i);
}
__device__ __forceinline__ void row_adds(const ForkPlan& f, const BlockOf& div, int S, int i, uint32_t (&v)[3]) {
  const int whole = div(f.kept[i]), stay = stays(f, div, S, i), want = f.next[i] ? div(f.next[i] - 1) + 1 : 0;
  v[0] = want - stay;
  v[1] = f.next[i] - f.kept[i];
  v[2] = f.kept[i] != whole * S && stay == whole;
}
__device__ __forceinline__ ForkRow row_of(const ForkPlan& f, const BlockOf& div, int S, int i, const uint32_t* before) {
  return ForkRow{f.parent[i], f.kept[i],     f.next[i],           stays(f, div, S, i), before[0], before[1],
                 before[2],   f.kids[i],     f.shortest[i],       div(max(f.most[i], 0)),
                 f.owner[i] == INT_MAX ? -1 : div(f.most[i]),     f.length[i]};
}
// The sums of all rows, whether the call can be done, and its error.
__device__ __forceinline__ ForkSum sum_of(const kvmi_fork_args& a, int head, int count, int turn, const uint32_t* all,
                                          int bad, int32_t* error) {
  bad |= count < 0 || count > a.blocks || all[1] > (uint32_t)a.max_tokens;
  const bool fits = all[0] <= (uint32_t)max(count, 0);
  *error = bad ? KVMI_ERR_LENGTH : fits ? 0 : KVMI_ERR_NO_BLOCKS;
  return ForkSum{bad || !fits ? -1 : (int)all[0], all[1], all[2], (int)((uint32_t)head % (uint32_t)a.blocks), count, turn, 0};
}

// What becomes of the blocks that row r held.  n entries from k on: their shares and atomics are on
// their way in `begin`, and looked at in `end`, with what else there is to do between the two.
// Counts are sums of integers, so the order of the atomics does not matter: a block is free when all that
// held it have let go, which the last of them sees.  (A call that is refused clears them all the same.)
template <int n>
struct Settled {
  int b[n], holders[n], shares[n];
  uint32_t before[n];
};
struct Settler {
  const kvmi_fork_args& a;
  const ForkSpace& at;
  const ForkRow& row;
  int have, listed;
  const int* list;
  int32_t* counts;
  bool foreign;

  template <int n>
  __device__ __forceinline__ void begin(int k, Settled<n>& s) {
#pragma unroll
    for (int x = 0; x < n; ++x) {
      int holders = k + x == row.own_column;
      if (k + x < row.shortest)
        holders += row.kids;
      else if (k + x < row.longest)
        for (int c = 0; c < listed; ++c) holders += list[c] > k + x;
      // (where a row goes on in its partly filled block, nobody else may hold it)
      const bool changes = k + x < have && (holders != 1 || k + x == row.own_column);
      const bool inside = (uint32_t)s.b[x] < (uint32_t)a.blocks;
      foreign |= changes && !inside;
      s.holders[x] = changes && inside ? holders : -1;
      s.shares[x] = s.holders[x] == 0 || s.holders[x] == 1 ? gld(a.shares + s.b[x]) : 0;
    }
    uint32_t* const words = (uint32_t*)a.workspace + at.words;
#pragma unroll
    for (int x = 0; x < n; ++x)
      if (s.holders[x] == 0)
        s.before[x] = atomicAdd(words + s.b[x], 0x10000u);
      else if (s.holders[x] > 1)
        atomicAdd(words + s.b[x], (uint32_t)(s.holders[x] - 1));
  }
  template <int n>
  __device__ __forceinline__ void end(const Settled<n>& s) {
#pragma unroll
    for (int x = 0; x < n; ++x) {
      if (s.holders[x] == 0 && (int)(s.before[x] >> 16) == s.shares[x])
        atomicAdd(counts + s.b[x] / kCounted, 1);
      foreign |= s.holders[x] == 1 && s.shares[x];
    }
  }
};
// The settler of row r, for which `child(i)` tells the whole blocks that row i keeps of it, -1 if it is no
// child.  `list` has room for all rows.
template <class F>
__device__ __forceinline__ Settler settler_of(const kvmi_fork_args& a, const BlockOf& div, const ForkSpace& at,
                                              const ForkRow& row, int turn, int* list, F child) {
  __shared__ int children;
  Settler s{a, at, row, row.length ? div(row.length - 1) + 1 : 0, 0, list,
            a.workspace + at.counts + (turn ? at.counted : 0), false};
  if (row.kids && row.shortest < row.longest && row.shortest < s.have) {
    // children that keep more and less: who holds a block between is counted
    if (threadIdx.x == 0) children = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.rows; i += kThreads) {
      const int keeps = child(i);
      if (keeps >= 0) list[atomicAdd(&children, 1)] = keeps;
    }
    __syncthreads();
    s.listed = children;
  }
  return s;
}
// Rows are read four entries at a time where they are aligned so.
__device__ __forceinline__ Settled<4> four(const uint4& v) {
  return Settled<4>{{(int)v.x, (int)v.y, (int)v.z, (int)v.w}, {-1, -1, -1, -1}, {}, {}};
}

// Part blockIdx.y of row r: its entries, slots and copy.  `ahead`: the parent's first entries, where rows
// are read in fours.
__device__ __forceinline__ void fork_row(const kvmi_fork_args& a, const BlockOf& div, bool in_place, const ForkSpace& at,
                                         const ForkRow& row, const ForkSum& all, int r, bool fours,
                                         const uint4& ahead) {
  const int R = a.rows, C = a.columns, N = a.blocks, S = a.block_size, tid = threadIdx.x;
  const int step = kThreads * gridDim.y, lane = blockIdx.y * kThreads + tid;
  int32_t* const out = (in_place ? a.workspace + at.tables : a.out_tables) + (int64_t)r * C;
  if (r == 0 && lane == 0) a.starts[0] = 0;
  if (all.taken < 0) {
    if (!in_place)
      for (int k = lane; k < C; k += step) gst(out + k, gld(a.tables + (int64_t)r * C + k));
    for (int64_t k = (int64_t)r * step + lane; k < a.max_tokens; k += (int64_t)R * step) gst(a.slots + k, (int64_t)-1);
    if (lane == 0) {
      if (!in_place) a.out_lengths[r] = gld(a.lengths + r);  // (row.length is 0 where it is out of range)
      a.starts[r + 1] = 0;
      int32_t* const copy = a.copies + 3 * (int64_t)r;
      copy[0] = copy[1] = copy[2] = -1;
    }
    return;
  }
  const int whole = div(row.kept), rest = row.kept - whole * S, want = row.next ? div(row.next - 1) + 1 : 0;
  const int stay = row.stay;
  const uint32_t from = ring_at(all.head, row.takes, N);
  const int32_t* const source = a.tables + (int64_t)max(row.parent, 0) * C;
  auto entry = [&](int k) -> int32_t {
    return k >= want ? -1 : gld(k < stay ? source + k : a.free_blocks + ring_at(from, k - stay, N));
  };
  if (fours) {
    for (int k = 4 * lane; k < C; k += 4 * step) {
      uint4 v = make_uint4(~0u, ~0u, ~0u, ~0u);
      if (k + 4 <= stay) {
        v = k == 4 * lane ? ahead : gld((const uint4*)(source + k));
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
  int64_t* const slots = a.slots + row.tokens;
  for (int i = lane; i < row.next - row.kept; i += step) {
    const int pos = row.kept + i, k = div(pos);
    gst(slots + i, (int64_t)entry(k) * S + (pos - k * S));
  }
  if (r == R - 1)
    for (int64_t k = (int64_t)all.tokens + lane; k < a.max_tokens; k += step) gst(a.slots + k, (int64_t)-1);
  if (lane == 0) {
    (in_place ? a.workspace + at.lengths : a.out_lengths)[r] = row.next;
    a.starts[r + 1] = (int)row.tokens + (row.next - row.kept);
    // copies first, in the order of their rows
    const bool copies = rest && stay == whole;
    const int b = copies ? gld(source + whole) : -1, fresh = copies ? entry(whole) : -1;
    int32_t* const to = a.copies + 3 * (int64_t)(copies ? row.copies : all.copies + (r - row.copies));
    to[0] = b;
    to[1] = fresh;
    to[2] = copies ? rest : -1;
  }
}
// The rest of what row r held, behind the first four entries of each thread.
__device__ __forceinline__ void settle_rest(Settler& settler, int r, bool fours) {
  const int step = kThreads * gridDim.y, lane = blockIdx.y * kThreads + threadIdx.x;
  const int32_t* const old = settler.a.tables + (int64_t)r * settler.a.columns;
  if (fours) {
    for (int k = 4 * (lane + step); k < settler.have; k += 4 * step) {
      Settled<4> s = four(gld((const uint4*)(old + k)));
      settler.begin(k, s);
      settler.end(s);
    }
  } else {
    for (int k = lane; k < settler.have; k += step) {
      Settled<1> s{{gld(old + k)}, {}, {}, {}};
      settler.begin(k, s);
      settler.end(s);
    }
  }
}
__device__ __forceinline__ bool in_fours(const kvmi_fork_args& a, const ForkSpace& at, bool in_place) {
  const void* const out = in_place ? a.workspace + at.tables : a.out_tables;
  return (a.columns & 3) == 0 && (((uintptr_t)a.tables | (uintptr_t)out) & 15) == 0;
}

// Up to kFused rows: every workgroup (row, part) plans them all for itself, while its entries are on
// their way, and no workgroup waits for another.  A chain of a trip to memory, the plan in the LDS,
// the sums, the entries out of the ring, and the atomics' answers: 4 rows of 32 blocks 6.4 us, 256 rows of
// up to 750 blocks 9.9 (7.2 without the atomics, of which it makes some 60,000).  Rows that are made in
// place: 256 rows 10.6, and 0.1 us more to bring them back; 64 rows of up to 8192 blocks 18.6 and 1.0 more.
constexpr int kFused = 256;
__global__ __launch_bounds__(kThreads) void fork_fused_kernel(kvmi_fork_args a, BlockOf div, bool in_place) {
  __shared__ int lds[8 * kFused + 1], list[kFused];
  const int R = a.rows, C = a.columns, tid = threadIdx.x, r = blockIdx.x;
  const ForkSpace at = fork_space(a.blocks, R, C);
  const bool fours = in_fours(a, at, in_place);
  const int head = gld(a.state), count = gld(a.state + 1), turn = gld(a.workspace + at.turn);
  const int k = 4 * (blockIdx.y * kThreads + tid);
  uint4 old = make_uint4(0, 0, 0, 0), source = old;
  if (fours && k < C) {
    int p = a.parents ? a.parents[r] : r;
    p = p < 0 || p >= R ? r : p;
    old = gld((const uint4*)(a.tables + (int64_t)r * C + k));
    source = gld((const uint4*)(a.tables + (int64_t)p * C + k));
  }
  const ForkPlan f = plan_rows<kThreads>(a, div, lds);
  // the row's own plan but for what the rows before it take; its blocks' holders are on their way
  // while that is summed, by every wave for itself
  const uint32_t none[3] = {0, 0, 0};
  ForkRow row = row_of(f, div, a.block_size, r, none);
  Settler settler = settler_of(a, div, at, row, turn, list, [&](int i) { return f.parent[i] == r ? div(f.kept[i]) : -1; });
  Settled<4> held = four(old);
  if (fours && k < settler.have) settler.begin(k, held);
  uint32_t sum[6] = {0, 0, 0, 0, 0, 0};
  for (int i = tid & 63; i < R; i += 64) {
    uint32_t v[3];
    row_adds(f, div, a.block_size, i, v);
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      sum[x] = add_sat(sum[x], v[x]);
      sum[3 + x] = add_sat(sum[3 + x], i < r ? v[x] : 0);
    }
  }
#pragma unroll
  for (int x = 0; x < 6; ++x) sum[x] = wave_sum(sum[x]);
  int32_t error;
  const ForkSum all = sum_of(a, head, count, turn, sum, *f.bad, &error);
  row.takes = sum[3];
  row.tokens = sum[4];
  row.copies = sum[5];
  if (r == 0 && blockIdx.y == 0 && tid == 0) {
    flag_error(a.err, error);
    *(ForkSum*)(a.workspace + at.sum) = all;
  }
  fork_row(a, div, in_place, at, row, all, r, fours, source);
  settler.end(held);
  settle_rest(settler, r, fours);
  if (settler.foreign) flag_error(a.err, KVMI_ERR_BLOCK_ID);
}

// More rows: one workgroup plans them, the others read their rows' plans.  1024 rows of up to 500 blocks: 5.9
// and 15.9 us (some 6 of it the atomics).  Rows of up to 750 blocks, us a call with this launch or planned
// by every workgroup for itself: 128 rows 14.1 / 11.8, 256 15.8 / 13.8, 384 18.1 / 17.0, 512 18.8 / 18.2, 768
// 23.8 / 24.2, 1024 27.5 / 29.1; 256 keeps the other kernel's LDS at 9 KB a workgroup.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(kvmi_fork_args a, BlockOf div) {
  extern __shared__ int plan_lds[];
  __shared__ uint32_t wave_sums[3][kPlanThreads / 64], carry[3];
  const int R = a.rows, tid = threadIdx.x, head = gld(a.state), count = gld(a.state + 1);
  const ForkSpace at = fork_space(a.blocks, R, a.columns);
  const int turn = gld(a.workspace + at.turn);
  const ForkPlan f = plan_rows<kPlanThreads>(a, div, plan_lds);
  if (tid < 3) carry[tid] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < R; i0 += kPlanThreads) {
    const int i = i0 + tid;
    uint32_t v[3] = {0, 0, 0}, before[3];
    if (i < R) row_adds(f, div, a.block_size, i, v);
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      before[x] = wave_scan(v[x]);
      if ((tid & 63) == 63) wave_sums[x][tid >> 6] = before[x];
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      uint32_t s = carry[x];
      for (int w = 0; w < (tid >> 6); ++w) s = add_sat(s, wave_sums[x][w]);
      before[x] = add_sat(s, before[x]) - v[x];  // (a saturated sum is refused)
    }
    if (i < R) {
      const ForkRow row = row_of(f, div, a.block_size, i, before);
      uint4* const to = (uint4*)(a.workspace + at.rows + 12 * (int64_t)i);
#pragma unroll
      for (int w = 0; w < 3; ++w) gst(to + w, ((const uint4*)&row)[w]);
    }
    __syncthreads();
    if (tid < 3) {
      uint32_t s = carry[tid];
      for (int w = 0; w < kPlanThreads / 64; ++w) s = add_sat(s, wave_sums[tid][w]);
      carry[tid] = s;
    }
    __syncthreads();
  }
  if (tid == 0) {
    int32_t error;
    const ForkSum all = sum_of(a, head, count, turn, carry, *f.bad, &error);
    flag_error(a.err, error);
    *(ForkSum*)(a.workspace + at.sum) = all;
  }
}
__global__ __launch_bounds__(kThreads) void fork_rows_kernel(kvmi_fork_args a, BlockOf div, bool in_place) {
  __shared__ int list[kMostForkRows];
  const int R = a.rows, C = a.columns, r = blockIdx.x;
  const ForkSpace at = fork_space(a.blocks, R, C);
  const bool fours = in_fours(a, at, in_place);
  const int k = 4 * (blockIdx.y * kThreads + threadIdx.x);
  const ForkRow* const rows = (const ForkRow*)(a.workspace + at.rows);
  uint4 old = make_uint4(0, 0, 0, 0), source = old;
  if (fours && k < C) old = gld((const uint4*)(a.tables + (int64_t)r * C + k));
  const ForkRow row = rows[r];
  const ForkSum all = *(const ForkSum*)(a.workspace + at.sum);
  if (fours && k < C) source = gld((const uint4*)(a.tables + (int64_t)max(row.parent, 0) * C + k));
  Settler settler = settler_of(a, div, at, row, all.turn, list, [&](int i) { return rows[i].parent == r ? div(rows[i].kept) : -1; });
  Settled<4> held = four(old);
  if (fours && k < settler.have) settler.begin(k, held);
  fork_row(a, div, in_place, at, row, all, r, fours, source);
  settler.end(held);
  settle_rest(settler, r, fours);
  if (settler.foreign) flag_error(a.err, KVMI_ERR_BLOCK_ID);
}

// Workgroup g < ranges goes through 1024 block ids: their new shares, and the free ones behind the
// ring's last, after those of the ranges before.  The other workgroups bring rows that are made in
// place from the workspace to their table.  34,000 blocks 3.9 us, 100,000 4.9: loads, two sums over the
// workgroup, stores.
__global__ __launch_bounds__(kThreads) void fork_blocks_kernel(kvmi_fork_args a, int ranges, bool in_place) {
  __shared__ uint32_t sums[2][kWaves];
  const int N = a.blocks, tid = threadIdx.x, g = blockIdx.x;
  const ForkSpace at = fork_space(N, a.rows, a.columns);
  const ForkSum call = *(const ForkSum*)(a.workspace + at.sum);
  const int taken = call.taken;
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
  const int count = call.count < 0 ? 0 : min(call.count, N);
  const int32_t* const counts = a.workspace + at.counts + (call.turn ? at.counted : 0);
  int32_t* const others = a.workspace + at.counts + (call.turn ? 0 : at.counted);
  uint32_t held[4], word[4];  // (a refused call has counted, too)
  int shares[4];
  const int first = g * kRange + 4 * tid;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const bool in = first + x < N;
    held[x] = in ? gld((const uint32_t*)a.workspace + at.words + first + x) : 0;
    word[x] = taken < 0 ? 0 : held[x];
    shares[x] = in ? gld(a.shares + first + x) : 0;
  }
  uint32_t sum[2] = {0, 0};  // freed before this range, and in all
  for (int i = tid; i < at.counted; i += kThreads) {
    const uint32_t v = gld(counts + i);
    sum[1] += v;
    if (i < g * (kRange / kCounted)) sum[0] += v;
  }
  block_sums(sum, sums);
  uint32_t free = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) free += word[x] >> 16 && (int)(word[x] >> 16) > shares[x];
  uint32_t place[1] = {free};
  before_in_block(place, sums);
  place[0] += sum[0];
  const uint32_t tail = ring_at(call.head, count, N);
  bool lost = false;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if (first + x >= N) break;
    const int gone = (int)(word[x] >> 16), b = first + x;
    const int now = max(0, shares[x] + (int)(word[x] & 0xffffu) - gone);
    if (!in_place || now != shares[x]) a.out_shares[b] = now;
    if (held[x]) a.workspace[at.words + b] = 0;
    if (gone && gone > shares[x]) {
      if (place[0] < (uint32_t)(N - count))
        a.free_blocks[ring_at(tail, place[0], N)] = b;
      else
        lost = true;
      ++place[0];
    }
  }
  if (lost) flag_error(a.err, KVMI_ERR_LENGTH);
  const int mine = g * (kRange / kCounted) + tid;
  if (tid < kRange / kCounted && mine < at.counted) others[mine] = 0;
  if (g == 0 && tid == 0) {  // (the other workgroups have state and turn from `call`)
    a.workspace[at.turn] = !call.turn;
    const int back = min((int)sum[1], N - count);
    a.out_state[0] = taken < 0 ? a.state[0] : (int)ring_at(call.head, taken, N);
    a.out_state[1] = taken < 0 ? call.count : count - taken + back;
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
// aligned), eight loads of a thread before its stores.  200 blocks of 64 KB in 32 layers 150 to 160 us (5.2 to
// 5.6 TB/s read and written: memory); 24 pieces of 8 KB in 28 layers 8.3: the list, the base, the rows, the
// stores, one after the other.
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

// Four launches (three for small pools): marks, counts, places, names.  Each is a trip or two to memory: a
// pool of 65,536 with 512 rows 3.8 + 2.2 + 5.9 + 5.4 us, one of 1,024 with 16 rows 2.4 + 4.4 + 2.7.

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

// Pools of up to kSelf ids: every workgroup adds up all marks for itself (32 KB out of the L2 at the most)
// instead of reading counts that a launch before it has made.  A thread takes the same power of two of ids,
// 16 or more, so ranges begin with a thread.  16,384 blocks: a call in 13.5 us, 15.0 with the counts; 65,536:
// 18.8, 16.5 with them.
constexpr int kSelf = 16384, kSelfRanges = kSelf / kRange;
__device__ __forceinline__ void count_all(const uint8_t* space, const CompactSpace& at, int N, uint32_t (*sums)[kWaves],
                                          uint32_t (*ranges)[kSelfRanges + 1], uint32_t (&total)[2]) {
  int log2 = 4;
  while ((kThreads << log2) < N) ++log2;
  const int first = threadIdx.x << log2;
  uint32_t v[2] = {0, 0};
  for (int i = first; i < min(first + (1 << log2), N); i += 16) {  // (the marks reach to a multiple of 16)
    const uint4 h = gld((const uint4*)(space + at.held + i)), f = gld((const uint4*)(space + at.free + i));
    v[0] += __popc(h.x) + __popc(h.y) + __popc(h.z) + __popc(h.w);
    v[1] += __popc(h.x | f.x) + __popc(h.y | f.y) + __popc(h.z | f.z) + __popc(h.w | f.w);
  }
  total[0] = v[0];
  total[1] = v[1];
  before_in_block(v, sums);
  if (first % kRange == 0 && first < kSelf) {
    ranges[0][first / kRange] = v[0];
    ranges[1][first / kRange] = v[1];
  }
  if (threadIdx.x == kThreads - 1) {  // (ranges behind the last hold nothing)
    const int last = (kThreads << log2) / kRange;
    ranges[0][last] = v[0] + total[0];
    ranges[1][last] = v[1] + total[1];
  }
  block_sums(total, sums);
}

// Workgroup g: the places of 1024 ids among the held blocks and in the pool.  The pool's first n ids
// stay or are taken (n: held blocks), so the number of moves is that of the free ones among them:
// those of the ranges below the one where n falls, and some in it, which each looks up for itself.
__global__ __launch_bounds__(kThreads) void compact_rank_kernel(kvmi_compact_args a, int ranges) {
  __shared__ uint32_t sums[2][kWaves], starts[2][kSelfRanges + 1], mine[2], cut[3];
  const int N = a.blocks, tid = threadIdx.x, g = blockIdx.x, first = g * kRange + 4 * tid;
  const CompactSpace at = compact_space(N);
  uint8_t* const space = (uint8_t*)a.workspace;
  const uint32_t* const counts = (const uint32_t*)(space + at.counts);
  uint32_t free;
  const uint32_t held = marks_of(space, at, N, first, &free), pool = held | free;
  int shares[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) shares[x] = (held >> (8 * x) & 1) && first + x < N ? gld(a.shares + first + x) : 0;
  // held, and in the pool: in all, before this range, and before the one in which the pool's n-th id falls
  uint32_t total[2] = {0, 0};
  if (tid == 0) cut[0] = 0x7fffffff;
  if (N <= kSelf) {
    count_all(space, at, N, sums, starts, total);
    if (tid < ranges) {
      const uint32_t u = starts[1][tid];
      if (u < total[0] && starts[1][tid + 1] >= total[0]) {
        cut[0] = tid;
        cut[1] = starts[0][tid];
        cut[2] = u;
      }
      if (tid == g) {
        mine[0] = starts[0][g];
        mine[1] = u;
      }
    }
  } else {
    for (int i = tid; i < ranges; i += kThreads) {
      total[0] += gld(counts + 2 * i);
      total[1] += gld(counts + 2 * i + 1);
    }
    block_sums(total, sums);
    uint32_t carry[2] = {0, 0};
    for (int i0 = 0; i0 < ranges; i0 += kThreads) {
      const int i = i0 + tid;
      const uint32_t h = i < ranges ? gld(counts + 2 * i) : 0, u = i < ranges ? gld(counts + 2 * i + 1) : 0;
      uint32_t before[2] = {h, u};
      before_in_block(before, sums);
      before[0] += carry[0];
      before[1] += carry[1];
      if (i == g) {
        mine[0] = before[0];
        mine[1] = before[1];
      }
      if (before[1] < total[0] && before[1] + u >= total[0]) {
        cut[0] = i;
        cut[1] = before[0];
        cut[2] = before[1];
      }
      if (i0 + kThreads < ranges) {
        uint32_t all[2] = {h, u};
        block_sums(all, sums);
        carry[0] += all[0];
        carry[1] += all[1];
      }
    }
  }
  const uint32_t n = total[0];
  // this range's places; both counts fit half a word
  uint32_t place[1] = {(uint32_t)__popc(held) | (uint32_t)__popc(pool) << 16};
  before_in_block(place, sums);  // (its barriers are for `mine` and `cut` too)
  uint32_t h = mine[0] + (place[0] & 0xffffu), u = mine[1] + (place[0] >> 16);
  uint32_t moves = 0;
  if (cut[0] != 0x7fffffff) {
    uint32_t cut_free;
    const uint32_t cut_held = marks_of(space, at, N, cut[0] * kRange + 4 * tid, &cut_free), cut_pool = cut_held | cut_free;
    uint32_t rank[1] = {(uint32_t)__popc(cut_pool)};
    before_in_block(rank, sums);
    rank[0] += cut[2];
    uint32_t low[1] = {0};  // held in the range below the cut
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (!(cut_pool >> (8 * x) & 1)) continue;
      low[0] += rank[0] < n && (cut_held >> (8 * x) & 1);
      ++rank[0];
    }
    block_sums(low, sums);
    moves = n - cut[1] - low[0];
  }
  int32_t* const names = (int32_t*)(space + at.names);
  const uint32_t left = total[1] - n;  // free blocks afterwards
  int bits = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if (first + x >= N) break;
    const int b = first + x;
    const bool is_held = held >> (8 * x) & 1, in_pool = pool >> (8 * x) & 1;
    if (is_held && (free >> (8 * x) & 1)) bits |= KVMI_ERR_BLOCK_ID;
    const bool high = in_pool && u >= n, moved = high && is_held, taken = in_pool && !high && !is_held;
    const uint32_t i = h - (n - moves);  // of a block that moves
    gst(names + b, moved ? -1 - (int)i : b);
    if (!taken) gst(a.out_shares + b, moved ? 0 : shares[x]);  // (what is taken has those of the block that comes)
    if (taken) gst((int32_t*)(space + at.to) + (u - h), b);
    if (moved) gst((int32_t*)(space + at.from) + i, b);
    if (moved) gst((int32_t*)(space + at.shares) + i, shares[x]);
    if (high) gst(a.out_free + (u - n), b);
    if ((uint32_t)b >= left) gst(a.out_free + b, -1);
    h += is_held;
    u += in_pool;
  }
  flag_error(a.err, bits);
  if (g == 0 && tid == 0) {
    *(uint32_t*)(space + at.moves) = moves;
    a.out_state[0] = 0;
    a.out_state[1] = (int)left;
  }
}

// The rows under the new names; the list of moves, and the marks cleared.
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
  const int moves = gld((const int32_t*)(space + at.moves));
  const int first = (int)(blockIdx.x - rows) * kRange;
  for (int i = first + tid; i < min(N / 2, first + kRange); i += kThreads) {
    const bool moved = i < moves;
    const int b = moved ? gld(to + i) : -1;
    gst(a.copies + 3 * (int64_t)i, moved ? gld((const int32_t*)(space + at.from) + i) : -1);
    gst(a.copies + 3 * (int64_t)i + 1, b);
    gst(a.copies + 3 * (int64_t)i + 2, moved ? a.block_size : -1);
    if (moved) gst(a.out_shares + b, gld((const int32_t*)(space + at.shares) + i));
  }
  if (first + 4 * tid < N) {  // the marks are left zero for the next call
    gst((uint32_t*)(space + at.held + first + 4 * tid), 0u);
    gst((uint32_t*)(space + at.free + first + 4 * tid), 0u);
  }
}

}  // namespace
}  // namespace kvmi

extern "C" int64_t kvmi_fork_workspace_bytes(int32_t blocks, int32_t rows, int32_t columns) {
  if (blocks < 1 || blocks > kvmi::kMostBlocks || rows < 0 || columns < 1) return KVMI_EINVAL;
  return 4 * kvmi::fork_space(blocks, rows, columns).size;
}

extern "C" int kvmi_fork_tables(const kvmi_fork_args* args, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!args) return KVMI_EINVAL;
  const kvmi_fork_args& a = *args;
  if (a.rows < 0 || a.rows > kMostForkRows || a.columns < 1 || a.blocks < 1 || a.blocks > kMostBlocks ||
      a.block_size < 1 || a.max_tokens < 0 ||
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
  if (a.new_lengths == a.out_lengths || a.parents == a.out_lengths || (uintptr_t)a.workspace % 16 ||
      a.workspace_bytes < kvmi_fork_workspace_bytes(a.blocks, a.rows, a.columns))
    return KVMI_EINVAL;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t most = std::max<int64_t>((a.columns + 1023) / 1024, ((int64_t)a.max_tokens + 4095) / 4096);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(most, std::min(64, 2048 / a.rows)));
  const BlockOf div = block_of(a.block_size);
  const dim3 grid((unsigned)a.rows, (unsigned)parts);
  if (a.rows <= kFused) {
    hipLaunchKernelGGL(fork_fused_kernel, grid, dim3(kThreads), 0, st, a, div, in_place);
  } else {
    hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 32 * (size_t)a.rows + 4, st, a, div);
    hipLaunchKernelGGL(fork_rows_kernel, grid, dim3(kThreads), 0, st, a, div, in_place);
  }
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
  if (blocks < 1 || blocks > kvmi::kMostBlocks) return KVMI_EINVAL;
  return kvmi::compact_space(blocks).size;
}

extern "C" int kvmi_compact_tables(const kvmi_compact_args* args, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!args) return KVMI_EINVAL;
  const kvmi_compact_args& a = *args;
  if (a.rows < 0 || a.columns < 1 || a.blocks < 1 || a.blocks > kMostBlocks || a.block_size < 1) return KVMI_EINVAL;
  if ((int64_t)a.columns * a.block_size > kMostPlaces || (int64_t)a.blocks * a.block_size > 0x7fffffffLL ||
      (int64_t)a.columns * a.rows > 0x7fffffffLL)
    return KVMI_EINVAL;
  if ((a.rows && (!a.lengths || !a.tables || !a.out_tables)) || !a.shares || !a.free_blocks || !a.state ||
      !a.out_shares || !a.out_free || !a.out_state || (a.blocks > 1 && !a.copies) || !a.workspace)
    return KVMI_EINVAL;
  const bool in_place = a.out_shares == a.shares;
  if ((a.rows && in_place != (a.out_tables == a.tables)) || in_place != (a.out_free == a.free_blocks) ||
      in_place != (a.out_state == a.state) || (uintptr_t)a.workspace % 16 ||
      a.workspace_bytes < kvmi_compact_workspace_bytes(a.blocks))
    return KVMI_EINVAL;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int ranges = ranges_of(a.blocks), parts = std::min(64, (a.columns + 1023) / 1024);
  const int64_t rows = (int64_t)a.rows * parts;
  if (rows + ranges > 0x7fffffffLL) return KVMI_EINVAL;
  const BlockOf div = block_of(a.block_size);
  hipLaunchKernelGGL(compact_mark_kernel, dim3((unsigned)(rows + ranges)), dim3(kThreads), 0, st, a, div, parts);
  if (a.blocks > kSelf) hipLaunchKernelGGL(compact_count_kernel, dim3((unsigned)ranges), dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(compact_rank_kernel, dim3((unsigned)ranges), dim3(kThreads), 0, st, a, ranges);
  hipLaunchKernelGGL(compact_name_kernel, dim3((unsigned)(rows + ranges)), dim3(kThreads), 0, st, a, div, parts);
  return launched();
}
