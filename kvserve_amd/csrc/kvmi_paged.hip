// Decode-instance upkeep of the paged cache: block tables and slot maps from request
// lengths, new keys and values written by slot, accepted drafts kept.
#include "kvmi_common.hpp"

#include <algorithm>

namespace kvmi {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void flag_error(int32_t* err, int32_t bits) {
  if (err && bits) atomicOr(err, bits);
}

// Sum over the workgroup, given to every thread.
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* lds) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// ---------------------------------------------------------------- block tables
struct Need {  // what one request's change of length asks for
  int now, next, have, want;
  bool bad;
  __device__ int take() const { return want > have ? want - have : 0; }
  __device__ int give() const { return have > want ? have - want : 0; }
  __device__ int tokens() const { return next > now ? next - now : 0; }
};
__device__ __forceinline__ Need need_of(const kvmi_tables_args& a, const BlockOf& div, int now, int next) {
  Need n;
  const int top = a.columns * a.block_size;
  n.bad = (uint32_t)now > (uint32_t)top || (uint32_t)next > (uint32_t)top;
  if (n.bad) next = now = now < 0 ? 0 : now > top ? top : now;
  n.now = now;
  n.next = next;
  n.have = now ? div(now - 1) + 1 : 0;
  n.want = next ? div(next - 1) + 1 : 0;
  return n;
}
__device__ __forceinline__ Need need_of(const kvmi_tables_args& a, const BlockOf& div, int r) {
  return need_of(a, div, a.lengths[r], a.new_lengths[r]);
}
// Place of the i-th entry behind `base` in a ring of N (base < N, i <= N).
__device__ __forceinline__ uint32_t ring_at(uint32_t base, uint32_t i, uint32_t N) {
  const uint32_t x = base + i;
  return x < N ? x : x - N;
}

// Workgroup (r, y) makes part y of request r's table row and slots.  No workgroup waits for
// another: each adds up what the requests before its own ask for and give back (R lengths out
// of the L2, a few microseconds less than a scan kernel and a second launch would take), and
// from those sums it knows its place in the ring, so that a slot needs no table entry that
// another workgroup writes.  A ring has room for every block of the pool, so the places behind
// the last free block never reach the head's: blocks returned here are not read here.  In a ring
// that has no such room, blocks past its free places are dropped and reported, not written over
// the free ones that other workgroups read.
// 1024 requests of all sorts, rows of 1024, 420 Ki new tokens: 8.8 us (1.8 by its 8.8 MB: bound by
// instructions and the chain lengths, ring, stores); 256 that grow by 8 tokens: 4.2.  With lengths
// and state written over, where every workgroup adds to the ticket and the last one walks all
// requests again, 8.0 for those 256 and 32 for 1024 that grow by 33 (7.4 into other tensors).
__global__ __launch_bounds__(kThreads) void tables_kernel(kvmi_tables_args a, BlockOf div) {
  __shared__ uint32_t sums[3][4];
  __shared__ int64_t lds[4];
  __shared__ int last;
  const int r = blockIdx.x, tid = threadIdx.x;
  const Need n = need_of(a, div, r);
  const int N = a.ring;
  const int head = (int)((uint32_t)a.state[0] % (uint32_t)N);
  const int given = a.state[1], count = given < 0 ? 0 : given > N ? N : given;

  // What the requests before this one take, give back and grow by.  Blocks add up to less than
  // the table's entries, 2^31; tokens stay at 2^32 - 1, past any slot map.
  uint32_t before[3] = {0, 0, 0};
  for (int i0 = 0; i0 < r; i0 += 4 * kThreads) {  // four loads at a time
    int now[4], next[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = min(i0 + u * kThreads + tid, r - 1);
      if (i0 + u * kThreads < r) {
        now[u] = gld(a.lengths + i);
        next[u] = gld(a.new_lengths + i);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u * kThreads < r) {
        const Need m = need_of(a, div, now[u], next[u]);
        if (i0 + u * kThreads + tid < r) {
          before[0] += m.take();
          before[1] += m.give();
          before[2] = add_sat(before[2], m.tokens());
        }
      }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    before[0] += __shfl_xor(before[0], d, 64);
    before[1] += __shfl_xor(before[1], d, 64);
    before[2] = add_sat(before[2], __shfl_xor(before[2], d, 64));
  }
  if ((tid & 63) == 0)
#pragma unroll
    for (int x = 0; x < 3; ++x) sums[x][tid >> 6] = before[x];
  __syncthreads();
  const int64_t take = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
  const int64_t give = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
  const int64_t tokens = add_sat(add_sat(sums[2][0], sums[2][1]), add_sat(sums[2][2], sums[2][3]));

  const bool fits = take + n.take() <= count;
  const bool granted = fits || n.take() == 0;
  const int keep = granted ? n.want : n.have;
  const bool in_place = a.out_tables == a.tables;
  const int32_t* const old = a.tables + (int64_t)r * a.columns;
  int32_t* const out = a.out_tables + (int64_t)r * a.columns;
  const int step = kThreads * gridDim.y, lane = blockIdx.y * kThreads + tid;
  // where this request takes blocks (looked at only where it fits: take <= N) and gives them back
  const uint32_t from = ring_at(head, fits ? (uint32_t)take : 0, N);
  const uint32_t to = (uint32_t)((uint64_t)(head + (int64_t)count + give) % (uint32_t)N);
  const int back = keep + (int)max((int64_t)0, min((int64_t)n.have - keep, N - count - give));  // keep .. back - 1

  // the table row: blocks kept, blocks taken, and -1 behind them; the blocks given back go
  // behind the last free one
  const int lo = in_place ? min(n.have, keep) : 0;
  const int hi = in_place ? max(n.have, keep) : a.columns;
  auto entry = [&](int k) -> int32_t {  // the row's entry k
    if (k < min(n.have, keep)) return gld(old + k);
    if (k < keep) return gld(a.free_blocks + ring_at(from, k - n.have, N));
    return -1;
  };
  if (!in_place && (a.columns & 3) == 0 && (((uintptr_t)a.tables | (uintptr_t)a.out_tables) & 15) == 0) {
    // four entries a thread: most of a row is kept, or -1
    for (int k = 4 * lane; k < a.columns; k += 4 * step) {
      uint4 v = make_uint4(~0u, ~0u, ~0u, ~0u);
      if (k + 4 <= min(n.have, keep)) {
        v = gld((const uint4*)(old + k));
      } else if (k < keep) {
        v.x = entry(k);
        v.y = entry(k + 1);
        v.z = entry(k + 2);
        v.w = entry(k + 3);
      }
      gst((uint4*)(out + k), v);
    }
    for (int k = keep + lane; k < back; k += step) gst(a.free_blocks + ring_at(to, k - keep, N), gld(old + k));
  } else {
    for (int k = lo + lane; k < hi; k += step) {
      const int32_t had = k >= keep && k < back ? gld(old + k) : -1;
      if (k >= keep && k < back) gst(a.free_blocks + ring_at(to, k - keep, N), had);
      gst(out + k, entry(k));
    }
  }

  // the new tokens' slots
  const int64_t room = a.max_tokens - tokens;
  const int grown = room <= 0 ? 0 : (int)min((int64_t)n.tokens(), room);
  auto slot_of = [&](int i) -> int64_t {
    const int p = n.now + i, k = div(p);
    const int32_t id = gld(k < n.have ? old + k : a.free_blocks + ring_at(from, k - n.have, N));
    return (int64_t)id * a.block_size + (p - k * a.block_size);
  };
  int64_t* const slots = a.slots + tokens;
  int i = lane;
  if (granted)  // all of a thread's loads before its stores, where it has several
    for (; i + 3 * (int64_t)step < grown; i += 4 * step) {
      int64_t v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = slot_of(i + u * step);
#pragma unroll
      for (int u = 0; u < 4; ++u) gst(slots + i + u * step, v[u]);
    }
  for (; i < grown; i += step) gst(slots + i, granted ? slot_of(i) : (int64_t)-1);
  const int64_t upto = tokens + n.tokens();
  if (r == a.requests - 1)
    for (int64_t k = upto + lane; k < a.max_tokens; k += step) gst(a.slots + k, (int64_t)-1);
  if (blockIdx.y == 0 && tid == 0) {
    if (r == 0) a.starts[0] = 0;
    a.starts[r + 1] = upto > 0x7fffffff ? 0x7fffffff : (int)upto;
    flag_error(a.err, (granted ? 0 : KVMI_ERR_NO_BLOCKS) | (n.bad || upto > a.max_tokens ? KVMI_ERR_LENGTH : 0));
  }

  // Lengths and ring state.  They may lie over the inputs that other workgroups still read:
  // then the last workgroup to arrive here writes them all.  Else each request's first
  // workgroup writes its length, and the last request's the state.
  const bool over = a.out_lengths == a.lengths;
  if (over) {
    __syncthreads();
    if (tid == 0) last = atomicAdd(a.ticket, 1) == (int)(gridDim.x * gridDim.y) - 1;
    __syncthreads();
    if (!last) return;
  } else {
    if (blockIdx.y) return;
    if (tid == 0) a.out_lengths[r] = granted ? (n.bad ? a.lengths[r] : n.next) : n.now;
    if (r != a.requests - 1) return;
  }
  // taken = the asked-for sum up to the last request that fits; only where blocks ran short,
  // or where all lengths are still to be written, are the sums needed request by request
  const int64_t all_give = give + (granted ? n.give() : 0);
  int64_t taken = take + n.take(), returned = all_give;
  if (over || !fits) {
    int64_t asked = 0, fit = 0;
    returned = 0;
    for (int base = 0; base < a.requests; base += kThreads) {
      const int i = base + tid;
      Need m{};
      if (i < a.requests) m = need_of(a, div, i);
      // inclusive sum of take over this piece: within the wave, then over the waves
      int64_t s = m.take();
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int64_t t = __shfl_up(s, d, 64);
        if ((tid & 63) >= d) s += t;
      }
      __syncthreads();
      if ((tid & 63) == 63) lds[tid >> 6] = s;
      __syncthreads();
      int64_t carry = asked;
      for (int w = 0; w < (tid >> 6); ++w) carry += lds[w];
      const int64_t piece = lds[0] + lds[1] + lds[2] + lds[3];
      s += carry;
      const bool ok = s <= count;
      if (over && i < a.requests && !m.bad) a.out_lengths[i] = ok || m.take() == 0 ? m.next : m.now;
      fit += i < a.requests && ok ? m.take() : 0;
      returned += m.give();
      asked += piece;
    }
    taken = block_sum(fit, lds);
    returned = block_sum(returned, lds);
  }
  if (tid == 0) {
    const int64_t spare = N - count;
    if (given != count || returned > spare) flag_error(a.err, KVMI_ERR_LENGTH);
    a.out_state[0] = (int)((head + taken) % N);
    a.out_state[1] = (int)(count - taken + min(returned, spare));
    if (over) *a.ticket = 0;
  }
}

// ---------------------------------------------------------------- slot writes
struct WriteArgs {
  kvmi_cache cache;
  const uint16_t* rows[2];
  int64_t token_stride[2], head_stride[2];
  const int64_t* slots;
  int64_t tokens;
  int32_t* err;
  int lanes_log2;  // lanes of a token, a power of two up to the workgroup
  BlockOf block, head;  // by the block size, by a head's units
};

// A group of 2^lanes_log2 lanes copies one token's K and V rows in units of V (16 bytes, or 2
// where a stride or an address is not aligned): copies, bound by memory.  16384 tokens of 8 x 128:
// 28.6 us out of memory (4.7 TB/s read and written), 21.4 out of the caches; 96 tokens: 2.5.
template <class V>
__global__ __launch_bounds__(kThreads) void write_kernel(WriteArgs a) {
  constexpr int U = sizeof(V) / 2;
  const int per_head = a.cache.head_dim / U, per_part = a.cache.num_heads * per_head;
  const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int64_t tok = ((int64_t)blockIdx.x << (8 - a.lanes_log2)) + (threadIdx.x >> a.lanes_log2);
  if (tok >= a.tokens) return;
  const int64_t slot = a.slots[tok];
  const int S = a.cache.block_size;
  if (slot < 0 || slot >= (int64_t)a.cache.num_blocks * S) {
    if (slot != -1 && lane == 0) flag_error(a.err, KVMI_ERR_BLOCK_ID);
    return;
  }
  const int block = a.block((int)slot);
  const int64_t place = block * a.cache.block_stride +
                        (int64_t)((int)slot - block * S) * (a.cache.num_heads * a.cache.head_dim);
  for (int p = lane; p < 2 * per_part; p += lanes) {
    const int part = p >= per_part, q = p - part * per_part;
    const int head = a.head(q);
    const uint16_t* src = a.rows[part] + tok * a.token_stride[part] + head * a.head_stride[part] +
                          (int64_t)(q - head * per_head) * U;
    uint16_t* dst = (uint16_t*)a.cache.base + part * a.cache.part_stride + place + (int64_t)q * U;
    gst((V*)dst, gld((const V*)src));
  }
}

// ---------------------------------------------------------------- kept drafts
struct KeepArgs {
  kvmi_cache cache;
  void* const* bases;
  const int32_t* tables;
  const int32_t* lengths;
  const int32_t* accepted;
  int32_t* out_lengths;
  int32_t* err;
  int columns, width, layers;
  BlockOf block;
};
constexpr int kMaxPath = 1024;

// Lane i's value, i the same for all; lanes that have left count too, unlike in a shuffle.
__device__ __forceinline__ int64_t lane_value(int64_t v, int i) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)v, i) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32);
}

// Workgroup (request, layer).  The path is checked as a whole before anything moves.  A thread
// owns one 16-byte (or 2-byte) column of the row and walks the path in order, so no thread waits
// for another: path[i] >= i and the path increases, hence a row is read before, or in the same
// step as, it is overwritten.  Bound by its chain of loads (path, tables, rows; 28 layers of one
// request 2.9 us, 32 layers of 32 requests 8.7): a path of up to 64 is checked by every wave for
// itself, a draft a lane, without a barrier.
template <class V, bool SHORT>
__global__ __launch_bounds__(kThreads) void keep_kernel(KeepArgs a) {
  constexpr int U = sizeof(V) / 2, kStep = 8;
  __shared__ int64_t src[SHORT ? 1 : kMaxPath], dst[SHORT ? 1 : kMaxPath];
  __shared__ int count;
  const int r = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int32_t* path = a.accepted + (int64_t)r * a.width;
  const int32_t* const table = a.tables + (int64_t)r * a.columns;
  const int S = a.cache.block_size;
  const int64_t base = a.lengths[r], top = (int64_t)a.columns * S;
  const int64_t row = (int64_t)a.cache.num_heads * a.cache.head_dim;
  int bad = base < 0 || base > top ? KVMI_ERR_LENGTH : 0, n;
  int64_t lane_src = 0, lane_dst = 0;
  // draft i of the path, `before` the one ahead of it: where it lies and where it goes
  auto place = [&](int i, int draft, int before, int64_t* from_row, int64_t* to_row) {
    const int64_t from = base + draft, to = base + i;
    // (draft < i: the path does not increase, and `to` may lie behind the table's row)
    if ((i && draft <= before) || draft < i || from >= top) {
      bad |= KVMI_ERR_LENGTH;
      return;
    }
    const int fc = a.block((int)from), tc = a.block((int)to);
    const int32_t fb = gld(table + fc), tb = gld(table + tc);
    if (fb < 0 || fb >= a.cache.num_blocks || tb < 0 || tb >= a.cache.num_blocks) bad |= KVMI_ERR_BLOCK_ID;
    *from_row = (int64_t)fb * a.cache.block_stride + (from - (int64_t)fc * S) * row;
    *to_row = (int64_t)tb * a.cache.block_stride + (to - (int64_t)tc * S) * row;
  };
  if constexpr (SHORT) {
    const int draft = lane < a.width ? gld(path + lane) : -1, before = __shfl_up(draft, 1, 64);
    const uint64_t ends = __ballot(draft < 0);
    n = ends ? __builtin_ctzll(ends) : 64;
    if (!bad && lane < n) place(lane, draft, before, &lane_src, &lane_dst);
    if (bad && layer == 0 && tid < 64) flag_error(a.err, bad);
    bad = __ballot(bad) != 0;
  } else {
    if (tid == 0) count = a.width;
    __syncthreads();
    for (int i = tid; i < a.width; i += kThreads)
      if (path[i] < 0) atomicMin(&count, i);
    __syncthreads();
    n = count;
    if (!bad)
      for (int i = tid; i < n; i += kThreads) place(i, path[i], i ? path[i - 1] : -1, &src[i], &dst[i]);
    if (bad && layer == 0) flag_error(a.err, bad);
    bad = __syncthreads_or(bad);
  }
  if (layer == 0 && tid == 0) a.out_lengths[r] = (int)base + (bad ? 0 : n);
  if (bad) return;
  auto from_row = [&](int i) -> int64_t { return SHORT ? lane_value(lane_src, i) : src[i]; };
  auto to_row = [&](int i) -> int64_t { return SHORT ? lane_value(lane_dst, i) : dst[i]; };
  const int per_part = a.cache.num_heads * a.cache.head_dim / U, all = 2 * per_part;
  const int64_t layer_base = (int64_t)(uintptr_t)gld((const int64_t*)a.bases + layer);
  for (int p0 = 0; p0 < all; p0 += kThreads) {
    const int p = p0 + tid, part = p >= per_part;
    uint16_t* col = (uint16_t*)layer_base + part * a.cache.part_stride + (int64_t)(p - part * per_part) * U;
    for (int i0 = 0; i0 < n; i0 += kStep) {
      V held[kStep];
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        if (i0 + i >= n) break;
        const int64_t from = from_row(i0 + i);
        if (p < all && from != to_row(i0 + i)) held[i] = gld((const V*)(col + from));
      }
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        if (i0 + i >= n) break;
        const int64_t to = to_row(i0 + i);
        if (p < all && from_row(i0 + i) != to) gst((V*)(col + to), held[i]);
      }
    }
  }
}

bool cache_ok(const kvmi_cache* c, bool base) {
  return c && (!base || c->base) && c->num_blocks >= 1 && c->block_size >= 1 && c->num_heads >= 1 && c->head_dim >= 1 &&
         c->part_stride >= 0 && c->block_stride >= (int64_t)c->block_size * c->num_heads * c->head_dim &&
         (int64_t)c->num_blocks * c->block_size < 0x7fffffffLL && (int64_t)c->num_heads * c->head_dim < (1 << 24);
}
bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
bool strides16(const kvmi_cache* c) {
  return c->head_dim % 8 == 0 && c->part_stride % 8 == 0 && c->block_stride % 8 == 0;
}
int launched() { return hipGetLastError() == hipSuccess ? KVMI_OK : KVMI_ELAUNCH; }

}  // namespace
}  // namespace kvmi

extern "C" int kvmi_build_tables(const kvmi_tables_args* args, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!args) return KVMI_EINVAL;
  const kvmi_tables_args& a = *args;
  if (a.requests < 0 || a.columns < 1 || a.ring < 1 || a.block_size < 1 || a.max_tokens < 0) return KVMI_EINVAL;
  if ((int64_t)a.columns * a.block_size > kMostPlaces || (int64_t)a.ring * a.block_size > 0x7fffffffLL ||
      (int64_t)a.columns * a.requests > 0x7fffffffLL)
    return KVMI_EINVAL;
  if (a.requests == 0) return KVMI_OK;
  if (!a.lengths || !a.new_lengths || !a.tables || !a.free_blocks || !a.state || !a.out_tables || !a.out_lengths ||
      !a.out_state || !a.starts || (a.max_tokens && !a.slots))
    return KVMI_EINVAL;
  const bool over = a.out_lengths == a.lengths;
  if (over != (a.out_state == a.state) || (over && !a.ticket) || a.new_lengths == a.out_lengths) return KVMI_EINVAL;
  // One request may own most of the tokens: where the requests alone do not fill the chip,
  // several workgroups share one, 4096 slots each.  Every part adds up the requests before its
  // own again, so there are no more than that needs (64 parts of 1024 requests took 153 us).
  const int64_t parts = std::max<int64_t>(
      1, std::min<int64_t>(((int64_t)a.max_tokens + 4095) / 4096, std::min(64, 2048 / a.requests)));
  hipLaunchKernelGGL(tables_kernel, dim3((unsigned)a.requests, (unsigned)parts), dim3(kThreads), 0,
                     reinterpret_cast<hipStream_t>(stream), a, block_of(a.block_size));
  return launched();
}

extern "C" int kvmi_write_kv(const kvmi_cache* cache, const void* key, const void* value, int64_t key_token_stride,
                             int64_t key_head_stride, int64_t value_token_stride, int64_t value_head_stride,
                             const int64_t* slots, int64_t tokens, int32_t* err, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!cache_ok(cache, true) || tokens < 0) return KVMI_EINVAL;
  if (tokens == 0) return KVMI_OK;
  if (!key || !value || !slots) return KVMI_EINVAL;
  WriteArgs a{*cache,
              {(const uint16_t*)key, (const uint16_t*)value},
              {key_token_stride, value_token_stride},
              {key_head_stride, value_head_stride},
              slots,
              tokens,
              err,
              8,
              block_of(cache->block_size),
              {}};
  const bool wide = strides16(cache) && aligned16(cache->base) && aligned16(key) && aligned16(value) &&
                    key_token_stride % 8 == 0 && key_head_stride % 8 == 0 && value_token_stride % 8 == 0 &&
                    value_head_stride % 8 == 0;
  const int units = 2 * cache->num_heads * cache->head_dim / (wide ? 8 : 1);
  a.head = block_of(wide ? cache->head_dim / 8 : cache->head_dim);
  while (a.lanes_log2 > 0 && (1 << (a.lanes_log2 - 1)) >= units) --a.lanes_log2;
  const int64_t per_wg = kThreads >> a.lanes_log2, grid = (tokens + per_wg - 1) / per_wg;
  if (grid > 0x7fffffffLL) return KVMI_EINVAL;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (wide)
    hipLaunchKernelGGL((write_kernel<uint4>), dim3((unsigned)grid), dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((write_kernel<uint16_t>), dim3((unsigned)grid), dim3(kThreads), 0, st, a);
  return launched();
}

extern "C" int kvmi_keep_drafts(const kvmi_cache* cache, void* const* bases, int32_t layers, const int32_t* tables,
                                int32_t columns, const int32_t* lengths, const int32_t* accepted, int32_t requests,
                                int32_t width, int32_t* out_lengths, int32_t* err, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!cache_ok(cache, false) || layers < 1 || layers > 65535 || columns < 1 || requests < 0 || width < 0 ||
      width > kMaxPath || (int64_t)columns * cache->block_size > kMostPlaces)
    return KVMI_EINVAL;
  if (requests == 0) return KVMI_OK;
  if (!bases || !tables || !lengths || !out_lengths || (width && !accepted) || lengths == out_lengths)
    return KVMI_EINVAL;
  KeepArgs a{*cache, bases, tables, lengths, accepted, out_lengths, err, columns, width, layers,
             block_of(cache->block_size)};
  const dim3 grid((unsigned)requests, (unsigned)layers);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // `cache->base` tells how the bases are aligned: the caller passes the OR of all of them
  const bool wide = strides16(cache) && aligned16(cache->base);
  if (width <= 64 && wide)
    hipLaunchKernelGGL((keep_kernel<uint4, true>), grid, dim3(kThreads), 0, st, a);
  else if (width <= 64)
    hipLaunchKernelGGL((keep_kernel<uint16_t, true>), grid, dim3(kThreads), 0, st, a);
  else if (wide)
    hipLaunchKernelGGL((keep_kernel<uint4, false>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((keep_kernel<uint16_t, false>), grid, dim3(kThreads), 0, st, a);
  return launched();
}
