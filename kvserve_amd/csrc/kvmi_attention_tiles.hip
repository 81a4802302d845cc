// Attention over the paged cache for many rows: tiles of 128 or 256 query rows against 64 keys.
//
// The rows of a KV head are its queries' heads, row m = query m / G, head m % G.  A wave holds
// 32 rows as the columns of its matrix products:
//   S^T = K Q^T     [64 keys][32 rows], operands K (LDS, 16 bytes a lane) and Q (registers)
//   O^T += V^T P^T  [D][32 rows], V^T by transposing reads of V's rows in LDS
// so that a lane has half of one row's scores, the softmax needs one exchange between the two
// halves of the wave, and the scores, rounded to the type, are the second product's operand
// where they lie: its key order within 16 is the one in which the first product left them.
//
// Work: 64 products of 32x32x16 a wave and tile at 128 channels, 2048 cycles of the matrix unit
// for the two waves of a SIMD, against about 135 vector instructions and 32 exponentials each.  A
// prompt of 8192 tokens, 32 heads over 8, 128 channels runs in 564 us (0.98 PFLOP/s, the matrix
// unit busy 45 % of the time; 64 channels: 0.80, 192: 0.74, 256: 0.59), 8 trees of 64 drafts with 8
// heads a KV head over 28 Ki tokens in 569 us (856 TFLOP/s), 96 trees of 26 drafts with 7 heads over
// 200 to 2000 tokens of 64 channels in 55 us.  Bound by issue and latency of two waves a SIMD (three
// at 64 channels); where few workgroups are left, by one's chain of tiles, 1.0 (64 channels) to
// 1.35 us (128) each.
#include "kvmi_attention.hpp"

namespace kvmi {
namespace {

constexpr int kKeys = 64;
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u32x2v read_transposed(const uint8_t* p) {
  return __builtin_bit_cast(
      u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

__device__ __forceinline__ void to_lds(const uint16_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((const KVMI_GLOBAL void*)from, (__attribute__((address_space(3))) void*)to, 16, 0,
                                   0);
}

// The order of a product's N instructions: AHEAD of their operands, READS reads of LDS each, are
// on their way before the first, then one more behind each.  (Left to itself the scheduler reads
// two and waits for both: 5 % slower.)
template <int N, int READS, int AHEAD>
__device__ __forceinline__ void interleave() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
  for (int k = 0; k < N - AHEAD; ++k) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x8, AHEAD, 0);
}

// Where chunk c (8 channels) of a key's row lies in its row in LDS.  The rows are PC chunks
// without gaps, since loads that go straight to LDS write 1 KiB in order, and are turned so that
// the reads meet every bank once: K's, one chunk of 16 keys, by single chunks, V's, 4 chunks of
// 4 keys, by 4.
template <int PC>
struct Turn {
  static constexpr int kPer = PC % 16 == 0 ? 16 : PC % 8 == 0 ? 8 : 4;  // gcd(PC, 16)
  static constexpr bool kPow2 = (PC & (PC - 1)) == 0;
  static __device__ __forceinline__ int key(int row) { return row / (16 / kPer) % kPer; }
  static __device__ __forceinline__ int value(int row) { return kPer < 8 ? 0 : kPer == 8 ? row / 2 % 2 * 4 : row % 4 * 4; }
  static __device__ __forceinline__ int place(int c, int turn) {
    if (kPow2) return c ^ turn;
    return c + turn >= PC ? c + turn - PC : c + turn;
  }
  static __device__ __forceinline__ int chunk(int place, int turn) {
    if (kPow2) return place ^ turn;
    return place < turn ? place - turn + PC : place - turn;
  }
};

// NT: 32-channel tiles of a head, D <= 32 * NT.
// WHOLE: D == 32 * NT, no channels to leave out.
// W: waves, of 32 rows each.
template <int DT, int NT, bool WHOLE, int W>
__global__ __launch_bounds__(64 * W, NT <= 4 ? 2 : 1) void attend_tiles_kernel(kvmi_attention_args a, AttendPlan plan) {
  constexpr int PC = 4 * NT, RS = 16 * PC, kPart = kKeys * RS;  // chunks and bytes of a row, bytes of a tile
  using T = Turn<PC>;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kPart];  // K and V of two tiles
  // of tile t in place t % 8 each key's offset in the cache, in place t % 2 the keys with a value
  // that is not finite
  __shared__ int64_t offs[8][kKeys];
  __shared__ uint32_t odd[2][2];

  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int threads = 64 * W, kRows = 32 * W, NP = PC / W;  // NP: a wave's instructions to load a K or V tile
  // Workgroups go to the XCDs in turn: all of a request's KV head go to one, one after the other,
  // so that its L2 has their keys (trees of 7 x 26 rows 56.7 -> 54.2 us); the last rows, which see
  // the most, first.
  const int per_pair = plan.row_tiles * plan.splits, in_xcd = blockIdx.x >> 3, nth = plan.tiles(in_xcd);
  const int pair = nth * 8 + (blockIdx.x & 7), y = in_xcd - nth * per_pair, r = plan.heads(pair);
  if (r >= a.requests) return;
  const int head = pair - r * a.cache.num_heads, part = y / plan.row_tiles;
  const int tile = plan.row_tiles - 1 - (y - part * plan.row_tiles);
  const Request q = request_of(a, r, tid == 0);
  const int D = a.cache.head_dim, H = a.cache.num_heads, G = a.query_heads / H;
  const int M = min(q.queries, a.max_query) * G, m0 = tile * kRows;
  if (m0 >= M) return;
  const int parts = parts_of(plan, q.length);
  if (part >= parts) return;
  const uint64_t* const masks = a.mask;
  const uint16_t* const keys = (const uint16_t*)a.cache.base + head * D;
  const uint16_t* const values = keys + a.cache.part_stride;

  // keys that any row of the workgroup sees end at `end`; those before `all` are seen by all
  const int last_row = min(m0 + kRows, M) - 1;
  const int end = masks ? q.length : min(q.length, q.prefix + plan.group(last_row) + 1);
  const int all = masks ? q.prefix : q.prefix + plan.group(m0) + 1;
  const int w0 = m0 + 32 * wave;
  const int w_all = masks ? q.prefix : q.prefix + plan.group(w0) + 1;
  const int tiles = (q.length + kKeys - 1) / kKeys;
  const int t0 = part_begin(tiles, part, parts);
  const int t1 = min(part_begin(tiles, part + 1, parts), (end + kKeys - 1) / kKeys);
  const int hiding = min(all, end) >> 6;  // the first tile with a key that some row does not see
  // this wave's: its rows see nothing from tile w1 on
  const int w_end = masks ? end : min(end, q.prefix + plan.group(min(w0 + 31, M - 1)) + 1);
  const int w1 = w0 >= M ? t0 : min(t1, (w_end + kKeys - 1) / kKeys), w_hiding = min(w_all, q.length) >> 6;

  const float c = a.scale * kLog2e;
  float mx = -INFINITY, l = 0;
  f32x16 o[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int x = 0; x < 16; ++x) o[n][x] = 0;

  // Every 4th tile each of the first 4 waves looks one of the next 4 tiles' keys up, a key a lane; the ids are
  // loaded ahead of a tile's loads, and waited for without waiting for those.
  const int32_t* const table = a.tables + (int64_t)r * a.columns;
  int place = 0, id = 0;
  auto look_up = [&](int t) {
    const int p = (t + wave) * kKeys + lane, at = plan.block(p < end ? p : 0);
    place = p < end ? p - at * a.cache.block_size : 0;
    id = gld(table + at);
  };
  auto note = [&](int t) { offs[(t + wave) & 7][lane] = row_offset(a, id, place); };
  const bool looks = W == 4 || wave < 4;
  if (t0 < t1 && looks) look_up(t0);

  // this lane's row
  const int m = min(w0 + col, M - 1), qi = plan.group(m), qh = head * G + m - qi * G;
  const int64_t row = q.first + qi;
  const uint64_t* const mask = masks ? masks + row * a.mask_words : nullptr;
  u32x4v qf[2 * NT];
  {
    const uint16_t* qp = (const uint16_t*)a.query + row * a.query_token_stride + qh * a.query_head_stride;
#pragma unroll
    for (int k = 0; k < 2 * NT; ++k) {
      const int d = 16 * k + 8 * half;
      qf[k] = d < D ? ld16(qp + d) : u32x4v{0, 0, 0, 0};
    }
  }

  // pieces of 16 bytes in the order of LDS, 64 an instruction; NT instructions of K's and of V's
  // a wave where there are 4 waves
  auto load = [&](int t) {
    uint8_t* const kb = lds + (t & 1) * 2 * kPart + wave * 1024;
    int64_t off[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) off[k] = offs[t & 7][((k * W + wave) * 64 + lane) / PC];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int idx = (k * W + wave) * 64 + lane, key = idx / PC, at = idx - key * PC;
      const int ck = T::chunk(at, T::key(key)), cv = T::chunk(at, T::value(key));
      if (WHOLE || ck * 8 < D) to_lds(keys + ck * 8 + off[k], kb + k * W * 1024);
      if (WHOLE || cv * 8 < D) to_lds(values + cv * 8 + off[k], kb + kPart + k * W * 1024);
    }
  };

  if (t0 < t1) {
    if (!WHOLE) {  // channels behind the head's are zero once and for all
      for (int x = tid; x < 4 * kKeys * PC; x += threads) {
        const int row = x / PC, place = x - row * PC, key = row & 63;
        if (T::chunk(place, row & 64 ? T::value(key) : T::key(key)) * 8 >= D)
          *(u32x4v*)(lds + x * 16) = u32x4v{0, 0, 0, 0};
      }
    }
    if (tid < 4) odd[tid >> 1][tid & 1] = 0;
    if (looks) note(t0);
    __syncthreads();
    load(t0);
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < 2 * NT; ++k) arrive(qf[k]);
  for (int t = t0; t < t1; ++t) {
    const bool look = looks && ((t - t0) & 3) == 0;
    if (look) look_up(t + 4);
    // (two pairs of waves a SIMD, W = 8, all wait at one barrier: their loads go behind the first
    // product's reads, 5 % faster; two workgroups of 4 waves, which run apart, are 5 % slower so)
    if (t + 1 < t1 && (W == 4 || t >= w1)) load(t + 1);
    uint32_t bad0 = 0, bad1 = 0;
    if (t >= hiding) {
      // some row does not see some key here: its weight is zero, and so must its product be.
      // Values that are not finite leave the tile, and go to the rows that see them below.
      uint8_t* const vb = lds + (t & 1) * 2 * kPart + kPart;
#pragma unroll 1
      for (int x = tid; x < kKeys * PC; x += threads) {
        const int key = x / PC;
        const u32x4v v = *(const u32x4v*)(vb + x * 16);
        u32x4v f = {0, 0, 0, 0};
        if (t * kKeys + key < end) {
#pragma unroll
          for (int y = 0; y < 4; ++y) f[y] = finite2<DT>(v[y]);
          if (f[0] != v[0] || f[1] != v[1] || f[2] != v[2] || f[3] != v[3])
            atomicOr(&odd[t & 1][key >> 5], 1u << (key & 31));
        }
        *(u32x4v*)(vb + x * 16) = f;
      }
      __syncthreads();
      bad0 = __builtin_amdgcn_readfirstlane(odd[t & 1][0]);
      bad1 = __builtin_amdgcn_readfirstlane(odd[t & 1][1]);
      if (tid < 2) odd[(t + 1) & 1][tid] = 0;
    }
    const int p0 = t * kKeys;
    if (t < w1) {
      const uint8_t* const kb = lds + (t & 1) * 2 * kPart;
      const uint8_t* const vb = kb + kPart;
      f32x16 s[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int x = 0; x < 16; ++x) s[b][x] = 0;
#pragma unroll
      for (int k = 0; k < 2 * NT; ++k) {
        const uint8_t* const kp = kb + col * RS + T::place(2 * k + half, T::key(col)) * 16;  // key + 32 turns alike
#pragma unroll
        for (int b = 0; b < 2; ++b) s[b] = mma32<DT>(*(const u32x4v*)(kp + 32 * b * RS), qf[k], s[b]);
      }
      interleave<4 * NT, 1, 4>();
      if constexpr (W == 8) {
        __builtin_amdgcn_sched_barrier(0);
        if (t + 1 < t1) load(t + 1);
      }
      uint64_t seen = ~0ull;
      if (t >= w_hiding) {
        seen = seen_bits(q, mask, a.mask_words, qi, p0);
        const uint64_t mine = seen >> (4 * half);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            s[b][x] = (mine >> (32 * b + 8 * (x / 4) + x % 4)) & 1 ? s[b][x] : -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int x = 0; x < 16; ++x) top = fmaxf(top, s[b][x]);
      top = join32(top, Larger()) * c;
      const bool raise = top > mx + kRaise;
      if (__ballot(raise)) {
        const float f = raise ? __builtin_amdgcn_exp2f(mx - top) : 1.0f;
        mx = raise ? top : mx;
        l *= f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[n][x] *= f;
      }
      const float ms = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int x = 0; x < 16; ++x) s[b][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][x], c, -ms));
      float sum[4] = {0, 0, 0, 0};
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int x = 0; x < 16; ++x) sum[x & 3] += s[b][x];
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      u32x4v pf[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          pf[k][x] = pack2<DT>(s[k >> 1][8 * (k & 1) + 2 * x], s[k >> 1][8 * (k & 1) + 2 * x + 1]);
      uint64_t bad = bad0 | (uint64_t)bad1 << 32;
#pragma unroll 1
      while (bad) {  // values that are not finite, to the rows that see them only
        const int key = __builtin_ctzll(bad), at = (key >> 5) * 16 + ((key >> 3) & 3) * 4 + (key & 3);
        bad &= bad - 1;
        float p = 0;
#pragma unroll
        for (int x = 0; x < 32; ++x) p = x == at ? s[x >> 4][x & 15] : p;
        p = __shfl(p, col + 32 * ((key >> 2) & 1), 64);
        const bool sees = (seen >> key) & 1;
        const uint16_t* const vp = values + offs[t & 7][key];
        const int d0 = 4 * here(half);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const u32x2v v = ld8(vp + min(d0 + 32 * n + 8 * x, D - 4));
#pragma unroll
            for (int y = 0; y < 4; ++y)
              o[n][4 * x + y] += sees ? odd_term<DT>(p, v[y >> 1] >> (16 * (y & 1))) : 0.0f;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      const int vrow = 4 * half + (lane & 15) / 4;
      const uint8_t* const vl = vb + vrow * RS + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int n = 0; n < NT; ++n) {  // key + 4 turns alike
          const uint8_t* const vp = vl + T::place(4 * n, T::value(vrow)) * 16 + 16 * k * RS;
          const u32x2v lo = read_transposed(vp), hi = read_transposed(vp + 8 * RS);
          o[n] = mma32<DT>(u32x4v{lo.x, lo.y, hi.x, hi.y}, pf[k], o[n]);
        }
      interleave<4 * NT, 2, 2>();
    }
    if (look) note(t + 4);
    __syncthreads();
  }

  l = join32(l, Plus());
  if (w0 + col >= M) return;
  const int64_t out_row = row * a.query_heads + qh;
  if (parts == 1) {
    const float f = l == 0 ? 0.0f : 1.0f / l;
    uint16_t* const op = (uint16_t*)a.out + out_row * D;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int d = 32 * n + 8 * x + 4 * half;
        if (d < D)
          gst((uint2*)(op + d), make_uint2(pack2<DT>(o[n][4 * x] * f, o[n][4 * x + 1] * f),
                                           pack2<DT>(o[n][4 * x + 2] * f, o[n][4 * x + 3] * f)));
      }
    if (a.lse && half == 0) a.lse[out_row] = l == 0 ? -INFINITY : (mx + __builtin_amdgcn_logf(l)) / kLog2e;
  } else {
    float* const op = plan.sums + (out_row * plan.splits + part) * D;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int d = 32 * n + 8 * x + 4 * half;
        if (d < D)
          *(KVMI_GLOBAL f32x4*)(op + d) = f32x4{o[n][4 * x], o[n][4 * x + 1], o[n][4 * x + 2], o[n][4 * x + 3]};
      }
    if (half == 0) plan.stats[out_row * plan.splits + part] = make_float2(mx, l);
  }
}

template <int DT, int NT, int W>
void launch(const kvmi_attention_args& a, const AttendPlan& p, hipStream_t st) {
  const int64_t pairs = ((int64_t)a.requests * a.cache.num_heads + 7) / 8 * 8;
  const dim3 grid((unsigned)(pairs * p.row_tiles * p.splits)), threads(64 * W);
  if (a.cache.head_dim == 32 * NT)
    hipLaunchKernelGGL((attend_tiles_kernel<DT, NT, true, W>), grid, threads, 0, st, a, p);
  else
    hipLaunchKernelGGL((attend_tiles_kernel<DT, NT, false, W>), grid, threads, 0, st, a, p);
}
template <int DT>
void launch(const kvmi_attention_args& a, const AttendPlan& p, hipStream_t st) {
  switch ((a.cache.head_dim + 31) / 32) {
    case 1:
    case 2: return launch<DT, 2, 4>(a, p, st);
    case 3: return launch<DT, 3, 4>(a, p, st);
    case 4: return p.waves == 8 ? launch<DT, 4, 8>(a, p, st) : launch<DT, 4, 4>(a, p, st);
    case 5: return launch<DT, 5, 4>(a, p, st);
    case 6: return launch<DT, 6, 4>(a, p, st);
    default: return launch<DT, 8, 4>(a, p, st);
  }
}

}  // namespace

int attend_tiles(const kvmi_attention_args& a, const AttendPlan& plan, hipStream_t st) {
  if (a.dtype == KVMI_DTYPE_BF16)
    launch<KVMI_DTYPE_BF16>(a, plan, st);
  else
    launch<KVMI_DTYPE_FP16>(a, plan, st);
  return hipGetLastError() == hipSuccess ? KVMI_OK : KVMI_ELAUNCH;
}

}  // namespace kvmi
