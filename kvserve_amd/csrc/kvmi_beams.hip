// Beam search's selection: the best continuations over a request's beams and the vocabulary.
#include "kvmi_paged.hpp"

#include <algorithm>
#include <cmath>

namespace kvmi {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMostCount = 64;  // the lanes of a wave: their largest values bound the count-th
constexpr int kRoom = 1024;     // candidates that a workgroup ranks at once
constexpr double kFar = 600.0;  // logits up to here are summed as they are: exp(600) times any vocabulary is finite

template <class T>
struct Logits;
template <>
struct Logits<__bf16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float at(const uint4& v, int i) {
    const uint32_t u = (&v.x)[i >> 1];
    return i & 1 ? bf_hi(u) : bf_lo(u);
  }
  static __device__ __forceinline__ uint32_t bits(const void* row, int64_t i) { return gld((const uint16_t*)row + i); }
  static constexpr uint32_t kNone = 0xff80;  // -inf
};
template <>
struct Logits<_Float16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float at(const uint4& v, int i) {
    const uint32_t u = (&v.x)[i >> 1];
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? u >> 16 : u));
  }
  static __device__ __forceinline__ uint32_t bits(const void* row, int64_t i) { return gld((const uint16_t*)row + i); }
  static constexpr uint32_t kNone = 0xfc00;
};
template <>
struct Logits<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float at(const uint4& v, int i) { return __uint_as_float((&v.x)[i]); }
  static __device__ __forceinline__ uint32_t bits(const void* row, int64_t i) { return gld((const uint32_t*)row + i); }
  static constexpr uint32_t kNone = 0xff800000;
};

// A vector of a row of V logits that begins at element e; outside the row -inf, and nothing is read
// there.
template <class T>
__device__ __forceinline__ uint4 load_logits(const void* row, int64_t e, int64_t V) {
  using L = Logits<T>;
  if (e >= 0 && e + L::kVec <= V) return gld((const uint4*)((const T*)row + e));
  uint4 v;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (L::kVec == 4) {
      (&v.x)[w] = e + w >= 0 && e + w < V ? L::bits(row, e + w) : L::kNone;
    } else {
      const int64_t a = e + 2 * w;
      const uint32_t lo = a >= 0 && a < V ? L::bits(row, a) : L::kNone;
      const uint32_t hi = a + 1 >= 0 && a + 1 < V ? L::bits(row, a + 1) : L::kNone;
      (&v.x)[w] = lo | hi << 16;
    }
  }
  return v;
}

// exp(x) for |x| <= 700: 2^(n + r), n whole and |r| <= 1/2, with a polynomial of degree 7 for 2^r
// (the smallest largest relative error, 4.0e-11, found by exchange).  In 64 bits since the order of two
// beams' candidates hangs on the difference of their rows' sums: with 32 bits (1e-7 off) one of
// some hundred calls of 64 requests would order two of them otherwise.  64-bit multiply-adds issue at
// the rate of 32-bit ones here.
__device__ __forceinline__ double exp_near(double x) {
  const double magic = 0x1.8p52, per = 0x1.71547652b82fep+0;  // log2(e)
  const double t = __builtin_fma(x, per, magic);              // its low word is n
  const double r = __builtin_fma(x, per, -(t - magic));
  double p = 0x1.fe17831d6aba5p-17;
  p = __builtin_fma(p, r, 0x1.446a1fdacb1dbp-13);
  p = __builtin_fma(p, r, 0x1.5d8a7088fda2cp-10);
  p = __builtin_fma(p, r, 0x1.3b29dc40d6655p-7);
  p = __builtin_fma(p, r, 0x1.c6b08aaf2e313p-5);
  p = __builtin_fma(p, r, 0x1.ebfbe0a4be818p-3);
  p = __builtin_fma(p, r, 0x1.62e42ff116290p-1);
  p = __builtin_fma(p, r, 0x1.ffffffffabbcdp-1);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
  return __builtin_bit_cast(double, (uint64_t)((uint32_t)(bits >> 32) + (n << 20)) << 32 | (uint32_t)bits);
}

// The order of floats as that of unsigned words; zeros are one.
__device__ __forceinline__ uint32_t order_of(float x) { return f2key(x + 0.0f); }

// The largest of the wave, NaN if one is NaN, in every lane.
__device__ __forceinline__ float wave_maximum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = __builtin_elementwise_maximum(x, __shfl_xor(x, d, 64));
  return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}

// A word that at least `count` of the wave's 64 lanes hold or exceed, near the count-th largest: as
// soon as exactly `count` do.
__device__ __forceinline__ uint32_t wave_bound(uint32_t key, int count) {
  uint32_t lo = 0, hi = 0xffffffffu;  // `count` lanes are at lo or more; fewer at hi
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    const int n = __popcll(__ballot(key >= mid));
    if (n >= count) lo = mid;
    if (n < count) hi = mid;
    if (n == count) break;
  }
  return lo;
}

// Sum of the flags of the threads before this one, and of all, in `all`.
__device__ __forceinline__ int before_in_block(int n, int* lds, int* all) {
  int s = n;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int t = __shfl_up(s, d, 64);
    if ((threadIdx.x & 63) >= d) s += t;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  int carry = 0;
  for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) carry += lds[w];
  *all = lds[0] + lds[1] + lds[2] + lds[3];
  return s - n + carry;
}

struct SelectArgs {
  kvmi_select_args a;
  int tiles;       // of a row
  double2* sums;   // [rows][tiles]: (s, m), the tile's sum of exp(x) is s exp(m); s NaN where it is not finite
  uint64_t* keys;  // [rows][tiles][count]: (order, ~token), best first; 0 behind the last
};

// Workgroup (tile, row): NV vectors a thread, all of them in registers: their sum of exp, and the
// `count` best.  At least `count` elements reach the count-th largest of a wave's 64 largest (one a
// lane), so those below it cannot be among the best; the few that reach it, by the waves' highest
// such bound, are ranked against each other.  Where too many do (ties, or large ones in few
// lanes) the count-th largest itself is found by bisection.
template <class T, int NV>
__global__ __launch_bounds__(kThreads) void select_tile_kernel(SelectArgs s) {
  using L = Logits<T>;
  constexpr int VEC = L::kVec;
  __shared__ uint64_t best[kRoom];
  __shared__ double part_sum[kWaves], part_at[kWaves];
  __shared__ uint32_t bounds[kWaves];
  __shared__ int found, scan[kWaves];
  const int tid = threadIdx.x, wave = tid >> 6, tile = blockIdx.x, count = s.a.count;
  const int64_t row = blockIdx.y, V = s.a.vocab;
  // a row whose score is not finite has no candidates
  const float score = gld(s.a.scores + row);
  if (!(__builtin_fabsf(score) < INFINITY)) return;
  const T* const logits = (const T*)s.a.logits + row * s.a.row_stride;
  // vectors lie on 16-byte places, whatever the row's
  const int64_t shift = (int64_t)((uintptr_t)logits % 16 / sizeof(T));
  const int64_t first = (int64_t)tile * (kThreads * NV * VEC) - shift;
  uint4 x[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) x[j] = load_logits<T>(logits, first + (int64_t)(j * kThreads + tid) * VEC, V);
  if (tid == 0) found = 0;

  float top[NV], lane_top = -INFINITY;
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    top[j] = L::at(x[j], 0);
#pragma unroll
    for (int i = 1; i < VEC; ++i) top[j] = __builtin_elementwise_maximum(top[j], L::at(x[j], i));
    lane_top = __builtin_elementwise_maximum(lane_top, top[j]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += exp_near((double)fmaxf(L::at(x[j], i), -700.0f));
  }
  const float high = wave_maximum(lane_top);
  double at = 0.0;
  if (!(__builtin_fabsf(high) <= (float)kFar)) {
    // far from zero: exp(x - high); a wave without anything finite has no sum, and one with NaN or
    // +inf says so
    sum = 0.0;
    if (high == -INFINITY) {
      at = -INFINITY;
    } else if (high < INFINITY) {
      at = high;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum += exp_near(fmax((double)L::at(x[j], i) - at, -700.0));
    } else {
      sum = (double)NAN;
    }
  }
  sum = wave_sum(sum);
  if ((tid & 63) == 0) {
    part_sum[wave] = sum;
    part_at[wave] = at;
  }
  const uint32_t floor = order_of(-INFINITY) + 1;  // -inf is no candidate
  const uint32_t wave_low = wave_bound(order_of(lane_top), count);
  if ((tid & 63) == 0) bounds[wave] = max(wave_low, floor);
  __syncthreads();
  uint32_t bound = max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3]));
  if (tid == 0) {
    const double m = fmax(fmax(part_at[0], part_at[1]), fmax(part_at[2], part_at[3]));
    double all = 0.0;
    for (int w = 0; w < kWaves; ++w)
      all += part_at[w] == m ? part_sum[w] : part_at[w] == -INFINITY ? 0.0 : part_sum[w] * exp(part_at[w] - m);
    s.sums[row * s.tiles + tile] = make_double2(all, m);
  }
  const float least = key2f(bound);
  auto token_of = [&](int j, int i) { return (uint32_t)(first + (int64_t)(j * kThreads + tid) * VEC + i); };
  auto keep = [&](float v, uint32_t token) {
    const int n = atomicAdd(&found, 1);
    if (n < kRoom) best[n] = (uint64_t)order_of(v) << 32 | (uint32_t)~token;
  };
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (top[j] >= least) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (L::at(x[j], i) >= least) keep(L::at(x[j], i), token_of(j, i));
    }
  __syncthreads();
  if (found > kRoom) {
    // the count-th largest: at least `count` elements are at lo or more, fewer at hi
    uint32_t lo = bound, hi = 0xffffffffu;
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      int n = 0, all;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) n += order_of(L::at(x[j], i)) >= mid;
      before_in_block(n, scan, &all);
      if (all >= count)
        lo = mid;
      else
        hi = mid;
    }
    __syncthreads();
    if (tid == 0) found = 0;
    __syncthreads();
    // fewer than `count` above it, and of those at it the first ones
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (order_of(L::at(x[j], i)) > lo) keep(L::at(x[j], i), token_of(j, i));
    __syncthreads();
    int left = count - found;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      int n = 0, all;
#pragma unroll
      for (int i = 0; i < VEC; ++i) n += order_of(L::at(x[j], i)) == lo;
      int before = before_in_block(n, scan, &all);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (order_of(L::at(x[j], i)) == lo && before++ < left) keep(L::at(x[j], i), token_of(j, i));
      left -= all;  // (may go below zero: then none is taken)
    }
    __syncthreads();
  }
  const int n = found;
  uint64_t* const out = s.keys + (row * s.tiles + tile) * count;
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t mine = best[i];
    int rank = 0;
    for (int k = 0; k < n; ++k) rank += best[k] > mine;
    if (rank < count) gst(out + rank, mine);
  }
  for (int i = n + tid; i < count; i += kThreads) gst(out + i, (uint64_t)0);
}

struct Candidate {
  double value;
  uint64_t key;  // (order, ~token)
  int beam;
};
// Whether a comes before b.
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  if (a.value != b.value) return a.value > b.value;
  return a.beam != b.beam ? a.beam < b.beam : a.key > b.key;
}

// Workgroup: a request.  The rows' sums of all tiles, then the tiles' best, 1024 at a time with the
// best so far: those below the count-th largest of 64 lanes' best, or below the count-th so far, drop
// out, the others are ranked against each other.
__global__ __launch_bounds__(kThreads) void select_join_kernel(SelectArgs s) {
  constexpr int kEach = 4, kRound = kEach * kThreads;
  __shared__ Candidate list[kRound + kMostCount], best[kMostCount];
  __shared__ double lse[kMostCount];
  __shared__ uint32_t bounds[kWaves];
  __shared__ int found;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = blockIdx.x;
  const int B = s.a.beams, count = s.a.count, tiles = s.tiles;
  for (int b = wave; b < B; b += kWaves) {
    const int64_t row = (int64_t)r * B + b;
    const float score = gld(s.a.scores + row);
    double value = -INFINITY;
    if (__builtin_fabsf(score) < INFINITY) {
      double m = -INFINITY, sum = 0.0;
      for (int t = lane; t < tiles; t += 64) m = fmax(m, s.sums[row * tiles + t].y);
#pragma unroll
      for (int d = 32; d; d >>= 1) m = fmax(m, __shfl_xor(m, d, 64));
      for (int t = lane; t < tiles; t += 64) {
        const double2 p = s.sums[row * tiles + t];
        sum += p.y == m ? p.x : p.y == -INFINITY ? 0.0 : p.x * exp(p.y - m);
      }
      sum = wave_sum(sum);
      value = sum != sum ? (double)NAN : sum > 0.0 ? log(sum) + m : -INFINITY;
    } else {
      if (score != -INFINITY && lane == 0) flag_error(s.a.err, KVMI_ERR_NOT_FINITE);
    }
    if (value != value && lane == 0) flag_error(s.a.err, KVMI_ERR_NOT_FINITE);
    if (lane == 0) lse[b] = value;
  }
  if (tid == 0) found = 0;
  __syncthreads();
  int have = 0;
  const int64_t per_beam = (int64_t)tiles * count, all = B * per_beam;
  for (int64_t begin = 0; begin < all; begin += kRound) {
    Candidate c[kEach];
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
      const int64_t i = begin + x * kThreads + tid;
      c[x].value = -INFINITY;
      if (i < all) {
        c[x].beam = (int)(i / per_beam);
        const double sum = lse[c[x].beam];
        if (__builtin_fabs(sum) < INFINITY) {  // (else nothing was written)
          c[x].key = gld(s.keys + r * all + i);
          if (c[x].key) {
            const double v = (double)gld(s.a.scores + (int64_t)r * B + c[x].beam) +
                             ((double)key2f((uint32_t)(c[x].key >> 32)) - sum);
            if ((float)v > -INFINITY) c[x].value = v;
          }
        }
      }
      top = fmaxf(top, (float)c[x].value);
    }
    const uint32_t floor = order_of(-INFINITY) + 1, low = wave_bound(order_of(top), count);
    if (lane == 0) bounds[wave] = max(low, floor);
    __syncthreads();
    uint32_t bound = max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3]));
    if (have == count) bound = max(bound, order_of((float)best[count - 1].value));
#pragma unroll
    for (int x = 0; x < kEach; ++x)
      if (order_of((float)c[x].value) >= bound) list[atomicAdd(&found, 1)] = c[x];
    __syncthreads();
    const int fresh = found;
    if (fresh) {
      for (int i = tid; i < have; i += kThreads) list[fresh + i] = best[i];
      __syncthreads();
      const int n = fresh + have;
      for (int i = tid; i < n; i += kThreads) {
        const Candidate mine = list[i];
        int rank = 0;
        for (int k = 0; k < n; ++k) rank += before(list[k], mine);
        if (rank < count) best[rank] = mine;
      }
      have = min(n, count);
    }
    __syncthreads();
    if (tid == 0) found = 0;
    __syncthreads();
  }
  if (wave) return;
  const bool there = lane < have;
  const int64_t parent = there ? (int64_t)r * B + best[lane].beam : -1;
  const int token = there ? (int)~(uint32_t)best[lane].key : -1;
  const float value = there ? (float)best[lane].value : -INFINITY;
  if (lane < count) {
    const int64_t at = (int64_t)r * count + lane;
    gst(s.a.all_parents + at, (int32_t)parent);
    gst(s.a.all_tokens + at, token);
    gst(s.a.all_scores + at, value);
  }
  // those that go on
  const bool on = there && (s.a.end_token < 0 || token != s.a.end_token);
  const uint64_t going = __ballot(on);
  const int place = __popcll(going & ((1ull << lane) - 1));
  if (on && place < B) {
    const int64_t at = (int64_t)r * B + place;
    gst(s.a.parents + at, (int32_t)parent);
    gst(s.a.tokens + at, token);
    gst(s.a.next_scores + at, value);
  }
  if (lane >= __popcll(going) && lane < B) {
    const int64_t at = (int64_t)r * B + lane;
    gst(s.a.parents + at, -1);
    gst(s.a.tokens + at, -1);
    gst(s.a.next_scores + at, -INFINITY);
  }
}

// Vectors a thread: as many as leave the chip full.
struct Shape {
  int nv, tiles;
};
inline Shape shape_of(const kvmi_select_args& a) {
  const int vec = a.dtype == KVMI_DTYPE_FP32 ? 4 : 8;
  Shape s;
  for (s.nv = 8; s.nv > 1; s.nv /= 2)
    if ((int64_t)a.requests * a.beams * a.vocab >= 1024LL * kThreads * s.nv * vec) break;
  const int64_t tile = (int64_t)kThreads * s.nv * vec;
  s.tiles = (int)((a.vocab + vec - 1 + tile - 1) / tile);  // (a row may begin inside a vector)
  return s;
}
bool select_ok(const kvmi_select_args& a) {
  return a.requests >= 0 && a.beams >= 1 && a.count >= a.beams && a.count <= kMostCount && a.vocab >= 1 &&
         a.vocab <= kMostPlaces && a.end_token >= -1 && a.row_stride >= 0 &&
         (int64_t)a.requests * a.beams <= 65535 &&
         (a.dtype == KVMI_DTYPE_BF16 || a.dtype == KVMI_DTYPE_FP16 || a.dtype == KVMI_DTYPE_FP32);
}
template <class T>
void launch_tiles(const SelectArgs& s, int nv, hipStream_t st) {
  const dim3 grid((unsigned)s.tiles, (unsigned)(s.a.requests * s.a.beams));
  switch (nv) {
    case 8: hipLaunchKernelGGL((select_tile_kernel<T, 8>), grid, dim3(kThreads), 0, st, s); break;
    case 4: hipLaunchKernelGGL((select_tile_kernel<T, 4>), grid, dim3(kThreads), 0, st, s); break;
    case 2: hipLaunchKernelGGL((select_tile_kernel<T, 2>), grid, dim3(kThreads), 0, st, s); break;
    default: hipLaunchKernelGGL((select_tile_kernel<T, 1>), grid, dim3(kThreads), 0, st, s); break;
  }
}

}  // namespace
}  // namespace kvmi

extern "C" int64_t kvmi_select_workspace_bytes(const kvmi_select_args* args) {
  using namespace kvmi;
  if (!args || !select_ok(*args)) return KVMI_EINVAL;
  return (int64_t)args->requests * args->beams * shape_of(*args).tiles * (16 + 8 * (int64_t)args->count);
}

extern "C" int kvmi_select_beams(const kvmi_select_args* args, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!args || !select_ok(*args)) return KVMI_EINVAL;
  const kvmi_select_args& a = *args;
  if (a.requests == 0) return KVMI_OK;
  if (!a.logits || !a.scores || !a.parents || !a.tokens || !a.next_scores || !a.all_parents || !a.all_tokens ||
      !a.all_scores || !a.workspace || !aligned16(a.workspace) ||
      (uintptr_t)a.logits % (a.dtype == KVMI_DTYPE_FP32 ? 4 : 2) || a.workspace_bytes < kvmi_select_workspace_bytes(args))
    return KVMI_EINVAL;
  const Shape shape = shape_of(a);
  SelectArgs s;
  s.a = a;
  s.tiles = shape.tiles;
  s.sums = (double2*)a.workspace;
  s.keys = (uint64_t*)(s.sums + (int64_t)a.requests * a.beams * s.tiles);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a.dtype == KVMI_DTYPE_BF16)
    launch_tiles<__bf16>(s, shape.nv, st);
  else if (a.dtype == KVMI_DTYPE_FP16)
    launch_tiles<_Float16>(s, shape.nv, st);
  else
    launch_tiles<float>(s, shape.nv, st);
  hipLaunchKernelGGL(select_join_kernel, dim3((unsigned)a.requests), dim3(kThreads), 0, st, s);
  return launched();
}
