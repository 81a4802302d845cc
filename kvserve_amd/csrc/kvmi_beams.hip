// Beam search's selection: the best continuations over a request's beams and the vocabulary.
#include "kvmi_paged.hpp"

#include <algorithm>
#include <cmath>

namespace kvmi {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMostCount = 64;  // (a lane each, where the best are listed)
constexpr int kVectors = 128;   // of 16 bytes, in which a tile's candidates are looked for; at least kMostCount
constexpr int kRoom = 8 * kVectors;  // candidates that are ranked at once
constexpr double kFar = 600.0;  // logits up to here are summed as they are: exp(600) times any vocabulary is finite

// Word w of a vector, w known only at run time.
__device__ __forceinline__ uint32_t word_of(const u32x4v& v, int w) {
  return w & 2 ? (w & 1 ? v.w : v.z) : (w & 1 ? v.y : v.x);
}

// The types of logits: element i of a vector, or of its word, and what stands for no logit.
template <class T>
struct Logits;
template <>
struct Logits<__bf16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float at(const u32x4v& v, int i) {
    return of(v[i >> 1], i);
  }
  static __device__ __forceinline__ uint32_t bits(const void* row, int64_t i) { return gld((const uint16_t*)row + i); }
  static __device__ __forceinline__ float of(uint32_t word, int i) { return i & 1 ? bf_hi(word) : bf_lo(word); }
  static __device__ __forceinline__ uint32_t word(const u32x4v& v, int i) { return word_of(v, i >> 1); }
  static constexpr uint32_t kNone = 0xff80;  // -inf
  static constexpr int kZeros = 16;          // bits at the end of a value in 32 bits that are all alike
};
template <>
struct Logits<_Float16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float at(const u32x4v& v, int i) {
    return of(v[i >> 1], i);
  }
  static __device__ __forceinline__ uint32_t bits(const void* row, int64_t i) { return gld((const uint16_t*)row + i); }
  static __device__ __forceinline__ float of(uint32_t word, int i) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? word >> 16 : word));
  }
  static __device__ __forceinline__ uint32_t word(const u32x4v& v, int i) { return word_of(v, i >> 1); }
  static constexpr uint32_t kNone = 0xfc00;
  static constexpr int kZeros = 13;
};
template <>
struct Logits<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float at(const u32x4v& v, int i) { return __uint_as_float(v[i]); }
  static __device__ __forceinline__ uint32_t bits(const void* row, int64_t i) { return gld((const uint32_t*)row + i); }
  static __device__ __forceinline__ float of(uint32_t word, int) { return __uint_as_float(word); }
  static __device__ __forceinline__ uint32_t word(const u32x4v& v, int i) { return word_of(v, i); }
  static constexpr uint32_t kNone = 0xff800000;
  static constexpr int kZeros = 0;
};

// A vector of a row that begins at any of its elements.  Vectors go by places in the row, not in memory, so
// that equal rows have equal sums, to the last bit, wherever they begin.  (The hardware loads 16 bytes from
// any address: 64 requests x 8 beams x 100003 in bf16 51.4 us a call, 54.4 with vectors on 16-byte places.)
typedef u32x4v AnyPlace __attribute__((aligned(2)));
template <class T>
__device__ __forceinline__ u32x4v load_vector(const T* p) {
  return *(const KVMI_GLOBAL AnyPlace*)p;
}
// A vector of a row of V logits that begins at element e; behind the row -inf, and nothing is read
// there.
template <class T>
__device__ __forceinline__ u32x4v load_logits(const void* row, int64_t e, int64_t V) {
  using L = Logits<T>;
  if (e + L::kVec <= V) return load_vector((const T*)row + e);
  u32x4v v;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (L::kVec == 4) {
      v[w] = e + w < V ? L::bits(row, e + w) : L::kNone;
    } else {
      const int64_t a = e + 2 * w;
      const uint32_t lo = a < V ? L::bits(row, a) : L::kNone;
      const uint32_t hi = a + 1 < V ? L::bits(row, a + 1) : L::kNone;
      v[w] = lo | hi << 16;
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
  // 2^n: n added to the exponent, in the upper word alone
  const u32x2v t_words = __builtin_bit_cast(u32x2v, t);
  u32x2v words = __builtin_bit_cast(u32x2v, p);
  words.y += t_words.x << 20;
  return __builtin_bit_cast(double, words);
}

// The order of floats as that of unsigned words; zeros are one.
__device__ __forceinline__ uint32_t order_of(float x) { return f2key(x + 0.0f); }

// The wave's reductions go from row to row of 16 lanes in registers (10 cycles a step where an exchange
// over the LDS takes 60) and end in lane 63.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t from_lane(uint32_t mine, uint32_t none) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)mine, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float maximum_with(float x) {
  return __builtin_elementwise_maximum(x, __uint_as_float(from_lane<CTRL, ROWS>(__float_as_uint(x), __float_as_uint(x))));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double sum_with(double x) {
  const u32x2v w = __builtin_bit_cast(u32x2v, x);
  const u32x2v other = {from_lane<CTRL, ROWS>(w.x, 0), from_lane<CTRL, ROWS>(w.y, 0)};
  return x + __builtin_bit_cast(double, other);
}
// The largest of the wave, NaN if one is NaN.
__device__ __forceinline__ float wave_maximum(float x) {
  x = maximum_with<0x111, 0xf>(x);  // the lane 1, 2, 4, 8 before in the row
  x = maximum_with<0x112, 0xf>(x);
  x = maximum_with<0x114, 0xf>(x);
  x = maximum_with<0x118, 0xf>(x);
  x = maximum_with<0x142, 0xa>(x);  // the last lane of the row before, of the half before
  x = maximum_with<0x143, 0xc>(x);
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
// The sum of the wave, in lane 63.
__device__ __forceinline__ double wave_sum(double x) {
  x = sum_with<0x111, 0xf>(x);
  x = sum_with<0x112, 0xf>(x);
  x = sum_with<0x114, 0xf>(x);
  x = sum_with<0x118, 0xf>(x);
  x = sum_with<0x142, 0xa>(x);
  return sum_with<0x143, 0xc>(x);
}

// Of 64 words, one a lane: the smallest of the largest of each 16 neighbours (`wide`), or of each 4.  So
// many words as there are such groups reach it.
__device__ __forceinline__ uint32_t least_of_groups(uint32_t x, bool wide) {
  x = max(x, from_lane<0xb1, 0xf>(x, x));  // lanes 1, 2 away within four
  x = max(x, from_lane<0x4e, 0xf>(x, x));
  const uint32_t y4 = from_lane<0x124, 0xf>(x, x);  // 4, 8 away within the row of 16
  x = wide ? max(x, y4) : min(x, y4);
  const uint32_t y8 = from_lane<0x128, 0xf>(x, x);
  x = wide ? max(x, y8) : min(x, y8);
  const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
  const uint32_t c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
  return min(min(a, b), min(c, d));
}

// A word that at least `count` of N words a lane reach, and not many more, where they differ.
// `count` reach lo; no word is above `most`.
template <int N>
__device__ __forceinline__ uint32_t near_bound(const uint32_t (&key)[N], int count, uint32_t lo, uint32_t most) {
  // fewer than `count` are at hi or above (NaN may have any place: hi stays above lo, so the loop ends)
  uint64_t hi = (uint64_t)max(most, lo) + 1;
  while (hi - lo > 1) {
    const uint32_t mid = (uint32_t)(lo + (hi - lo) / 2);
    int n = 0;
#pragma unroll
    for (int x = 0; x < N; ++x) n += __popcll(__ballot(key[x] >= mid));
    if (n >= count) {
      lo = mid;
      if (n <= count + count / 2) break;
    } else {
      hi = mid;
    }
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
  BlockOf per_row;  // by a row's keys
};

// Candidates that are ranked against each other: 2^l lanes for each of n, at most 16.
__device__ __forceinline__ int rankers_log2(int n, int threads) {
  int l = 0;
  while (l < 4 && (2 * n << l) <= threads) ++l;
  return l;
}

// Workgroup (tile, row): NV vectors a thread, all of them in registers: their sum of exp, and the
// `count` best.  At least `count` elements reach the count-th largest of the threads' 256 largest, so
// those below it cannot be among the best; the few that reach it, or a word a little below it, are
// ranked against each other.  Where too many do (ties, or large ones in few threads) the count-th
// largest itself is found by bisection.
// 64 requests x 8 beams x 131072 in bf16: 45 to 47 us; reading alone takes 22, the vector unit's 18
// instructions an element, a tile's end among them, about 35 at 1.9 ns each (multiply-adds of 64 bits
// issue like those of 32): bound by instructions.
template <class T, int NV>
__global__ __launch_bounds__(kThreads) void select_tile_kernel(SelectArgs s) {
  using L = Logits<T>;
  constexpr int VEC = L::kVec;
  __shared__ uint64_t best[kRoom];
  __shared__ double part_sum[kWaves], part_at[kWaves];
  __shared__ uint32_t tops[kThreads], lows[kWaves], highs[kWaves];
  __shared__ u32x4v hit[kVectors];
  __shared__ int hit_at[kVectors];
  __shared__ int found, vectors, scan[kWaves];
  const int tid = threadIdx.x, wave = tid >> 6, tile = blockIdx.x, count = s.a.count;
  const int64_t row = blockIdx.y, V = s.a.vocab;
  // a row whose score is not finite has no candidates, and is not read but where a call is so small
  // that one load after the other would be its time
  const float score = gld(s.a.scores + row);
  if (NV > 1 && !(__builtin_fabsf(score) < INFINITY)) return;
  const T* const logits = (const T*)s.a.logits + row * s.a.row_stride;
  const int64_t first = (int64_t)tile * (kThreads * NV * VEC);
  u32x4v x[NV];
  if (first + kThreads * NV * VEC <= V) {
    const T* const from = logits + first + tid * VEC;
#pragma unroll
    for (int j = 0; j < NV; ++j) x[j] = load_vector(from + j * (kThreads * VEC));
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) x[j] = load_logits<T>(logits, first + (int64_t)(j * kThreads + tid) * VEC, V);
  }
  if (NV == 1 && !(__builtin_fabsf(score) < INFINITY)) return;
  // What is seldom done goes through the tile in memory again, f(vector, j): unpacked from registers it
  // would take twice those of what is always done.
  auto over_tile = [&](auto f) {
#pragma unroll 1
    for (int j = 0; j < NV; ++j) f(load_logits<T>(logits, first + (int64_t)(j * kThreads + tid) * VEC, V), j);
  };
  if (tid == 0) found = vectors = 0;

  float top[NV], lane_top = -INFINITY;
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    top[j] = L::at(x[j], 0);
#pragma unroll
    for (int i = 1; i < VEC; ++i) top[j] = __builtin_elementwise_maximum(top[j], L::at(x[j], i));
    lane_top = __builtin_elementwise_maximum(lane_top, top[j]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += exp_near((double)__builtin_elementwise_maximum(L::at(x[j], i), -700.0f));
    // (a vector's values are done with here: summed behind all the largest, they would all be kept, and
    // take half the waves of a SIMD)
    asm volatile("" : "+v"(sum));
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
      over_tile([&](const u32x4v& v, int) {
#pragma unroll 1
        for (int i = 0; i < VEC; ++i) sum += exp_near(fmax((double)L::of(L::word(v, i), i) - at, -700.0));
      });
    } else {
      sum = (double)NAN;
    }
  }
  sum = wave_sum(sum);
  if ((tid & 63) == 63) {
    part_sum[wave] = sum;
    part_at[wave] = at;
  }
  const uint32_t top_key = order_of(lane_top) >> L::kZeros;
  const uint32_t low = least_of_groups(top_key, count <= 4 * kWaves);
  tops[tid] = top_key;
  if ((tid & 63) == 0) {
    lows[wave] = low;
    highs[wave] = order_of(high) >> L::kZeros;
  }
  __syncthreads();
  uint32_t all_tops[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all_tops[w] = tops[w * 64 + (tid & 63)];
  const uint32_t bound = max(
      near_bound(all_tops, count, min(min(lows[0], lows[1]), min(lows[2], lows[3])),
                 max(max(highs[0], highs[1]), max(highs[2], highs[3]))) << L::kZeros,
      order_of(-INFINITY) + 1);  // -inf is no candidate
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
    if (n < kRoom) best[n] = (uint64_t)order_of(v) << 32 | (uint32_t)~token;  // (more only if the logits change meanwhile)
  };
  // the vectors that reach the bound, then their elements, spread over the threads
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (top[j] >= least) {
      const int n = atomicAdd(&vectors, 1);
      if (n < kVectors) {
        hit[n] = x[j];
        hit_at[n] = j * kThreads + tid;
      }
    }
  __syncthreads();
  const int hits = vectors;
  if (hits <= kVectors)
    for (int i = tid; i < hits * VEC; i += kThreads) {
      const float v = L::of(((const uint32_t*)hit)[i * (int)sizeof(T) / 4], i);
      if (v >= least) keep(v, (uint32_t)(first + (int64_t)hit_at[i / VEC] * VEC + i % VEC));
    }
  __syncthreads();
  if (hits > kVectors) {
    // the count-th largest: at least `count` elements are at lo or more, fewer at hi
    uint32_t lo = bound, hi = 0xffffffffu;
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const float at_mid = key2f(mid);  // (NaN past +inf: nothing reaches it)
      int n = 0, all;
      over_tile([&](const u32x4v& v, int) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) n += L::at(v, i) >= at_mid;
      });
      before_in_block(n, scan, &all);
      if (all >= count)
        lo = mid;
      else
        hi = mid;
    }
    // fewer than `count` above it, found by the comparison that they were counted with (which NaN never
    // passes: its words lie above +inf's, and any number of them may be there), and of those at it the first
    const float above = key2f(lo + 1);
    over_tile([&](const u32x4v& v, int j) {
#pragma unroll 1
      for (int i = 0; i < VEC; ++i) {
        const float y = L::of(L::word(v, i), i);
        if (y >= above) keep(y, token_of(j, i));
      }
    });
    __syncthreads();
    int left = count - min(found, count);
    __syncthreads();
    over_tile([&](const u32x4v& v, int j) {
      int n = 0, all;
#pragma unroll
      for (int i = 0; i < VEC; ++i) n += order_of(L::at(v, i)) == lo;
      int before = before_in_block(n, scan, &all);
#pragma unroll 1
      for (int i = 0; i < VEC; ++i)
        if (order_of(L::of(L::word(v, i), i)) == lo && before++ < left) keep(L::of(L::word(v, i), i), token_of(j, i));
      left -= all;  // (may go below zero: then none is taken)
    });
    __syncthreads();
  }
  const int n = min(found, kRoom);
  uint64_t* const out = s.keys + (row * s.tiles + tile) * count;
  const int log2 = rankers_log2(n, kThreads), parts = 1 << log2, part = tid & (parts - 1);
  for (int i0 = 0; i0 < n; i0 += kThreads >> log2) {
    const int i = i0 + (tid >> log2);
    const uint64_t mine = best[min(i, n - 1)];
    int rank = 0;
    for (int k = part; k < n; k += parts) rank += best[k] > mine;
    for (int d = parts / 2; d; d /= 2) rank += __shfl_xor(rank, d, 64);
    if (i < n && part == 0 && rank < count) gst(out + rank, mine);
  }
  for (int i = n + tid; i < count; i += kThreads) gst(out + i, (uint64_t)0);
}

// The sum of a row's exponentials as s exp(m), and two of them together.
struct Sum {
  double s, m;
};
__device__ __forceinline__ Sum join(const Sum& a, const Sum& b) {
  if (a.m == b.m) return Sum{a.s + b.s, a.m};
  const double m = fmax(a.m, b.m);  // (a sum at -inf is 0)
  return Sum{(a.m == m ? a.s : a.m == -INFINITY ? 0.0 : a.s * exp(a.m - m)) +
                 (b.m == m ? b.s : b.m == -INFINITY ? 0.0 : b.s * exp(b.m - m)),
             m};
}

constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / 64, kEach = 4, kRound = kEach * kJoinThreads;

// Workgroup: a request.  The rows' sums of all tiles, then the tiles' best, kRound at a time with the
// best so far: those below the count-th largest of 64 lanes' best, or below the count-th so far, drop
// out, the others are ranked against each other, each by several lanes where they are few.  A chain
// of loads and of barriers, 5.2 us for 4 beams x 16 tiles x 8 and 6.0 for 64 requests of 8 x 4 x 16: the first
// round's keys are on their way while the sums are made.
__global__ __launch_bounds__(kJoinThreads) void select_join_kernel(SelectArgs s) {
  struct Candidates {
    double value[kRound + kMostCount];
    uint64_t key[kRound + kMostCount];  // (order, ~token)
    uint8_t beam[kRound + kMostCount];
  };
  __shared__ Candidates list;
  __shared__ double best_value[kMostCount], lse[kMostCount];
  __shared__ uint64_t best_key[kMostCount];
  __shared__ uint8_t best_beam[kMostCount];
  __shared__ uint32_t bounds[kJoinWaves];
  __shared__ float scores[kMostCount];
  __shared__ int found;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = blockIdx.x;
  const int B = s.a.beams, count = s.a.count, tiles = s.tiles;
  const int all = B * tiles * count;  // (at most 64 * 64 * tiles: select_ok)
  const uint64_t* const keys = s.keys + (int64_t)r * all;
  uint64_t key[kEach];
#pragma unroll
  for (int x = 0; x < kEach; ++x) key[x] = x * kJoinThreads + tid < all ? gld(keys + x * kJoinThreads + tid) : 0;

  // log-sums: 2^group lanes a row
  int group = 0;
  while ((1 << group) < tiles && group < 6) ++group;
  const int member = tid & ((1 << group) - 1);
  if (tid == 0) found = 0;
  for (int b = tid >> group; b < B; b += kJoinThreads >> group) {
    const int64_t row = (int64_t)r * B + b;
    const float score = gld(s.a.scores + row);
    const bool used = __builtin_fabsf(score) < INFINITY;
    Sum sum{0.0, -INFINITY};
    for (int t = member; t < tiles; t += 1 << group) {
      const double2 p = s.sums[row * tiles + t];  // (anything, where the row is not used)
      if (used) sum = join(sum, Sum{p.x, p.y});
    }
    for (int d = 1 << group >> 1; d; d /= 2) sum = join(sum, Sum{__shfl_xor(sum.s, d, 64), __shfl_xor(sum.m, d, 64)});
    if (member == 0) {
      const double value = sum.s != sum.s ? (double)NAN : sum.s > 0.0 ? log(sum.s) + sum.m : -INFINITY;
      lse[b] = value;
      scores[b] = score;
      if (used ? value != value : score != -INFINITY) flag_error(s.a.err, KVMI_ERR_NOT_FINITE);
    }
  }
  __syncthreads();
  int have = 0;
  for (int begin = 0; begin < all; begin += kRound) {
    double value[kEach];
    int beam[kEach];
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
      const int i = begin + x * kJoinThreads + tid;
      value[x] = -INFINITY;
      if (begin) key[x] = i < all ? gld(keys + i) : 0;
      if (i < all) {
        beam[x] = s.per_row(i);
        const double sum = lse[beam[x]];
        if (__builtin_fabs(sum) < INFINITY && key[x]) {  // (a row without a sum has no keys)
          const double v = (double)scores[beam[x]] + ((double)key2f((uint32_t)(key[x] >> 32)) - sum);
          if ((float)v > -INFINITY) value[x] = v;
        }
      }
      top = fmaxf(top, (float)value[x]);
    }
    const uint32_t floor = order_of(-INFINITY) + 1, tops[1] = {order_of(top)};
    const uint32_t least = count <= 16 ? least_of_groups(tops[0], count <= 4) : 0;  // (16 groups, or 4)
    const uint32_t low = near_bound(tops, count, least, order_of(wave_maximum(top)));
    if (lane == 0) bounds[wave] = max(low, floor);
    __syncthreads();
    uint32_t bound = have == count ? order_of((float)best_value[count - 1]) : floor;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) bound = max(bound, bounds[w]);
#pragma unroll
    for (int x = 0; x < kEach; ++x)
      if (order_of((float)value[x]) >= bound) {
        const int at = atomicAdd(&found, 1);
        list.value[at] = value[x];
        list.key[at] = key[x];
        list.beam[at] = (uint8_t)beam[x];
      }
    __syncthreads();
    const int fresh = found, n = fresh + have;
    if (fresh) {
      if (have) {
        if (tid < have) {
          list.value[fresh + tid] = best_value[tid];
          list.key[fresh + tid] = best_key[tid];
          list.beam[fresh + tid] = best_beam[tid];
        }
        __syncthreads();
      }
      const int log2 = rankers_log2(n, kJoinThreads), parts = 1 << log2, part = tid & (parts - 1);
      for (int i0 = 0; i0 < n; i0 += kJoinThreads >> log2) {
        const int i = i0 + (tid >> log2);
        int rank = 0;
        double mine = 0.0;
        uint64_t my_key = 0;
        int my_beam = 0;
        if (i < n) {
          mine = list.value[i];
          my_key = list.key[i];
          my_beam = list.beam[i];
          for (int k = part; k < n; k += parts) {
            const double other = list.value[k];
            rank += other > mine;
            if (other == mine && k != i) {  // the lower beam, then the larger logit, then the lower token
              const int other_beam = list.beam[k];
              rank += other_beam != my_beam ? other_beam < my_beam : list.key[k] > my_key;
            }
          }
        }
        for (int d = parts / 2; d; d /= 2) rank += __shfl_xor(rank, d, 64);
        if (i < n && part == 0 && rank < count) {
          best_value[rank] = mine;
          best_key[rank] = my_key;
          best_beam[rank] = (uint8_t)my_beam;
        }
      }
      have = min(n, count);
    }
    __syncthreads();
    if (begin + kRound < all) {
      if (tid == 0) found = 0;
      __syncthreads();
    }
  }
  if (wave) return;
  const bool there = lane < have;
  const int64_t parent = there ? (int64_t)r * B + best_beam[lane] : -1;
  const int token = there ? (int)~(uint32_t)best_key[lane] : -1;
  const float value = there ? (float)best_value[lane] : -INFINITY;
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

// Vectors a thread: as many as leave 384 workgroups, for what a tile does besides its sums costs the
// same for any tile (us a call with its join: 32 rows x 4 beams x 131072 21.9 at 8 vectors, 25.6 at 4; 8 x 4: 13.9 at 4, 18.1
// at 1; 13 x 5 x 50021: 15.0 at 4 in 455 workgroups, 15.1 at 2, 17.0 at 8); 16 only where 1536 are left, six
// for a CU, whose loads and sums overlap (64 x 8 x 131072: 52.6 in 2048 workgroups, 56.4 at 8; but 16 x 4 x
// 152064 in 32 bits 21.7 in 640, 19.1 at 8).
struct Shape {
  int nv, tiles;
};
inline Shape shape_of(const kvmi_select_args& a) {
  const int vec = a.dtype == KVMI_DTYPE_FP32 ? 4 : 8;
  Shape s;
  const int64_t vectors = (int64_t)a.requests * a.beams * a.vocab / vec;
  for (s.nv = 16; s.nv > 1; s.nv /= 2)
    if (vectors >= (s.nv == 16 ? 1536LL : 384LL) * kThreads * s.nv) break;
  const int64_t tile = (int64_t)kThreads * s.nv * vec;
  s.tiles = (int)(((int64_t)a.vocab + tile - 1) / tile);
  return s;
}
bool select_ok(const kvmi_select_args& a) {
  return a.requests >= 0 && a.beams >= 1 && a.count >= a.beams && a.count <= kMostCount && a.vocab >= 1 &&
         a.vocab <= kMostPlaces && a.end_token >= -1 && a.row_stride >= 0 &&
         (int64_t)a.requests * a.beams <= 65535 && (int64_t)a.beams * a.count * (a.vocab / 1024 + 2) <= 0x7fffffffLL - kRound &&
         (a.dtype == KVMI_DTYPE_BF16 || a.dtype == KVMI_DTYPE_FP16 || a.dtype == KVMI_DTYPE_FP32);
}
template <class T>
void launch_tiles(const SelectArgs& s, int nv, hipStream_t st) {
  const dim3 grid((unsigned)s.tiles, (unsigned)(s.a.requests * s.a.beams));
  switch (nv) {
    case 16: hipLaunchKernelGGL((select_tile_kernel<T, 16>), grid, dim3(kThreads), 0, st, s); break;
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
  s.per_row = block_of(s.tiles * a.count);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a.dtype == KVMI_DTYPE_BF16)
    launch_tiles<__bf16>(s, shape.nv, st);
  else if (a.dtype == KVMI_DTYPE_FP16)
    launch_tiles<_Float16>(s, shape.nv, st);
  else
    launch_tiles<float>(s, shape.nv, st);
  hipLaunchKernelGGL(select_join_kernel, dim3((unsigned)a.requests), dim3(kJoinThreads), 0, st, s);
  return launched();
}
