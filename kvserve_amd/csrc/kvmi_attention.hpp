// What the attention kernels over the paged cache share: a request's ranges, the split of its
// keys over workgroups, number formats and matrix instructions, and the way in which places
// that some rows do not see are kept out of those rows' sums.
#pragma once

#include "kvmi_common.hpp"

namespace kvmi {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
// A row's running maximum is raised only when a score passes it by 2^8: weights up to 256 cost
// no bits (they keep their relative step in bf16, and gain some in fp16, whose small ones are
// subnormal), and most tiles then leave the sums as they are.  Decided for each row by itself,
// so that what one row sees never changes another's rounding.
constexpr float kRaise = 8.0f;

// How the keys of a request are split over workgroups and where the parts go.
struct AttendPlan {
  BlockOf block, group;  // by the block size, by the query heads of a KV head
  BlockOf tiles, heads;  // tiles kernel: by row_tiles * splits, by the KV heads
  int waves;      // of a workgroup
  int row_tiles;  // tiles kernel: row tiles of a KV head, 32 rows a wave
  int splits;     // the most parts of a request
  int chunk;      // keys that a part should have
  float* sums;    // [query row][query head][splits][D] unnormalised sums, where splits > 1
  float2* stats;  // [query row][query head][splits] maximum (in powers of two) and sum
};

struct Request {
  int first, queries;  // query rows first .. first + queries - 1
  int length, prefix;  // cached tokens, and those before the queries (negative: fewer than queries)
};
__device__ __forceinline__ Request request_of(const kvmi_attention_args& a, int r, bool report) {
  int s0 = cld(a.starts + r), s1 = cld(a.starts + r + 1), len = cld(a.lengths + r), err = 0;
  if (s0 < 0 || s1 < s0 || s1 > a.total_queries || s1 - s0 > a.max_query) err |= KVMI_ERR_LENGTH;
  s0 = min(max(s0, 0), a.total_queries);
  s1 = min(max(s1, s0), a.total_queries);
  const int top = a.columns * a.cache.block_size;
  if (len < 0 || len > top) err |= KVMI_ERR_LENGTH;
  len = min(max(len, 0), top);
  if (err && report && a.err) atomicOr(a.err, err);
  return Request{s0, s1 - s0, len, len - (s1 - s0)};
}
// Parts that a request of so many tokens has.
__device__ __forceinline__ int parts_of(const AttendPlan& p, int length) {
  return min(p.splits, max(1, (int)(((uint32_t)length + (uint32_t)p.chunk - 1) / (uint32_t)p.chunk)));
}

// Where part `part` of `parts` of n tiles begins (n < 2^26, 64 parts at most).
__device__ __forceinline__ int part_begin(int n, int part, int parts) {
  return parts == 1 ? n * part : (int)((uint32_t)n * (uint32_t)part / (uint32_t)parts);
}

// Element offset of a token's row from the part's base, from its block's id and its place in the
// block.  A bad id is reported and the nearest block read in its place.
__device__ __forceinline__ int64_t row_offset(const kvmi_attention_args& a, int id, int place) {
  if (id < 0 || id >= a.cache.num_blocks) {
    if (a.err) atomicOr(a.err, KVMI_ERR_BLOCK_ID);
    id = min(max(id, 0), a.cache.num_blocks - 1);
  }
  return (int64_t)id * a.cache.block_stride + (int64_t)((uint32_t)place * (uint32_t)(a.cache.num_heads * a.cache.head_dim));
}

// Bit k: query i of the request (its mask row at `mask`, or null: the causal chain) sees token
// p0 + k.
__device__ __forceinline__ uint64_t seen_bits(const Request& q, const uint64_t* mask, int words, int i, int p0) {
  const int n = (mask ? q.length : min(q.length, q.prefix + i + 1)) - p0;
  uint64_t v = n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
  if (mask) {
    const int j = p0 - q.prefix;  // the draft that bit 0 stands for
    uint64_t m = 0;
    if (j < 0) {
      m = j <= -64 ? ~0ull : (1ull << -j) - 1;
      if (j > -64) m |= gld(mask) << -j;
    } else {
      const int w = j >> 6, s = j & 63;
      if (w < words) m = gld(mask + w) >> s;
      if (s && w + 1 < words) m |= gld(mask + w + 1) << (64 - s);
    }
    v &= m;
  }
  return v;
}

// ---------------------------------------------------------------- formats
template <int DT>
__device__ __forceinline__ float to_f32(uint32_t x) {
  if constexpr (DT == KVMI_DTYPE_BF16) return bf16_to_f32(x);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)x);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {  // rounded to nearest, ties to even
  if constexpr (DT == KVMI_DTYPE_BF16) return pack_bf16x2(lo, hi);
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, (h2){(_Float16)lo, (_Float16)hi});
}
// The two values of a word with infinities and NaN as zero.
template <int DT>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  constexpr uint32_t lo = DT == KVMI_DTYPE_BF16 ? 0x7f80u : 0x7c00u, hi = lo << 16;
  w = (w & hi) == hi ? w & 0xffffu : w;
  return (w & lo) == lo ? w & 0xffff0000u : w;
}
// p * x where x, the low 16 bits, is not finite; else 0.
template <int DT>
__device__ __forceinline__ float odd_term(float p, uint32_t x) {
  constexpr uint32_t e = DT == KVMI_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  return (x & e) == e ? p * to_f32<DT>(x & 0xffffu) : 0.0f;
}
// A value needed from here on: a load of it is waited for here, not at a first use inside a loop,
// where the wait would be for the loop's own loads too.
__device__ __forceinline__ void arrive(u32x4v& v) { asm volatile("" : "+v"(v)); }
// A value that is taken anew where it stands: keeps what a rare path computes from it inside
// that path.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <int DT>
__device__ __forceinline__ f32x16 mma32(u32x4v a, u32x4v b, f32x16 c) {
  if constexpr (DT == KVMI_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0,
                                                  0);
}
template <int DT>
__device__ __forceinline__ f32x4 mma16(u32x4v a, u32x4v b, f32x4 c) {
  if constexpr (DT == KVMI_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0,
                                                  0);
}
__device__ __forceinline__ u32x4v ld16(const uint16_t* p) { return *(const KVMI_GLOBAL u32x4v*)p; }
__device__ __forceinline__ u32x2v ld8(const uint16_t* p) { return *(const KVMI_GLOBAL u32x2v*)p; }

// Over lanes 32 (16) apart.
template <class F>
__device__ __forceinline__ float join32(float x, F f) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
template <class F>
__device__ __forceinline__ float join16(float x, F f) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
struct Larger {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Plus {
  __device__ float operator()(float a, float b) const { return a + b; }
};

int attend_tiles(const kvmi_attention_args& a, const AttendPlan& plan, hipStream_t st);

}  // namespace kvmi
