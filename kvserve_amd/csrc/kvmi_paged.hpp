// Shared by the paged cache's operators: error bits, places in the ring of free blocks, checks of
// a cache's description.
#pragma once

#include "kvmi_common.hpp"

namespace kvmi {
namespace {

__device__ __forceinline__ void flag_error(int32_t* err, int32_t bits) {
  if (err && bits) atomicOr(err, bits);
}
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
// Place of the i-th entry behind `base` in a ring of N (base < N, i <= N).
__device__ __forceinline__ uint32_t ring_at(uint32_t base, uint32_t i, uint32_t N) {
  const uint32_t x = base + i;
  return x < N ? x : x - N;
}

inline bool cache_ok(const kvmi_cache* c, bool base) {
  return c && (!base || c->base) && c->num_blocks >= 1 && c->block_size >= 1 && c->num_heads >= 1 && c->head_dim >= 1 &&
         c->part_stride >= 0 && c->block_stride >= (int64_t)c->block_size * c->num_heads * c->head_dim &&
         (int64_t)c->num_blocks * c->block_size < 0x7fffffffLL && (int64_t)c->num_heads * c->head_dim < (1 << 24);
}
inline bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
inline bool strides16(const kvmi_cache* c) {
  return c->head_dim % 8 == 0 && c->part_stride % 8 == 0 && c->block_stride % 8 == 0;
}
inline int launched() { return hipGetLastError() == hipSuccess ? KVMI_OK : KVMI_ELAUNCH; }

}  // namespace
}  // namespace kvmi
