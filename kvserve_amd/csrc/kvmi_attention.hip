// Attention of drafted (or any last) tokens over the paged cache.
#include "kvmi_common.hpp"

namespace kvmi {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <int DT>
__device__ __forceinline__ float to_f32(uint16_t x) {
  if constexpr (DT == KVMI_DTYPE_BF16) return bf16_to_f32(x);
  return (float)__builtin_bit_cast(_Float16, x);
}
template <int DT>
__device__ __forceinline__ uint16_t from_f32(float x) {
  if constexpr (DT == KVMI_DTYPE_BF16) return (uint16_t)f32_to_bf16_bits(x);
  return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// One wave a query row: 64 keys at a time, a lane a key for the scores, a lane four channels
// for the sums.
template <int DT>
__global__ __launch_bounds__(64) void attend_kernel(kvmi_attention_args a) {
  __shared__ float q[256], w[64];
  __shared__ int64_t at[64];
  const int lane = threadIdx.x, r = blockIdx.y;
  const int i = blockIdx.x / a.query_heads, head = blockIdx.x % a.query_heads;
  const int D = a.cache.head_dim, S = a.cache.block_size;
  int s0 = a.starts[r], s1 = a.starts[r + 1], err = 0;
  if (s0 < 0 || s1 < s0 || s1 > a.total_queries || s1 - s0 > a.max_query) err |= KVMI_ERR_LENGTH;
  s0 = min(max(s0, 0), a.total_queries);
  s1 = min(max(s1, s0), a.total_queries);
  int L = a.lengths[r];
  const int top = a.columns * S;
  if (L < 0 || L > top) err |= KVMI_ERR_LENGTH;
  L = min(max(L, 0), top);
  if (err && a.err && lane == 0) atomicOr(a.err, err);
  const int T = s1 - s0, prefix = L - T;
  if (i >= T) return;
  const int64_t row = s0 + i;
  const uint16_t* qp = (const uint16_t*)a.query + row * a.query_token_stride + head * a.query_head_stride;
  for (int d = lane; d < D; d += 64) q[d] = to_f32<DT>(qp[d]);
  __syncthreads();
  const uint16_t* base = (const uint16_t*)a.cache.base + (head / (a.query_heads / a.cache.num_heads)) * D;
  const float c = a.scale * kLog2e;
  float m = -INFINITY, l = 0, o[4] = {0, 0, 0, 0};
  const int end = a.mask ? L : min(L, prefix + i + 1);
  for (int p0 = 0; p0 < end; p0 += 64) {
    const int p = p0 + lane;
    bool seen = p < end;
    int64_t off = 0;
    float s = -INFINITY;
    if (seen) {
      int id = a.tables[(int64_t)r * a.columns + p / S];
      if (id < 0 || id >= a.cache.num_blocks) {
        if (a.err) atomicOr(a.err, KVMI_ERR_BLOCK_ID);
        id = min(max(id, 0), a.cache.num_blocks - 1);
      }
      off = (int64_t)id * a.cache.block_stride + (int64_t)(p % S) * a.cache.num_heads * D;
      const int j = p - prefix;
      if (a.mask && j >= 0)
        seen = j < a.mask_words * 64 && ((a.mask[row * a.mask_words + j / 64] >> (j % 64)) & 1);
    }
    if (seen) {
      s = 0;
      for (int d = 0; d < D; ++d) s += q[d] * to_f32<DT>(base[off + d]);
      s *= c;
    }
    float mx = s;
#pragma unroll
    for (int d = 32; d; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
    const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.0f : mn;
    const float f = __builtin_amdgcn_exp2f(m - ms), x = seen ? __builtin_amdgcn_exp2f(s - ms) : 0.0f;
    m = mn;
    l = l * f + x;
    __syncthreads();
    w[lane] = x;
    at[lane] = seen ? off : -1;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] *= f;
    for (int t = 0; t < 64; ++t) {
      if (at[t] < 0) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (lane + 64 * k < D) o[k] += w[t] * to_f32<DT>(base[a.cache.part_stride + at[t] + lane + 64 * k]);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d, 64);
  uint16_t* out = (uint16_t*)a.out + (row * a.query_heads + head) * D;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 64 * k < D) out[lane + 64 * k] = from_f32<DT>(l == 0 ? 0.0f : o[k] / l);
  if (a.lse && lane == 0)
    a.lse[row * a.query_heads + head] = l == 0 ? -INFINITY : (m + __builtin_amdgcn_logf(l)) / kLog2e;
}

bool attention_ok(const kvmi_attention_args* a) {
  if (!a) return false;
  const kvmi_cache& c = a->cache;
  if (!c.base || c.num_blocks < 1 || c.block_size < 1 || c.num_heads < 1 || c.head_dim < 8 || c.head_dim > 256 ||
      c.head_dim % 8 || c.part_stride < 0 || c.part_stride % 8 || c.block_stride % 8 ||
      c.block_stride < (int64_t)c.block_size * c.num_heads * c.head_dim || (uintptr_t)c.base % 16)
    return false;
  if (a->requests < 0 || a->requests > 65535 || a->columns < 1 || a->total_queries < 0 || a->max_query < 0 ||
      a->max_length < 0 || a->query_heads < 1 || a->query_heads % c.num_heads ||
      (a->dtype != KVMI_DTYPE_BF16 && a->dtype != KVMI_DTYPE_FP16) || !(a->scale > 0) || a->scale > 3.0e38f)
    return false;
  if ((int64_t)a->columns * c.block_size > 0x7fffffffLL || (int64_t)c.num_blocks * c.block_size > 0x7fffffffLL ||
      (int64_t)a->max_query * a->query_heads > 0x7fffffffLL)
    return false;
  if (a->mask && a->mask_words < 1) return false;
  return true;
}

}  // namespace
}  // namespace kvmi

extern "C" int64_t kvmi_attention_workspace_bytes(const kvmi_attention_args* args) {
  return kvmi::attention_ok(args) ? 0 : KVMI_EINVAL;
}

extern "C" int kvmi_tree_attention(const kvmi_attention_args* args, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!attention_ok(args)) return KVMI_EINVAL;
  const kvmi_attention_args& a = *args;
  if (a.requests == 0 || a.total_queries == 0 || a.max_query == 0) return KVMI_OK;
  if (!a.query || !a.out || !a.tables || !a.lengths || !a.starts || (uintptr_t)a.query % 16 ||
      a.query_token_stride % 8 || a.query_head_stride % 8)
    return KVMI_EINVAL;
  const dim3 grid((unsigned)(a.max_query * a.query_heads), (unsigned)a.requests);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a.dtype == KVMI_DTYPE_BF16)
    hipLaunchKernelGGL((attend_kernel<KVMI_DTYPE_BF16>), grid, dim3(64), 0, st, a);
  else
    hipLaunchKernelGGL((attend_kernel<KVMI_DTYPE_FP16>), grid, dim3(64), 0, st, a);
  return hipGetLastError() == hipSuccess ? KVMI_OK : KVMI_ELAUNCH;
}
