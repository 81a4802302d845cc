// Attention of drafted (or any last) tokens over the paged cache: the kernel for few rows, the
// joining of split sums, and the entry points.
#include "kvmi_attention.hpp"

#include <algorithm>

namespace kvmi {
namespace {

constexpr int kStep = 32;  // keys a wave takes at a time

// Few rows (16 * R at most a KV head): bound by reading the cache.  Each wave takes every NW-th
// 32 keys of the workgroup's part straight from memory into registers:
//   S^T = K Q^T     a lane has 16 bytes of key l % 16, four lanes 64 bytes of one
//   O^T += V^T P^T  a lane loads 16 bytes of each of its 8 keys, 16 lanes a whole row of 128
//                   channels; pairs of keys are brought together by byte permutes, and the
//                   output row of tile j is channel 8 * row + j
// so that keys and values do not go through LDS and, but for the queries below, no wave waits for
// another before their sums are joined at the end; a wave's own row offsets go through LDS.  64
// requests of 1 to 12 Ki tokens, 32 heads over 8, 128 channels: 323 us with the join, 5.1 TB/s, as
// fast as a copy reads and writes; 32 rows 3.7 TB/s, 256 channels 4.2; one token over 512, a chain
// of loads, 7.6 us with the join in a graph.
// N8 / N4: panels of 128 / 64 channels.  Past 16 rows, and from 129 to 192 channels, the queries
// stay in LDS (one barrier) and are read again for every 32 keys: with them in registers a wave
// would not fit its 256.  Past 192 channels it does not fit them either way, and has a SIMD's 512 to
// itself.
// WHOLE: D is all of the panels' channels.
template <int DT, int N8, int N4, int R, bool WHOLE>
__global__ __launch_bounds__((N8 == 2 ? 256 : 512), (N8 == 2 ? 1 : 2)) void attend_rows_kernel(kvmi_attention_args a,
                                                                                             AttendPlan plan) {
  constexpr bool kShared = (N8 + N4 > 1 || R > 1) && N8 < 2;
  constexpr int KS = 4 * N8 + 2 * N4, OT = 8 * N8 + 4 * N4;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // [waves][16 rows][D] sums
  __shared__ int64_t offs[8][2][kStep];
  __shared__ float2 stat[8][16 * R];
  // chunk c of row m at c ^ (m % 16): 16 rows' reads meet every bank once
  constexpr int kRowChunks = KS > 4 ? 32 : 16;
  __shared__ __attribute__((aligned(16))) uint8_t shared_q[kShared ? 16 * R * kRowChunks * 16 : 16];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const int head = blockIdx.x, part = blockIdx.y, r = blockIdx.z;
  const Request q = request_of(a, r, threadIdx.x == 0);
  const int D = a.cache.head_dim, H = a.cache.num_heads, G = a.query_heads / H;
  const int M = min(q.queries, a.max_query) * G;
  if (M == 0) return;
  const int parts = parts_of(plan, q.length);
  if (part >= parts) return;
  const uint16_t* const keys = (const uint16_t*)a.cache.base + head * D;
  const uint16_t* const values = keys + a.cache.part_stride;

  u32x4v qf[R][kShared ? 1 : KS];
  int qi[R];
  const uint64_t* mask[R];
#pragma unroll
  for (int x = 0; x < R; ++x) {
    const int m = min(16 * x + col, M - 1);
    qi[x] = plan.group(m);
    const int64_t row = q.first + qi[x];
    mask[x] = a.mask ? a.mask + row * a.mask_words : nullptr;
    const uint16_t* qp = (const uint16_t*)a.query + row * a.query_token_stride +
                         (head * G + m - qi[x] * G) * a.query_head_stride;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int d = 32 * k + 8 * g;
      const u32x4v v = d < D ? ld16(qp + d) : u32x4v{0, 0, 0, 0};
      if constexpr (kShared) {
        if (wave == 0) *(u32x4v*)(shared_q + ((16 * x + col) * kRowChunks + ((4 * k + g) ^ col)) * 16) = v;
      } else {
        qf[x][k] = v;
      }
    }
  }
  if constexpr (kShared) __syncthreads();
  // A panel's last two chunks may lie behind the head's channels: there the keys' loads repeat the
  // first 8, and are left out of the product, since an infinity times the query's zero is NaN.
  // (4 us of 121 at 256 channels, one wave a SIMD, so that whole heads have kernels of their own)
  auto key = [&](int k, u32x4v v) -> u32x4v {
    return WHOLE || k < KS - 2 || 32 * k + 8 * g < D ? v : u32x4v{0, 0, 0, 0};
  };
  auto query = [&](int x, int k, int at) -> u32x4v {  // `at`: the lane's column, taken anew
    if constexpr (kShared)
      return *(const u32x4v*)(shared_q + ((16 * x + at) * kRowChunks + ((4 * k + g) ^ at)) * 16);
    else
      return qf[x][k];
  };
  const float c = a.scale * kLog2e;
  float mx[R], l[R];
  f32x4 o[R][OT];
#pragma unroll
  for (int x = 0; x < R; ++x) {
    mx[x] = -INFINITY;
    l[x] = 0;
#pragma unroll
    for (int j = 0; j < OT; ++j) o[x][j] = f32x4{0, 0, 0, 0};
  }

  const int end = q.length, all = a.mask ? q.prefix : q.prefix + 1;  // seen by some row, by all
  const int steps = (q.length + kStep - 1) / kStep;
  const int t0 = part_begin(steps, part, parts) + wave, t1 = part_begin(steps, part + 1, parts);

  auto lookup = [&](int t) -> int64_t {
    const int p = t * kStep + (lane & 31);
    if (t >= t1 || p >= end) return 0;
    const int at = plan.block(p);
    return row_offset(a, gld(a.tables + (int64_t)r * a.columns + at), p - at * a.cache.block_size);
  };
  u32x4v kf[2][KS], v8[8][N8 ? N8 : 1];
  u32x2v v4[8];
  auto load_keys = [&](const int64_t* at) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint16_t* kp = keys + at[16 * b + col];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d = 32 * k + 8 * g;
        kf[b][k] = ld16(kp + (d < D ? d : 0));
      }
    }
  };
  auto load_values = [&](const int64_t* at) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t* vp = values + at[16 * (i >> 2) + 4 * g + (i & 3)];
#pragma unroll
      for (int n = 0; n < N8; ++n) {
        const int d = 128 * n + 8 * col;
        v8[i][n] = ld16(vp + (d < D ? d : 0));
      }
      if constexpr (N4 != 0) {
        const int d = 128 * N8 + 4 * col;
        v4[i] = ld8(vp + (d < D ? d : 0));
      }
    }
  };

  int64_t* const mine = offs[wave][0];
  if (t0 < t1) {
    if (lane < kStep) mine[lane] = lookup(t0);
    __builtin_amdgcn_wave_barrier();
    load_keys(mine);
    load_values(mine);
  }
  int buf = 0;
  for (int t = t0; t < t1; t += waves) {
    const int p0 = t * kStep;
    if (lane < kStep) mine[(buf ^ 1) * kStep + lane] = lookup(t + waves);
    f32x4 s[R][2];
    const int at = kShared ? here(col) : col;
#pragma unroll
    for (int x = 0; x < R; ++x) {
      s[x][0] = s[x][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4v v = query(x, k, at);
#pragma unroll
        for (int b = 0; b < 2; ++b) s[x][b] = mma16<DT>(key(k, kf[b][k]), v, s[x][b]);
      }
    }
    __builtin_amdgcn_wave_barrier();
    const int64_t* const next = mine + (buf ^ 1) * kStep;
    load_keys(next);
    const bool masked = p0 + kStep > all || p0 + kStep > end;
    uint32_t seen[R];
#pragma unroll
    for (int x = 0; x < R; ++x) {
      seen[x] = ~0u;
      if (masked) {
        seen[x] = (uint32_t)seen_bits(q, mask[x], a.mask_words, qi[x], p0);
        const uint32_t v = seen[x] >> (4 * g);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[x][b][i] = (v >> (16 * b + i)) & 1 ? s[x][b][i] : -INFINITY;
      }
    }
    u32x4v pf[R];
#pragma unroll
    for (int x = 0; x < R; ++x) {
      float top = fmaxf(fmaxf(fmaxf(s[x][0][0], s[x][0][1]), fmaxf(s[x][0][2], s[x][0][3])),
                        fmaxf(fmaxf(s[x][1][0], s[x][1][1]), fmaxf(s[x][1][2], s[x][1][3])));
      top = join32(join16(top, Larger()), Larger()) * c;
      const bool raise = top > mx[x] + kRaise;
      if (__ballot(raise)) {
        const float f = raise ? __builtin_amdgcn_exp2f(mx[x] - top) : 1.0f;
        mx[x] = raise ? top : mx[x];
        l[x] *= f;
#pragma unroll
        for (int j = 0; j < OT; ++j) o[x][j] *= f;
      }
      const float ms = mx[x] == -INFINITY ? 0.0f : mx[x];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[x][b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][b][i], c, -ms));
        l[x] += (s[x][b][0] + s[x][b][1]) + (s[x][b][2] + s[x][b][3]);
        pf[x][2 * b] = pack2<DT>(s[x][b][0], s[x][b][1]);
        pf[x][2 * b + 1] = pack2<DT>(s[x][b][2], s[x][b][3]);
      }
    }
    if (masked) {
      // a weight of zero has to give zero: values past the end, and those that are not finite,
      // leave the product; the latter then go to the rows that see them
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = 16 * (i >> 2) + 4 * g + (i & 3);
        bool odd = false;
        const bool in = p0 + key < end;
#pragma unroll
        for (int n = 0; n < N8; ++n)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t f = in ? finite2<DT>(v8[i][n][w]) : 0;
            odd |= in && f != v8[i][n][w];
            v8[i][n][w] = f;
          }
        if constexpr (N4 != 0) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t f = in ? finite2<DT>(v4[i][w]) : 0;
            odd |= in && f != v4[i][w];
            v4[i][w] = f;
          }
        }
        const uint64_t b = __ballot(odd);
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if ((b >> (16 * y)) & 0xffff) bad |= 1u << (16 * (i >> 2) + 4 * y + (i & 3));
      }
      bad = __builtin_amdgcn_readfirstlane(bad);
#pragma unroll 1
      while (bad) {
        const int key = __builtin_ctz(bad), at = (key >> 4) * 4 + (key & 3);
        bad &= bad - 1;
        const uint16_t* const vp = values + mine[buf * kStep + key];
#pragma unroll
        for (int x = 0; x < R; ++x) {
          float p = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) p = i == at ? s[x][i >> 2][i & 3] : p;
          p = __shfl(p, col + 16 * ((key >> 2) & 3), 64);
          const bool sees = (seen[x] >> key) & 1;
          const int g0 = here(g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int n = 0; n < N8; ++n) {
              const u32x4v v = ld16(vp + min(128 * n + 8 * (4 * g0 + i), D - 8));
#pragma unroll
              for (int j = 0; j < 8; ++j)
                o[x][8 * n + j][i] += sees ? odd_term<DT>(p, v[j >> 1] >> (16 * (j & 1))) : 0.0f;
            }
            if constexpr (N4 != 0) {
              const u32x2v v = ld8(vp + min(128 * N8 + 4 * (4 * g0 + i), D - 4));
#pragma unroll
              for (int j = 0; j < 4; ++j)
                o[x][8 * N8 + j][i] += sees ? odd_term<DT>(p, v[j >> 1] >> (16 * (j & 1))) : 0.0f;
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < OT; ++j) {
      const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
      u32x4v f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (j < 8 * N8)
          f[w] = __builtin_amdgcn_perm(v8[2 * w + 1][j >> 3][(j & 7) >> 1], v8[2 * w][j >> 3][(j & 7) >> 1], sel);
        else
          f[w] = __builtin_amdgcn_perm(v4[2 * w + 1][(j & 3) >> 1], v4[2 * w][(j & 3) >> 1], sel);
      }
#pragma unroll
      for (int x = 0; x < R; ++x) o[x][j] = mma16<DT>(f, pf[x], o[x][j]);
    }
    load_values(next);
    buf ^= 1;
  }

  // the waves' sums, brought to their common maximum and added up in the waves' order, 16 rows at
  // a time (32 at once take the LDS of two workgroups)
  const int DP = D + 4;
  float* const sums = (float*)lds;
#pragma unroll
  for (int x = 0; x < R; ++x) {
    l[x] = join32(join16(l[x], Plus()), Plus());
    if (g == 0) stat[wave][16 * x + col] = make_float2(mx[x], l[x]);
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < R; ++x) {
    const int rows = min(M - 16 * x, 16);
    if (rows <= 0) break;
    if (x) __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < waves; ++w) top = fmaxf(top, stat[w][16 * x + col].x);
    const float f = mx[x] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx[x] - top);
    if (col < rows) {
      float* const dst = sums + (wave * 16 + col) * DP;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int n = 0; n < 2 * N8; ++n) {
          const int d = 128 * (n >> 1) + 8 * (4 * g + i) + 4 * (n & 1), j = 4 * n;
          if (d < D) *(f32x4*)(dst + d) = f32x4{o[x][j][i], o[x][j + 1][i], o[x][j + 2][i], o[x][j + 3][i]} * f;
        }
        if constexpr (N4 != 0) {
          constexpr int j = 8 * N8;
          const int d = 128 * N8 + 4 * (4 * g + i);
          if (d < D) *(f32x4*)(dst + d) = f32x4{o[x][j][i], o[x][j + 1][i], o[x][j + 2][i], o[x][j + 3][i]} * f;
        }
      }
    }
    __syncthreads();
    // D / 4 lanes, or the next power of two, a row
    const int lanes_log2 = D > 128 ? 6 : D > 64 ? 5 : D > 32 ? 4 : D > 16 ? 3 : 2;
    for (int e = threadIdx.x; e < rows << lanes_log2; e += blockDim.x) {
      const int at = e >> lanes_log2, d = 4 * (e - (at << lanes_log2)), m = 16 * x + at;
      if (d >= D) continue;
      float most = -INFINITY, total = 0;
      for (int w = 0; w < waves; ++w) most = fmaxf(most, stat[w][m].x);
      f32x4 v = {0, 0, 0, 0};
      for (int w = 0; w < waves; ++w) {
        const float2 s = stat[w][m];
        total += s.y == 0 ? 0.0f : s.y * __builtin_amdgcn_exp2f(s.x - most);  // (0: saw nothing)
        v += *(const f32x4*)(sums + (w * 16 + at) * DP + d);
      }
      const int i = plan.group(m);
      const int64_t out_row = (int64_t)(q.first + i) * a.query_heads + head * G + m - i * G;
      if (parts == 1) {
        const float f = total == 0 ? 0.0f : 1.0f / total;
        gst((uint2*)((uint16_t*)a.out + out_row * D + d),
            make_uint2(pack2<DT>(v[0] * f, v[1] * f), pack2<DT>(v[2] * f, v[3] * f)));
        if (a.lse && d == 0) a.lse[out_row] = total == 0 ? -INFINITY : (most + __builtin_amdgcn_logf(total)) / kLog2e;
      } else {
        *(KVMI_GLOBAL f32x4*)(plan.sums + (out_row * plan.splits + part) * D + d) = v;
        if (d == 0) plan.stats[out_row * plan.splits + part] = make_float2(most, total);
      }
    }
  }
}

// The parts of each query head of a request that was split, joined in their order (3 us for 8
// parts of 32 rows, 7 for the 19 MB of 1900 queries' parts).  D / 4 lanes,
// or the next power of two, a row.
template <int DT>
__global__ __launch_bounds__(256) void join_kernel(kvmi_attention_args a, AttendPlan plan, int lanes_log2) {
  const int r = blockIdx.y, D = a.cache.head_dim;
  const Request q = request_of(a, r, false);
  const int parts = parts_of(plan, q.length);
  if (parts == 1) return;
  const int d = 4 * (threadIdx.x & ((1 << lanes_log2) - 1)), per = 256 >> lanes_log2;
  const int rows = min(q.queries, a.max_query) * a.query_heads;
  if (d >= D) return;
  for (int e = (int)blockIdx.x * per + (threadIdx.x >> lanes_log2); e < rows; e += (int)gridDim.x * per) {
    const int64_t row = (int64_t)q.first * a.query_heads + e;
    const float2* const stats = plan.stats + row * plan.splits;
    const float* const sums = plan.sums + row * plan.splits * D + d;
    // kAtOnce parts' loads together, then their sums with a running maximum
    constexpr int kAtOnce = 8;
    float top = -INFINITY, total = 0;
    f32x4 v = {0, 0, 0, 0};
    for (int s0 = 0; s0 < parts; s0 += kAtOnce) {
      float2 st[kAtOnce];
      f32x4 x[kAtOnce];
#pragma unroll
      for (int s = 0; s < kAtOnce; ++s) {
        const int at = min(s0 + s, parts - 1);
        st[s] = stats[at];
        x[s] = *(const KVMI_GLOBAL f32x4*)(sums + (int64_t)at * D);
        if (s0 + s >= parts) st[s] = make_float2(-INFINITY, 0);
      }
      float most = top;
#pragma unroll
      for (int s = 0; s < kAtOnce; ++s) most = fmaxf(most, st[s].x);
      const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - most);
      total *= f;
      v *= f;
      top = most;
#pragma unroll
      for (int s = 0; s < kAtOnce; ++s)
        if (st[s].y != 0) {  // 0: saw nothing; a part of NaN scores has a NaN sum and no maximum
          const float g = __builtin_amdgcn_exp2f(st[s].x - top);
          total += st[s].y * g;
          v += x[s] * g;
        }
    }
    const float f = total == 0 ? 0.0f : 1.0f / total;
    gst((uint2*)((uint16_t*)a.out + row * D + d),
        make_uint2(pack2<DT>(v[0] * f, v[1] * f), pack2<DT>(v[2] * f, v[3] * f)));
    if (a.lse && d == 0) a.lse[row] = total == 0 ? -INFINITY : (top + __builtin_amdgcn_logf(total)) / kLog2e;
  }
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
  if ((int64_t)a->columns * c.block_size > kMostPlaces || (int64_t)c.num_blocks * c.block_size > 0x7fffffffLL ||
      (int64_t)a->max_query * a->query_heads > kMostPlaces ||
      (int64_t)c.block_size * c.num_heads * c.head_dim > 0x7fffffffLL)
    return false;
  if (a->mask && a->mask_words < 1) return false;
  return true;
}

struct Choice {
  bool rows;     // the kernel for few rows
  int row_groups;
  AttendPlan plan;
};
int64_t parts_bytes(const kvmi_attention_args& a, int splits) {
  const int64_t rows = (int64_t)a.total_queries * a.query_heads * splits;
  return splits == 1 ? 0 : rows * (a.cache.head_dim * 4 + 8);
}
Choice choose(const kvmi_attention_args& a) {
  Choice c{};
  const int G = a.query_heads / a.cache.num_heads, D = a.cache.head_dim;
  const int64_t rows = (int64_t)a.max_query * G;
  c.row_groups = rows <= 16 ? 1 : 2;
  c.rows = rows <= (D <= 128 ? 32 : 16);
  const int64_t length = a.max_length < 1 ? 1 : a.max_length;
  c.plan.block = block_of(a.cache.block_size);
  c.plan.group = block_of(G);
  c.plan.waves = 4;
  c.plan.row_tiles = 1;
  // Row tiles that have rows: requests may differ in queries, but not add up to more than all.
  auto tiles_of = [&](int tile) -> int64_t {
    return std::min<int64_t>(a.requests * ((rows + tile - 1) / tile), (int64_t)a.total_queries * G / tile + a.requests);
  };
  int64_t tiles = a.requests;
  if (!c.rows) {
    // Tiles of 256 rows where those alone fill every CU twice over, for 97 to 128 channels, whose
    // 4 waves have half a CU's registers: a tile of keys is loaded once for both halves (a prompt
    // of 8192: 577 -> 555 us; 64 channels, three workgroups of 4 waves a CU: 332 -> 368), and are
    // mostly full.
    const bool full = rows >= 1024 || (rows + 127) / 128 % 2 == 0;
    if (D > 96 && D <= 128 && full && tiles_of(256) * a.cache.num_heads >= 512) c.plan.waves = 8;
    c.plan.row_tiles = (int)((rows + 32 * c.plan.waves - 1) / (32 * c.plan.waves));
    tiles = tiles_of(32 * c.plan.waves);
  }
  const int64_t groups = tiles * a.cache.num_heads;
  // Keys are split until there are workgroups for the chip, one a CU for few rows (a workgroup
  // then keeps 4 waves' loads in flight) and two for tiles, but not below the part at which the
  // join costs more than it saves: 64 keys of few rows (512 keys of one token in a graph: 7.5 us in
  // 8 parts, 8.3 in 4, 8.8 in 16, 9.6 whole), 256 of tiles.  Few rows are split at 704 keys in any
  // case, against requests of unequal lengths and a last round of workgroups that leaves the chip
  // half empty.  That is a compromise of four batches, two of which would have more (us at 512 / 704
  // / 1024 / 1536 keys: 64 requests of 1 to 12 Ki 333 / 325 / 325 / 329, 64 of 1 to 8 Ki and 64
  // channels 128 / 127 / 140 / 132, 32 of 256 channels 123 / 119 / 135 / 108, 256 of up to 3 Ki
  // 357 / 340 / 333 / 350).  Tiles of a ragged batch are not split below the longest request: every
  // finer part costs more than the chains it cuts (96 trees over 200 to 2000 tokens whole 54.7, at
  // 1024 / 768 / 512 keys 64.2 / 58.7 / 65.2).
  const bool even = (int64_t)a.requests * c.plan.row_tiles <= tiles;  // all have the most queries
  const int64_t room = c.rows ? 256 : 512, want = std::max<int64_t>(1, (room + (even ? 0 : groups - 1)) / groups);
  c.plan.chunk = (int)std::max<int64_t>((length + want - 1) / want, c.rows ? 64 : 256);
  if (c.rows) {
    c.plan.chunk = std::min(c.plan.chunk, 704);
    c.plan.waves = std::min(4, (c.plan.chunk + kStep - 1) / kStep);
  }
  int64_t splits = std::min<int64_t>((length + c.plan.chunk - 1) / c.plan.chunk, 64);
  while (splits > 1 && parts_bytes(a, (int)splits) > (1LL << 31)) splits /= 2;
  c.plan.splits = (int)splits;
  c.plan.tiles = block_of(c.plan.row_tiles * (int)splits);
  c.plan.heads = block_of(a.cache.num_heads);
  return c;
}

template <int DT>
void launch_rows(const kvmi_attention_args& a, const Choice& c, hipStream_t st) {
  const int D = a.cache.head_dim;
  const dim3 grid((unsigned)a.cache.num_heads, (unsigned)c.plan.splits, (unsigned)a.requests);
  const dim3 threads((unsigned)(64 * c.plan.waves));
  const size_t lds = (size_t)c.plan.waves * 16 * (D + 4) * 4;
#define KVMI_ROWS(N8, N4, R)                                                                       \
  do {                                                                                             \
    if (D == 128 * N8 + 64 * N4)                                                                   \
      hipLaunchKernelGGL((attend_rows_kernel<DT, N8, N4, R, true>), grid, threads, lds, st, a, c.plan);  \
    else                                                                                           \
      hipLaunchKernelGGL((attend_rows_kernel<DT, N8, N4, R, false>), grid, threads, lds, st, a, c.plan); \
  } while (0)
  if (D > 192)
    KVMI_ROWS(2, 0, 1);
  else if (D > 128)
    KVMI_ROWS(1, 1, 1);
  else if (D > 64 && c.row_groups == 1)
    KVMI_ROWS(1, 0, 1);
  else if (D > 64)
    KVMI_ROWS(1, 0, 2);
  else if (c.row_groups == 1)
    KVMI_ROWS(0, 1, 1);
  else
    KVMI_ROWS(0, 1, 2);
#undef KVMI_ROWS
}

}  // namespace
}  // namespace kvmi

extern "C" int64_t kvmi_attention_workspace_bytes(const kvmi_attention_args* args) {
  using namespace kvmi;
  if (!attention_ok(args)) return KVMI_EINVAL;
  if (args->requests == 0 || args->total_queries == 0 || args->max_query == 0) return 0;
  return parts_bytes(*args, choose(*args).plan.splits);
}

extern "C" int kvmi_attention_kernels(const kvmi_attention_args* args, int32_t* shape) {
  using namespace kvmi;
  if (!attention_ok(args) || args->requests == 0 || args->total_queries == 0 || args->max_query == 0)
    return KVMI_EINVAL;
  const Choice c = choose(*args);
  if (shape) {
    shape[0] = c.plan.waves;
    shape[1] = c.rows ? 16 * c.row_groups : 32 * c.plan.waves;
    shape[2] = c.plan.splits;
    shape[3] = c.plan.chunk;
  }
  return c.rows ? KVMI_ATTENTION_ROWS : KVMI_ATTENTION_TILES;
}

extern "C" int kvmi_tree_attention(const kvmi_attention_args* args, kvmi_stream_t stream) {
  using namespace kvmi;
  if (!attention_ok(args)) return KVMI_EINVAL;
  const kvmi_attention_args& a = *args;
  if (a.requests == 0 || a.total_queries == 0 || a.max_query == 0) return KVMI_OK;
  if (!a.query || !a.out || !a.tables || !a.lengths || !a.starts || (uintptr_t)a.query % 16 ||
      (uintptr_t)a.out % 16 || a.query_token_stride % 8 || a.query_head_stride % 8)
    return KVMI_EINVAL;
  Choice c = choose(a);
  const int64_t space = parts_bytes(a, c.plan.splits);
  // the tiles kernel's workgroups are numbered in 31 bits
  if ((!c.rows && ((int64_t)a.requests * a.cache.num_heads + 7) / 8 * 8 * c.plan.row_tiles * c.plan.splits > 0x7fffffffLL) ||
      (space && (!a.workspace || a.workspace_bytes < space || (uintptr_t)a.workspace % 16)))
    return KVMI_EINVAL;
  c.plan.sums = (float*)a.workspace;
  c.plan.stats = (float2*)((uint8_t*)a.workspace +
                           (int64_t)a.total_queries * a.query_heads * c.plan.splits * a.cache.head_dim * 4);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool bf16 = a.dtype == KVMI_DTYPE_BF16;
  if (!c.rows) {
    const int rc = attend_tiles(a, c.plan, st);
    if (rc != KVMI_OK) return rc;
  } else if (bf16) {
    launch_rows<KVMI_DTYPE_BF16>(a, c, st);
  } else {
    launch_rows<KVMI_DTYPE_FP16>(a, c, st);
  }
  if (c.plan.splits > 1) {
    int lanes_log2 = 1;
    while ((4 << lanes_log2) < a.cache.head_dim) ++lanes_log2;
    const int per = 256 >> lanes_log2;
    const int64_t rows = (int64_t)a.max_query * a.query_heads;
    // (requests of fewer queries than the most leave workgroups without rows)
    const int64_t most = std::max<int64_t>(1, 4096 / a.requests);
    const dim3 grid((unsigned)std::min((rows + per - 1) / per, most), (unsigned)a.requests);
    if (bf16)
      hipLaunchKernelGGL((join_kernel<KVMI_DTYPE_BF16>), grid, dim3(256), 0, st, a, c.plan, lanes_log2);
    else
      hipLaunchKernelGGL((join_kernel<KVMI_DTYPE_FP16>), grid, dim3(256), 0, st, a, c.plan, lanes_log2);
  }
  return hipGetLastError() == hipSuccess ? KVMI_OK : KVMI_ELAUNCH;
}
