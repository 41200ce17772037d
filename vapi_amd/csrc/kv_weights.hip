// Running attention weights: the columns' sums of a step's softmax.
//
//   w[g, k] = decay w[g, k] + sum_r exp2(s[r, k] - lse[r])
//
// over the rows r = (query, query head of g) of one sequence and kv head, with
// s the scores in log2 units and lse[r] = log2 sum_k exp2 s[r, k]. The sum over
// a row's keys has to be known before the first of its weights is, so there are
// two passes over K Q^T and nothing but (m, l) of each row between them:
//  1. weights_lse: a workgroup takes up to 16 MT rows and a chunk of keys, its
//     four waves every fourth 16-key tile; a lane keeps a running maximum and
//     sum of its own over the keys it sees, joined across lanes and waves at
//     the end: (m, l) per row and chunk.
//  2. weights_sum: a wave holds KT 16-key tiles of K in registers, walks the
//     rows that see them and adds up exp2(s - lse) per key; the 16 lanes of a
//     key are added at the end. Each weight has one owner: no atomics, a fixed
//     order.
// S^T = K Q^T as in the attention kernels (lane (col, g) holds keys 4 g .. +3
// of row col), straight from HBM/L2 into MFMA operands. Pass 2 reads K again:
// from L2 or the last-level cache where a call's K fits them.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "q8.hpp"

namespace vk {

// What K is stored as: the rows' own 16-bit type or a format of 8-bit codes.
constexpr int kK16 = -1;

struct WeightArgs {
  const char* k;
  const float* k_scale;  // 8-bit pools
  const char* q;
  const uint32_t *cu_q, *cu_k, *table, *index;
  float* w;
  float2* ml;  // [batch][kvh][row_cap][n_chunk]
  uint64_t blk_b, head_b;  // bytes
  uint32_t tok_b, sblk, last_blk, bs_shift, max_blocks;
  uint64_t row_stride, head_stride;
  uint32_t n_rows, width;
  uint32_t kvh, num_heads, hd, last_queries;
  FastDiv group;
  uint32_t row_cap, n_chunk, chunk_keys;
  float scale_log2, decay;
  int32_t wl, wr;
};

// One (sequence, kv head): its rows and keys.
struct WeightSeg {
  uint32_t seq, h, q0, n_rows;  // q0: the first query taken
  int32_t len_k, pos0;          // pos0: its position
  uint32_t state_row;
  bool ok;
};
__device__ __forceinline__ WeightSeg weight_seg(const WeightArgs& a, uint32_t seg) {
  WeightSeg s;
  s.seq = seg / a.kvh;
  s.h = seg - s.seq * a.kvh;
  const uint32_t end = a.cu_q[s.seq + 1], len_q = end - a.cu_q[s.seq];
  s.len_k = (int32_t)(a.cu_k[s.seq + 1] - a.cu_k[s.seq]);
  const uint32_t n_q = a.last_queries ? min(len_q, a.last_queries) : len_q;
  s.q0 = end - n_q;
  // (Rows past what the workspace was sized for, which no valid call has, are
  // left out.)
  s.n_rows = min(n_q * a.group.d, a.row_cap);
  s.pos0 = s.len_k - (int32_t)n_q;
  s.state_row = a.index ? a.index[s.seq] : s.seq;
  s.ok = n_q > 0 && s.len_k > 0 && s.state_row < a.n_rows;
  s.len_k = min(s.len_k, (int32_t)a.width);
  return s;
}

// The d of chunk c's eight elements in lane group g, for Q and K alike (8-bit
// codes come 16 to a load).
template <int F>
__device__ __forceinline__ uint32_t weight_d(int c, uint32_t g) {
  return F == kK16 ? 32 * c + 8 * g : 64 * (c / 2) + 16 * g + 8 * (c % 2);
}

// Q operand of 16 rows from `first` (rows past the segment's repeat its last).
template <typename T, int F, int D>
__device__ __forceinline__ void weight_q(uint4 (&q)[D / 32], const WeightArgs& a,
                                         const WeightSeg& s, uint32_t row, uint32_t g) {
  row = min(row, s.n_rows - 1);
  const uint32_t j = a.group.div(row), c = row - j * a.group.d;
  const T* p = (const T*)a.q +
               ((uint64_t)(s.q0 + j) * a.num_heads + s.h * a.group.d + c) * a.hd;
#pragma unroll
  for (int c2 = 0; c2 < D / 32; ++c2) {
    const uint32_t d = weight_d<F>(c2, g);
    q[c2] = d < a.hd ? *(const uint4*)(p + d) : make_uint4(0u, 0u, 0u, 0u);
  }
}

// A 16-key tile as it is stored, and its scale. Keys past the last repeat it.
template <int F, int D>
struct WeightTile {
  uint4 w[F == kK16 ? D / 32 : D / 64];
  float scale;
};
template <int F, int D>
__device__ __forceinline__ void weight_load(WeightTile<F, D>& t, const WeightArgs& a,
                                            const WeightSeg& s, int32_t key, uint32_t col,
                                            uint32_t g) {
  using ConstU32 = const __attribute__((address_space(4))) uint32_t;
  using ConstF32 = const __attribute__((address_space(4))) float;
  const int32_t last = s.len_k - 1;
  const int32_t ts = __builtin_amdgcn_readfirstlane(min(key, last & ~15));
  ConstU32* tab = (ConstU32*)(a.table + (uint64_t)s.seq * a.max_blocks);
  const uint32_t blk = min(tab[min((uint32_t)ts >> a.bs_shift, a.max_blocks - 1)], a.last_blk);
  const uint32_t off = (uint32_t)ts & ((1u << a.bs_shift) - 1);
  const char* p = a.k + blk * a.blk_b + s.h * a.head_b + (uint64_t)off * a.tok_b +
                  (uint32_t)min((int32_t)col, last - ts) * a.tok_b;
  t.scale = 1.f;
  if constexpr (F != kK16) t.scale = ((ConstF32*)a.k_scale)[(uint64_t)blk * a.sblk + s.h];
  constexpr int N = F == kK16 ? D / 32 : D / 64;
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const uint32_t b = 64 * c + 16 * g;  // bytes into the row
    t.w[c] = b < a.hd * (F == kK16 ? 2 : 1) ? *(const uint4*)(p + b) : make_uint4(0u, 0u, 0u, 0u);
  }
}
// The tile as MFMA operands (codes unscaled).
template <typename T, int F, int D>
__device__ __forceinline__ void weight_operand(const WeightTile<F, D>& t, uint4 (&k)[D / 32]) {
  if constexpr (F == kK16) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) k[c] = t.w[c];
  } else {
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 w = t.w[c];
      const uint2 a0 = q8_expand4<T, F, false>(w.x, 1.f), a1 = q8_expand4<T, F, false>(w.y, 1.f);
      const uint2 b0 = q8_expand4<T, F, false>(w.z, 1.f), b1 = q8_expand4<T, F, false>(w.w, 1.f);
      k[2 * c] = make_uint4(a0.x, a0.y, a1.x, a1.y);
      k[2 * c + 1] = make_uint4(b0.x, b0.y, b1.x, b1.y);
    }
  }
}
template <typename T, int D>
__device__ __forceinline__ floatx4 weight_dot(const uint4 (&k)[D / 32], const uint4 (&q)[D / 32]) {
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < D / 32; ++c) acc = mfma16x16x32<T>(k[c], q[c], acc);
  return acc;
}

// Keys that a query at `pos` sees: [lo, hi].
__device__ __forceinline__ int32_t weight_lo(const WeightArgs& a, int32_t pos) {
  return a.wl >= 0 ? max(0, pos - a.wl) : 0;
}
__device__ __forceinline__ int32_t weight_hi(const WeightArgs& a, int32_t pos, int32_t len_k) {
  return a.wr >= 0 ? (int32_t)min((int64_t)len_k - 1, (int64_t)pos + a.wr) : len_k - 1;
}

constexpr int kWeightWaves = 4;

// ---- pass 1 --------------------------------------------------------------------

// Grid: (row tiles x chunks, segments).
template <typename T, int F, int D, int MT>
__global__ __launch_bounds__(64 * kWeightWaves) void weights_lse(WeightArgs a) {
  __shared__ float2 part[kWeightWaves][16 * MT];
  const WeightSeg s = weight_seg(a, blockIdx.y);
  if (!s.ok) return;
  const uint32_t tile = blockIdx.x / a.n_chunk, chunk = blockIdx.x - tile * a.n_chunk;
  const uint32_t row0 = tile * 16 * MT;
  if (row0 >= s.n_rows) return;
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int32_t wave = (int32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint4 q[MT][D / 32];
  int32_t lo[MT], hi[MT];
  float m[MT], l[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const uint32_t row = row0 + 16 * t + col;
    weight_q<T, F, D>(q[t], a, s, row, g);
    const int32_t pos = s.pos0 + (int32_t)a.group.div(min(row, s.n_rows - 1));
    lo[t] = weight_lo(a, pos), hi[t] = weight_hi(a, pos, s.len_k);
    m[t] = kNegBig, l[t] = 0.f;
  }
  // The keys any row of the tile sees, and those all of them see.
  const uint32_t row1 = min(row0 + 16 * MT, s.n_rows) - 1;
  const int32_t p0 = s.pos0 + (int32_t)a.group.div(row0), p1 = s.pos0 + (int32_t)a.group.div(row1);
  const int32_t all_lo = weight_lo(a, p1), all_hi = weight_hi(a, p0, s.len_k);
  const int32_t c0 = (int32_t)(chunk * a.chunk_keys);
  const int32_t c1 = (int32_t)min((int64_t)c0 + a.chunk_keys, (int64_t)s.len_k) - 1;
  const int32_t k0 = max(c0, weight_lo(a, p0) & ~15), k1 = min(c1, weight_hi(a, p1, s.len_k));
  WeightTile<F, D> next;
  int32_t key = k0 + 16 * wave;
  weight_load<F, D>(next, a, s, key, col, g);
  for (; key <= k1; key += 16 * kWeightWaves) {
    uint4 k[D / 32];
    weight_operand<T, F, D>(next, k);
    const float by = next.scale * a.scale_log2;
    weight_load<F, D>(next, a, s, key + 16 * kWeightWaves, col, g);
    const bool whole = key >= all_lo && key + 15 <= all_hi;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const floatx4 acc = weight_dot<T, D>(k, q[t]);
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int32_t at = key + 4 * (int32_t)g + i;
        x[i] = whole || (at >= lo[t] && at <= hi[t]) ? acc[i] * by : -INFINITY;
      }
      const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      if (__any(mx > m[t] + kRescaleSlack)) {
        const float mn = fmaxf(m[t], mx);
        l[t] *= fast_exp2(m[t] - mn);
        m[t] = mn;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) l[t] += fast_exp2(x[i] - m[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const float mx = wave_max_g(m[t]);
    const float sum = wave_sum_g(l[t] * fast_exp2(m[t] - mx));
    if (g == 0) part[wave][16 * t + col] = make_float2(mx, sum);
  }
  __syncthreads();
  const uint32_t r = threadIdx.x;
  if (r < 16 * MT && row0 + r < s.n_rows) {
    float mx = kNegBig, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWeightWaves; ++w) mx = fmaxf(mx, part[w][r].x);
#pragma unroll
    for (int w = 0; w < kWeightWaves; ++w) sum += part[w][r].y * fast_exp2(part[w][r].x - mx);
    a.ml[((uint64_t)blockIdx.y * a.row_cap + row0 + r) * a.n_chunk + chunk] =
        make_float2(mx, sum);
  }
}

// ---- pass 2 --------------------------------------------------------------------

// lse of a row from its chunks' (m, l); +infinity (weights of 0) where it saw
// no key.
__device__ __forceinline__ float weight_join(const float2* ml, uint32_t n) {
  float mx = kNegBig, sum = 0.f;
  for (uint32_t c = 0; c < n; ++c) {
    const float2 x = ml[c];
    const float mn = fmaxf(mx, x.x);
    sum = sum * fast_exp2(mx - mn) + x.y * fast_exp2(x.x - mn);
    mx = mn;
  }
  return sum > 0.f ? mx + __builtin_amdgcn_logf(sum) : INFINITY;
}

constexpr uint32_t kWeightJoinRows = 1024;  // rows whose lse a workgroup joins in LDS

// Grid: (key tiles of 16 KT x 4 waves, segments).
template <typename T, int F, int D, int KT, bool kJoin>
__global__ __launch_bounds__(64 * kWeightWaves) void weights_sum(WeightArgs a) {
  __shared__ float lse_lds[kJoin ? kWeightJoinRows : 1];
  const WeightSeg s = weight_seg(a, blockIdx.y);
  const int32_t wg0 = (int32_t)(blockIdx.x * 16 * KT * kWeightWaves);
  if (!s.ok || wg0 >= s.len_k) return;
  const float2* ml = a.ml + (uint64_t)blockIdx.y * a.row_cap * a.n_chunk;
  if constexpr (kJoin) {
    for (uint32_t r = threadIdx.x; r < s.n_rows; r += 64 * kWeightWaves)
      lse_lds[r] = weight_join(ml + (uint64_t)r * a.n_chunk, a.n_chunk);
    __syncthreads();
  }
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int32_t wave = (int32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t key0 = wg0 + 16 * KT * wave;
  if (key0 >= s.len_k) return;
  uint4 k[KT][D / 32];
  float by[KT], sum[KT][4];
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    WeightTile<F, D> raw;
    weight_load<F, D>(raw, a, s, key0 + 16 * t, col, g);
    weight_operand<T, F, D>(raw, k[t]);
    by[t] = raw.scale * a.scale_log2;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[t][i] = 0.f;
  }
  // The queries that see any of these keys: pos >= key0 - wr, pos <= last + wl.
  const int32_t key1 = min(key0 + 16 * KT, s.len_k) - 1;
  const int32_t n_q = (int32_t)a.group.div(s.n_rows - 1) + 1;
  const int32_t j0 = a.wr >= 0 ? (int32_t)max((int64_t)0, (int64_t)key0 - a.wr - s.pos0) : 0;
  const int32_t j1 =
      a.wl >= 0 ? (int32_t)min((int64_t)n_q - 1, (int64_t)key1 + a.wl - s.pos0) : n_q - 1;
  if (j0 <= j1) {
    const uint32_t r0 = ((uint32_t)j0 * a.group.d) & ~15u;
    const uint32_t r1 = min(((uint32_t)j1 + 1) * a.group.d, s.n_rows);
    uint4 next[D / 32];
    weight_q<T, F, D>(next, a, s, r0 + col, g);
    for (uint32_t r = r0; r < r1; r += 16) {
      uint4 q[D / 32];
#pragma unroll
      for (int c = 0; c < D / 32; ++c) q[c] = next[c];
      const uint32_t row = min(r + col, s.n_rows - 1);
      float lse;
      if constexpr (kJoin) {
        lse = lse_lds[row];
      } else {
        const float2 x = ml[row];
        lse = x.y > 0.f ? x.x + __builtin_amdgcn_logf(x.y) : INFINITY;
      }
      if (r + col >= s.n_rows) lse = INFINITY;
      weight_q<T, F, D>(next, a, s, r + 16 + col, g);
      const int32_t pos = s.pos0 + (int32_t)a.group.div(row);
      const int32_t lo = weight_lo(a, pos), hi = weight_hi(a, pos, s.len_k);
      const bool whole = __all(key0 >= lo && key0 + 16 * KT - 1 <= hi);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const floatx4 acc = weight_dot<T, D>(k[t], q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t at = key0 + 16 * t + 4 * (int32_t)g + i;
          const float x = __builtin_fmaf(acc[i], by[t], -lse);
          sum[t][i] += fast_exp2(whole || (at >= lo && at <= hi) ? x : -INFINITY);
        }
      }
    }
  }
  // Over the 16 rows of a lane group; lane col then writes key 4 g + col.
  float* w = a.w + s.state_row * a.row_stride + s.h * a.head_stride;
#pragma unroll
  for (int t = 0; t < KT; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = sum[t][i];
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) x += __shfl_xor(x, o);
      sum[t][i] = x;
    }
    const float x = col == 0 ? sum[t][0] : col == 1 ? sum[t][1] : col == 2 ? sum[t][2] : sum[t][3];
    const int32_t at = key0 + 16 * t + 4 * (int32_t)g + (int32_t)col;
    if (col < 4 && at < s.len_k) w[at] = a.decay == 0.f ? x : w[at] * a.decay + x;
  }
}

// ---- host ------------------------------------------------------------------------

struct WeightPlan {
  uint32_t row_cap, row_tiles, n_chunk, chunk_keys;
  int mt, kt;
  size_t bytes;
};

// Rows per workgroup of pass 1 (16 mt): enough to use a K tile many times where
// there are many rows. Chunks of keys: as many as give pass 1 about kWeightWgs
// workgroups, where the rows are few enough for pass 2 to join them.
constexpr uint64_t kWeightWgs = 2048;
static WeightPlan weight_plan(uint32_t batch, uint32_t kvh, uint32_t group, uint32_t hd,
                              uint32_t max_q, uint32_t max_k, uint32_t last) {
  WeightPlan p;
  const uint64_t n_q = last ? std::min(max_q, last) : max_q;
  const uint64_t rows = n_q * group;
  p.row_cap = (uint32_t)std::min<uint64_t>(rows, 0x7FFFFFF0u);
  const int most = hd > 128 ? 4 : 8;
  p.mt = rows <= 16 ? 1 : rows <= 64 ? 4 : most;
  p.row_tiles = (p.row_cap + 16 * p.mt - 1) / (16 * p.mt);
  p.kt = rows <= 64 ? 1 : 4;
  const uint64_t wgs = std::max<uint64_t>((uint64_t)p.row_tiles * batch * kvh, 1);
  uint64_t n = p.row_cap <= kWeightJoinRows ? std::max<uint64_t>(kWeightWgs / wgs, 1) : 1;
  uint64_t keys = (((uint64_t)max_k + n - 1) / n + 63) & ~63ull;
  keys = std::max<uint64_t>(keys, p.row_cap <= kWeightJoinRows ? 256 : 64);
  p.chunk_keys = (uint32_t)keys;
  p.n_chunk = (uint32_t)std::max<uint64_t>(((uint64_t)max_k + keys - 1) / keys, 1);
  p.bytes = (size_t)batch * kvh * p.row_cap * p.n_chunk * sizeof(float2);
  return p;
}

template <typename T, int F, int D>
static void launch_weights_d(const WeightArgs& a, const WeightPlan& p, uint32_t segs,
                             uint32_t max_k, hipStream_t s) {
  const dim3 block(64 * kWeightWaves), g1(p.row_tiles * p.n_chunk, segs);
  if (p.mt == 1) hipLaunchKernelGGL((weights_lse<T, F, D, 1>), g1, block, 0, s, a);
  else if (p.mt == 4) hipLaunchKernelGGL((weights_lse<T, F, D, 4>), g1, block, 0, s, a);
  else if constexpr (D <= 128) hipLaunchKernelGGL((weights_lse<T, F, D, 8>), g1, block, 0, s, a);
  const uint32_t keys = 16 * p.kt * kWeightWaves;
  const dim3 g2((max_k + keys - 1) / keys, segs);
  const bool join = p.row_cap <= kWeightJoinRows;
  if (p.kt == 1) hipLaunchKernelGGL((weights_sum<T, F, D, 1, true>), g2, block, 0, s, a);
  else if (join) hipLaunchKernelGGL((weights_sum<T, F, D, 4, true>), g2, block, 0, s, a);
  else hipLaunchKernelGGL((weights_sum<T, F, D, 4, false>), g2, block, 0, s, a);
}
template <typename T, int F>
static void launch_weights(const WeightArgs& a, const WeightPlan& p, uint32_t segs, uint32_t max_k,
                           hipStream_t s) {
  if (a.hd <= 64) launch_weights_d<T, F, 64>(a, p, segs, max_k, s);
  else if (a.hd <= 128) launch_weights_d<T, F, 128>(a, p, segs, max_k, s);
  else launch_weights_d<T, F, 256>(a, p, segs, max_k, s);
}

int check_weights(const vapi_kv_weights* w, uint32_t batch, uint32_t kvh, const char* who) {
  if (!w || !w->data) VK_FAIL(VAPI_KV_EINVAL, "%s: null weights", who);
  if (((uintptr_t)w->data & 3) || ((uintptr_t)w->index & 3))
    VK_FAIL(VAPI_KV_EINVAL, "%s: weights and their index must be 4-byte aligned", who);
  if (w->head_stride < w->width && kvh > 1)
    VK_FAIL(VAPI_KV_EINVAL, "%s: weights' head stride %llu < their width %u", who,
            (unsigned long long)w->head_stride, w->width);
  if (w->rows > 1 && w->row_stride < (kvh - 1) * w->head_stride + w->width)
    VK_FAIL(VAPI_KV_EINVAL, "%s: weights' row stride %llu < a row's extent", who,
            (unsigned long long)w->row_stride);
  if (!w->index && batch > w->rows)
    VK_FAIL(VAPI_KV_EINVAL, "%s: %u sequences but %u rows of weights", who, batch, w->rows);
  return 0;
}

struct WeightCall {
  const void* q;
  const uint32_t *cu_q, *cu_k, *table;
  uint32_t batch, max_blocks, max_q, max_k, num_heads;
  float scale;
  int32_t wl, wr;
  uint32_t last;
  float decay;
  const vapi_kv_weights* w;
  void* ws;
  size_t ws_bytes;
};

// The checks that do not depend on the kind of pool; *todo is false where there
// is nothing to launch.
static int weight_checks(const WeightCall& c, uint32_t kvh, uint32_t hd, uint32_t num_blocks,
                         const char* who, WeightPlan* plan, bool* todo) {
  *todo = false;
  if (c.num_heads == 0 || c.num_heads % kvh)
    VK_FAIL(VAPI_KV_EINVAL, "%s: %u query heads is not a multiple of %u kv heads", who,
            c.num_heads, kvh);
  if (int rc = check_weights(c.w, c.batch, kvh, who)) return rc;
  if (!(c.decay >= 0.f) || !std::isfinite(c.decay))
    VK_FAIL(VAPI_KV_EINVAL, "%s: decay %g", who, (double)c.decay);
  if (c.max_k > c.w->width)
    VK_FAIL(VAPI_KV_EINVAL, "%s: max_seqlen_k %u exceeds the weights' width %u", who, c.max_k,
            c.w->width);
  if (c.batch == 0 || c.max_q == 0 || c.max_k == 0) return 0;
  if (!c.q || !c.cu_q || !c.cu_k || !c.table)
    VK_FAIL(VAPI_KV_EINVAL, "%s: null device pointer", who);
  if ((uintptr_t)c.q & 15) VK_FAIL(VAPI_KV_EINVAL, "%s: q must be 16-byte aligned", who);
  if (num_blocks == 0) VK_FAIL(VAPI_KV_EINVAL, "%s: keys in an empty pool", who);
  if (c.max_blocks == 0) VK_FAIL(VAPI_KV_EINVAL, "%s: block table width 0", who);
  const uint64_t segs = (uint64_t)c.batch * kvh, n_q = c.last ? std::min(c.max_q, c.last) : c.max_q;
  if (segs > 65535 || n_q * (c.num_heads / kvh) > 0x3FFFFFFFu || c.max_k > 0x3FFFFFFFu)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: a batch of %u x %u kv heads with %u queries of %u heads", who,
            c.batch, kvh, c.max_q, c.num_heads);
  *plan = weight_plan(c.batch, kvh, c.num_heads / kvh, hd, c.max_q, c.max_k, c.last);
  if ((uint64_t)plan->row_tiles * plan->n_chunk > 0x7FFFFFFFu)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: batch too large for one launch", who);
  if (c.ws_bytes < plan->bytes || !c.ws)
    VK_FAIL(VAPI_KV_ESPACE, "%s: workspace %zu bytes < %zu", who, c.ws_bytes, plan->bytes);
  if ((uintptr_t)c.ws & 15)
    VK_FAIL(VAPI_KV_EINVAL, "%s: the workspace must be 16-byte aligned", who);
  *todo = true;
  return 0;
}

static WeightArgs weight_args(const WeightCall& c, const WeightPlan& p, uint32_t kvh, uint32_t hd,
                              uint32_t block_size, uint32_t num_blocks) {
  WeightArgs a{};
  a.q = (const char*)c.q;
  a.cu_q = c.cu_q, a.cu_k = c.cu_k, a.table = c.table, a.index = c.w->index;
  a.w = c.w->data;
  a.ml = (float2*)c.ws;
  a.last_blk = num_blocks - 1;
  while ((1u << a.bs_shift) < block_size) ++a.bs_shift;
  a.max_blocks = c.max_blocks;
  a.row_stride = c.w->row_stride, a.head_stride = c.w->head_stride;
  a.n_rows = c.w->rows;
  // Keys past max_seqlen_k, which no valid call has, are left out.
  a.width = std::min(c.w->width, c.max_k);
  a.kvh = kvh, a.num_heads = c.num_heads, a.hd = hd, a.last_queries = c.last;
  a.group = FastDiv(c.num_heads / kvh);
  a.row_cap = p.row_cap, a.n_chunk = p.n_chunk, a.chunk_keys = p.chunk_keys;
  a.scale_log2 = c.scale * kLog2e;
  a.decay = c.decay;
  a.wl = c.wl < 0 ? -1 : c.wl;
  a.wr = c.wr < 0 ? -1 : c.wr;
  return a;
}

}  // namespace vk

using namespace vk;

extern "C" {

size_t vapi_kv_attention_weights_workspace_size(uint32_t batch, uint32_t num_kv_heads,
                                                uint32_t num_heads, uint32_t head_dim,
                                                uint32_t max_seqlen_q, uint32_t max_seqlen_k,
                                                uint32_t last_queries) {
  if (num_kv_heads == 0 || num_heads == 0 || num_heads % num_kv_heads || batch == 0 ||
      max_seqlen_q == 0 || max_seqlen_k == 0)
    return 0;
  return weight_plan(batch, num_kv_heads, num_heads / num_kv_heads, head_dim, max_seqlen_q,
                     max_seqlen_k, last_queries)
      .bytes;
}

int vapi_kv_attention_weights(const vapi_kv_pool* pool, uint32_t layer, const void* q,
                              const uint32_t* cu_seqlens_q, const uint32_t* cu_seqlens_k,
                              const uint32_t* block_table, uint32_t batch, uint32_t max_blocks,
                              uint32_t max_seqlen_q, uint32_t max_seqlen_k, uint32_t num_heads,
                              float scale, int32_t window_left, int32_t window_right,
                              uint32_t last_queries, float decay, const vapi_kv_weights* weights,
                              void* workspace, size_t workspace_bytes, vapi_stream_t stream) {
  const char* who = "vapi_kv_attention_weights";
  if (int rc = check_pool(pool, who)) return rc;
  if (layer >= pool->num_layers)
    VK_FAIL(VAPI_KV_EINVAL, "%s: layer %u of %u", who, layer, pool->num_layers);
  if (!pool->v) VK_FAIL(VAPI_KV_EINVAL, "%s: a K-only pool is not attended over", who);
  if (pool->dtype != VAPI_KV_BF16 && pool->dtype != VAPI_KV_F16)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: f16 and bf16 pools only", who);
  if (pool->head_dim % 8 || pool->head_dim > 256)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: head_dim %u is not a multiple of 8 up to 256", who,
            pool->head_dim);
  if (pool->block_size < 16 || (pool->block_size & (pool->block_size - 1)))
    VK_FAIL(VAPI_KV_EUNSUP, "%s: block_size %u is not a power of two from 16", who,
            pool->block_size);
  const WeightCall c{q, cu_seqlens_q, cu_seqlens_k, block_table, batch, max_blocks, max_seqlen_q,
                     max_seqlen_k, num_heads, scale, window_left, window_right, last_queries,
                     decay, weights, workspace, workspace_bytes};
  WeightPlan p;
  bool todo;
  if (int rc = weight_checks(c, pool->num_kv_heads, pool->head_dim, pool->num_blocks, who, &p,
                             &todo))
    return rc;
  if (!todo) return 0;
  const Geom g = make_geom(pool);
  WeightArgs a = weight_args(c, p, g.kvh, g.d, g.block_size, g.num_blocks);
  a.k = layer_ptrs(pool, layer).k;
  a.blk_b = g.blk * 2, a.head_b = g.head * 2, a.tok_b = (uint32_t)g.tok * 2;
  const uint32_t segs = batch * g.kvh;
  if (pool->dtype == VAPI_KV_BF16) launch_weights<bf16_t, kK16>(a, p, segs, max_seqlen_k, hs(stream));
  else launch_weights<f16_t, kK16>(a, p, segs, max_seqlen_k, hs(stream));
  VK_LAUNCHED(who);
  return 0;
}

int vapi_kv_q8_attention_weights(const vapi_kv_q8_pool* pool, uint32_t layer, const void* q,
                                 const uint32_t* cu_seqlens_q, const uint32_t* cu_seqlens_k,
                                 const uint32_t* block_table, uint32_t batch, uint32_t max_blocks,
                                 uint32_t max_seqlen_q, uint32_t max_seqlen_k, uint32_t num_heads,
                                 float scale, int32_t window_left, int32_t window_right,
                                 uint32_t last_queries, float decay,
                                 const vapi_kv_weights* weights, void* workspace,
                                 size_t workspace_bytes, vapi_stream_t stream) {
  const char* who = "vapi_kv_q8_attention_weights";
  if (int rc = check_q8_pool(pool, layer, who)) return rc;
  const WeightCall c{q, cu_seqlens_q, cu_seqlens_k, block_table, batch, max_blocks, max_seqlen_q,
                     max_seqlen_k, num_heads, scale, window_left, window_right, last_queries,
                     decay, weights, workspace, workspace_bytes};
  WeightPlan p;
  bool todo;
  if (int rc = weight_checks(c, pool->num_kv_heads, pool->head_dim, pool->num_blocks, who, &p,
                             &todo))
    return rc;
  if (!todo) return 0;
  const Q8Geom g = q8_geom(pool);
  const Q8Ptrs ptr = q8_ptrs(pool, layer);
  WeightArgs a = weight_args(c, p, g.kvh, g.d, g.block_size, g.num_blocks);
  a.k = ptr.k, a.k_scale = ptr.ks, a.sblk = g.sblk;
  a.blk_b = g.blk, a.head_b = g.head, a.tok_b = g.tok;
  const uint32_t segs = batch * g.kvh;
  const bool bf16 = pool->dtype == VAPI_KV_BF16, e4m3 = pool->format == VAPI_KV_Q8_E4M3;
  const hipStream_t s = hs(stream);
  if (bf16 && e4m3) launch_weights<bf16_t, VAPI_KV_Q8_E4M3>(a, p, segs, max_seqlen_k, s);
  else if (bf16) launch_weights<bf16_t, VAPI_KV_Q8_INT8>(a, p, segs, max_seqlen_k, s);
  else if (e4m3) launch_weights<f16_t, VAPI_KV_Q8_E4M3>(a, p, segs, max_seqlen_k, s);
  else launch_weights<f16_t, VAPI_KV_Q8_INT8>(a, p, segs, max_seqlen_k, s);
  VK_LAUNCHED(who);
  return 0;
}

}  // extern "C"
