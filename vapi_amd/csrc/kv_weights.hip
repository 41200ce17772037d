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
//     rows that see them (Q staged in LDS for the workgroup's four waves) and
//     adds up exp2(s - lse) per key; the 16 lanes of a key are added at the end.
//     Many rows go in parts, whose sums weights_add adds in order. Each weight has
//     one owner: no atomics, a fixed order.
// S^T = K Q^T as in the attention kernels: lane (col, g) holds keys 4 g .. +3 of
// row col. Up to 16 rows (single tokens) the scores themselves are kept and pass 2
// is a sum over them (weights_stored).
//
// What bounds it. Single tokens: HBM, K once (129 MB in 31 us, 4.2 TB/s, of 37 us
// with pass 2). Many rows: three fresh prompts of 700-2,000 tokens (32 q / 8 kv
// heads, f16; 30 GFLOP of scores) take 56 + 54 + 6 us. By the counters the vector
// units issue in 59% of a SIMD's busy time in pass 1 and 62% in pass 2 (about 7
// instructions a score, an exponential among them) and the matrix cores are busy in
// 25% and 29%; a wave issues in 38 and 40% of its life and waits for results in 36
// and 34%, which the 2.7 and 2.5 waves a SIMD do not cover. So half is vector work,
// and the rest waits that more waves would hide, had they registers.
// Few rows over long contexts: latency, ~4 us of dependent loads before a workgroup's
// first product in each pass (a prompt's last 32 queries over 6,500 keys, 28 q / 4
// kv heads: 16 + 12 + 4 us).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "q8.hpp"

namespace vk {

typedef uint32_t uint32x4 __attribute__((ext_vector_type(4)));

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
  uint32_t row_cap, n_chunk, chunk_keys, key_cap, part_rows;
  float* part;    // [part][segment][key_cap] sums of pass 2
  float* scores;  // [segment][row_cap][key_cap] (kept scores)
  float scale_log2;  // of the absolute scale; a negative one flips Q's signs
  uint32_t q_sign;
  float decay;
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

// Pieces past head_dim as zeros: one uniform branch around selects (a branch per
// piece waits for its load before the next is issued).
template <int F, int D>
__device__ __forceinline__ void weight_zero(uint4 (&x)[D / 32], uint32_t hd, uint32_t g) {
  if (hd < D) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint32_t keep = weight_d<F>(c, g) < hd ? 0xFFFFFFFFu : 0u;
      x[c] = make_uint4(x[c].x & keep, x[c].y & keep, x[c].z & keep, x[c].w & keep);
    }
  }
}

// Rows of Q by their distance from `first`, a uniform row of the segment: row
// (query j, head c of the group) lies row + j (heads - group) rows of Q further.
struct WeightQ {
  const char* base;
  uint32_t first, j0, skip, row_b;
};
__device__ __forceinline__ WeightQ weight_q_from(const WeightArgs& a, const WeightSeg& s,
                                                 uint32_t first) {
  WeightQ w;
  w.first = first, w.j0 = a.group.div(first);
  w.skip = a.num_heads - a.group.d, w.row_b = 2 * a.hd;
  w.base = a.q + ((uint64_t)(s.q0 + w.j0) * a.num_heads + s.h * a.group.d +
                  (first - w.j0 * a.group.d)) * w.row_b;
  return w;
}
// Bytes from the base (at most 64 rows on: the heads, up to 65,535, keep it in 32
// bits), of the segment's last row for rows past it.
__device__ __forceinline__ uint32_t weight_q_row(const WeightQ& w, const WeightArgs& a,
                                                 const WeightSeg& s, uint32_t row) {
  row = min(row, s.n_rows - 1);
  return (row - w.first + (a.group.div(row) - w.j0) * w.skip) * w.row_b;
}

// Q operand of a row (rows past the segment's repeat its last).
template <int F, int D>
__device__ __forceinline__ void weight_q(uint4 (&q)[D / 32], const WeightQ& w, const WeightArgs& a,
                                         const WeightSeg& s, uint32_t row, uint32_t g) {
  const uint32_t at = weight_q_row(w, a, s, row);
#pragma unroll
  for (int c2 = 0; c2 < D / 32; ++c2) {
    const uint4 x =
        *(const uint4*)(w.base + (at + min(2 * weight_d<F>(c2, g), w.row_b - 16)));
    q[c2] = make_uint4(x.x ^ a.q_sign, x.y ^ a.q_sign, x.z ^ a.q_sign, x.w ^ a.q_sign);
  }
  weight_zero<F, D>(q, a.hd, g);
}

// A 16-key tile as it is stored, and its scale, on its way to MFMA operands
// through LDS. An operand's lane wants 16 bytes of one of 16 rows, so loading it
// straight takes two instructions (or four) for each 128-byte line, and L1 stalls
// on the second while the first is on its way: with 8 KiB a wave outstanding, the
// latency of 1,155 cycles held a read of K to 4.2 TB/s. Here consecutive lanes
// load consecutive 16-byte pieces (each line by one instruction); the wave writes
// them to its own LDS, piece c of row r at c ^ swizzle(r) so that the reads meet
// no bank twice, and reads the operands back.
template <int F, int D>
struct WeightTile {
  static constexpr int kPieces = D / (F == kK16 ? 8 : 16);  // of a row
  static constexpr int N = kPieces / 4;
  uint32x4 w[N];
  float scale;
  __device__ static __forceinline__ uint32_t place(uint32_t row, uint32_t piece) {
    return row * kPieces + (piece ^ (kPieces == 4 ? row >> 1 & 3 : row & 7));
  }
};
// Keys past the last repeat it, pieces past head_dim the row's last (they meet
// zeros of Q). Every load is unconditional: one under a branch makes the
// compiler wait for all loads in flight.
// kNt: streaming loads, where no other workgroup reads the tile.
__device__ __forceinline__ int32_t weight_tile(const WeightSeg& s, int32_t key) {
  return __builtin_amdgcn_readfirstlane(min(key, (s.len_k - 1) & ~15));
}
__device__ __forceinline__ uint32_t weight_block(const WeightArgs& a, const WeightSeg& s,
                                                 int32_t key) {
  using ConstU32 = const __attribute__((address_space(4))) uint32_t;
  ConstU32* tab = (ConstU32*)(a.table + (uint64_t)s.seq * a.max_blocks);
  return min(tab[min((uint32_t)weight_tile(s, key) >> a.bs_shift, a.max_blocks - 1)], a.last_blk);
}
template <int F, int D, bool kNt>
__device__ __forceinline__ void weight_load(WeightTile<F, D>& t, const WeightArgs& a,
                                            const WeightSeg& s, int32_t key, uint32_t blk,
                                            uint32_t lane) {
  using ConstF32 = const __attribute__((address_space(4))) float;
  using Tile = WeightTile<F, D>;
  const int32_t last = s.len_k - 1, ts = weight_tile(s, key);
  const uint32_t off = (uint32_t)ts & ((1u << a.bs_shift) - 1);
  const char* p = a.k + blk * a.blk_b + s.h * a.head_b + (uint64_t)off * a.tok_b;
  t.scale = 1.f;
  if constexpr (F != kK16) t.scale = ((ConstF32*)a.k_scale)[(uint64_t)blk * a.sblk + s.h];
  const uint32_t end = a.hd * (F == kK16 ? 2 : 1) - 16;
#pragma unroll
  for (int i = 0; i < Tile::N; ++i) {
    const uint32_t row = (64 * i + lane) / Tile::kPieces, piece = lane % Tile::kPieces;
    t.w[i] = load_kv<kNt>(
        (const uint32x4*)(p + min((int32_t)row, last - ts) * a.tok_b + min(16 * piece, end)));
  }
}
template <int F, int D>
__device__ __forceinline__ void weight_stage(uint32x4* lds, const WeightTile<F, D>& t,
                                             uint32_t lane) {
  using Tile = WeightTile<F, D>;
#pragma unroll
  for (int i = 0; i < Tile::N; ++i)
    lds[Tile::place((64 * i + lane) / Tile::kPieces, lane % Tile::kPieces)] = t.w[i];
}
// Log2 units per unit of a tile's products. Positive even where a block's scale is
// 0 (its codes are): a masked score, -infinity, stays one.
template <int F, int D>
__device__ __forceinline__ float weight_unit(const WeightTile<F, D>& t, const WeightArgs& a) {
  return F == kK16 ? a.scale_log2 : fmaxf(t.scale * a.scale_log2, 1e-37f);
}
// The staged tile as MFMA operands (codes unscaled). A 16-bit pool's pieces past
// head_dim are zeroed: they may repeat an infinity (codes are finite).
template <typename T, int F, int D>
__device__ __forceinline__ void weight_operand(const uint32x4* lds, uint4 (&k)[D / 32], uint32_t hd,
                                               uint32_t col, uint32_t g) {
  using Tile = WeightTile<F, D>;
  if constexpr (F == kK16) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) k[c] = __builtin_bit_cast(uint4, lds[Tile::place(col, 4 * c + g)]);
    weight_zero<F, D>(k, hd, g);
  } else {
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 w = __builtin_bit_cast(uint4, lds[Tile::place(col, 4 * c + g)]);
      const uint2 a0 = q8_expand4<T, F, false>(w.x, 1.f), a1 = q8_expand4<T, F, false>(w.y, 1.f);
      const uint2 b0 = q8_expand4<T, F, false>(w.z, 1.f), b1 = q8_expand4<T, F, false>(w.w, 1.f);
      k[2 * c] = make_uint4(a0.x, a0.y, a1.x, a1.y);
      k[2 * c + 1] = make_uint4(b0.x, b0.y, b1.x, b1.y);
    }
  }
}
// The wave's LDS writes before its reads (a wave's LDS operations run in order;
// this holds the compiler to it).
__device__ __forceinline__ void weight_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
}

// Keys that a query at `pos` sees: [lo, hi].
__device__ __forceinline__ int32_t weight_lo(const WeightArgs& a, int32_t pos) {
  return a.wl >= 0 ? max(0, pos - a.wl) : 0;
}
__device__ __forceinline__ int32_t weight_hi(const WeightArgs& a, int32_t pos, int32_t len_k) {
  return a.wr >= 0 ? min(len_k - 1, pos + a.wr) : len_k - 1;
}

constexpr int kWeightWaves = 4;
constexpr uint32_t kWeightChunk = 256;  // pass 1's chunks of keys are multiples of this

// Tiles a wave of pass 1 loads at a time: 4 KiB of K where few rows use them
// (with four workgroups a CU the next step's 4 KiB of 16 waves are in flight; 8
// and 16 KiB a wave measured 1 and 3 us slower of 37), one where many rows do.
template <int F, int D, int MT>
constexpr int weight_step() {
  const int n = MT == 1 ? 4096 / (16 * D * (F == kK16 ? 2 : 1)) : 1;
  return n < 1 ? 1 : n;
}

// ---- pass 1 --------------------------------------------------------------------

// Every grid has the segments fastest, so that the round-robin dealing over the
// XCDs gives each of them work of every sequence (with the chunks fastest, eight
// chunks put the ends of all long sequences on one XCD; the three fresh prompts
// 285 -> 207 us).
// Grid: (segments, row tiles x chunks). kStore: the scores are kept (then one
// row tile, MT = 1).
template <typename T, int F, int D, int MT, bool kStore>
__global__ __launch_bounds__(64 * kWeightWaves) void weights_lse(WeightArgs a) {
  constexpr int ST = weight_step<F, D, MT>();
  __shared__ float2 part[kWeightWaves][16 * MT];
  __shared__ uint32x4 stage[kWeightWaves][ST][16 * WeightTile<F, D>::kPieces];
  // (Chunk by chunk the sequences are turned by five, which has no factor in common
  // with the usual batches: otherwise all chunks of a long one land on the same CUs.
  // 16 sequences of 256-8,192 keys 41.3 -> 37.3, the one batch measured.)
  const uint32_t turn = (uint32_t)((uint64_t)(5 * a.kvh) * blockIdx.y % gridDim.x);
  const uint32_t seg = (blockIdx.x + turn) % gridDim.x;
  const WeightSeg s = weight_seg(a, seg);
  if (!s.ok) return;
  // The last rows see the most keys: their workgroups start first.
  const uint32_t back = blockIdx.y / a.n_chunk, chunk = blockIdx.y - back * a.n_chunk;
  const uint32_t row0 = (gridDim.y / a.n_chunk - 1 - back) * 16 * MT;
  if (row0 >= s.n_rows) return;
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int32_t wave = (int32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint4 q[MT][D / 32];
  int32_t lo[MT], hi[MT];
  float m[MT], l[MT];
  const WeightQ rows = weight_q_from(a, s, row0);
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const uint32_t row = row0 + 16 * t + col;
    weight_q<F, D>(q[t], rows, a, s, row, g);
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
  // (From a whole step of the chunk's, which is a multiple of every step: the walk
  // then ends at the chunk's end. From any other tile its last step would take keys
  // of the next chunk, which counts them too.)
  static_assert(kWeightChunk % (16 * ST) == 0, "chunks are whole steps");
  const int32_t k0 = max(c0, weight_lo(a, p0) & ~(16 * ST - 1));
  const int32_t k1 = min(c1, weight_hi(a, p1, s.len_k));
  // Stores past the buffer (rows and keys that are not there) are dropped.
  const uint32_t kept = kStore ? s.n_rows * a.key_cap * (uint32_t)sizeof(float) : 0;
  const auto store = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.scores + (uint64_t)seg * a.row_cap * a.key_cap), 0, (int)kept, 0x00027000);
  // The next step loads into the registers that staging has just freed, while
  // this one is computed from LDS. (One loop body: a second one for a second set
  // of registers doubles the code, which short walks fetch once.)
  WeightTile<F, D> buf[ST];
  int32_t key = k0 + 16 * ST * wave;
  uint32_t blk[ST];  // the next step's table entries: their loads come before the tiles'
#pragma unroll
  for (int tt = 0; tt < ST; ++tt) {
    weight_load<F, D, kStore>(buf[tt], a, s, key + 16 * tt, weight_block(a, s, key + 16 * tt), lane);
    blk[tt] = weight_block(a, s, key + 16 * (ST * kWeightWaves + tt));
  }
  while (key <= k1) {
    float by[ST];
#pragma unroll
    for (int tt = 0; tt < ST; ++tt) {
      weight_stage<F, D>(stage[wave][tt], buf[tt], lane);
      by[tt] = weight_unit(buf[tt], a);
    }
    weight_fence();
#pragma unroll
    for (int tt = 0; tt < ST; ++tt) {
      weight_load<F, D, kStore>(buf[tt], a, s, key + 16 * (ST * kWeightWaves + tt), blk[tt], lane);
      blk[tt] = weight_block(a, s, key + 16 * (2 * ST * kWeightWaves + tt));
    }
    const bool whole = key >= all_lo && key + 16 * ST - 1 <= all_hi;
    floatx4 x[ST][MT];  // products; times by[tt] the scores
    float mx[MT];
    bool grow = false;
#pragma unroll
    for (int tt = 0; tt < ST; ++tt) {
      uint4 k[D / 32];
      weight_operand<T, F, D>(stage[wave][tt], k, a.hd, col, g);
#pragma unroll
      for (int t = 0; t < MT; ++t) x[tt][t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int t = 0; t < MT; ++t) x[tt][t] = mfma16x16x32<T>(k[c], q[t][c], x[tt][t]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int32_t at = key + 16 * tt + 4 * (int32_t)g + i;
            if (!(at >= lo[t] && at <= hi[t])) x[tt][t][i] = -INFINITY;
          }
        }
        const float top =
            by[tt] * max_nc(max3_nc(x[tt][t][0], x[tt][t][1], x[tt][t][2]), x[tt][t][3]);
        mx[t] = tt == 0 ? top : max_nc(mx[t], top);
      }
      if constexpr (kStore) {
        const int32_t at = key + 16 * tt + 4 * (int32_t)g;
        const uint32_t to = at <= k1 ? (col * a.key_cap + (uint32_t)at) * 4 : 0xFFFFFFF0u;
        const floatx4 v = x[tt][0] * by[tt];
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint32x4, v), store, (int)to, 0,
                                               0);
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) grow |= mx[t] > m[t] + kRescaleSlack;
    if (__any(grow)) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const float mn = max_nc(m[t], mx[t]);
        l[t] *= fast_exp2(m[t] - mn);
        m[t] = mn;
      }
    }
#pragma unroll
    for (int tt = 0; tt < ST; ++tt)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = fast_exp2(__builtin_fmaf(x[tt][t][i], by[tt], -m[t]));
        l[t] += (p[0] + p[1]) + (p[2] + p[3]);
      }
    weight_fence();
    key += 16 * ST * kWeightWaves;
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
    a.ml[((uint64_t)seg * a.row_cap + row0 + r) * a.n_chunk + chunk] =
        make_float2(mx, sum);
  }
}

// ---- pass 2 --------------------------------------------------------------------

// lse of a row from its chunks' (m, l); +infinity (weights of 0) where it saw
// no key, or NaN (a test of the bits: the compiler takes NaN as absent). Eight
// loads at a time.
__device__ __forceinline__ float weight_join(const float2* ml, uint32_t n) {
  float mx = kNegBig, sum = 0.f;
  for (uint32_t c0 = 0; c0 < n; c0 += 8) {
    float2 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = c0 + j < n ? ml[c0 + j] : make_float2(kNegBig, 0.f);
    float mn = mx;
#pragma unroll
    for (int j = 0; j < 8; ++j) mn = fmaxf(mn, x[j].x);
    sum *= fast_exp2(mx - mn);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += x[j].y * fast_exp2(x[j].x - mn);
    mx = mn;
  }
  return __float_as_uint(sum) - 1u < 0x7f7fffffu ? mx + __builtin_amdgcn_logf(sum) : INFINITY;
}

constexpr uint32_t kWeightJoinRows = 512;  // rows whose lse a workgroup holds in LDS
// 16-key tiles a wave of pass 2 holds. More of them read Q less often, fewer leave
// registers for more waves: three fresh prompts (above) 55.8 / 53.5 / 66.9 us at 2 /
// 3 / 4, a prompt's last 32 queries 13.8 / 12.0 / 16.2. (Measured at head_dim 128;
// the other sizes take the same.)
constexpr int kWeightKt = 3;
constexpr uint32_t kWeightBlock = 64;       // rows whose Q a workgroup of pass 2 stages

// Joins the segment's rows [r0, r1) into lds; every thread calls it.
__device__ __forceinline__ void weight_lse_rows(float* lds, const WeightArgs& a, uint32_t seg,
                                                uint32_t r0, uint32_t r1) {
  const float2* ml = a.ml + (uint64_t)seg * a.row_cap * a.n_chunk;
  for (uint32_t r = r0 + threadIdx.x; r < r1; r += 64 * kWeightWaves)
    lds[r - r0] = weight_join(ml + (uint64_t)r * a.n_chunk, a.n_chunk);
  __syncthreads();
}

__device__ __forceinline__ void weight_write(const WeightArgs& a, float* w, float x) {
  *w = a.decay == 0.f ? x : *w * a.decay + x;
}

// The sum over each 16 lanes, in all of them.
__device__ __forceinline__ float row_sum(float x) {
#define VK_ROTATE(N)                                                                       \
  x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), \
                                                             0x120 + N, 0xF, 0xF, true))
  VK_ROTATE(8);
  VK_ROTATE(4);
  VK_ROTATE(2);
  VK_ROTATE(1);
#undef VK_ROTATE
  return x;
}

// Grid: (segments, key tiles of 16 KT x 4 waves, parts of the rows). With more
// than one part the sums go to a.part, which weights_add adds up.
template <typename T, int F, int D>
__global__ __launch_bounds__(64 * kWeightWaves) void weights_sum(WeightArgs a) {
  constexpr int KT = kWeightKt, PR = D / 8;  // 16-byte pieces of a Q row
  constexpr int N = kWeightBlock * PR / (64 * kWeightWaves);
  __shared__ float lse_lds[kWeightJoinRows];
  // The rows' Q, a block of them for all four waves (two blocks in turn); before
  // the first, each wave's K on its way to operands.
  __shared__ uint32x4 lds[2][kWeightBlock * PR];
  static_assert(kWeightWaves * 16 * WeightTile<F, D>::kPieces <= 2 * kWeightBlock * PR, "K's place");
  const WeightSeg s = weight_seg(a, blockIdx.x);
  const int32_t wg0 = (int32_t)(blockIdx.y * 16 * KT * kWeightWaves);
  if (!s.ok || wg0 >= s.len_k) return;
  // This part's rows, and of them those that see any key of the workgroup:
  // pos >= first key - wr, pos <= last key + wl.
  uint32_t r0 = blockIdx.z * a.part_rows, r1 = min(r0 + a.part_rows, s.n_rows);
  const int32_t wg1 = min(wg0 + 16 * KT * kWeightWaves, s.len_k) - 1;
  if (a.wr >= 0) {
    const int64_t j = (int64_t)wg0 - a.wr - s.pos0;
    if (j > 0) r0 = max(r0, (uint32_t)min(j * a.group.d, (int64_t)s.n_rows) & ~15u);
  }
  if (a.wl >= 0) {
    const int64_t j = (int64_t)wg1 + a.wl - s.pos0 + 1;
    r1 = (uint32_t)max((int64_t)0, min((int64_t)r1, j * a.group.d));
  }
  float* part = a.part + ((uint64_t)blockIdx.z * gridDim.x + blockIdx.x) * a.key_cap;
  if (r0 >= r1 && gridDim.z > 1) {  // nothing sees them (of a causal prompt, half)
    if (wg0 + (int32_t)threadIdx.x <= wg1) part[wg0 + threadIdx.x] = 0.f;
    return;
  }
  r1 = max(r0, r1);
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int32_t wave = (int32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t key0 = wg0 + 16 * KT * wave;
  uint4 k[KT][D / 32];
  float by[KT], sum[KT][4];
  {
    uint32x4* const place = &lds[0][0] + wave * 16 * WeightTile<F, D>::kPieces;
    WeightTile<F, D> raw[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t)
      weight_load<F, D, false>(raw[t], a, s, key0 + 16 * t, weight_block(a, s, key0 + 16 * t), lane);
    weight_lse_rows(lse_lds, a, blockIdx.x, r0, min(r0 + kWeightJoinRows, r1));
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      weight_stage<F, D>(place, raw[t], lane);
      weight_fence();
      weight_operand<T, F, D>(place, k[t], a.hd, col, g);
      weight_fence();
      by[t] = __uint_as_float(__float_as_uint(weight_unit(raw[t], a)) ^ (a.q_sign << 16));
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[t][i] = 0.f;
    }
    __syncthreads();
  }
  uint32_t q_at[D / 32];  // this lane's pieces among a tile of 16 rows
#pragma unroll
  for (int c = 0; c < D / 32; ++c) q_at[c] = col * PR + ((weight_d<F>(c, g) / 8) ^ (col & 7));
  // A block's Q pieces in registers: loaded a block ahead, then put in LDS.
  uint32x4 held[N];
  const uint32_t in_row = min(16 * (threadIdx.x % PR), 2 * a.hd - 16);
  auto fetch = [&](uint32_t first) __attribute__((always_inline)) {
    const WeightQ rows = weight_q_from(a, s, first);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t row = first + (64 * kWeightWaves * i + threadIdx.x) / PR;
      held[i] = *(const uint32x4*)(rows.base + (weight_q_row(rows, a, s, row) + in_row));
    }
  };
  // Of this wave's keys: rows [some0, some1) see any, [all0, all1) all of them
  // (pos >= key - wr, pos <= key + wl). Worked out here once: per tile of rows they
  // were most of the loop's scalar instructions.
  auto row_at = [&](int64_t pos) {
    return (uint32_t)min(max((pos - s.pos0) * a.group.d, (int64_t)r0), (int64_t)r1);
  };
  const int32_t key1 = key0 + 16 * KT - 1;
  const bool held_all = key1 < s.len_k;  // (else never whole)
  const uint32_t some0 = a.wr >= 0 ? row_at((int64_t)key0 - a.wr) & ~15u : r0;
  const uint32_t some1 = key0 >= s.len_k ? r0 : a.wl >= 0 ? row_at((int64_t)key1 + a.wl + 1) : r1;
  const uint32_t all0 = a.wr >= 0 ? row_at((int64_t)key1 - a.wr) : r0;
  const uint32_t all1 = !held_all ? r0 : a.wl >= 0 ? row_at((int64_t)key0 + a.wl + 1) : r1;
  uint32_t turn = 0, lse0 = r0;  // lse0: the row of lse_lds's first
  static_assert(kWeightJoinRows % kWeightBlock == 0, "lse_lds holds whole blocks");
  if (r0 < r1) fetch(r0);
  for (uint32_t first = r0; first < r1; first += kWeightBlock, turn ^= 1) {
    if (first - lse0 == kWeightJoinRows) {
      lse0 = first;
      __syncthreads();  // the last rows' readers
      weight_lse_rows(lse_lds, a, blockIdx.x, lse0, min(lse0 + kWeightJoinRows, r1));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t at = 64 * kWeightWaves * i + threadIdx.x, row = at / PR, piece = at % PR;
      if (a.hd < D) held[i] &= 8 * piece < a.hd ? 0xFFFFFFFFu : 0u;
      lds[turn][row * PR + (piece ^ (row & 7))] = held[i];
    }
    if (first + kWeightBlock < r1) fetch(first + kWeightBlock);
    // (One barrier a block: a wave that writes a buffer again has passed the
    // barrier that every wave reaches after reading it.)
    lds_barrier();
    {
      const uint32_t end = min(first + kWeightBlock, some1);
#pragma unroll 1
      for (uint32_t r = max(first, some0); r < end; r += 16) {
        // (Rows past r1 see nothing here, whatever they hold.)
        const bool whole = r >= all0 && r + 16 <= all1;
        uint4 q[D / 32];
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          q[c] = __builtin_bit_cast(uint4, lds[turn][(r - first) * PR + q_at[c]]);
        const float lse = lse_lds[r - lse0 + col];  // (a part is whole tiles)
        floatx4 acc[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) acc[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int t = 0; t < KT; ++t) acc[t] = mfma16x16x32<T>(k[t][c], q[c], acc[t]);
        float x[KT][4];
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[t][i] = __builtin_fmaf(acc[t][i], by[t], -lse);
        if (!whole) {
          const int32_t pos = s.pos0 + (int32_t)a.group.div(r + col);
          const int32_t lo = weight_lo(a, pos);
          const int32_t hi = r + col < r1 ? weight_hi(a, pos, s.len_k) : -1;
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int32_t at = key0 + 16 * t + 4 * (int32_t)g + i;
              x[t][i] = at >= lo && at <= hi ? x[t][i] : -INFINITY;
            }
        }
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[t][i] += fast_exp2(x[t][i]);
      }
    }
  }
  // Over the 16 rows of a lane group; lane col then writes key 4 g + col.
  float* w = a.w + s.state_row * a.row_stride + s.h * a.head_stride;
#pragma unroll
  for (int t = 0; t < KT; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum[t][i] = row_sum(sum[t][i]);
    }
    const float x = col == 0 ? sum[t][0] : col == 1 ? sum[t][1] : col == 2 ? sum[t][2] : sum[t][3];
    const int32_t at = key0 + 16 * t + 4 * (int32_t)g + (int32_t)col;
    if (col < 4 && at < s.len_k) {
      if (gridDim.z > 1) part[at] = x;
      else weight_write(a, w + at, x);
    }
  }
}

// Grid: (segments, keys / 256): the parts' sums, in order.
__global__ __launch_bounds__(256) void weights_add(WeightArgs a, uint32_t parts) {
  const WeightSeg s = weight_seg(a, blockIdx.x);
  const int32_t at = (int32_t)(blockIdx.y * 256 + threadIdx.x);
  if (!s.ok || at >= s.len_k) return;
  float x = 0.f;
  for (uint32_t p = 0; p < parts; ++p)
    x += a.part[((uint64_t)p * gridDim.x + blockIdx.x) * a.key_cap + at];
  weight_write(a, a.w + s.state_row * a.row_stride + s.h * a.head_stride + at, x);
}

// Pass 2 over stored scores. Grid: (segments, keys / 1,024); a thread sums four
// keys over the segment's rows (at most 16).
__global__ __launch_bounds__(64 * kWeightWaves) void weights_stored(WeightArgs a) {
  __shared__ float lse[16];
  const WeightSeg s = weight_seg(a, blockIdx.x);
  if (!s.ok || (int32_t)(blockIdx.y * 1024) >= s.len_k) return;
  const int32_t at = (int32_t)(blockIdx.y * 1024 + 4 * threadIdx.x);
  const float* scores = a.scores + (uint64_t)blockIdx.x * a.row_cap * a.key_cap + at;
  weight_lse_rows(lse, a, blockIdx.x, 0, s.n_rows);
  if (at >= s.len_k) return;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  // (Pass 1 visits every key from the 16-key tile of the first that some row sees.)
  const int32_t last = s.pos0 + (int32_t)a.group.div(s.n_rows - 1);
  const bool seen = at >= (weight_lo(a, s.pos0) & ~15) && at <= weight_hi(a, last, s.len_k);
  for (uint32_t r = 0; seen && r < s.n_rows; ++r) {
    const float4 x = *(const float4*)(scores + (uint64_t)r * a.key_cap);
    sum[0] += fast_exp2(x.x - lse[r]), sum[1] += fast_exp2(x.y - lse[r]);
    sum[2] += fast_exp2(x.z - lse[r]), sum[3] += fast_exp2(x.w - lse[r]);
  }
  float* w = a.w + s.state_row * a.row_stride + s.h * a.head_stride + at;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < s.len_k) weight_write(a, w + i, sum[i]);
}

// ---- host ------------------------------------------------------------------------

struct WeightPlan {
  uint32_t row_cap, row_tiles, n_chunk, chunk_keys, key_cap, parts, part_rows;
  int mt;
  bool store;
  size_t ml_bytes, bytes;
};

// Rows a workgroup of pass 1 takes (16 mt): one tile for single tokens, else
// enough to use each K tile many times. Chunks of keys give pass 1 about
// kWeightWgs workgroups where the rows alone do not, parts of the rows pass 2.
// Up to 16 rows and kStoreBytes the scores are kept between the passes: 8 bytes
// a score moved instead of K read again (16 sequences of 256-8,192 keys, 32 q /
// 8 kv heads, bf16: pass 2 53.6 -> 7.1 us).
constexpr uint64_t kWeightWgs = 1024;
constexpr uint64_t kStoreBytes = 256ull << 20;
// Each part holds a sum a key: at most this much of them. Where it binds, pass 2
// has at least 43,000 workgroups of 192 keys (half of it, 8 M sums), enough without
// more parts.
constexpr uint64_t kPartBytes = 64ull << 20;
static WeightPlan weight_plan(uint32_t batch, uint32_t kvh, uint32_t group, uint32_t hd,
                              uint32_t max_q, uint32_t max_k, uint32_t last) {
  WeightPlan p;
  const uint64_t segs = (uint64_t)batch * kvh;
  const uint64_t n_q = last ? std::min(max_q, last) : max_q;
  const uint64_t rows = n_q * group;
  p.row_cap = (uint32_t)std::min<uint64_t>(rows, 0x7FFFFFF0u);
  p.mt = rows <= 16 ? 1 : 4;
  p.row_tiles = (p.row_cap + 16 * p.mt - 1) / (16 * p.mt);
  p.key_cap = (max_k + 63) & ~63u;
  p.store = rows <= 16 && segs * rows * p.key_cap * sizeof(float) <= kStoreBytes;
  auto up = [](uint64_t x, uint64_t y) { return (x + y - 1) / y; };
  const uint64_t want = std::max<uint64_t>(up(kWeightWgs, p.row_tiles * segs), 1);
  const uint64_t keys = std::max<uint64_t>(up(max_k, want), 1);
  p.chunk_keys = (uint32_t)(up(keys, kWeightChunk) * kWeightChunk);
  p.n_chunk = (uint32_t)std::max<uint64_t>(up(max_k, p.chunk_keys), 1);
  const uint64_t blocks = up(max_k, 16 * kWeightKt * kWeightWaves);
  // (Parts of at most kWeightJoinRows rows where kPartBytes takes them: the rows
  // of a causal prompt's late parts are many, of its early ones few.)
  uint64_t parts = std::max<uint64_t>(up(kWeightWgs, blocks * segs), 1);
  parts = std::max(std::min<uint64_t>(parts, up(rows, 128)), up(rows, kWeightJoinRows));
  parts = std::min(parts, std::max<uint64_t>(kPartBytes / (segs * p.key_cap * sizeof(float)), 1));
  p.part_rows = (uint32_t)(up(up(rows, parts), 16) * 16);
  p.parts = p.store ? 1 : (uint32_t)up(rows, p.part_rows);
  p.ml_bytes = (segs * p.row_cap * p.n_chunk * sizeof(float2) + 255) & ~(size_t)255;
  p.bytes = p.ml_bytes;
  if (p.store) p.bytes += segs * rows * p.key_cap * sizeof(float);
  else if (p.parts > 1) p.bytes += p.parts * segs * p.key_cap * sizeof(float);
  return p;
}

template <typename T, int F, int D>
static void launch_weights_d(const WeightArgs& a, const WeightPlan& p, uint32_t segs,
                             uint32_t max_k, hipStream_t s) {
  const dim3 block(64 * kWeightWaves), g1(segs, p.row_tiles * p.n_chunk);
  if (p.store) {
    hipLaunchKernelGGL((weights_lse<T, F, D, 1, true>), g1, block, 0, s, a);
    hipLaunchKernelGGL(weights_stored, dim3(segs, (max_k + 1023) / 1024), block, 0, s, a);
    return;
  }
  if (p.mt == 1) hipLaunchKernelGGL((weights_lse<T, F, D, 1, false>), g1, block, 0, s, a);
  else hipLaunchKernelGGL((weights_lse<T, F, D, 4, false>), g1, block, 0, s, a);
  const uint32_t keys = 16 * kWeightKt * kWeightWaves;
  hipLaunchKernelGGL((weights_sum<T, F, D>), dim3(segs, (max_k + keys - 1) / keys, p.parts), block,
                     0, s, a);
  if (p.parts > 1)
    hipLaunchKernelGGL(weights_add, dim3(segs, (max_k + 255) / 256), dim3(256), 0, s, a, p.parts);
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
  // (Grids: 2^32 threads in x, 65,535 workgroups of the fewest keys, pass 2's, in y.)
  if (segs > 0xFFFFFFu || c.num_heads > 65535 || n_q * (c.num_heads / kvh) > 0x3FFFFFFFu ||
      c.max_k > 65535u * 16 * kWeightKt * kWeightWaves)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: a batch of %u x %u kv heads with %u queries of %u heads, %u keys",
            who, c.batch, kvh, c.max_q, c.num_heads, c.max_k);
  *plan = weight_plan(c.batch, kvh, c.num_heads / kvh, hd, c.max_q, c.max_k, c.last);
  if ((uint64_t)plan->row_tiles * plan->n_chunk > 65535 || plan->parts > 65535)
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
  a.key_cap = p.key_cap, a.part_rows = p.part_rows;
  a.part = a.scores = (float*)((char*)c.ws + p.ml_bytes);
  a.scale_log2 = fmaxf(fabsf(c.scale) * kLog2e, 1e-30f);
  a.q_sign = c.scale < 0.f ? 0x80008000u : 0u;
  a.decay = c.decay;
  a.wl = window_arg(c.wl);
  a.wr = window_arg(c.wr);
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
