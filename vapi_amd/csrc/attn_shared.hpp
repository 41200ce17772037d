// Attention of a batch whose sequences share the blocks of long prefixes.
//
// softmax over [0, n) splits at any key: with (m, l, o) of the keys before and after
// it (maximum, sum of exponentials, their weighted sum of V), the row's output is
// (o1 2^(m1 - m) + o2 2^(m2 - m)) / (l1 2^(m1 - m) + l2 2^(m2 - m)), m = max(m1, m2).
// So the keys that a group of sequences shares are attended by all of the group's
// queries at once, as the rows of one matrix product that reads each key once, and
// every sequence attends the rest of its keys for itself:
//  * decode rows by the stream of attn_decode.hpp, from their first own key on;
//  * everything else in tiles of rows: a group's queries (of all its sequences, and
//    of all query heads of a kv head) over the shared keys, and the queries of a
//    sequence that brings several over its own keys. Both are nodes here: rows, a
//    range of keys, and a block table.
// A merge then joins each row's partials.
//
// Tiles are cut into ranges of equal work, one workgroup each: the work of a launch
// is the run of 32-key steps over (kv head, node, row tile), and range r takes its
// r-th part. Tiles whose rows are joined with others' results (groups', and those of
// sequences with shared keys) write partials even where a range holds all of them;
// the others write the output there. With `before` the number of such joined tiles
// before a tile in step order, a piece's partial is slot 2 r + before, + 1 if it is
// not the first of its range: slots grow from one written piece to the next, so they
// are distinct. The piece that starts a tile describes it for the merge: the joined
// tile number `before`, or range r's open tile (a range leaves at most one open).
#pragma once

#include "attn_decode.hpp"
#include "attn_prefill.hpp"

namespace vk {

constexpr int kShWaves = 4;
constexpr uint32_t kShThreads = 64 * kShWaves;
template <int D>
constexpr int sh_row_tiles() { return D == 256 ? 1 : 2; }
constexpr uint32_t sh_rows(uint32_t d) { return 16u * (d == 256 ? 1 : 2) * kShWaves; }
constexpr uint32_t kShMinSteps = 4;       // of a range, in launches of few steps
constexpr uint32_t kShMaxNodes = 4096;    // their plan is in LDS
constexpr uint32_t kShMaxRanges = 512;

struct ShTile {
  uint32_t valid, r0, r1;  // the ranges that hold it
  uint32_t node, tile, kh;
  uint32_t slot0, before;  // its first piece's slot; of range r's, for r > r0: 2 r + before
};

struct SharedArgs {
  // Groups, in device memory: group i's queries are entries offsets[i] ..
  // offsets[i + 1] of rows (rows of q) and seqs, its keys [0, keys[i]).
  const uint32_t *offsets, *rows, *seqs, *keys;
  uint32_t n_groups, n_rows;
  uint32_t n_nodes;     // the groups, then the sequences of a.pf_seqs
  uint32_t max_joined;  // joined tiles of a kv head, at most
  uint32_t ranges;
  // Blocks of node i at tables[i * table_width ..] (null: a.table's rows).
  const uint32_t* tables;
  uint32_t table_width;
  uint32_t last_blk;
  const char *k, *v;  // the pool they lie in
  uint64_t blk_e, head_e;
  uint32_t tok_e;
  // Workspace: the joined tiles of a kv head, joined tiles, ranges' open tiles; the
  // first tile of a sequence's own node; partials.
  uint32_t* n_joined;
  ShTile *joined, *open;
  uint32_t* own;
  char* part;
};

// a: the decode's arguments (kvh and group of virtual kv heads).
__device__ __forceinline__ uint32_t sh_heads(const AttnArgs& a) { return a.kvh / a.kv_parts.d; }

struct ShNode {
  uint32_t first, tokens;  // rows of its queries: entries of rows, or rows of q
  uint32_t seq;            // own nodes: the sequence; groups: one of theirs
  int32_t k0, k1;          // its keys
};
__device__ __forceinline__ ShNode sh_node(const AttnArgs& a, const SharedArgs& sh, uint32_t i) {
  ShNode n{0, 0, 0, 0, 0};
  if (i < sh.n_groups) {
    const uint32_t e0 = min(sh.offsets[i], sh.n_rows), e1 = min(sh.offsets[i + 1], sh.n_rows);
    n.first = e0;
    n.k1 = shared_keys(a, sh.keys[i]);
    if (e1 <= e0 || n.k1 <= 0) return n;
    n.seq = sh.seqs[e0];
    if (n.seq < a.batch) n.tokens = e1 - e0;
    return n;
  }
  n.seq = a.pf_seqs ? a.pf_seqs[i - sh.n_groups] : i - sh.n_groups;
  if (n.seq >= a.batch) return n;
  n.first = a.cu_q[n.seq];
  const uint32_t len_q = a.cu_q[n.seq + 1] - n.first;
  n.k1 = (int32_t)(a.cu_k[n.seq + 1] - a.cu_k[n.seq]);
  n.k0 = shared_keys(a, a.shared[n.seq]);
  if (len_q >= a.pf_min_q) n.tokens = len_q;
  return n;
}
// Steps of each of its tiles, at most (the last's).
__device__ __forceinline__ uint32_t sh_node_steps(const AttnArgs& a, const ShNode& n, bool group) {
  int32_t lo = n.k0, sinks = 0;
  if (!group) {
    if (a.wl >= 0) lo = max(lo, n.k1 - (int32_t)n.tokens - a.wl);
    if (n.k0 == 0) sinks = a.sinks;
  }
  if (lo >= n.k1) return 1;
  const KeySteps<true> ks(lo, n.k1 - 1, sinks, 32);
  return (uint32_t)ks.last / 32 + 1;
}

// The plan, in LDS: tiles, steps and joined tiles of the nodes before each (n_nodes + 1
// of each, one array after the other).
__device__ __forceinline__ void sh_plan(const AttnArgs& a, const SharedArgs& sh, uint32_t rows,
                                        uint32_t* tiles) {
  __shared__ uint32_t tot[3][kShWaves];
  const uint32_t N1 = sh.n_nodes + 1;
  uint32_t *steps = tiles + N1, *joined = steps + N1;
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t per = (sh.n_nodes + kShThreads - 1) / kShThreads;
  const uint32_t i0 = min(tid * per, sh.n_nodes), i1 = min(i0 + per, sh.n_nodes);
  uint32_t sum[3] = {0u, 0u, 0u}, inc[3];
  for (uint32_t i = i0; i < i1; ++i) {
    const ShNode n = sh_node(a, sh, i);
    const uint32_t nt = (uint32_t)(((uint64_t)n.tokens * a.g_real + rows - 1) / rows);
    const uint32_t ns = nt * sh_node_steps(a, n, i < sh.n_groups);
    const uint32_t nj = i < sh.n_groups || n.k0 > 0 ? nt : 0u;
    tiles[i] = nt, steps[i] = ns, joined[i] = nj;
    sum[0] += nt, sum[1] += ns, sum[2] += nj;
  }
#pragma unroll
  for (int x = 0; x < 3; ++x) {
    inc[x] = sum[x];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(inc[x], o);
      if (lane >= (uint32_t)o) inc[x] += y;
    }
    if (lane == 63) tot[x][wave] = inc[x];
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 3; ++x) {
    uint32_t* arr = tiles + x * N1;
    uint32_t run = inc[x] - sum[x];
    for (uint32_t w = 0; w < wave; ++w) run += tot[x][w];
    for (uint32_t i = i0; i < i1; ++i) {
      const uint32_t v = arr[i];
      arr[i] = run;
      run += v;
    }
    if (tid == kShThreads - 1) arr[sh.n_nodes] = run;
  }
  __syncthreads();
}

// The query of row r of a node: its row of q, sequence and position (false: none).
struct ShRow {
  uint32_t q, seq, head;  // head: of the kv head's group
  int32_t pos, len_k;
};
__device__ __forceinline__ bool sh_row(const AttnArgs& a, const SharedArgs& sh, const ShNode& n,
                                       bool group, uint32_t r, ShRow& w) {
  const uint32_t G = a.g_real, j = r / G;
  if (j >= n.tokens) return false;
  w.head = r - j * G;
  w.q = group ? sh.rows[n.first + j] : n.first + j;
  w.seq = group ? sh.seqs[n.first + j] : n.seq;
  if (w.seq >= a.batch) return false;
  const uint32_t q0 = a.cu_q[w.seq], len_q = a.cu_q[w.seq + 1] - q0;
  w.len_k = (int32_t)(a.cu_k[w.seq + 1] - a.cu_k[w.seq]);
  w.pos = w.len_k - (int32_t)len_q + (int32_t)(w.q - q0);
  return w.q - q0 < len_q;
}

// Counts [u0, u1) of the c of a node's tile at kv head kh (its share of the steps),
// to the partial `pb`, or to the output if pb is null.
template <typename T, int D, bool kPad>
__device__ __forceinline__ void sh_piece(const AttnArgs& a, const SharedArgs& sh, uint32_t node,
                                         uint32_t tile, uint32_t kh, uint32_t u0, uint32_t u1,
                                         uint32_t c, char* pb) {
  constexpr int RT = sh_row_tiles<D>(), W = kShWaves, KC = D / 32, DT = D / 16;
  constexpr uint32_t kRows = 16 * RT * W;
  constexpr int kLoadsPerStep = D >= 128 ? 2 * D / (16 * W) : 2;
  // (Three separate objects a tensor: see prefill_piece.)
  __shared__ __attribute__((aligned(16))) uint16_t kb0[32 * D], kb1[32 * D], kb2[32 * D];
  __shared__ __attribute__((aligned(16))) uint16_t vb0[32 * D], vb1[32 * D], vb2[32 * D];
  __shared__ int4 span[W];
  const bool group = node < sh.n_groups;
  const ShNode n = sh_node(a, sh, node);
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t col = lane & 15, g = lane >> 4;
  const uint32_t row0 = tile * kRows + wave * 16 * RT;
  const int32_t sinks = n.k0 ? 0 : a.sinks;

  // This lane's rows: what they see, and Q^T.
  uint4 qf[RT][KC];
  int32_t lo[RT], cnt[RT];
  // Over the workgroup's rows: the least and largest first key + 1, last key + 2.
  constexpr uint32_t kNone = 0x7FFFFFFFu;
  uint32_t ext[4] = {kNone, 0u, kNone, 0u};
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    ShRow w;
    const bool live = sh_row(a, sh, n, group, row0 + 16 * t + col, w);
    lo[t] = 0, cnt[t] = 0;
    if (live) {
      int32_t hi;
      key_range(w.pos, w.len_k, a.wl, a.wr, lo[t], hi);
      lo[t] = max(lo[t], n.k0);
      hi = max(min(hi, n.k1 - 1), -1);
      cnt[t] = max(hi - lo[t] + 1, 0);
      const uint32_t l1 = (uint32_t)lo[t] + 1, h2 = (uint32_t)(hi + 2);
      ext[0] = min(ext[0], l1), ext[1] = max(ext[1], l1);
      ext[2] = min(ext[2], h2), ext[3] = max(ext[3], h2);
    }
    const T* qrow = (const T*)a.q +
                    ((uint64_t)(live ? w.q : 0) * a.num_heads + kh * a.g_real + (live ? w.head : 0)) *
                        (kPad ? a.hd : D);
#pragma unroll
    for (int x = 0; x < KC; ++x) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (live && (!kPad || 32 * x + 8 * g < a.hd)) {
        u = *(const uint4*)(qrow + 32 * x + 8 * g);
        u.x ^= a.q_sign, u.y ^= a.q_sign, u.z ^= a.q_sign, u.w ^= a.q_sign;
      }
      qf[t][x] = u;
    }
  }
  {
    auto least = [](uint32_t x, uint32_t y) { return min(x, y); };
    auto most = [](uint32_t x, uint32_t y) { return max(x, y); };
    const uint32_t e0 = wave_reduce(ext[0], least), e1 = wave_reduce(ext[1], most);
    const uint32_t e2 = wave_reduce(ext[2], least), e3 = wave_reduce(ext[3], most);
    if (lane == 0) span[wave] = make_int4((int32_t)e0, (int32_t)e1, (int32_t)e2, (int32_t)e3);
  }
  __syncthreads();
  int4 e = span[0];
#pragma unroll
  for (int w = 1; w < W; ++w) {
    e.x = min(e.x, span[w].x), e.y = max(e.y, span[w].y);
    e.z = min(e.z, span[w].z), e.w = max(e.w, span[w].w);
  }
  // Keys that some row sees [klo, khi], and that all rows see [full_lo, full_hi].
  const int32_t klo = __builtin_amdgcn_readfirstlane(e.x) - 1;
  const int32_t full_lo = __builtin_amdgcn_readfirstlane(e.y) - 1;
  const int32_t full_hi = __builtin_amdgcn_readfirstlane(e.z) - 2;
  const int32_t khi = __builtin_amdgcn_readfirstlane(e.w) - 2;
  const KeySteps<true> ks(klo, khi, sinks, 32);
  const int32_t all = full_lo >= 0 && khi >= klo ? ks.last / 32 + 1 : 0;
  const int32_t a0 = (int32_t)pf_step_at(u0, c, (uint32_t)all);
  const int32_t a1 = (int32_t)pf_step_at(u1, c, (uint32_t)all);
  int32_t s0_ = 32 * a0;
  const int32_t s_last = 32 * a1 - 32;

  const uint32_t* __restrict__ tab =
      sh.tables ? sh.tables + (uint64_t)node * sh.table_width
                : a.table + (uint64_t)n.seq * a.max_blocks;
  AttnArgs p = a;  // (the fields that loads use)
  p.blk_e = sh.blk_e, p.head_e = sh.head_e, p.tok_e = sh.tok_e, p.last_blk = sh.last_blk;
  p.max_blocks = sh.tables ? sh.table_width : a.max_blocks;
  const T* kb = (const T*)sh.k + kh * sh.head_e;
  const T* vb = (const T*)sh.v + kh * sh.head_e;

  float m_run[RT], l_run[RT];
  floatx4 o[RT][DT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m_run[t] = kNegBig;
    l_run[t] = 0.f;
#pragma unroll
    for (int k = 0; k < DT; ++k) o[t][k] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  uint32_t k_off[2][KC];
#pragma unroll
  for (int tt = 0; tt < 2; ++tt)
#pragma unroll
    for (int x = 0; x < KC; ++x) k_off[tt][x] = pf_chunk<D>(16 * tt + col, 4 * x + g);
  const uint32_t vj = col >> 2, vq = col & 3;
  uint32_t v_off[DT][2];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      v_off[t][h] = pf_chunk<D>(16 * h + 4 * g + vj, 2 * t + (vq >> 1)) + 4 * (vq & 1);

  auto load = [&](uint16_t* kd, uint16_t* vd, int32_t at) __attribute__((always_inline)) {
    pf_dma<T, D, W, kPad>(kd, vd, tab, kb, vb, p, ks.key(at), KeyReads(ks, at, klo, khi, sinks), tid,
                          wave);
  };
  // The 32-key step of prefill_piece: scores, online softmax, O^T += V^T P^T, the
  // step after next on its way.
  auto step = [&](auto cur) __attribute__((always_inline)) {
    constexpr int B = decltype(cur)::value;
    uint16_t* const kbuf = B == 0 ? kb0 : B == 1 ? kb1 : kb2;
    uint16_t* const vbuf = B == 0 ? vb0 : B == 1 ? vb1 : vb2;
    uint16_t* const knext = B == 0 ? kb2 : B == 1 ? kb0 : kb1;
    uint16_t* const vnext = B == 0 ? vb2 : B == 1 ? vb0 : vb1;
    const int32_t at = __builtin_amdgcn_readfirstlane(s0_), s0 = ks.key(at);
    load(knext, vnext, min(at + 64, s_last));
    const bool masked = !(s0 >= full_lo && s0 + 31 <= full_hi);
    const uint32_t vbase = lds_addr(vbuf);
    constexpr int NB = (DT + 1) / 2;
    uint2 r[NB][4];
    auto issue = [&](int b) __attribute__((always_inline)) {
      uint32_t ad[4];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) ad[2 * k + h] = vbase + 2 * v_off[2 * b + k][h];
      ds_read_tr16_issue4(r[b], ad);
    };
    float sc[RT][8];
    {
      floatx4 acc[RT][2];
      KTile<D> kt;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int x = 0; x < KC; ++x) {
          kt.k[tt][x] = *(const uint4*)(kbuf + k_off[tt][x]);
          if (kPad && 32 * x + 8 * g >= a.hd) kt.k[tt][x] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int t = 0; t < RT; ++t) qk_scores<T, D>(kt, qf[t], acc[t]);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[t][4 * tt + i] = acc[t][tt][i];
        if (masked) {
          const int32_t key = s0 + 4 * (int32_t)g, top = min(sinks, lo[t] + cnt[t]);
          const uint32_t base = (uint32_t)(key - lo[t]), m = (uint32_t)cnt[t];
#pragma unroll
          for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!(base + 16 * tt + i < m || key + 16 * tt + i < top))
                sc[t][4 * tt + i] = -INFINITY;
        }
      }
    }
    issue(0);
    float mx[RT];
    bool grow = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      mx[t] = max3_nc(max3_nc(sc[t][0], sc[t][1], sc[t][2]), max3_nc(sc[t][3], sc[t][4], sc[t][5]),
                      max_nc(sc[t][6], sc[t][7])) * a.scale_log2;
      grow |= mx[t] > m_run[t] + kRescaleSlack;
    }
    if (__any(grow)) {
#pragma unroll
      for (int t = 0; t < RT; ++t) rescale_rows<D>(mx[t], o[t], m_run[t], l_run[t]);
    }
    uint4 pf[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) pf[t] = exp_pack<T>(sc[t], m_run[t], l_run[t], a.scale_log2);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (b + 1 < NB) {
        issue(b + 1);
        lgkm_wait<4>(r[b]);
      } else {
        lgkm_wait<0>(r[b]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint4 vf = make_uint4(r[b][2 * k].x, r[b][2 * k].y, r[b][2 * k + 1].x,
                                    r[b][2 * k + 1].y);
#pragma unroll
        for (int t = 0; t < RT; ++t) o[t][2 * b + k] = mfma16x16x32<T>(vf, pf[t], o[t][2 * b + k]);
      }
    }
    wait_vmcnt<kLoadsPerStep>();
    ring_barrier();
    s0_ += 32;
  };
  if (s0_ <= s_last) {  // (uniform)
    load(kb0, vb0, s0_);
    load(kb1, vb1, min(s0_ + 32, s_last));
    wait_vmcnt<kLoadsPerStep>();
    ring_barrier();
    while (true) {
      step(std::integral_constant<int, 0>{});
      if (s0_ > s_last) break;
      step(std::integral_constant<int, 1>{});
      if (s0_ > s_last) break;
      step(std::integral_constant<int, 2>{});
      if (s0_ > s_last) break;
    }
  }
  wait_vmcnt<0>();  // no load may land in LDS after the workgroup ends

#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const float lt = wave_sum_g(l_run[t]);
    const float inv = lt > 0.f ? 1.f / lt : 0.f;
    const uint32_t row = wave * 16 * RT + 16 * t + col;  // of the tile
    if (pb) {
      // Per row (m in scaled log2 units, l), then o / l (pf_part_bytes).
      if (g == 0) *(float2*)(pb + (uint64_t)row * 8) = make_float2(m_run[t], lt);
      float* po = (float*)(pb + (uint64_t)kRows * 8) + (uint64_t)row * D;
#pragma unroll
      for (int k = 0; k < DT; ++k)
        *(float4*)(po + 16 * k + 4 * g) = make_float4(o[t][k][0] * inv, o[t][k][1] * inv,
                                                      o[t][k][2] * inv, o[t][k][3] * inv);
      continue;
    }
    const uint32_t r = tile * kRows + row, j = r / a.g_real;
    if (j >= n.tokens) continue;
    T* orow = (T*)a.out + ((uint64_t)(n.first + j) * a.num_heads + kh * a.g_real + (r - j * a.g_real)) *
                              (kPad ? a.hd : D);
#pragma unroll
    for (int k = 0; k < DT; ++k)
      if (!kPad || 16 * k + 4 * g < a.hd)
        *(uint2*)(orow + 16 * k + 4 * g) = make_uint2(pack2<T>(o[t][k][0] * inv, o[t][k][1] * inv),
                                                      pack2<T>(o[t][k][2] * inv, o[t][k][3] * inv));
  }
}

// Workgroup `bid` of sh.ranges. lds: 3 (n_nodes + 1) words.
template <typename T, int D, bool kPad>
__device__ __forceinline__ void sh_range(const AttnArgs& a, const SharedArgs& sh, uint32_t* lds,
                                         uint32_t bid) {
  constexpr uint32_t kRows = sh_rows(D);
  const uint32_t N = sh.n_nodes, kvh = sh_heads(a);
  const uint32_t *tiles = lds, *steps = lds + N + 1, *joined = steps + N + 1;
  sh_plan(a, sh, kRows, lds);
  const uint32_t S = __builtin_amdgcn_readfirstlane(steps[N]);
  const uint32_t n_joined = __builtin_amdgcn_readfirstlane(joined[N]);
  const bool fits = n_joined <= sh.max_joined;  // (as every plan of the host's)
  if (bid == 0 && threadIdx.x == 0) *sh.n_joined = fits ? n_joined : 0u;
  const uint64_t total = (uint64_t)S * kvh;
  const uint32_t nr = (uint32_t)min((uint64_t)sh.ranges, (total + kShMinSteps - 1) / kShMinSteps);
  if (bid >= nr || !fits) {
    if (threadIdx.x == 0) sh.open[bid].valid = 0;
    return;
  }
  // An eighth of the ranges, one after the other, to an XCD: its row tiles of a kv
  // head and node read the same keys at about the same time.
  const uint32_t x = bid % 8, r = x * (nr / 8) + min(x, nr % 8) + bid / 8;
  uint64_t at = total * r / nr;
  const uint64_t end = total * (r + 1) / nr;
  uint32_t kh = (uint32_t)(at / S), rest = (uint32_t)(at - (uint64_t)kh * S);
  uint32_t lo = 0, hi = N;  // steps[lo] <= rest < steps[hi]
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (__builtin_amdgcn_readfirstlane(steps[mid]) <= rest) lo = mid;
    else hi = mid;
  }
  uint32_t node = lo;
  uint32_t t0 = __builtin_amdgcn_readfirstlane(tiles[node]);
  uint32_t nt = __builtin_amdgcn_readfirstlane(tiles[node + 1]) - t0;
  uint32_t s0 = __builtin_amdgcn_readfirstlane(steps[node]);
  uint32_t c = (__builtin_amdgcn_readfirstlane(steps[node + 1]) - s0) / nt;
  uint32_t tile = (rest - s0) / c, u0 = rest - s0 - tile * c;
  bool open = false;
  uint32_t after = 0;  // 1 past the range's first piece
  while (true) {
    const uint32_t u1 = (uint32_t)min((uint64_t)c, u0 + (end - at));
    const uint32_t j0 = __builtin_amdgcn_readfirstlane(joined[node]);
    const bool joins = __builtin_amdgcn_readfirstlane(joined[node + 1]) > j0;
    const uint32_t before = kh * n_joined + j0 + (joins ? tile : 0u);
    const uint32_t slot = 2 * r + after + before;
    const bool whole = u0 == 0 && u1 == c;
    if (u0 == 0 && (joins || !whole) && threadIdx.x == 0) {
      const uint32_t last = (uint32_t)min(((at + c) * nr + total - 1) / total, (uint64_t)nr) - 1;
      const ShTile d{1u, r, last, node, tile, kh, slot, before};
      (joins ? sh.joined[before] : sh.open[r]) = d;
      if (joins && node >= sh.n_groups && kh == 0 && tile == 0) {
        const uint32_t li = node - sh.n_groups;
        sh.own[a.pf_seqs ? a.pf_seqs[li] : li] = j0;
      }
    }
    open = open || (u0 == 0 && !joins && !whole);
    sh_piece<T, D, kPad>(a, sh, node, tile, kh, u0, u1, c,
                         joins || !whole ? sh.part + (uint64_t)slot * pf_part_bytes(kRows, D)
                                         : nullptr);
    after = 1;
    at += u1 - u0;
    if (at >= end) break;
    u0 = 0;
    if (++tile == nt) {
      tile = 0;
      do {
        if (++node == N) node = 0, ++kh;
        t0 = __builtin_amdgcn_readfirstlane(tiles[node]);
        nt = __builtin_amdgcn_readfirstlane(tiles[node + 1]) - t0;
      } while (nt == 0);
      s0 = __builtin_amdgcn_readfirstlane(steps[node]);
      c = (__builtin_amdgcn_readfirstlane(steps[node + 1]) - s0) / nt;
    }
    __syncthreads();  // the ring and span are used again
  }
  if (!open && threadIdx.x == 0) sh.open[r].valid = 0;
}

// Joins the partials of the rows of row block `block` of item `i` (the joined tiles of
// all kv heads, at most kvh * max_joined of them, then the ranges' open tiles): thread
// (row, four outputs). nwg: the decode's workgroups.
template <typename T, int D>
__device__ __forceinline__ void sh_merge(const AttnArgs& a, const SharedArgs& sh, uint32_t nwg,
                                         uint32_t i, uint32_t block) {
  constexpr uint32_t kRows = sh_rows(D), kTpr = D / 4, kRpw = 256 / kTpr;
  const uint32_t n_joined = *sh.n_joined, kvh = sh_heads(a);
  const uint32_t most = sh.max_joined * kvh;
  if (i < most && i >= n_joined * kvh) return;
  const ShTile d = i < most ? sh.joined[i] : sh.open[i - most];
  if (!d.valid || d.node >= sh.n_nodes) return;
  const uint32_t kh = d.kh, G = a.g_real;
  const uint32_t row = block * kRpw + threadIdx.x / kTpr, dq = (threadIdx.x % kTpr) * 4;
  const bool group = d.node < sh.n_groups;
  const ShNode n = sh_node(a, sh, d.node);
  if (!group && n.k0 > 0) return;  // joined with its group's
  ShRow w;
  if (!sh_row(a, sh, n, group, d.tile * kRows + row, w) || dq >= a.hd) return;
  const uint64_t stride = pf_part_bytes(kRows, D);
  // The partials: ranges d.r0 .. d.r1 of this tile, then of the sequence's own keys:
  // ranges of its tile, or the decode stream's of its segment.
  uint32_t np = d.r1 - d.r0 + 1, no = 0;
  ShTile e{};  // the own tile
  uint32_t orow = 0;
  auto slot_of = [](const ShTile& t, uint32_t j) { return j ? 2 * (t.r0 + j) + t.before : t.slot0; };
  uint64_t sl = 0;           // or the stream's first
  bool stream = false;
  if (group) {
    const uint32_t first = a.cu_q[w.seq], len_q = a.cu_q[w.seq + 1] - first;
    if (len_q < a.pf_min_q) {
      if (w.len_k > shared_keys(a, a.shared[w.seq])) {
        const uint32_t v = w.head / a.group;  // the virtual kv head of the group's part
        const uint32_t seg = w.seq * a.kvh + kh * a.kv_parts.d + v;
        const uint2 rr = *(const uint2*)(a.seg_ranges + 2 * seg);
        if (rr.y < nwg * kDecodeWavesPerWG && rr.x <= rr.y) {
          stream = true;
          no = rr.y - rr.x + 1;
          sl = ((uint64_t)rr.x * a.kv_parts.d + seg) * a.group + (w.head - v * a.group);
        }
      }
    } else {
      const uint32_t r = (w.q - first) * G + w.head;
      const uint32_t t = sh.own[w.seq] + r / kRows;
      if (t < n_joined) {
        e = sh.joined[kh * n_joined + t];
        // (A sequence that the list leaves out has no tile of its own.)
        if (e.node >= sh.n_groups && e.node < sh.n_nodes && e.tile == r / kRows &&
            sh_node(a, sh, e.node).seq == w.seq) {
          no = e.r1 - e.r0 + 1;
          orow = r % kRows;
        }
      }
    }
  }
  constexpr uint32_t kB = 8;  // partials per round trip
  float M = kNegBig, L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t s0 = 0; s0 < np + no; s0 += kB) {
    float2 ml[kB];
    float4 x[kB];
    float by[kB];
#pragma unroll
    for (uint32_t u = 0; u < kB; ++u) {
      const bool in = s0 + u < np + no;
      const uint32_t j = in ? s0 + u : 0;
      const bool own_part = j >= np;
      const float *pm, *px;
      if (own_part && stream) {
        const uint64_t slot = sl + (uint64_t)(j - np) * a.kv_parts.d * a.group;
        pm = a.ws_ml + slot * 2;
        px = a.ws_o + slot * D + dq;
      } else {
        const char* pb =
            sh.part + (uint64_t)(own_part ? slot_of(e, j - np) : slot_of(d, j)) * stride;
        const uint32_t rw = own_part ? orow : row;
        pm = (const float*)(pb + (uint64_t)rw * 8);
        px = (const float*)(pb + (uint64_t)kRows * 8) + (uint64_t)rw * D + dq;
      }
      ml[u] = *(const float2*)pm;
      x[u] = *(const float4*)px;
      // Tiles' partials hold o / l, the stream's o.
      by[u] = own_part && stream ? 1.f : ml[u].y;
      if (!in) ml[u].y = 0.f;
    }
    float Mn = M;
#pragma unroll
    for (uint32_t u = 0; u < kB; ++u)
      if (ml[u].y > 0.f) Mn = fmaxf(Mn, ml[u].x);
    const float f = fast_exp2(M - Mn);
    L *= f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= f;
#pragma unroll
    for (uint32_t u = 0; u < kB; ++u) {
      if (!(ml[u].y > 0.f)) continue;  // a share with no visible key (its o is stale)
      const float e = fast_exp2(ml[u].x - Mn), wgt = by[u] * e;
      L += ml[u].y * e;
      o[0] += x[u].x * wgt, o[1] += x[u].y * wgt, o[2] += x[u].z * wgt, o[3] += x[u].w * wgt;
    }
    M = Mn;
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  T* dst = (T*)a.out + ((uint64_t)w.q * a.num_heads + kh * G + w.head) * a.hd + dq;
  *(uint2*)dst = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
}

// ---- launch (attn_shared.hip) ----------------------------------------------------

// What a call needs past the decode's workspace.
size_t shared_workspace_bytes(const vapi_kv_prefixes* p, uint32_t batch, uint32_t kvh,
                              uint32_t group, uint32_t head_dim, uint32_t n_pf, uint32_t max_q);
// Refusals by the plan and the sizes: 0 or an error code with a message. n_pf: the
// sequences whose queries run as tiles (0 if no sequence has several).
int shared_check(const vapi_kv_prefixes* p, uint32_t batch, uint32_t kvh, uint32_t group,
                 uint32_t head_dim, uint32_t n_pf, uint32_t max_q, uint32_t max_k, const char* who);
// The groups and `ws` of a call over a's pool (a: the decode's arguments).
SharedArgs shared_args(const vapi_kv_prefixes* p, const AttnArgs& a, uint32_t head_dim,
                       uint32_t n_pf, uint32_t max_q, char* ws);
// The decode stream over the rows' own keys.
void launch_decode_shared(const AttnArgs& a, uint32_t head_dim, bool bf16, hipStream_t s);
// The tiles of a launch; then the merge of their partials and the stream's.
void launch_shared_tiles(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                         hipStream_t s);
void launch_shared_merge(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                         bool decode, hipStream_t s);

}  // namespace vk
