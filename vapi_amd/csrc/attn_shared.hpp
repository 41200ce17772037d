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
// is the run of 32-key steps over (kv head, node, row tile), kShTileSteps more to a
// tile, and range r takes its r-th part. Tiles whose rows are joined with others'
// results (groups', and those of sequences with shared keys) write partials even where
// a range holds all of them; the others write the output there. With `before` the
// number of such joined tiles before a tile in step order, a piece's partial is slot
// 2 r + before, + 1 if it is not the first of its range: slots grow from one written
// piece to the next, so they are distinct and nothing is atomic. The piece that starts
// a tile describes it for the merge: the joined tile number `before`, or range r's open
// tile (a range leaves at most one open).
//
// Measured, us a call (without sharing), 32 q / 8 kv heads of 128 in bf16: 64 sequences
// over 4,096 shared keys 43.2 (172), 4-8 queries each of 16 over 3,200 45.4 (72); 64 q
// heads, 128 sequences over 32,768 224-230 (2,485), 620 TFLOP/s. Long prefixes are bound
// by the tiles' step (25% MFMA, 29% VALU, waits at 2 waves a SIMD), short ones by round
// trips, 4-10 us each while the stream keeps HBM's queues full, and by the merge, 6-15.
#pragma once

#include "attn_decode.hpp"
#include "attn_prefill.hpp"
#include "q8.hpp"

namespace vk {

constexpr int kShWaves = 4;
constexpr uint32_t kShThreads = 64 * kShWaves;
template <int D>
constexpr int sh_row_tiles() { return D == 256 ? 1 : 2; }
constexpr uint32_t sh_rows(uint32_t d) { return 16u * (d == 256 ? 1 : 2) * kShWaves; }
constexpr uint32_t kShMinSteps = 8;       // of a range, in launches of few steps
// What a tile costs beside its steps (its rows, its first loads, its results: 5-6 us, a
// step 1-1.4): counted as work, so that ranges of many short tiles are not the longest.
constexpr uint32_t kShTileSteps = 5;
// Their plan (32 bytes each) is in LDS, beside 128 KiB of queries and ring at D = 256.
constexpr uint32_t kShMaxNodes = 1000;
constexpr uint32_t kShMaxRanges = 512;

struct __attribute__((aligned(16))) ShTile {
  uint32_t valid, r0, r1;  // the ranges that hold it
  uint32_t tile;
  uint32_t kh, slot0, before;  // its first piece's slot; of range r's, for r > r0: 2 r + before
  uint32_t seq;                // own nodes: the sequence; groups: ~0
  uint32_t first, tokens;      // the node's rows
  uint32_t pad[2];
};
// A query of a group as the merge needs it.
struct __attribute__((aligned(16))) ShQuery {
  uint32_t q;     // its row of q, ~0: none
  uint32_t seq;
  uint32_t kind;  // where its own keys' partials are: ShOwn
  uint32_t tok;   // its number among its sequence's queries
};
enum ShOwn : uint32_t { kOwnNone, kOwnStream, kOwnTiles };

struct SharedArgs {
  // Groups, in device memory: group i's queries are entries offsets[i] ..
  // offsets[i + 1] of rows (rows of q) and seqs, its keys [0, keys[i]).
  const uint32_t *offsets, *rows, *seqs, *keys;
  uint32_t n_groups, n_rows;
  uint32_t n_nodes;     // the groups, then the sequences of a.pf_seqs
  uint32_t max_joined;   // joined tiles of a kv head, at most
  uint32_t max_grouped;  // the groups' of them (the first, in step order)
  uint32_t ranges;
  const float *ks, *vs;  // 8-bit pools: the layer's scales, sblk a block
  uint32_t sblk;
  uint32_t lds_rows;  // whether every query of the groups has an entry in LDS
  // Workspace: the joined tiles of a kv head, {the groups', the sequences' own}; joined
  // tiles, max_grouped of each kv head for the groups and then the rest for each; the
  // ranges' open tiles; the first joined tile of a sequence's own node (of sequences that
  // have one: what the others' words hold is of earlier calls); the groups' queries;
  // partials.
  uint32_t* n_tiles;
  ShTile *joined, *open;
  uint32_t* own;
  ShQuery* queries;
  char* part;
};

// a: the decode's arguments (kvh and group of virtual kv heads).
__device__ __forceinline__ uint32_t sh_heads(const AttnArgs& a) { return a.kvh / a.kv_parts.d; }

struct ShNode {
  uint32_t first, tokens;  // rows of its queries: entries of rows, or rows of q
  uint32_t seq;            // own nodes: the sequence; groups: one of theirs (sh_plan)
  int32_t k0, k1;          // its keys
};
__device__ __forceinline__ ShNode sh_node(const AttnArgs& a, const SharedArgs& sh, uint32_t i) {
  ShNode n{0, 0, 0, 0, 0};
  if (i < sh.n_groups) {
    const uint32_t e0 = min(sh.offsets[i], sh.n_rows), e1 = min(sh.offsets[i + 1], sh.n_rows);
    n.first = e0;
    n.k1 = shared_keys(a, sh.keys[i]);
    if (e1 <= e0 || n.k1 <= 0) return n;
    n.tokens = e1 - e0;
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

// Entry e of the groups' lists: its row of q (~0: it names none), its sequence, and the
// keys that its mask leaves.
struct ShEntry {
  uint32_t q, seq;
  int32_t lo, hi;
};
__device__ __forceinline__ ShEntry sh_entry(const AttnArgs& a, const SharedArgs& sh, uint32_t e,
                                            ShQuery* info = nullptr) {
  ShEntry x{sh.rows[e], sh.seqs[e], 0, -1};
  const bool in = x.seq < a.batch;
  const uint32_t s = in ? x.seq : 0;
  const uint32_t q0 = a.cu_q[s], len_q = a.cu_q[s + 1] - q0;
  const int32_t len_k = (int32_t)(a.cu_k[s + 1] - a.cu_k[s]);
  const uint32_t tok = x.q - q0;
  if (!in || tok >= len_q) x.q = ~0u;
  else key_range(len_k - (int32_t)len_q + (int32_t)tok, len_k, a.wl, a.wr, x.lo, x.hi);
  if (info) {
    const bool past = len_k > shared_keys(a, a.shared[s]);
    *info = ShQuery{x.q, s, len_q >= a.pf_min_q ? kOwnTiles : past ? kOwnStream : kOwnNone, tok};
  }
  return x;
}

// The plan, in LDS: tiles, steps and joined tiles of the nodes before each (n_nodes + 1
// of each, one array after the other), then the nodes. `entries`: the groups' queries, if
// they are in LDS. A group's keys are those of the sequence of its first entry that names
// a query (none: of any).
constexpr size_t sh_plan_bytes(uint32_t n_nodes) {
  return 3 * ((size_t)n_nodes + 1) * sizeof(uint32_t) + n_nodes * sizeof(ShNode);
}
__device__ __forceinline__ void sh_plan(const AttnArgs& a, const SharedArgs& sh, uint32_t rows,
                                        uint32_t* tiles, const ShEntry* entries) {
  __shared__ uint32_t tot[3][kShWaves];
  const uint32_t N1 = sh.n_nodes + 1;
  uint32_t *steps = tiles + N1, *joined = steps + N1;
  ShNode* nodes = (ShNode*)(joined + N1);
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t per = (sh.n_nodes + kShThreads - 1) / kShThreads;
  const uint32_t i0 = min(tid * per, sh.n_nodes), i1 = min(i0 + per, sh.n_nodes);
  uint32_t sum[3] = {0u, 0u, 0u}, inc[3];
  for (uint32_t i = i0; i < i1; ++i) {
    const ShNode n = sh_node(a, sh, i);
    const uint32_t nt = (uint32_t)(((uint64_t)n.tokens * a.g_real + rows - 1) / rows);
    const uint32_t ns = nt * (sh_node_steps(a, n, i < sh.n_groups) + kShTileSteps);
    const uint32_t nj = i < sh.n_groups || n.k0 > 0 ? nt : 0u;
    tiles[i] = nt, steps[i] = ns, joined[i] = nj;
    nodes[i] = n;
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
  auto entry = [&](uint32_t e) { return sh.lds_rows ? entries[e] : sh_entry(a, sh, e); };
  for (uint32_t i = i0; i < i0 + per; ++i) {
    ShEntry x{0, 0, 0, 0};
    if (i < min(i1, sh.n_groups) && nodes[i].tokens) {
      x = entry(nodes[i].first);
      nodes[i].seq = x.q != ~0u ? x.seq : 0u;
    }
    // Groups whose first entry names none, one after the other by all of the wave.
    for (uint64_t dead = __ballot(x.q == ~0u); dead; dead &= dead - 1) {
      const uint32_t node = __shfl(i, __builtin_ctzll(dead));
      const uint32_t first = nodes[node].first, end = first + nodes[node].tokens;
      for (uint32_t e = first; e < end; e += 64) {
        const ShEntry y = entry(min(e + lane, end - 1));
        const uint64_t live = __ballot(y.q != ~0u);
        if (!live) continue;
        if (lane == (uint32_t)__builtin_ctzll(live)) nodes[node].seq = y.seq;
        break;
      }
    }
  }
  __syncthreads();
}

// A thread's chunks are the same rows and columns of every step (ShSlots), so that a
// step whose keys are all read as they are costs no address arithmetic per lane.
template <int D, int W, bool kPad>
struct ShSlots {
  static constexpr uint32_t CPR = D / 8;             // chunks a row
  static constexpr int N = D >= 128 ? D / (16 * W) : 1;
  static_assert((64 * W / CPR) % 8 == 0 || N == 1, "slots of a thread are 8 or 16 rows apart");
  uint32_t r0, col[N], off[N];  // off: bytes from the 16-key tile's first row
  __device__ __forceinline__ ShSlots(uint32_t tid, uint32_t tok_e, uint32_t hd) {
    const uint32_t slot0 = D >= 128 || W == 4 ? tid : tid & 255;  // (W == 8, D == 64: see issue)
    r0 = slot0 / CPR;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint32_t r = r0 + (64 * W / CPR) * j;
      uint32_t p = (slot0 % CPR) ^ pf_swz<D>(r);
      if (kPad && 8 * p >= hd) p = 0;
      col[j] = 8 * p;
      off[j] = ((r & 15) * tok_e + 8 * p) * 2;
    }
  }
};
template <typename T, int D, int W, bool kPad, typename Reads>
__device__ __forceinline__ void sh_issue(const ShSlots<D, W, kPad>& sl, uint16_t* kdst,
                                         uint16_t* vdst, const T* kb, const T* vb, uint32_t blk0,
                                         uint32_t blk1, uint64_t blk_e, uint32_t tok_e,
                                         uint32_t block_size, int32_t s0, const Reads& rd,
                                         uint32_t wave) {
  constexpr uint32_t CPR = D / 8;
  const int32_t ts0 = rd.tile(s0), ts1 = rd.tile(s0 + 16);
  const uint64_t off0 = (uint64_t)blk0 * blk_e + (uint64_t)((uint32_t)ts0 & (block_size - 1)) * tok_e;
  const uint64_t off1 = (uint64_t)blk1 * blk_e + (uint64_t)((uint32_t)ts1 & (block_size - 1)) * tok_e;
  auto all = [&](auto whole) __attribute__((always_inline)) {
    auto one = [&](const T* base_t, uint16_t* buf, int j, uint32_t wslot0)
                   __attribute__((always_inline)) {
      // A wave's slots cover 64 / CPR whole rows of one 16-key tile.
      const bool second = wslot0 / CPR >= 16;
      const char* base = (const char*)(base_t + (second ? off1 : off0));
      uint32_t off = sl.off[j];
      if constexpr (!decltype(whole)::value) {
        const uint32_t r = sl.r0 + (64 * W / CPR) * j;
        off = (rd.row((int32_t)(r & 15), second ? ts1 : ts0) * tok_e + sl.col[j]) * 2;
      }
      __builtin_amdgcn_global_load_lds((const void*)(base + off), (LdsVoid*)(buf + wslot0 * 8), 16, 0,
                                       0);
    };
    if constexpr (D >= 128) {
#pragma unroll
      for (int j = 0; j < D / (16 * W); ++j) {
        one(kb, kdst, j, 64 * wave + 64 * W * j);
        one(vb, vdst, j, 64 * wave + 64 * W * j);
      }
    } else if constexpr (W == 8) {
      if (wave < 4) one(kb, kdst, 0, 64 * wave);
      else one(vb, vdst, 0, 64 * (wave - 4));
    } else {
      one(kb, kdst, 0, 64 * wave);
      one(vb, vdst, 0, 64 * wave);
    }
  };
  if (rd.whole(s0)) all(std::true_type{});
  else all(std::false_type{});
}

// A thread's codes of a step: 16 of a row at a time (D == 64: of K in the first half of
// the workgroup, of V in the other), and the scales of their block.
template <int D>
struct ShCodes {
  static constexpr uint32_t CPR = D / 16;     // chunks of 16 codes a row
  static constexpr int N = D == 256 ? 2 : 1;  // chunks of a tensor
  uint4 k[N], v[N];
  float ks[N], vs[N];
};

// Four ds_read_b64_tr_b16 issued without waiting (results valid only after a later
// lgkm wait that names the same registers): the d tiles at a0 and a1, their keys 0 .. 15
// and, 16 rows on (the swizzle repeats), 16 .. 31.
template <int D>
__device__ __forceinline__ void sh_read_tr16(uint2 (&r)[4], uint32_t a0, uint32_t a1) {
  __asm__ volatile(
      "ds_read_b64_tr_b16 %0, %4\n\t"
      "ds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
      "ds_read_b64_tr_b16 %2, %5\n\t"
      "ds_read_b64_tr_b16 %3, %5 offset:%6"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
      : "v"(a0), "v"(a1), "n"(16 * D * 2)
      : "memory");
}
// Counts [u0, u1) of the c of a node's tile at kv head kh (its share of the steps),
// to the partial `pb`, or to the output if pb is null. F: the format of an 8-bit pool's
// codes, kShValues where the pool holds values of T. Codes come through registers, three
// steps ahead, and are expanded into the ring a step before they are used (exactly: every
// code times its scale is a value of T): 128 columns of 32 keys are 16 codes of K and of V
// a thread. (Expanded by a launch of its own into a 16-bit pool in the workspace, 32
// sequences over 5,008 keys, 32 kv heads, took 26 us more: 41 MB read, 82 written, 82
// read again.)
constexpr int kShValues = -1;
template <typename T, int D, bool kPad, int F>
__device__ __forceinline__ void sh_piece(const AttnArgs& a, const SharedArgs& sh, uint32_t node,
                                         const ShNode* nodes, const ShEntry* entries,
                                         uint32_t tile, uint32_t kh, uint32_t u0, uint32_t u1,
                                         uint32_t c, char* pb) {
  constexpr int RT = sh_row_tiles<D>(), W = kShWaves, KC = D / 32, DT = D / 16;
  constexpr uint32_t kRows = 16 * RT * W;
  constexpr int kLoadsPerStep = D >= 128 ? 2 * D / (16 * W) : 2;
  constexpr bool kCodes = F != kShValues;
  using E = std::conditional_t<kCodes, uint8_t, T>;  // of the pool
  // (Three separate objects a tensor: see prefill_piece.)
  __shared__ __attribute__((aligned(16))) uint16_t kb0[32 * D], kb1[32 * D], kb2[32 * D];
  __shared__ __attribute__((aligned(16))) uint16_t vb0[32 * D], vb1[32 * D], vb2[32 * D];
  __shared__ int2 span[W];
  const bool group = node < sh.n_groups;
  ShNode n;
  n.first = __builtin_amdgcn_readfirstlane(nodes[node].first);
  n.tokens = __builtin_amdgcn_readfirstlane(nodes[node].tokens);
  n.seq = __builtin_amdgcn_readfirstlane(nodes[node].seq);
  n.k0 = __builtin_amdgcn_readfirstlane(nodes[node].k0);
  n.k1 = __builtin_amdgcn_readfirstlane(nodes[node].k1);
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t col = lane & 15, g = lane >> 4;
  const uint32_t row0 = tile * kRows + wave * 16 * RT;
  const int32_t sinks = n.k0 ? 0 : a.sinks;

  const uint32_t* __restrict__ tab = a.table + (uint64_t)n.seq * a.max_blocks;
  const uint32_t width = a.max_blocks - 1;
  const E* kb = (const E*)a.k + kh * a.head_e;
  const E* vb = (const E*)a.v + kh * a.head_e;
  // The keys [klo, khi] that the tile's rows see, this share of their steps, and the
  // share's first two on their way.
  int32_t klo = 0, khi = -1, s0_ = 0, s_last = -32;
  KeySteps<true> ks(0, 0, 0, 32);
  // A step's blocks are looked up a step before its loads are issued, so that a wave
  // does not wait for the table there.
  auto lookup = [&](int32_t at) __attribute__((always_inline)) {
    using ConstU32 = const __attribute__((address_space(4))) uint32_t;
    const KeyReads rd(ks, at, klo, khi, sinks);
    const int32_t s0 = ks.key(at);
    return make_uint2(((ConstU32*)tab)[min((uint32_t)rd.tile(s0) >> a.bs_shift, width)],
                      ((ConstU32*)tab)[min((uint32_t)rd.tile(s0 + 16) >> a.bs_shift, width)]);
  };
  const ShSlots<D, W, kPad> slots(tid, a.tok_e, a.hd);
  auto load = [&](uint16_t* kd, uint16_t* vd, int32_t at, uint2 blk) __attribute__((always_inline)) {
    if constexpr (!kCodes)
      sh_issue<T, D, W, kPad>(slots, kd, vd, kb, vb, min(blk.x, a.last_blk), min(blk.y, a.last_blk),
                              a.blk_e, a.tok_e, a.block_size, ks.key(at),
                              KeyReads(ks, at, klo, khi, sinks), wave);
  };
  using Codes = ShCodes<D>;
  Codes c0, c1, c2;
  const uint32_t slot_c = D == 64 ? tid & 127 : tid, row_c = slot_c / Codes::CPR;
  const uint32_t col_c = slot_c % Codes::CPR;  // in chunks
  auto load_codes = [&](Codes& x, int32_t at, uint2 blk) __attribute__((always_inline)) {
    using ConstF32 = const __attribute__((address_space(4))) float;
    const KeyReads rd(ks, at, klo, khi, sinks);
    const int32_t s0 = ks.key(at);
    const uint32_t d = kPad && 16 * col_c >= a.hd ? 0 : 16 * col_c;
#pragma unroll
    for (int j = 0; j < Codes::N; ++j) {
      // (A wave's rows lie in one 16-key tile, so in one block.)
      const bool second = D == 256 ? j == 1 : D == 128 ? wave >= 2 : wave & 1;
      const uint32_t b = min(second ? blk.y : blk.x, a.last_blk);
      const int32_t ts = rd.tile(second ? s0 + 16 : s0);
      const uint64_t off = (uint64_t)b * a.blk_e +
                           (uint64_t)((uint32_t)ts & (a.block_size - 1)) * a.tok_e +
                           (rd.row((int32_t)(row_c & 15), ts) * a.tok_e + d);
      const uint64_t si = (uint64_t)b * sh.sblk + kh;
      if constexpr (D == 64) {
        x.k[j] = *(const uint4*)((wave < 2 ? kb : vb) + off);
        x.ks[j] = ((ConstF32*)(wave < 2 ? sh.ks : sh.vs))[si];
      } else {
        x.k[j] = *(const uint4*)(kb + off), x.v[j] = *(const uint4*)(vb + off);
        x.ks[j] = ((ConstF32*)sh.ks)[si], x.vs[j] = ((ConstF32*)sh.vs)[si];
      }
    }
  };
  auto expand = [&](const Codes& x, uint16_t* kd, uint16_t* vd) __attribute__((always_inline)) {
    auto put = [&](uint16_t* buf, int j, uint4 w, float s) __attribute__((always_inline)) {
      const uint32_t r = row_c + 16 * j;
      const uint2 e0 = q8_expand4<T, F, true>(w.x, s), e1 = q8_expand4<T, F, true>(w.y, s);
      const uint2 e2 = q8_expand4<T, F, true>(w.z, s), e3 = q8_expand4<T, F, true>(w.w, s);
      *(uint4*)(buf + pf_chunk<D>(r, 2 * col_c)) = make_uint4(e0.x, e0.y, e1.x, e1.y);
      *(uint4*)(buf + pf_chunk<D>(r, 2 * col_c + 1)) = make_uint4(e2.x, e2.y, e3.x, e3.y);
    };
#pragma unroll
    for (int j = 0; j < Codes::N; ++j) {
      if constexpr (D == 64) {
        if (wave < 2) put(kd, j, x.k[j], x.ks[j]);
        else put(vd, j, x.k[j], x.ks[j]);
      } else {
        put(kd, j, x.k[j], x.ks[j]), put(vd, j, x.v[j], x.vs[j]);
      }
    }
  };
  // The next step's rows are in the ring, all waves'.
  auto ring_ready = [&]() __attribute__((always_inline)) {
    if constexpr (kCodes) __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    else wait_vmcnt<kLoadsPerStep>();
    ring_barrier();
  };
  uint2 blk{0, 0};  // of the step whose loads are issued next
  auto begin = [&](int32_t lo_, int32_t hi_) __attribute__((always_inline)) {
    // (Windows past all of the node's keys leave the sinks' steps, or none.)
    klo = window_first(lo_, hi_, 32), khi = hi_;
    ks = KeySteps<true>(klo, khi, sinks, 32);
    const uint32_t all = (uint32_t)(ks.last / 32 + 1);
    s0_ = 32 * (int32_t)pf_step_at(u0, c, all);
    s_last = 32 * (int32_t)pf_step_at(u1, c, all) - 32;
    if (s0_ <= s_last) {  // (uniform)
      const uint2 b0 = lookup(s0_), b1 = lookup(min(s0_ + 32, s_last));
      const uint2 b2 = lookup(min(s0_ + 64, s_last));
      if constexpr (kCodes) {
        blk = lookup(min(s0_ + 96, s_last));
        load_codes(c0, s0_, b0);
        load_codes(c1, min(s0_ + 32, s_last), b1);
        load_codes(c2, min(s0_ + 64, s_last), b2);
      } else {
        blk = b2;
        load(kb0, vb0, s0_, b0);
        load(kb1, vb1, min(s0_ + 32, s_last), b1);
      }
    }
  };
  // Without a left window the keys follow from the node: the first loads need not wait
  // for the rows' lengths (shared keys past a row's position are masked).
  if (a.wl < 0) {
    const uint32_t r_end = min((tile + 1) * kRows, n.tokens * a.g_real);
    const int32_t p_last = n.k1 - (int32_t)n.tokens + (int32_t)((r_end - 1) / a.g_real);
    begin(n.k0, group || a.wr < 0 ? n.k1 - 1 : min(n.k1 - 1, p_last + a.wr));
  }

  // This lane's rows: what they see, and Q^T.
  uint4 qf[RT][KC];
  int32_t lo[RT], cnt[RT];
  // Over the wave's rows: their largest first key + 1, least last key + 2; over those
  // and the other waves': the least first key + 1, the largest last key + 2.
  uint32_t lo_min = 0x7FFFFFFFu, lo_max = 0u, hi_min = 0x7FFFFFFFu, hi_max = 0u;
  const T* qrow[RT];
  bool live[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const uint32_t r = row0 + 16 * t + col, j = r / a.g_real;
    const bool in = j < n.tokens;
    uint32_t wq = n.first + (in ? j : 0);
    int32_t wlo, hi;
    key_range(n.k1 - (int32_t)n.tokens + (int32_t)j, n.k1, a.wl, a.wr, wlo, hi);
    if (group && in) {
      const uint32_t e = wq;
      if (sh.lds_rows) {
        wq = entries[e].q, wlo = entries[e].lo, hi = entries[e].hi;
      } else {
        const ShEntry x = sh_entry(a, sh, e);
        wq = x.q, wlo = x.lo, hi = x.hi;
      }
    }
    live[t] = in && wq != ~0u;
    lo[t] = 0, cnt[t] = 0;
    if (live[t]) {
      lo[t] = max(wlo, n.k0);
      hi = max(min(hi, n.k1 - 1), -1);
      cnt[t] = max(hi - lo[t] + 1, 0);
      const uint32_t l1 = (uint32_t)lo[t] + 1, h2 = (uint32_t)(hi + 2);
      lo_min = min(lo_min, l1), lo_max = max(lo_max, l1);
      hi_min = min(hi_min, h2), hi_max = max(hi_max, h2);
    }
    qrow[t] = (const T*)a.q + ((uint64_t)(live[t] ? wq : 0) * a.num_heads + kh * a.g_real +
                               (live[t] ? r - j * a.g_real : 0)) * (kPad ? a.hd : D);
  }
  auto least = [](uint32_t x, uint32_t y) { return min(x, y); };
  auto most = [](uint32_t x, uint32_t y) { return max(x, y); };
  const int32_t full_lo = (int32_t)__builtin_amdgcn_readfirstlane(wave_reduce(lo_max, most)) - 1;
  const int32_t full_hi = (int32_t)__builtin_amdgcn_readfirstlane(wave_reduce(hi_min, least)) - 2;
  const bool active = full_lo >= 0;  // a wave without rows only loads
  if (a.wl >= 0) {
    const uint32_t e0 = wave_reduce(lo_min, least), e1 = wave_reduce(hi_max, most);
    if (lane == 0) span[wave] = make_int2((int32_t)e0, (int32_t)e1);
    __syncthreads();
    int2 e = span[0];
#pragma unroll
    for (int w = 1; w < W; ++w) e.x = min(e.x, span[w].x), e.y = max(e.y, span[w].y);
    begin(__builtin_amdgcn_readfirstlane(e.x) - 1, __builtin_amdgcn_readfirstlane(e.y) - 2);
  }
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int x = 0; x < KC; ++x) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (live[t] && (!kPad || 32 * x + 8 * g < a.hd)) {
        u = *(const uint4*)(qrow[t] + 32 * x + 8 * g);
        u.x ^= a.q_sign, u.y ^= a.q_sign, u.z ^= a.q_sign, u.w ^= a.q_sign;
      }
      qf[t][x] = u;
    }

  float m_run[RT], l_run[RT];
  floatx4 o[RT][DT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m_run[t] = kNegBig;
    l_run[t] = 0.f;
#pragma unroll
    for (int k = 0; k < DT; ++k) o[t][k] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  uint32_t k_off[KC];
#pragma unroll
  for (int x = 0; x < KC; ++x) k_off[x] = pf_chunk<D>(col, 4 * x + g);
  const uint32_t vj = col >> 2, vq = col & 3;
  uint32_t v_off[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
    v_off[t] = 2 * (pf_chunk<D>(4 * g + vj, 2 * t + (vq >> 1)) + 4 * (vq & 1));

  // The 32-key step of prefill_piece: scores, online softmax, O^T += V^T P^T, the
  // step after next on its way.
  auto step = [&](auto cur) __attribute__((always_inline)) {
    constexpr int B = decltype(cur)::value;
    uint16_t* const kbuf = B == 0 ? kb0 : B == 1 ? kb1 : kb2;
    uint16_t* const vbuf = B == 0 ? vb0 : B == 1 ? vb1 : vb2;
    uint16_t* const knext = B == 0 ? kb2 : B == 1 ? kb0 : kb1;
    uint16_t* const vnext = B == 0 ? vb2 : B == 1 ? vb0 : vb1;
    const int32_t at = __builtin_amdgcn_readfirstlane(s0_), s0 = ks.key(at);
    if constexpr (kCodes) {
      Codes& x = B == 0 ? c1 : B == 1 ? c2 : c0;
      expand(x, B == 0 ? kb1 : B == 1 ? kb2 : kb0, B == 0 ? vb1 : B == 1 ? vb2 : vb0);
      load_codes(x, min(at + 128, s_last), blk);
      blk = lookup(min(at + 160, s_last));
    } else {
      load(knext, vnext, min(at + 64, s_last), blk);
      blk = lookup(min(at + 96, s_last));
    }
    s0_ += 32;
    if (!active) {
      ring_ready();
      return;
    }
    const bool masked = !(s0 >= full_lo && s0 + 31 <= full_hi);
    const uint32_t vbase = lds_addr(vbuf);
    constexpr int NB = (DT + 1) / 2;
    uint2 r[NB][4];
    auto issue = [&](int b) __attribute__((always_inline)) {
      sh_read_tr16<D>(r[b], vbase + v_off[2 * b], vbase + v_off[2 * b + 1]);
    };
    float sc[RT][8];
    {
      floatx4 acc[RT][2];
      KTile<D> kt;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int x = 0; x < KC; ++x) {
          kt.k[tt][x] = *(const uint4*)(kbuf + k_off[x] + 16 * D * tt);
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
    ring_ready();
  };
  if (s0_ <= s_last) {  // (uniform)
    if constexpr (kCodes) {
      expand(c0, kb0, vb0);
      load_codes(c0, min(s0_ + 96, s_last), blk);
      blk = lookup(min(s0_ + 128, s_last));
    }
    ring_ready();
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
    const uint32_t r = tile * kRows + row, j = r / a.g_real;
    if (j >= n.tokens) continue;
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
    const uint64_t head = (uint64_t)(n.first + j) * a.num_heads + kh * a.g_real + (r - j * a.g_real);
    T* orow = (T*)a.out + head * (kPad ? a.hd : D);
#pragma unroll
    for (int k = 0; k < DT; ++k)
      if (!kPad || 16 * k + 4 * g < a.hd)
        *(uint2*)(orow + 16 * k + 4 * g) = make_uint2(pack2<T>(o[t][k][0] * inv, o[t][k][1] * inv),
                                                      pack2<T>(o[t][k][2] * inv, o[t][k][3] * inv));
  }
}

// Workgroup `bid` of sh.ranges. lds: sh_plan_bytes, and with sh.lds_rows an entry for
// each of the groups' queries: read while nothing else runs yet, where a round trip to
// memory is short (beside the stream at work it takes 4 to 5 us).
template <typename T, int D, bool kPad, int F = kShValues>
__device__ __forceinline__ void sh_range(const AttnArgs& a, const SharedArgs& sh, uint32_t* lds,
                                         uint32_t bid) {
  constexpr uint32_t kRows = sh_rows(D);
  const uint32_t N = sh.n_nodes, kvh = sh_heads(a);
  const uint32_t *tiles = lds, *steps = lds + N + 1, *joined = steps + N + 1;
  const ShNode* nodes = (const ShNode*)(joined + N + 1);
  ShEntry* entries = (ShEntry*)(nodes + N);
  if (sh.lds_rows)
    for (uint32_t e = threadIdx.x; e < sh.n_rows; e += kShThreads) entries[e] = sh_entry(a, sh, e);
  for (uint32_t e = bid * kShThreads + threadIdx.x; e < sh.n_rows; e += sh.ranges * kShThreads)
    sh_entry(a, sh, e, sh.queries + e);
  sh_plan(a, sh, kRows, lds, entries);
  const uint32_t S = __builtin_amdgcn_readfirstlane(steps[N]);
  const uint32_t n_joined = __builtin_amdgcn_readfirstlane(joined[N]);
  const uint32_t n_grouped = __builtin_amdgcn_readfirstlane(joined[sh.n_groups]);
  const uint32_t max_own = sh.max_joined - sh.max_grouped;
  const bool fits = n_grouped <= sh.max_grouped && n_joined - n_grouped <= max_own;  // (every plan)
  if (bid == 0 && threadIdx.x == 0)
    *(uint2*)sh.n_tiles = fits ? make_uint2(n_grouped, n_joined - n_grouped) : make_uint2(0u, 0u);
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
      const bool group = node < sh.n_groups;
      const uint32_t t = j0 + tile;  // of the kv head's joined tiles
      uint4* d = (uint4*)(!joins  ? sh.open + r
                          : group ? sh.joined + kh * sh.max_grouped + t
                                  : sh.joined + kvh * sh.max_grouped + kh * max_own +
                                        (t - n_grouped));
      d[0] = make_uint4(1u, r, last, tile);
      d[1] = make_uint4(kh, slot, before, group ? ~0u : nodes[node].seq);
      d[2] = make_uint4(nodes[node].first, nodes[node].tokens, 0u, 0u);
      if (joins && !group && kh == 0 && tile == 0) sh.own[nodes[node].seq] = j0 - n_grouped;
    }
    open = open || (u0 == 0 && !joins && !whole);
    sh_piece<T, D, kPad, F>(a, sh, node, nodes, entries, tile, kh, u0, u1, c,
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

// Rows of a workgroup of the merge: threads of four outputs (NV == 1) or eight.
constexpr uint32_t sh_merge_rows(uint32_t d, int nv) { return 256 / (d / (4 * nv)); }

// Joins the partials of the rows of row block `block` of item `i` (the groups' tiles of
// all kv heads, at most kvh * max_grouped of them, then the ranges' open tiles): thread
// (row, 4 NV outputs). nwg: the decode's workgroups.
template <typename T, int D, int NV>
__device__ __forceinline__ void sh_merge(const AttnArgs& a, const SharedArgs& sh, uint32_t nwg,
                                         uint32_t i, uint32_t block) {
  constexpr uint32_t kRows = sh_rows(D), kTpr = D / (4 * NV), kRpw = sh_merge_rows(D, NV);
  const uint32_t kvh = sh_heads(a), most = sh.max_grouped * kvh, G = a.g_real;
  const bool group = i < most;
  const uint2 n_tiles = *(const uint2*)sh.n_tiles;
  const ShTile d = group ? sh.joined[i] : sh.open[i - most];
  if (group ? i % sh.max_grouped >= n_tiles.x : !d.valid) return;
  const uint32_t kh = d.kh;
  const uint32_t row = block * kRpw + threadIdx.x / kTpr, dq = (threadIdx.x % kTpr) * 4;
  const uint32_t r = d.tile * kRows + row, tok = r / G, head = r - tok * G;
  if (tok >= d.tokens || dq >= a.hd) return;
  ShQuery w{d.first + tok, d.seq, kOwnNone, tok};
  if (group) w = sh.queries[d.first + tok];
  const uint64_t stride = pf_part_bytes(kRows, D);
  auto slot_of = [](const ShTile& t, uint32_t j) { return j ? 2 * (t.r0 + j) + t.before : t.slot0; };
  constexpr uint32_t kB = 8 / NV;  // partials per round trip
  // The second four outputs are D / 2 on (past a.hd: the first again, not stored).
  const uint32_t d2 = NV > 1 && dq + D / 2 < a.hd ? D / 2 : 0;
  float M = kNegBig, L = 0.f, o[4 * NV] = {};
  uint2 ml[kB];  // (bits: weighs)
  float4 x[kB][NV];
  // Partials [j0, j0 + kB) of the n at (m, l) pm(j) and o px(j).
  auto fetch = [&](uint32_t j0, uint32_t n, auto at) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t u = 0; u < kB; ++u) {
      ml[u].y = 0u;
      if (j0 + u >= n) continue;
      const float *pm, *px;
      at(j0 + u, pm, px);
      ml[u] = *(const uint2*)pm;
#pragma unroll
      for (int v = 0; v < NV; ++v) x[u][v] = *(const float4*)(px + v * d2);
    }
  };
  // Joins what was fetched. kNormed: it is o / l (tiles'), else o (the stream's).
  auto join = [&](bool normed) __attribute__((always_inline)) {
    float Mn = M;
#pragma unroll
    for (uint32_t u = 0; u < kB; ++u)
      if (weighs(ml[u].y)) Mn = fmaxf(Mn, __uint_as_float(ml[u].x));
    const float f = fast_exp2(M - Mn);
    L *= f;
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) o[i] *= f;
#pragma unroll
    for (uint32_t u = 0; u < kB; ++u) {
      if (!weighs(ml[u].y)) continue;  // a share with no visible key (its o is stale)
      const float e = fast_exp2(__uint_as_float(ml[u].x) - Mn), l = __uint_as_float(ml[u].y);
      const float wgt = normed ? l * e : e;
      L += l * e;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        o[4 * v] += x[u][v].x * wgt, o[4 * v + 1] += x[u][v].y * wgt;
        o[4 * v + 2] += x[u][v].z * wgt, o[4 * v + 3] += x[u][v].w * wgt;
      }
    }
    M = Mn;
  };
  auto of_tile = [&](const ShTile& t, uint32_t r) {
    return [&, r](uint32_t j, const float*& pm, const float*& px) {
      const char* pb = sh.part + (uint64_t)slot_of(t, j) * stride;
      pm = (const float*)(pb + (uint64_t)r * 8);
      px = (const float*)(pb + (uint64_t)kRows * 8) + (uint64_t)r * D + dq;
    };
  };
  // The tile's partials are on their way while the row's own are looked up.
  const uint32_t np = d.r1 - d.r0 + 1;
  fetch(0, np, of_tile(d, row));
  if (w.q == ~0u) return;
  // Its own keys: ranges of its tile, or the decode stream's of its segment.
  uint32_t no = 0, orow = 0;
  ShTile e{};
  uint64_t sl = 0;
  const bool stream = w.kind == kOwnStream;
  if (stream) {
    const uint32_t v = head / a.group;  // the virtual kv head of the group's part
    const uint32_t seg = w.seq * a.kvh + kh * a.kv_parts.d + v;
    const uint2 rr = *(const uint2*)(a.seg_ranges + 2 * seg);
    if (rr.y < nwg * kDecodeWavesPerWG && rr.x <= rr.y) {
      no = rr.y - rr.x + 1;
      sl = (uint64_t)stream_slot(a.plan_parts, rr.x, seg) * a.group + (head - v * a.group);
    }
  } else if (w.kind == kOwnTiles) {
    const uint32_t row_own = w.tok * G + head, max_own = sh.max_joined - sh.max_grouped;
    const uint32_t t = sh.own[w.seq] + row_own / kRows;
    // (The call's own tiles, all of them written: a sequence that the list of prefill
    // sequences leaves out has none among them, whatever `own` holds for it.)
    if (t < n_tiles.y) {
      e = sh.joined[most + kh * max_own + t];
      if (e.seq == w.seq && e.tile == row_own / kRows) {
        no = e.r1 - e.r0 + 1;
        orow = row_own % kRows;
      }
    }
  }
  join(true);
  for (uint32_t j0 = kB; j0 < np; j0 += kB) {
    fetch(j0, np, of_tile(d, row));
    join(true);
  }
  for (uint32_t j0 = 0; j0 < no; j0 += kB) {
    if (stream)
      fetch(j0, no, [&](uint32_t j, const float*& pm, const float*& px) {
        const uint64_t slot = sl + (uint64_t)j * a.plan_parts * a.group;
        pm = a.ws_ml + slot * 2;
        px = a.ws_o + slot * D + dq;
      });
    else
      fetch(j0, no, of_tile(e, orow));
    join(!stream);
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  T* dst = (T*)a.out + ((uint64_t)w.q * a.num_heads + kh * G + head) * a.hd + dq;
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (v == 0 || d2)
      *(uint2*)(dst + v * d2) = make_uint2(pack2<T>(o[4 * v] * inv, o[4 * v + 1] * inv),
                                           pack2<T>(o[4 * v + 2] * inv, o[4 * v + 3] * inv));
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
                       uint32_t n_pf, char* ws);
// The decode rows' own keys (`decode`: the batch may have such rows), the tiles, and
// the merge of their partials.
void launch_shared(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                   bool decode, hipStream_t s);
// The same over an 8-bit pool (sh.ks, sh.vs and sh.sblk set).
void launch_q8_shared(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                      bool e4m3, bool decode, hipStream_t s);
// Their merge, and the dynamic LDS of a launch of nwg and `ranges` workgroups.
void launch_shared_merge(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                         bool decode, hipStream_t s);
size_t shared_lds(const AttnArgs& a, const SharedArgs& sh, uint32_t nwg, uint32_t ranges);

}  // namespace vk
