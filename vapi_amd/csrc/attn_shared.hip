// Launches of attention over shared prefixes (the device code is in attn_shared.hpp).
#include <algorithm>

#include "attn_shared.hpp"

namespace vk {

// Workgroups 0 .. nwg - 1 stream the decode rows' own keys (one to a CU, workgroup b on
// XCD b % 8), the others run ranges of tiles: HBM-bound waves and MFMA-bound ones side
// by side on a CU, and two workgroups of tiles to a CU where no stream runs.
template <typename T, int D, bool kPad, bool kNt>
__global__ __launch_bounds__(kShThreads, D == 256 ? 1 : 2) void paged_shared_stream(
    AttnArgs a, SharedArgs sh, uint32_t nwg) {
  static_assert(kShThreads == 64 * kDecodeWavesPerWG, "one workgroup size");
  extern __shared__ uint32_t plan[];
  if (blockIdx.x < nwg) {
    decode_stream_body<T, D, false, kPad, D / 16, kNt, true, true>(a, a.cu_q, a.cu_k, a.table, plan,
                                                                   blockIdx.x, nwg);
  } else {
    sh_range<T, D, kPad>(a, sh, plan, blockIdx.x - nwg);
  }
}

// Workgroups 0 .. merge_wgs - 1 join the stream's partials of rows without shared
// keys, the others those of tiles.
template <typename T, int D, int WPS, bool kPad, int NV>
__global__ __launch_bounds__(256) void paged_shared_merge(AttnArgs a, SharedArgs sh, uint32_t nwg,
                                                          uint32_t merge_wgs, uint32_t ns) {
  if (blockIdx.x < merge_wgs) {
    decode_merge_body<T, D, false, WPS, kPad, true>(a, nwg, merge_wgs, blockIdx.x, merge_wgs, ns);
    return;
  }
  // A workgroup to each row block of a group's tile, one to an open tile.
  constexpr uint32_t kBlocks = sh_rows(D) / sh_merge_rows(D, NV);
  const uint32_t i = blockIdx.x - merge_wgs, most = sh.max_grouped * sh_heads(a);
  if (i < most * kBlocks) {
    sh_merge<T, D, NV>(a, sh, nwg, i / kBlocks, i % kBlocks);
    return;
  }
  const uint32_t r = i - most * kBlocks;
  if (sh.open[r].valid)
    for (uint32_t b = 0; b < kBlocks; ++b) sh_merge<T, D, NV>(a, sh, nwg, most + r, b);
}

// Dynamic LDS with which two workgroups still share a CU (at head_dim 128, where the
// stream's queries and the tiles' ring take 64.3 KiB of the half).
constexpr size_t kShPlanLds = 15 * 1024;

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// Joined tiles of a kv head, at most: the groups' (each rounds up once), and those of
// members with several queries.
static uint64_t grouped_tiles(const vapi_kv_prefixes* p, uint32_t group, uint32_t head_dim) {
  return (uint64_t)p->n_rows * group / sh_rows(head_dim) + std::min(p->n_groups, p->n_rows);
}
static uint64_t joined_tiles(const vapi_kv_prefixes* p, uint32_t group, uint32_t head_dim,
                             uint32_t n_pf) {
  return grouped_tiles(p, group, head_dim) +
         (n_pf ? (uint64_t)p->n_rows * group / sh_rows(head_dim) + std::min(p->n_rows, n_pf) : 0);
}

// Workgroups of tiles: one to a CU (the stream's beside it), or two where each would
// have more than kShLongSteps steps: a step then takes 1.2-1.4 us instead of 1, a tile's
// fixed costs overlap, and half the partials are written where it is one. Us a call with
// 256 / 512: 64 sequences over 4,096 keys 43 / 58, three groups 55 / 62, 4-8 queries of 16
// over 3,200 47 / 49; 128 over 32,768 319 / 227, 1,050 queries of 28 152 / 119.
constexpr uint64_t kShLongSteps = 64;
static uint32_t shared_ranges(const vapi_kv_prefixes* p, uint32_t kvh, uint32_t group,
                              uint32_t head_dim, uint32_t n_pf) {
  const uint64_t steps =
      kvh * (grouped_tiles(p, group, head_dim) * (p->max_keys / 32 + kShTileSteps) +
             n_pf * (uint64_t)(kShTileSteps + kShMinSteps));
  const uint32_t one = kShMaxRanges / 2;
  return head_dim == 256 || steps < kShLongSteps * one ? one : kShMaxRanges;
}

struct SharedWs {
  size_t joined, open, own, queries, part, total;
};
static SharedWs shared_ws(uint32_t batch, uint32_t kvh, uint32_t head_dim, uint64_t joined,
                          uint32_t n_rows) {
  constexpr uint32_t ranges = kShMaxRanges;
  SharedWs w;
  w.joined = 256;
  w.open = w.joined + up256(kvh * joined * sizeof(ShTile));
  w.own = w.open + up256(ranges * sizeof(ShTile));
  w.queries = w.own + up256((size_t)batch * sizeof(uint32_t));
  w.part = w.queries + up256((size_t)n_rows * sizeof(ShQuery));
  w.total = w.part + (2 * ranges + kvh * joined + 1) * pf_part_bytes(sh_rows(head_dim), head_dim);
  return w;
}

size_t shared_workspace_bytes(const vapi_kv_prefixes* p, uint32_t batch, uint32_t kvh,
                              uint32_t group, uint32_t head_dim, uint32_t n_pf, uint32_t max_q) {
  return shared_ws(batch, kvh, head_dim, joined_tiles(p, group, head_dim, n_pf), p->n_rows)
      .total;
}

int shared_check(const vapi_kv_prefixes* p, uint32_t batch, uint32_t kvh, uint32_t group,
                 uint32_t head_dim, uint32_t n_pf, uint32_t max_q, uint32_t max_k,
                 const char* who) {
  if (!p) VK_FAIL(VAPI_KV_EINVAL, "%s: null prefixes", who);
  if (!p->start || !p->offsets ||
      (p->n_groups && p->n_rows && (!p->rows || !p->seqs || !p->keys)))
    VK_FAIL(VAPI_KV_EINVAL, "%s: null list of shared prefixes", who);
  if (p->max_keys > max_k)
    VK_FAIL(VAPI_KV_EINVAL, "%s: a prefix of %u keys, sequences of at most %u", who, p->max_keys,
            max_k);
  if (batch > decode_max_plan_seqs() || (uint64_t)p->n_groups + n_pf > kShMaxNodes)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: %u sequences, %u groups and %u prefill sequences", who, batch,
            p->n_groups, n_pf);
  // Steps of a kv head and threads of the merge (16 workgroups a joined tile) stay in
  // 32 bits.
  const uint64_t rows = sh_rows(head_dim), joined = joined_tiles(p, group, head_dim, n_pf);
  const uint64_t tiles =
      (uint64_t)p->n_rows * group / rows + p->n_groups +
      n_pf * (((uint64_t)max_q * group + rows - 1) / rows);
  if (tiles * ((uint64_t)max_k / 32 + 4 + kShTileSteps) > 0xFFFFFFFFull ||
      (joined + 1) * kvh > 0x7FFFFull)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: too many queries for one launch", who);
  return 0;
}

SharedArgs shared_args(const vapi_kv_prefixes* p, const AttnArgs& a, uint32_t head_dim,
                       uint32_t n_pf, char* ws) {
  SharedArgs sh{};
  sh.offsets = p->offsets, sh.rows = p->rows, sh.seqs = p->seqs, sh.keys = p->keys;
  // (Groups without rows or rows without groups are neither: their lists may be null.)
  sh.n_groups = p->n_rows ? p->n_groups : 0;
  sh.n_rows = p->n_groups ? p->n_rows : 0;
  sh.n_nodes = sh.n_groups + n_pf;
  sh.max_joined = (uint32_t)joined_tiles(p, a.g_real, head_dim, n_pf);
  sh.max_grouped = (uint32_t)grouped_tiles(p, a.g_real, head_dim);
  sh.ranges = shared_ranges(p, a.kvh / a.kv_parts.d, a.g_real, head_dim, n_pf);
  const SharedWs w = shared_ws(a.batch, a.kvh / a.kv_parts.d, head_dim, sh.max_joined,
                               p->n_rows);
  sh.lds_rows =
      sh.n_rows && sh_plan_bytes(sh.n_nodes) + sh.n_rows * sizeof(ShEntry) <= kShPlanLds;
  sh.n_tiles = (uint32_t*)ws;
  sh.joined = (ShTile*)(ws + w.joined);
  sh.open = (ShTile*)(ws + w.open);
  sh.own = (uint32_t*)(ws + w.own);
  sh.queries = (ShQuery*)(ws + w.queries);
  sh.part = ws + w.part;
  return sh;
}

#define VK_SH_ALL(FN)                                            \
  do {                                                           \
    if (bf16) {                                                  \
      if (head_dim == 256) FN(bf16_t, 256);                      \
      else if (head_dim == 128) FN(bf16_t, 128);                 \
      else FN(bf16_t, 64);                                       \
    } else {                                                     \
      if (head_dim == 256) FN(f16_t, 256);                       \
      else if (head_dim == 128) FN(f16_t, 128);                  \
      else FN(f16_t, 64);                                        \
    }                                                            \
  } while (0)

size_t shared_lds(const AttnArgs& a, const SharedArgs& sh, uint32_t nwg, uint32_t ranges) {
  const size_t plan =
      sh_plan_bytes(sh.n_nodes) + (sh.lds_rows ? sh.n_rows * sizeof(ShEntry) : 0);
  return std::max(ranges ? plan : 0, nwg ? (a.batch + 1) * sizeof(uint32_t) : 0);
}

static void launch_shared_stream(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim,
                                 bool bf16, uint32_t nwg, uint32_t ranges, hipStream_t s) {
  const size_t lds = shared_lds(a, sh, nwg, ranges);
  // (A group of query heads in parts reads its keys with ordinary loads: launch_stream.)
#define VK_SHT(T, DD)                                                                            \
  do {                                                                                           \
    constexpr auto once = paged_shared_stream<T, DD, false, true>;                               \
    constexpr auto once_pad = paged_shared_stream<T, DD, true, true>;                            \
    constexpr auto parts = paged_shared_stream<T, DD, true, false>;                              \
    hipLaunchKernelGGL(a.kv_parts.d > 1 ? parts : a.hd != DD ? once_pad : once, dim3(nwg + ranges), \
                       dim3(kShThreads), lds, s, a, sh, nwg);                                    \
  } while (0)
  VK_SH_ALL(VK_SHT);
#undef VK_SHT
}

void launch_shared(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                   bool decode, hipStream_t s) {
  const uint32_t nwg = decode ? a.num_waves / kDecodeWavesPerWG : 0;
  if (head_dim == 256 && decode) {  // one workgroup to a CU: one kind after the other
    launch_shared_stream(a, sh, head_dim, bf16, nwg, 0, s);
    launch_shared_stream(a, sh, head_dim, bf16, 0, sh.ranges, s);
  } else {
    launch_shared_stream(a, sh, head_dim, bf16, nwg, sh.ranges, s);
  }
  launch_shared_merge(a, sh, head_dim, bf16, decode, s);
}

void launch_shared_merge(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                         bool decode, hipStream_t s) {
  const uint32_t ns = decode_merge_slices(a.group, head_dim);
  bool wide = false;
  const uint32_t all = decode_merge_wgs(a.batch, a.kvh, &wide, ns);
  const uint32_t merge_wgs = decode ? all : 0u, nwg = a.num_waves / kDecodeWavesPerWG;
  // Four outputs a thread and eight partials a round trip, or where those workgroups do
  // not all run at once (four to a CU) eight and four: half the chains of lists, tiles
  // and partials. Us, with four / eight outputs: 1,050 queries of 28 sequences (32 heads,
  // 9 tiles a head) 21.7 / 14.5; 64 single queries 8.5 / 9.8, three groups 9.0 / 10.7.
  const uint32_t tiles = sh.max_grouped * (a.kvh / a.kv_parts.d);
  const int nv = tiles * (sh_rows(head_dim) / sh_merge_rows(head_dim, 1)) > 1024 ? 2 : 1;
  const uint32_t blocks = sh_rows(head_dim) / sh_merge_rows(head_dim, nv);
  // (Without sequences of their own tiles, no range has an open one.)
  const dim3 grid(merge_wgs + tiles * blocks +
                  (sh.n_nodes > sh.n_groups ? sh.ranges : 0u));
#define VK_SHM3(T, DD, WPS, NV)                                                   \
  hipLaunchKernelGGL((a.hd != DD ? paged_shared_merge<T, DD, WPS, true, NV>        \
                                 : paged_shared_merge<T, DD, WPS, false, NV>),     \
                     grid, dim3(256), 0, s, a, sh, nwg, merge_wgs, ns)
#define VK_SHM2(T, DD, WPS)          \
  do {                               \
    if (nv > 1) VK_SHM3(T, DD, WPS, 2); \
    else VK_SHM3(T, DD, WPS, 1);     \
  } while (0)
#define VK_SHM(T, DD)                          \
  do {                                         \
    if (wide) VK_SHM2(T, DD, (int)kMergeWaves); \
    else VK_SHM2(T, DD, 1);                    \
  } while (0)
  VK_SH_ALL(VK_SHM);
#undef VK_SHM
#undef VK_SHM2
#undef VK_SHM3
}

}  // namespace vk
