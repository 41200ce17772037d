// Launches of attention over shared prefixes (the device code is in attn_shared.hpp).
#include <algorithm>

#include "attn_shared.hpp"

namespace vk {

template <typename T, int D, bool kPad>
__global__ __launch_bounds__(kShThreads, D == 256 ? 1 : 2) void paged_shared_tiles(AttnArgs a,
                                                                                   SharedArgs sh) {
  extern __shared__ uint32_t plan[];
  sh_range<T, D, kPad>(a, sh, plan, blockIdx.x);
}

// Workgroups 0 .. merge_wgs - 1 join the stream's partials of rows without shared
// keys, the others those of tiles.
template <typename T, int D, int WPS, bool kPad>
__global__ __launch_bounds__(256) void paged_shared_merge(AttnArgs a, SharedArgs sh, uint32_t nwg,
                                                          uint32_t merge_wgs, uint32_t ns) {
  if (blockIdx.x < merge_wgs) {
    decode_merge_body<T, D, false, WPS, kPad, true>(a, nwg, merge_wgs, blockIdx.x, merge_wgs, ns);
    return;
  }
  constexpr uint32_t kBlocks = sh_rows(D) / (256 / (D / 4));
  const uint32_t i = blockIdx.x - merge_wgs;
  sh_merge<T, D>(a, sh, nwg, i / kBlocks, i % kBlocks);
}

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// Joined tiles of a kv head, at most: the groups' (each rounds up once), and those of
// members with several queries.
static uint64_t joined_tiles(const vapi_kv_prefixes* p, uint32_t group, uint32_t head_dim,
                             uint32_t n_pf) {
  const uint64_t t = (uint64_t)p->n_rows * group / sh_rows(head_dim);
  return t + std::min(p->n_groups, p->n_rows) + (n_pf ? t + std::min(p->n_rows, n_pf) : 0);
}

static uint32_t shared_ranges() {
  return std::min(kShMaxRanges, decode_num_waves() / kDecodeWavesPerWG);
}

struct SharedWs {
  size_t joined, open, own, part, total;
};
static SharedWs shared_ws(uint32_t batch, uint32_t kvh, uint32_t head_dim, uint64_t joined,
                          uint32_t ranges) {
  SharedWs w;
  w.joined = 256;
  w.open = w.joined + up256(kvh * joined * sizeof(ShTile));
  w.own = w.open + up256(ranges * sizeof(ShTile));
  w.part = w.own + up256((size_t)batch * sizeof(uint32_t));
  w.total = w.part + (2 * ranges + kvh * joined + 1) * pf_part_bytes(sh_rows(head_dim), head_dim);
  return w;
}

size_t shared_workspace_bytes(const vapi_kv_prefixes* p, uint32_t batch, uint32_t kvh,
                              uint32_t group, uint32_t head_dim, uint32_t n_pf, uint32_t max_q) {
  return shared_ws(batch, kvh, head_dim, joined_tiles(p, group, head_dim, n_pf), shared_ranges())
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
  // Steps of a kv head and workgroups of the merge stay in 32 bits.
  const uint64_t rows = sh_rows(head_dim), joined = joined_tiles(p, group, head_dim, n_pf);
  const uint64_t tiles =
      (uint64_t)p->n_rows * group / rows + p->n_groups +
      n_pf * (((uint64_t)max_q * group + rows - 1) / rows);
  if (tiles * ((uint64_t)max_k / 32 + 4) > 0xFFFFFFFFull || (joined + 1) * kvh > 0xFFFFFFull)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: too many queries for one launch", who);
  return 0;
}

SharedArgs shared_args(const vapi_kv_prefixes* p, const AttnArgs& a, uint32_t head_dim,
                       uint32_t n_pf, uint32_t max_q, char* ws) {
  SharedArgs sh{};
  sh.offsets = p->offsets, sh.rows = p->rows, sh.seqs = p->seqs, sh.keys = p->keys;
  sh.n_groups = p->n_rows ? p->n_groups : 0;
  sh.n_rows = p->n_rows;
  sh.n_nodes = sh.n_groups + n_pf;
  sh.max_joined = (uint32_t)joined_tiles(p, a.g_real, head_dim, n_pf);
  sh.ranges = shared_ranges();
  sh.last_blk = a.last_blk;
  sh.k = a.k, sh.v = a.v;
  sh.blk_e = a.blk_e, sh.head_e = a.head_e, sh.tok_e = a.tok_e;
  const SharedWs w = shared_ws(a.batch, a.kvh / a.kv_parts.d, head_dim, sh.max_joined, sh.ranges);
  sh.n_joined = (uint32_t*)ws;
  sh.joined = (ShTile*)(ws + w.joined);
  sh.open = (ShTile*)(ws + w.open);
  sh.own = (uint32_t*)(ws + w.own);
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

void launch_shared_tiles(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                         hipStream_t s) {
  const size_t lds = 3 * ((size_t)sh.n_nodes + 1) * sizeof(uint32_t);
#define VK_SHT(T, DD)                                                                          \
  hipLaunchKernelGGL((a.hd != DD ? paged_shared_tiles<T, DD, true>                             \
                                 : paged_shared_tiles<T, DD, false>),                          \
                     dim3(sh.ranges), dim3(kShThreads), lds, s, a, sh)
  VK_SH_ALL(VK_SHT);
#undef VK_SHT
}

void launch_shared_merge(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                         bool decode, hipStream_t s) {
  const uint32_t ns = decode_merge_slices(a.group, head_dim);
  bool wide = false;
  const uint32_t all = decode_merge_wgs(a.batch, a.kvh, &wide, ns);
  const uint32_t merge_wgs = decode ? all : 0u, nwg = a.num_waves / kDecodeWavesPerWG;
  const uint32_t items = sh.max_joined * (a.kvh / a.kv_parts.d) + sh.ranges;
  const dim3 grid(merge_wgs + items * (sh_rows(head_dim) / (256 / (head_dim / 4))));
#define VK_SHM2(T, DD, WPS)                                                                    \
  hipLaunchKernelGGL((a.hd != DD ? paged_shared_merge<T, DD, WPS, true>                        \
                                 : paged_shared_merge<T, DD, WPS, false>),                     \
                     grid, dim3(256), 0, s, a, sh, nwg, merge_wgs, ns)
#define VK_SHM(T, DD)                          \
  do {                                         \
    if (wide) VK_SHM2(T, DD, (int)kMergeWaves); \
    else VK_SHM2(T, DD, 1);                    \
  } while (0)
  VK_SH_ALL(VK_SHM);
#undef VK_SHM
#undef VK_SHM2
}

}  // namespace vk
