// Eviction by running attention weight: which keys of each (sequence, kv head)
// stay, and their rows moved into new blocks.
//
//  1. evict_select: a workgroup per (sequence, kv head) finds the weight of the
//     last key that stays by a radix select on order-preserving keys (8 bits a
//     pass, a histogram in LDS), then walks the positions in order and writes
//     the kept ones with their weights. Ties go to the earlier position: the
//     walk counts those equal to the threshold as it meets them.
//  2. evict_copy (any pool): 16-byte pieces of K and V rows, from each head's
//     own positions. evict_q8: a wave per (new block, kv head, K or V) takes
//     the rows' codes and scales, finds the block's scale from their largest
//     value and writes the codes under it.
#include <algorithm>

#include "q8.hpp"

namespace vk {

constexpr uint32_t kSelectThreads = 1024;

struct EvictArgs {
  const float* in;
  float* out;  // null: weights are not wanted
  const uint32_t *in_index, *out_index, *lens;
  uint64_t in_row, in_head, out_row, out_head;
  uint32_t in_rows, out_rows, in_width, out_width;
  int32_t* kept;
  uint32_t kvh, max_len, max_keep, budget, sinks, recent;
};

__device__ __forceinline__ uint32_t evict_len(const EvictArgs& a, uint32_t seq) {
  return min(a.lens[seq], a.max_len);
}

// Weights as unsigned numbers in the same order: NaN lowest, both zeros alike.
__device__ __forceinline__ uint32_t evict_key(float w) {
  const uint32_t u = __float_as_uint(w), mag = u & 0x7fffffffu;
  if (mag > 0x7f800000u) return 0u;
  if (mag == 0) return 0x80000000u;
  return u >> 31 ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select(EvictArgs a) {
  constexpr uint32_t kWaves = kSelectThreads / 64;
  __shared__ uint32_t hist[256], counts[2][kWaves], found[2];
  const uint32_t seq = blockIdx.x / a.kvh, h = blockIdx.x - seq * a.kvh;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t in_row = a.in_index ? a.in_index[seq] : seq;
  const uint32_t out_row = a.out ? (a.out_index ? a.out_index[seq] : seq) : 0;
  int32_t* kept = a.kept + (uint64_t)blockIdx.x * a.max_keep;
  // A row index past the state leaves the sequence out (no key is kept).
  const bool ok = in_row < a.in_rows;
  const uint32_t len = ok ? evict_len(a, seq) : 0;
  const float* w = a.in + in_row * a.in_row + h * a.in_head;
  float* out = a.out && out_row < a.out_rows ? a.out + out_row * a.out_row + h * a.out_head
                                             : nullptr;
  const uint32_t n = min(len, a.budget);
  // Always kept: [0, first) and [end, len); of [first, end) the `want` largest.
  const uint32_t first = min(a.sinks, len), end = len - min(a.recent, len - first);
  const uint32_t want = n - first - (len - end);
  uint32_t threshold = 0, equal = 0xFFFFFFFFu;  // all of them
  if (want < end - first) {
    // The want-th largest key: digit by digit, `equal` of the keys that share
    // the digits found so far are still wanted.
    uint32_t prefix = 0;
    equal = want;
    for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t above = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
      for (uint32_t i = first + tid; i < end; i += kSelectThreads) {
        const uint32_t key = evict_key(w[i]);
        if ((key & above) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid < 64) {
        // Lane l holds digits 255 - 4 l .. 252 - 4 l, from the largest down.
        uint32_t c[4], sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = hist[255 - (4 * lane + j)], sum += c[j];
        uint32_t run = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t y = __shfl_up(run, o);
          if (lane >= (uint32_t)o) run += y;
        }
        run -= sum;  // keys with larger digits than this lane's
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (run < equal && equal <= run + c[j])
            found[0] = 255 - (4 * lane + j), found[1] = equal - run;
          run += c[j];
        }
      }
      __syncthreads();
      prefix |= found[0] << shift;
      equal = found[1];
      __syncthreads();
    }
    threshold = prefix;
    if (want == 0) threshold = 0xFFFFFFFFu, equal = 0;
  }
  // In order of position: larger ones, and the first `equal` of the equal ones.
  uint32_t eq_before = 0, at = 0;
  for (uint32_t base = 0; base < len; base += kSelectThreads) {
    const uint32_t i = base + tid;
    const bool mid = i >= first && i < end;
    const float x = i < len ? w[i] : 0.f;
    const uint32_t key = evict_key(x);
    const uint64_t eq = __ballot(mid && key == threshold);
    if (lane == 0) counts[0][wave] = (uint32_t)__popcll(eq);
    __syncthreads();
    uint32_t rank = eq_before, total = eq_before;
    for (uint32_t v = 0; v < kWaves; ++v) {
      if (v < wave) rank += counts[0][v];
      total += counts[0][v];
    }
    eq_before = total;
    rank += (uint32_t)__popcll(eq & ((1ull << lane) - 1));
    const bool take = i < len && (!mid || key > threshold || (key == threshold && rank < equal));
    const uint64_t taken = __ballot(take);
    if (lane == 0) counts[1][wave] = (uint32_t)__popcll(taken);
    __syncthreads();
    uint32_t to = at;
    total = at;
    for (uint32_t v = 0; v < kWaves; ++v) {
      if (v < wave) to += counts[1][v];
      total += counts[1][v];
    }
    at = total;
    to += (uint32_t)__popcll(taken & ((1ull << lane) - 1));
    // to <= i: with out the same row as in, what is overwritten has been read.
    if (take && to < n) {
      kept[to] = (int32_t)i;
      if (out && to < a.out_width) out[to] = x;
    }
  }
  for (uint32_t j = n + tid; j < a.max_keep; j += kSelectThreads) kept[j] = -1;
  if (out && ok) {
    __syncthreads();
    for (uint32_t j = n + tid; j < a.out_width; j += kSelectThreads) out[j] = 0.f;
  }
}

// ---- rows into their new blocks ---------------------------------------------------

struct EvictMove {
  const uint32_t *src_table, *dst_table;
  const int32_t* kept;
  uint32_t src_blocks, dst_blocks, num_blocks, block_size;
  FastDiv bs;
  uint32_t max_keep, kvh;
  char *k, *v;
  uint64_t blk_b, head_b, tok_b;
  uint32_t row_bytes;
};

// Grid: (pieces of a head's kept rows, segments, K or V).
template <int C>
__global__ __launch_bounds__(256) void evict_copy(EvictMove a, FastDiv upr) {
  using V = typename Chunk<C>::T;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  const uint32_t j = upr.div(i), u = i - j * upr.d;
  if (j >= a.max_keep) return;
  const uint32_t seq = blockIdx.y / a.kvh, h = blockIdx.y - seq * a.kvh;
  const int32_t from = a.kept[(uint64_t)blockIdx.y * a.max_keep + j];
  if (from < 0) return;
  const uint32_t sb = a.bs.div((uint32_t)from), db = a.bs.div(j);
  const uint32_t src = min(a.src_table[(uint64_t)seq * a.src_blocks + min(sb, a.src_blocks - 1)],
                           a.num_blocks - 1);
  if (db >= a.dst_blocks) return;
  const uint32_t dst = a.dst_table[(uint64_t)seq * a.dst_blocks + db];
  if (dst >= a.num_blocks) return;
  char* base = (blockIdx.z ? a.v : a.k) + h * a.head_b + (uint64_t)u * C;
  const uint64_t so = ((uint32_t)from - sb * a.bs.d) * a.tok_b, d_o = (j - db * a.bs.d) * a.tok_b;
  *(V*)(base + dst * a.blk_b + d_o) = load_stream((const V*)(base + src * a.blk_b + so));
}

constexpr int kMoveRegs = 4;  // 16-code pieces a lane holds: 4,096 codes a wave
constexpr uint32_t kMoveWaves = 4;

// Grid: (new blocks / 4 waves, segments, K or V).
template <typename T, int F>
__global__ __launch_bounds__(64 * kMoveWaves) void evict_q8(EvictMove a, FastDiv upr, float* ks,
                                                             float* vs, uint32_t sblk) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t db = blockIdx.x * kMoveWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t j0 = db * a.block_size;
  if (j0 >= a.max_keep || db >= a.dst_blocks) return;
  const uint32_t seq = blockIdx.y / a.kvh, h = blockIdx.y - seq * a.kvh;
  const int32_t* kept = a.kept + (uint64_t)blockIdx.y * a.max_keep;
  if (kept[j0] < 0) return;  // the sequence keeps fewer
  const uint32_t dst = a.dst_table[(uint64_t)seq * a.dst_blocks + db];
  if (dst >= a.num_blocks) return;
  float* scales = blockIdx.z ? vs : ks;
  char* base = (blockIdx.z ? a.v : a.k) + h * a.head_b;
  const uint32_t total = a.block_size * upr.d;
  uint4 w[kMoveRegs];
  float s[kMoveRegs];
  auto load = [&](uint32_t first) {
#pragma unroll
    for (int r = 0; r < kMoveRegs; ++r) {
      const uint32_t i = first + 64 * r + lane, o = upr.div(i), c = i - o * upr.d;
      w[r] = make_uint4(0u, 0u, 0u, 0u);
      s[r] = 0.f;
      const int32_t from = i < total && j0 + o < a.max_keep ? kept[j0 + o] : -1;
      if (from >= 0) {
        const uint32_t sb = a.bs.div((uint32_t)from);
        const uint32_t src = min(
            a.src_table[(uint64_t)seq * a.src_blocks + min(sb, a.src_blocks - 1)], a.num_blocks - 1);
        w[r] = *(const uint4*)(base + src * a.blk_b +
                               ((uint32_t)from - sb * a.bs.d) * a.tok_b + 16 * c);
        const float x = scales[(uint64_t)src * sblk + h];
        s[r] = q8_inverse(x) > 0.f ? x : 0.f;
      }
    }
  };
  auto word = [](const uint4& x, int e) { return e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w; };
  float top = 0.f;
  for (uint32_t first = 0; first < total; first += 64 * kMoveRegs) {
    load(first);
#pragma unroll
    for (int r = 0; r < kMoveRegs; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x[4];
        q8_unpack4<F>(word(w[r], e), x);
        top = fmaxf(top, s[r] * fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])),
                                      fmaxf(fabsf(x[2]), fabsf(x[3]))));
      }
  }
  const float amax = __uint_as_float(wave_reduce(__float_as_uint(top), [](uint32_t p, uint32_t q) {
    return max(p, q);
  }));
  const float scale = q8_scale<T, F>(amax), inv = q8_inverse(scale);
  const bool again = total > 64 * kMoveRegs;
  for (uint32_t first = 0; first < total; first += 64 * kMoveRegs) {
    if (again) load(first);
#pragma unroll
    for (int r = 0; r < kMoveRegs; ++r) {
      const uint32_t i = first + 64 * r + lane;
      if (i >= total) continue;
      const uint32_t o = upr.div(i), c = i - o * upr.d;
      uint32_t out[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x[4];
        q8_unpack4<F>(word(w[r], e), x);
        // (Two products: s times 1 / scale may not be a number of its own.)
        out[e] = q8_pack4<F>(x[0] * s[r] * inv, x[1] * s[r] * inv, x[2] * s[r] * inv,
                             x[3] * s[r] * inv);
      }
      *(uint4*)(base + dst * a.blk_b + o * a.tok_b + 16 * c) =
          make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
  if (lane == 0) scales[(uint64_t)dst * sblk + h] = scale;
}

int check_weights(const vapi_kv_weights* w, uint32_t batch, uint32_t kvh, const char* who);

struct EvictCall {
  const vapi_kv_weights *in, *out;
  const uint32_t *lens, *src_table, *dst_table;
  uint32_t src_blocks, dst_blocks, batch, max_len, budget, sinks, recent;
  int32_t* kept;
};

static int evict_checks(const EvictCall& c, uint32_t kvh, uint32_t num_blocks, const char* who,
                        bool* todo) {
  *todo = false;
  if (int rc = check_weights(c.in, c.batch, kvh, who)) return rc;
  if (c.out)
    if (int rc = check_weights(c.out, c.batch, kvh, who)) return rc;
  if (c.budget == 0 || (uint64_t)c.sinks + c.recent > c.budget)
    VK_FAIL(VAPI_KV_EINVAL, "%s: a budget of %u keys for %u first and %u last ones", who, c.budget,
            c.sinks, c.recent);
  const uint32_t keep = std::min(c.budget, c.max_len);
  if (c.max_len > c.in->width)
    VK_FAIL(VAPI_KV_EINVAL, "%s: max_len %u exceeds the weights' width %u", who, c.max_len,
            c.in->width);
  if (c.out && keep > c.out->width)
    VK_FAIL(VAPI_KV_EINVAL, "%s: %u kept keys exceed the weights' width %u", who, keep,
            c.out->width);
  if (c.batch == 0 || c.max_len == 0) return 0;
  if (!c.lens || !c.src_table || !c.dst_table || !c.kept)
    VK_FAIL(VAPI_KV_EINVAL, "%s: null device pointer", who);
  if (num_blocks == 0) VK_FAIL(VAPI_KV_EINVAL, "%s: keys in an empty pool", who);
  if (c.src_blocks == 0 || c.dst_blocks == 0)
    VK_FAIL(VAPI_KV_EINVAL, "%s: block table width 0", who);
  if ((uint64_t)c.batch * kvh > 65535 || c.max_len > 0x3FFFFFFFu)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: a batch of %u x %u kv heads of up to %u keys", who, c.batch, kvh,
            c.max_len);
  *todo = true;
  return 0;
}

static void launch_evict_select(const EvictCall& c, uint32_t kvh, hipStream_t s) {
  EvictArgs a{};
  a.in = c.in->data, a.in_index = c.in->index;
  a.in_row = c.in->row_stride, a.in_head = c.in->head_stride;
  a.in_rows = c.in->rows, a.in_width = c.in->width;
  if (c.out) {
    a.out = c.out->data, a.out_index = c.out->index;
    a.out_row = c.out->row_stride, a.out_head = c.out->head_stride;
    a.out_rows = c.out->rows, a.out_width = c.out->width;
  }
  a.lens = c.lens, a.kept = c.kept, a.kvh = kvh, a.max_len = c.max_len;
  a.max_keep = std::min(c.budget, c.max_len);
  a.budget = c.budget, a.sinks = c.sinks, a.recent = c.recent;
  hipLaunchKernelGGL(evict_select, dim3(c.batch * kvh), dim3(kSelectThreads), 0, s, a);
}

static EvictMove evict_move(const EvictCall& c, uint32_t kvh, uint32_t num_blocks,
                            uint32_t block_size) {
  EvictMove m{};
  m.src_table = c.src_table, m.dst_table = c.dst_table, m.kept = c.kept;
  m.src_blocks = c.src_blocks, m.dst_blocks = c.dst_blocks;
  m.num_blocks = num_blocks, m.block_size = block_size, m.bs = FastDiv(block_size);
  m.max_keep = std::min(c.budget, c.max_len), m.kvh = kvh;
  return m;
}

}  // namespace vk

using namespace vk;

extern "C" {

int vapi_kv_evict(const vapi_kv_pool* pool, uint32_t layer, const vapi_kv_weights* in,
                  const vapi_kv_weights* out, const uint32_t* lens, const uint32_t* src_table,
                  uint32_t src_blocks, const uint32_t* dst_table, uint32_t dst_blocks,
                  uint32_t batch, uint32_t max_len, uint32_t budget, uint32_t sinks,
                  uint32_t recent, int32_t* kept, vapi_stream_t stream) {
  const char* who = "vapi_kv_evict";
  if (int rc = check_pool(pool, who)) return rc;
  if (layer >= pool->num_layers)
    VK_FAIL(VAPI_KV_EINVAL, "%s: layer %u of %u", who, layer, pool->num_layers);
  const EvictCall c{in, out, lens, src_table, dst_table, src_blocks, dst_blocks,
                    batch, max_len, budget, sinks, recent, kept};
  bool todo;
  if (int rc = evict_checks(c, pool->num_kv_heads, pool->num_blocks, who, &todo)) return rc;
  if (!todo) return 0;
  const Geom g = make_geom(pool);
  const LayerPtrs p = layer_ptrs(pool, layer);
  const uint32_t elt = (uint32_t)dtype_size(pool->dtype);
  EvictMove m = evict_move(c, g.kvh, g.num_blocks, g.block_size);
  m.k = p.k, m.v = p.v;
  m.blk_b = g.blk * elt, m.head_b = g.head * elt, m.tok_b = g.tok * elt;
  m.row_bytes = g.d * elt;
  const int chunk = chunk_bytes_for(m.row_bytes);
  const uint32_t upr = m.row_bytes / chunk;
  if ((uint64_t)m.max_keep * upr >= 0x7FFFFFFFull)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: %u kept keys of %u bytes", who, m.max_keep, m.row_bytes);
  launch_evict_select(c, g.kvh, hs(stream));
  const dim3 grid((m.max_keep * upr + 255) / 256, batch * g.kvh, pool->v ? 2 : 1);
#define VK_EVICT(C)                                                                       \
  case C:                                                                                 \
    hipLaunchKernelGGL((evict_copy<C>), grid, dim3(256), 0, hs(stream), m, FastDiv(upr)); \
    break
  switch (chunk) {
    VK_EVICT(16);
    VK_EVICT(8);
    VK_EVICT(4);
    VK_EVICT(2);
  }
#undef VK_EVICT
  VK_LAUNCHED(who);
  return 0;
}

int vapi_kv_q8_evict(const vapi_kv_q8_pool* pool, uint32_t layer, const vapi_kv_weights* in,
                     const vapi_kv_weights* out, const uint32_t* lens, const uint32_t* src_table,
                     uint32_t src_blocks, const uint32_t* dst_table, uint32_t dst_blocks,
                     uint32_t batch, uint32_t max_len, uint32_t budget, uint32_t sinks,
                     uint32_t recent, int32_t* kept, vapi_stream_t stream) {
  const char* who = "vapi_kv_q8_evict";
  if (int rc = check_q8_pool(pool, layer, who)) return rc;
  const EvictCall c{in, out, lens, src_table, dst_table, src_blocks, dst_blocks,
                    batch, max_len, budget, sinks, recent, kept};
  bool todo;
  if (int rc = evict_checks(c, pool->num_kv_heads, pool->num_blocks, who, &todo)) return rc;
  if (!todo) return 0;
  const Q8Geom g = q8_geom(pool);
  const Q8Ptrs p = q8_ptrs(pool, layer);
  EvictMove m = evict_move(c, g.kvh, g.num_blocks, g.block_size);
  m.k = p.k, m.v = p.v;
  m.blk_b = g.blk, m.head_b = g.head, m.tok_b = g.tok, m.row_bytes = g.d;
  launch_evict_select(c, g.kvh, hs(stream));
  const uint32_t nb = (m.max_keep + g.block_size - 1) / g.block_size;
  const dim3 grid((nb + kMoveWaves - 1) / kMoveWaves, batch * g.kvh, 2);
  const FastDiv upr(g.d / 16);
  const bool bf16 = pool->dtype == VAPI_KV_BF16, e4m3 = pool->format == VAPI_KV_Q8_E4M3;
#define VK_EVICT(T, F)                                                                       \
  hipLaunchKernelGGL((evict_q8<T, F>), grid, dim3(64 * kMoveWaves), 0, hs(stream), m, upr,   \
                     p.ks, p.vs, g.sblk)
  if (bf16 && e4m3) VK_EVICT(bf16_t, VAPI_KV_Q8_E4M3);
  else if (bf16) VK_EVICT(bf16_t, VAPI_KV_Q8_INT8);
  else if (e4m3) VK_EVICT(f16_t, VAPI_KV_Q8_E4M3);
  else VK_EVICT(f16_t, VAPI_KV_Q8_INT8);
#undef VK_EVICT
  VK_LAUNCHED(who);
  return 0;
}

}  // extern "C"
