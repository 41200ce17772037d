// Eviction by running attention weight: which keys of each (sequence, kv head)
// stay, and their rows moved into new blocks.
//
//  1. evict_select: a workgroup per (sequence, kv head) finds the weight of the
//     last key that stays by a radix select on order-preserving keys (a
//     histogram of a digit in LDS), then writes the kept positions in order with
//     their weights. Ties go to the earlier position: a prefix sum numbers those
//     equal to the threshold.
//  2. evict_copy (any pool): 16-byte pieces of K and V rows, from each head's
//     own positions. evict_q8: a wave per (new block, kv head, K or V) takes
//     the rows' codes and scales, finds the block's scale from their largest
//     value and writes the codes under it.
#include <algorithm>

#include "q8.hpp"

namespace vk {

struct EvictArgs {
  const float* in;
  float* out;  // null: weights are not wanted
  const uint32_t *in_index, *out_index, *lens;
  uint64_t in_row, in_head, out_row, out_head;
  uint32_t in_rows, out_rows, out_width;
  int32_t* kept;
  uint32_t kvh, max_len, max_keep, budget, sinks, recent;
};

__device__ __forceinline__ uint32_t evict_len(const EvictArgs& a, uint32_t seq) {
  return a.max_len ? min(a.lens[seq], a.max_len) : 0u;
}

// Weights as unsigned numbers in the same order: NaN lowest, both zeros alike.
__device__ __forceinline__ uint32_t evict_key(float w) {
  const uint32_t u = __float_as_uint(w), mag = u & 0x7fffffffu;
  if (mag > 0x7f800000u) return 0u;
  if (mag == 0) return 0x80000000u;
  return u >> 31 ? ~u : u | 0x80000000u;
}

// The weight of a key (a NaN for a NaN, +0 for either zero).
__device__ __forceinline__ float evict_weight(uint32_t key) {
  return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key);
}

// The sum of x over the lanes up to this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
#define VK_SHIFT(CTRL, ROWS) \
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false)
  VK_SHIFT(0x111, 0xF);  // row_shr:1, 2, 4, 8: within rows of 16 lanes
  VK_SHIFT(0x112, 0xF);
  VK_SHIFT(0x114, 0xF);
  VK_SHIFT(0x118, 0xF);
  VK_SHIFT(0x142, 0xA);  // row_bcast:15 and :31: the rows before
  VK_SHIFT(0x143, 0xC);
#undef VK_SHIFT
  return x;
}

// The sum of x over the threads before this one (in thread order), and over all
// of them; `waves` is LDS of a word a wave. Every thread calls it.
template <uint32_t NT>
__device__ __forceinline__ uint32_t evict_scan(uint32_t x, uint32_t* waves, uint32_t* total) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t run = wave_scan(x);
  __syncthreads();  // the words' last readers
  if (lane == 63) waves[wave] = run;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (uint32_t v = 0; v < NT / 64; ++v) {
    const uint32_t t = waves[v];
    before += v < wave ? t : 0u;
    all += t;
  }
  *total = all;
  return before + run - x;
}

constexpr uint32_t kSelectBins = 1u << 11;
constexpr uint32_t kSelectKeys = 12288;  // keys held in LDS (48 KiB)

// Up to kSelectKeys keys are read once and held in LDS, longer sequences walked in
// tiles of that many. Digits of 11, 11 and 10 bits from the top: three passes, and
// bins that part weights of one magnitude (8-bit digits hold little but the
// exponent, and a wave's adds to one bin queue up). NT threads: 256 for up to
// 4,096 keys, where barriers are most of the time, else 1,024. (Keys in
// registers, 16 a thread, unrolled: 16.8 against 10.9 us for 8 heads of 1,500
// keys; the code is fetched once.)
template <uint32_t NT>
__global__ __launch_bounds__(NT) void evict_select(EvictArgs a) {
  __shared__ uint32_t hist[kSelectBins], waves[NT / 64], found[2], keys[kSelectKeys];
  const uint32_t seq = blockIdx.x / a.kvh, h = blockIdx.x - seq * a.kvh;
  const uint32_t tid = threadIdx.x;
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
  const bool once = len <= kSelectKeys;
  auto load = [&](uint32_t base) {
    const uint32_t count = min(len - base, kSelectKeys);
#pragma unroll 4
    for (uint32_t i = tid; i < count; i += NT) keys[i] = evict_key(w[base + i]);
  };
  if (once) load(0);
  uint32_t threshold = 0, equal = 0xFFFFFFFFu;  // all of them
  if (want == 0) {
    threshold = 0xFFFFFFFFu, equal = 0;
  } else if (want < end - first) {
    // The want-th largest key: digit by digit, `equal` of the keys that share
    // the digits found so far are still wanted.
    uint32_t prefix = 0, mask = 0, shift = 32;
    equal = want;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const uint32_t bits = pass < 2 ? 11 : 10, digit = (1u << bits) - 1;
      shift -= bits;
      for (uint32_t i = tid; i < kSelectBins; i += NT) hist[i] = 0;
      __syncthreads();
      for (uint32_t base = 0; base < len; base += kSelectKeys) {
        if (!once) {
          __syncthreads();
          load(base);
        }
        // (A thread reads the keys that it put there.)
        const uint32_t count = min(len - base, kSelectKeys);
#pragma unroll 2
        for (uint32_t i = tid; i < count; i += NT) {
          const uint32_t key = keys[i], at = base + i;
          if (at >= first && at < end && (key & mask) == prefix)
            atomicAdd(&hist[key >> shift & digit], 1u);
        }
      }
      __syncthreads();
      // A thread's bins, from the largest down.
      constexpr uint32_t kOwn = kSelectBins / NT;
      uint32_t sum = 0;
#pragma unroll
      for (uint32_t j = 0; j < kOwn; ++j) sum += hist[kSelectBins - 1 - kOwn * tid - j];
      uint32_t total;
      uint32_t above = evict_scan<NT>(sum, waves, &total);
      if (above < equal && equal <= above + sum) {
        for (uint32_t j = 0; j < kOwn; ++j) {
          const uint32_t bin = kSelectBins - 1 - kOwn * tid - j, c = hist[bin];
          if (equal <= above + c) {
            found[0] = bin, found[1] = equal - above;
            break;
          }
          above += c;
        }
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= digit << shift;
      equal = found[1];
    }
    threshold = prefix;
  }
  // In order of position: larger ones, and the first `equal` of the equal ones. A
  // thread takes consecutive keys (an odd number, so that no two lanes meet in a
  // bank more often than they must).
  uint32_t eq_before = 0, at = 0;
  for (uint32_t base = 0; base < len; base += kSelectKeys) {
    __syncthreads();
    if (!once) {
      load(base);
      __syncthreads();
    }
    const uint32_t count = min(len - base, kSelectKeys);
    const uint32_t per = (count + NT - 1) / NT | 1u;
    const uint32_t i0 = min(tid * per, count), i1 = min(i0 + per, count);
    uint32_t eq = 0, sure = 0;  // equal to the threshold; taken whatever their rank
    for (uint32_t i = i0; i < i1; ++i) {
      const uint32_t p = base + i;
      const bool mid = p >= first && p < end;
      eq += mid && keys[i] == threshold;
      sure += !mid || keys[i] > threshold;
    }
    uint32_t total, rank = eq_before + evict_scan<NT>(eq, waves, &total);
    eq_before += total;
    // Of this thread's equal ones, those whose rank is below `equal`.
    const uint32_t of_eq = rank < equal ? min(eq, equal - rank) : 0u;
    uint32_t to = at + evict_scan<NT>(sure + of_eq, waves, &total);
    at += total;
    for (uint32_t i = i0; i < i1; ++i) {
      const uint32_t p = base + i, key = keys[i];
      bool take = p < first || p >= end || key > threshold;
      if (!take && key == threshold) take = rank++ < equal;
      // to <= p: with out the same row as in, what is overwritten has been read (the
      // keys in LDS hold the weights).
      if (take && to < a.max_keep) {
        kept[to] = (int32_t)p;
        if (out) out[to] = evict_weight(key);
      }
      to += take;
    }
  }
  for (uint32_t j = n + tid; j < a.max_keep; j += NT) kept[j] = -1;
  if (!out || !ok) return;
  __syncthreads();
  for (uint32_t j = n + tid; j < a.out_width; j += NT) out[j] = 0.f;
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

// Grid: (groups of kCopyRows kept rows a thread, segments, K or V): a thread copies
// one piece of kCopyRows rows, their addresses (kept position, table entry) and
// loads in flight together.
constexpr int kCopyRows = 4;
template <int C>
__global__ __launch_bounds__(256) void evict_copy(EvictMove a, FastDiv upr) {
  using V = typename Chunk<C>::T;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  const uint32_t r = upr.div(i), u = i - r * upr.d;
  const uint32_t seq = blockIdx.y / a.kvh, h = blockIdx.y - seq * a.kvh;
  const int32_t* kept = a.kept + (uint64_t)blockIdx.y * a.max_keep;
  const uint32_t* from = a.src_table + (uint64_t)seq * a.src_blocks;
  const uint32_t* to = a.dst_table + (uint64_t)seq * a.dst_blocks;
  char* base = (blockIdx.z ? a.v : a.k) + h * a.head_b + (uint64_t)u * C;
  // Row k of a thread lies `apart` rows from row k - 1.
  const uint32_t apart = (a.max_keep + kCopyRows - 1) / kCopyRows;
  if (r >= apart) return;
  int32_t pos[kCopyRows];
  uint32_t dst[kCopyRows];
#pragma unroll
  for (int k = 0; k < kCopyRows; ++k) {
    const uint32_t j = r + k * apart, db = a.bs.div(j);
    pos[k] = j < a.max_keep ? kept[j] : -1;
    dst[k] = j < a.max_keep && db < a.dst_blocks ? to[db] : 0xFFFFFFFFu;
  }
  const char* src[kCopyRows];
#pragma unroll
  for (int k = 0; k < kCopyRows; ++k) {
    const uint32_t p = (uint32_t)max(pos[k], 0), sb = a.bs.div(p);
    src[k] = base + min(from[min(sb, a.src_blocks - 1)], a.num_blocks - 1) * a.blk_b +
             (p - sb * a.bs.d) * a.tok_b;
  }
  V v[kCopyRows];
#pragma unroll
  for (int k = 0; k < kCopyRows; ++k) v[k] = load_stream((const V*)src[k]);
#pragma unroll
  for (int k = 0; k < kCopyRows; ++k) {
    const uint32_t j = r + k * apart;
    if (pos[k] >= 0 && dst[k] < a.num_blocks)
      *(V*)(base + dst[k] * a.blk_b + (j - a.bs.div(j) * a.bs.d) * a.tok_b) = v[k];
  }
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
      // A power of two, 1 where the scale stays. (Past 2^20 only rows of zeros
      // have it: a value of theirs would have made the new scale larger.)
      const float by = fminf(s[r] * inv, 0x1p20f);
      uint32_t out[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
      if (__any(by != 1.f)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x[4];
          q8_unpack4<F>(out[e], x);
          out[e] = q8_pack4_within<F>(x[0] * by, x[1] * by, x[2] * by, x[3] * by);
        }
      }
      if (i >= total) continue;
      const uint32_t o = upr.div(i), c = i - o * upr.d;
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
  if (c.batch == 0 || (c.max_len == 0 && !c.out)) return 0;
  // (Without keys nothing is read, kept or moved, but rows of `out` become zeros.)
  if (c.max_len && (!c.lens || !c.src_table || !c.dst_table || !c.kept))
    VK_FAIL(VAPI_KV_EINVAL, "%s: null device pointer", who);
  if (c.max_len && num_blocks == 0) VK_FAIL(VAPI_KV_EINVAL, "%s: keys in an empty pool", who);
  if (c.max_len && (c.src_blocks == 0 || c.dst_blocks == 0))
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
  a.in_rows = c.in->rows;
  if (c.out) {
    a.out = c.out->data, a.out_index = c.out->index;
    a.out_row = c.out->row_stride, a.out_head = c.out->head_stride;
    a.out_rows = c.out->rows, a.out_width = c.out->width;
  }
  a.lens = c.lens, a.kept = c.kept, a.kvh = kvh, a.max_len = c.max_len;
  a.max_keep = std::min(c.budget, c.max_len);
  a.budget = c.budget, a.sinks = c.sinks, a.recent = c.recent;
  if (c.max_len <= 4096)
    hipLaunchKernelGGL((evict_select<256>), dim3(c.batch * kvh), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((evict_select<1024>), dim3(c.batch * kvh), dim3(1024), 0, s, a);
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
  if (c.max_len == 0) {
    VK_LAUNCHED(who);
    return 0;
  }
  const uint32_t rows = (m.max_keep + kCopyRows - 1) / kCopyRows;
  const dim3 grid((rows * upr + 255) / 256, batch * g.kvh, pool->v ? 2 : 1);
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
  if (c.max_len == 0) {
    VK_LAUNCHED(who);
    return 0;
  }
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
