// 8-bit pools: the append, which picks and grows the blocks' scales, the
// gather, and the descriptor's checks.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "q8.hpp"

namespace vk {

int check_q8_pool(const vapi_kv_q8_pool* p, uint32_t layer, const char* who) {
  if (!p) VK_FAIL(VAPI_KV_EINVAL, "%s: null pool", who);
  if (p->format != VAPI_KV_Q8_E4M3 && p->format != VAPI_KV_Q8_INT8)
    VK_FAIL(VAPI_KV_EINVAL, "%s: unknown 8-bit format %u", who, p->format);
  if (dtype_size(p->dtype) == 0) VK_FAIL(VAPI_KV_EINVAL, "%s: unknown dtype %u", who, p->dtype);
  if (p->layout != VAPI_KV_LAYOUT_HND && p->layout != VAPI_KV_LAYOUT_NHD)
    VK_FAIL(VAPI_KV_EINVAL, "%s: unknown layout %u", who, p->layout);
  if (p->num_layers == 0 || p->block_size == 0 || p->num_kv_heads == 0 || p->head_dim == 0)
    VK_FAIL(VAPI_KV_EINVAL,
            "%s: empty pool geometry (layers %u, block_size %u, kv_heads %u, head_dim %u)", who,
            p->num_layers, p->block_size, p->num_kv_heads, p->head_dim);
  if (layer >= p->num_layers)
    VK_FAIL(VAPI_KV_EINVAL, "%s: layer %u of %u", who, layer, p->num_layers);
  if (p->dtype == VAPI_KV_F32)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: an 8-bit pool's rows are f16 or bf16", who);
  if (p->head_dim % 16 || p->head_dim > 256)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: head_dim %u is not a multiple of 16 up to 256", who, p->head_dim);
  if (p->block_size < 16 || p->block_size > kQ8MaxBlockSize ||
      (p->block_size & (p->block_size - 1)))
    VK_FAIL(VAPI_KV_EUNSUP, "%s: block_size %u is not a power of two from 16 to %u", who,
            p->block_size, kQ8MaxBlockSize);
  if (p->num_kv_heads > 65535)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: %u kv heads", who, p->num_kv_heads);
  if ((uint64_t)p->num_blocks * p->block_size >= 0xFFFFFFFFull)
    VK_FAIL(VAPI_KV_EINVAL, "%s: %u blocks of %u slots overflow u32 slots", who, p->num_blocks,
            p->block_size);
  if (p->scale_block_stride < p->num_kv_heads)
    VK_FAIL(VAPI_KV_EINVAL, "%s: %u scales a block for %u kv heads", who, p->scale_block_stride,
            p->num_kv_heads);
  const uint64_t codes =
      (uint64_t)p->num_blocks * p->block_size * p->num_kv_heads * p->head_dim;
  const uint64_t scales = (uint64_t)p->num_blocks * p->scale_block_stride * sizeof(float);
  if (p->num_layers > 1 &&
      (p->layer_stride_bytes < codes || p->scale_layer_stride_bytes < scales))
    VK_FAIL(VAPI_KV_EINVAL, "%s: layer strides %llu and %llu < layer sizes %llu and %llu", who,
            (unsigned long long)p->layer_stride_bytes,
            (unsigned long long)p->scale_layer_stride_bytes, (unsigned long long)codes,
            (unsigned long long)scales);
  if (p->num_blocks > 0 && (!p->k || !p->v || !p->k_scale || !p->v_scale))
    VK_FAIL(VAPI_KV_EINVAL, "%s: null pool pointer", who);
  if (((uintptr_t)p->k | (uintptr_t)p->v) & 15)
    VK_FAIL(VAPI_KV_EINVAL, "%s: K/V base pointers must be 16-byte aligned", who);
  if (((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) & 3)
    VK_FAIL(VAPI_KV_EINVAL, "%s: scale pointers must be 4-byte aligned", who);
  if (p->num_layers > 1 && ((p->layer_stride_bytes & 15) || (p->scale_layer_stride_bytes & 3)))
    VK_FAIL(VAPI_KV_EINVAL, "%s: layer strides %llu and %llu are not multiples of 16 and 4 bytes",
            who, (unsigned long long)p->layer_stride_bytes,
            (unsigned long long)p->scale_layer_stride_bytes);
  return 0;
}

// ---- append -------------------------------------------------------------------
//
// A block's scale depends on all the rows a call puts into it, so the unit of
// work is a (block, kv head, K or V) and a wave does one: it finds the block's
// tokens, reads their rows (16 bytes a lane) into registers, reduces their
// largest magnitude, settles the scale and writes the codes; where the scale
// grew it also re-rounds the rows that were there. The unit is owned by the
// wave, so nothing is atomic and the order of waves changes nothing.
//
// The unit belongs to the first of the block's tokens (its leader: the token
// before it, skipped ones aside, lies in another block). A workgroup looks at
// `chunk` tokens; its waves and those of the grid's y dimension share the
// units of the leaders among them.
//
// 4,096 rows of 8 x 128 in runs of 256 (24 MB read and written): 10.5 us, 2.3
// TB/s; what bounds it is the chain slot -> rows -> largest magnitude -> codes of
// one unit a wave, ~5 us with the launch, and the VALU's ~5 operations a value.

struct Q8AppendArgs {
  const char* src[2];  // K, V rows
  char* dst[2];
  float* scale[2];
  const uint32_t* slots;
  uint32_t n, chunk, num_slots, bs_shift, kvh, d;
  uint64_t blk, head;
  uint32_t tok, sblk;
  FastDiv upr;  // 8-element pieces of a row
};

constexpr uint32_t kAppendWaves = 4;
constexpr int kAppendRegs = 4;  // pieces a lane holds: a block of 16 x 128 in one go

template <typename T, int F>
__global__ __launch_bounds__(64 * kAppendWaves) void q8_append_kernel(Q8AppendArgs a) {
  __shared__ int32_t row_of[kAppendWaves][kQ8MaxBlockSize];
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int32_t* const rows = row_of[wave];
  const uint32_t bs = 1u << a.bs_shift;
  const uint32_t t0 = blockIdx.x * a.chunk;
  // The blocks of the 64 tokens from the first of this workgroup's on, and of the
  // 64 before (none: skipped, or past the pool).
  constexpr uint32_t kNone = 0xFFFFFFFFu;
  auto block_of = [&](uint32_t s) { return s < a.num_slots ? s >> a.bs_shift : kNone; };
  auto slot_at = [&](uint32_t t) { return t < a.n ? a.slots[t] : kNone; };
  const uint32_t slot = slot_at(t0 + lane);
  uint32_t back = block_of(lane < t0 ? a.slots[t0 - 1 - lane] : kNone);
  const uint32_t mine = block_of(slot);
  const uint64_t valid = __ballot(mine != kNone);
  const uint64_t own = a.chunk >= 64 ? ~0ull : (1ull << a.chunk) - 1;
  if ((valid & own) == 0) return;
  // The last valid token before this workgroup's.
  uint32_t before = kNone;
  for (uint32_t end = t0;;) {
    const uint64_t m = __ballot(back != kNone);
    if (m) before = __builtin_amdgcn_readlane(back, (uint32_t)__builtin_ctzll(m));
    if (m || end <= 64) break;
    end -= 64;
    back = block_of(lane < end ? a.slots[end - 1 - lane] : kNone);
  }
  const uint64_t below = valid & ((1ull << lane) - 1);
  const uint32_t prev = (uint32_t)__shfl((int)mine, below ? 63 - __builtin_clzll(below) : 0);
  uint64_t leaders = own & __ballot(mine != kNone && mine != (below ? prev : before));

  const uint32_t units = 2 * a.kvh;
  const uint32_t waves = gridDim.y * kAppendWaves;
  uint32_t u = blockIdx.y * kAppendWaves + wave;  // the unit among the leader's
  while (leaders) {
    const uint32_t li = (uint32_t)__builtin_ctzll(leaders);
    if (u >= units) {  // this wave's next unit is a later leader's
      u -= units;
      leaders &= leaders - 1;
      continue;
    }
    const uint32_t blk = __builtin_amdgcn_readlane(mine, li);
    // Which token brings each slot of the block (-1: none of this call's).
    for (uint32_t o = lane; o < bs; o += 64) rows[o] = -1;
    wait_lds();
    uint32_t sl = slot;
    uint64_t from = ~0ull << li;  // the window's tokens from the leader on
    for (uint32_t t = t0;;) {
      const uint32_t bl = block_of(sl);
      const uint64_t other = __ballot(bl != kNone && bl != blk) & from;
      if (bl == blk && (from >> lane & 1) && !(other & ((1ull << lane) - 1)))
        rows[sl & (bs - 1)] = (int32_t)(t + lane);
      t += 64;
      if (other || t >= a.n) break;
      sl = slot_at(t + lane);
      from = ~0ull;
    }
    wait_lds();
    const bool fresh = __builtin_amdgcn_readfirstlane(rows[0]) >= 0;
    for (; u < units; u += waves) {
      const uint32_t h = u >> 1, kv = u & 1;
      const T* src = (const T*)a.src[kv] + (uint64_t)h * a.d;
      char* dst = a.dst[kv] + blk * a.blk + h * a.head;
      float* sp = a.scale[kv] + (uint64_t)blk * a.sblk + h;
      const uint32_t total = bs * a.upr.d;
      const float held = *sp;
      // A scale no append wrote (NaN, a negative value) counts as none.
      const float s_old = fresh || q8_inverse(held) == 0.f ? 0.f : held;
      uint4 x[kAppendRegs];
      auto load = [&](uint32_t base) {
#pragma unroll
        for (int j = 0; j < kAppendRegs; ++j) {
          const uint32_t i = base + 64 * j + lane;
          x[j] = make_uint4(0u, 0u, 0u, 0u);
          if (i < total) {
            const uint32_t o = a.upr.div(i), c = i - o * a.upr.d;
            const int32_t t = rows[o];
            if (t >= 0) x[j] = *(const uint4*)(src + (uint64_t)t * a.kvh * a.d + 8 * c);
          }
        }
      };
      // An element as it is (two to a word), and as it is stored where some are
      // not numbers the format holds.
      auto raw = [](const uint4& v, int e) {
        const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
        return T{(uint16_t)(e & 1 ? w >> 16 : w & 0xffffu)};
      };
      // The largest magnitude: the bits of magnitudes order as they do.
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 most = {0, 0};
      for (uint32_t base = 0; base < total; base += 64 * kAppendRegs) {
        load(base);
#pragma unroll
        for (int j = 0; j < kAppendRegs; ++j) {
          const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
        }
      }
      uint32_t top = wave_reduce((uint32_t)max(most[0], most[1]),
                                 [](uint32_t p, uint32_t q) { return max(p, q); });
      // NaN, infinities and what rounds past the format's range are rare: such a
      // unit takes the long way round.
      const bool odd = top > q8_big_bits<T, F>();
      if (odd) {
        uint32_t big = 0;
        for (uint32_t base = 0; base < total; base += 64 * kAppendRegs) {
          if (total > 64 * kAppendRegs) load(base);
#pragma unroll
          for (int j = 0; j < kAppendRegs; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              big = max(big, __float_as_uint(q8_finite<T, F>(raw(x[j], e))) & 0x7fffffffu);
        }
        top = wave_reduce(big, [](uint32_t p, uint32_t q) { return max(p, q); });
      } else {
        top = __float_as_uint(to_f32(T{(uint16_t)top}));
      }
      const float s = fmaxf(s_old, q8_scale<T, F>(__uint_as_float(top)));
      const float inv = q8_inverse(s);
      const bool slow = odd || (F == VAPI_KV_Q8_INT8 && __uint_as_float(top) * inv >= 127.5f);
      // Rows of earlier calls: 0 in a block that starts here, shifted where
      // the scale grew, untouched otherwise.
      const bool rest = fresh || s != s_old;
      const float shift = s_old * inv;
      const bool again = total > 64 * kAppendRegs;  // the registers hold the last part only
      for (uint32_t base = 0; base < total; base += 64 * kAppendRegs) {
        if (again) load(base);
#pragma unroll
        for (int j = 0; j < kAppendRegs; ++j) {
          const uint32_t i = base + 64 * j + lane;
          if (i >= total) continue;
          const uint32_t o = a.upr.div(i), c = i - o * a.upr.d;
          uint2* p = (uint2*)(dst + (uint64_t)o * a.tok + 8 * c);
          if (rows[o] >= 0) {
            float v[8];
            if (slow) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = q8_finite<T, F>(raw(x[j], e)) * inv;
              *p = make_uint2(q8_pack4<F>(v[0], v[1], v[2], v[3]),
                              q8_pack4<F>(v[4], v[5], v[6], v[7]));
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = to_f32(raw(x[j], e)) * inv;
              *p = make_uint2(q8_pack4_within<F>(v[0], v[1], v[2], v[3]),
                              q8_pack4_within<F>(v[4], v[5], v[6], v[7]));
            }
          } else if (rest) {
            uint2 w = make_uint2(0u, 0u);
            if (shift > 0.f) {
              w = *p;
              float lo[4], hi[4];
              q8_unpack4<F>(w.x, lo);
              q8_unpack4<F>(w.y, hi);
              w = make_uint2(
                  q8_pack4<F>(lo[0] * shift, lo[1] * shift, lo[2] * shift, lo[3] * shift),
                  q8_pack4<F>(hi[0] * shift, hi[1] * shift, hi[2] * shift, hi[3] * shift));
            }
            *p = w;
          }
        }
      }
      if (lane == 0) *sp = s;
    }
    u -= units;
    leaders &= leaders - 1;
  }
}

// ---- gather -------------------------------------------------------------------

struct Q8GatherArgs {
  const char* src[2];
  const float* scale[2];
  char* out[2];
  const uint32_t* table;
  uint32_t n_table, num_blocks, bs_shift;
  uint64_t total;  // 16-element pieces of one tensor
  FastDiv upr, kvh;
  uint64_t blk, head;
  uint32_t tok, sblk;
};

// A thread expands 16 codes (16 bytes in, 32 out); y picks K or V.
template <typename T, int F>
__global__ __launch_bounds__(256) void q8_gather_kernel(Q8GatherArgs a, int first) {
  const int kv = first + (int)blockIdx.y;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.total) return;
  const uint32_t r = a.upr.div((uint32_t)i), c = (uint32_t)i - r * a.upr.d;
  const uint32_t pos = a.kvh.div(r), h = r - pos * a.kvh.d;
  const uint32_t blk = a.table[min(pos >> a.bs_shift, a.n_table - 1)];
  uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
  if (blk < a.num_blocks) {
    const uint32_t off = pos & ((1u << a.bs_shift) - 1);
    const uint4 w = load_stream(
        (const uint4*)(a.src[kv] + blk * a.blk + h * a.head + (uint64_t)off * a.tok + 16 * c));
    const float s = a.scale[kv][(uint64_t)blk * a.sblk + h];
    const uint2 p0 = q8_expand4<T, F, true>(w.x, s), p1 = q8_expand4<T, F, true>(w.y, s);
    const uint2 p2 = q8_expand4<T, F, true>(w.z, s), p3 = q8_expand4<T, F, true>(w.w, s);
    lo = make_uint4(p0.x, p0.y, p1.x, p1.y);
    hi = make_uint4(p2.x, p2.y, p3.x, p3.y);
  }
  uint4* out = (uint4*)a.out[kv] + 2 * i;
  out[0] = lo;
  out[1] = hi;
}

}  // namespace vk

using namespace vk;

#define VK_Q8_DISPATCH(pool, CALL)                                           \
  do {                                                                       \
    if ((pool)->dtype == VAPI_KV_BF16) {                                     \
      if ((pool)->format == VAPI_KV_Q8_E4M3) CALL(bf16_t, VAPI_KV_Q8_E4M3);  \
      else CALL(bf16_t, VAPI_KV_Q8_INT8);                                    \
    } else {                                                                 \
      if ((pool)->format == VAPI_KV_Q8_E4M3) CALL(f16_t, VAPI_KV_Q8_E4M3);   \
      else CALL(f16_t, VAPI_KV_Q8_INT8);                                     \
    }                                                                        \
  } while (0)

static uint32_t log2_of(uint32_t x) {
  uint32_t s = 0;
  while ((1u << s) < x) ++s;
  return s;
}

extern "C" {

int vapi_kv_q8_append(const vapi_kv_q8_pool* pool, uint32_t layer, const void* k_src,
                      const void* v_src, const uint32_t* slot_mapping, uint32_t n_tokens,
                      vapi_stream_t stream) {
  if (int rc = check_q8_pool(pool, layer, "vapi_kv_q8_append")) return rc;
  if (n_tokens == 0 || pool->num_blocks == 0) return 0;
  if (!k_src || !v_src || !slot_mapping)
    VK_FAIL(VAPI_KV_EINVAL, "vapi_kv_q8_append: null source or slot_mapping");
  if (((uintptr_t)k_src | (uintptr_t)v_src) & 15)
    VK_FAIL(VAPI_KV_EINVAL, "vapi_kv_q8_append: k_src and v_src must be 16-byte aligned");
  if (n_tokens > 0xFFFFFFFu)  // 2^32 threads in a grid
    VK_FAIL(VAPI_KV_EUNSUP, "vapi_kv_q8_append: %u tokens in one call", n_tokens);
  const Q8Geom g = q8_geom(pool);
  const Q8Ptrs p = q8_ptrs(pool, layer);
  Q8AppendArgs a;
  a.src[0] = (const char*)k_src, a.src[1] = (const char*)v_src;
  a.dst[0] = p.k, a.dst[1] = p.v;
  a.scale[0] = p.ks, a.scale[1] = p.vs;
  a.slots = slot_mapping;
  a.n = n_tokens;
  a.num_slots = g.num_blocks * g.block_size;
  a.bs_shift = log2_of(g.block_size);
  a.kvh = g.kvh, a.d = g.d;
  a.blk = g.blk, a.head = g.head, a.tok = g.tok, a.sblk = g.sblk;
  a.upr = FastDiv(g.d / 8);
  // Tokens a workgroup looks at. Few tokens are mostly single ones of decode rows,
  // a unit each (64 tokens, 8 kv heads: 7.4 us one to a workgroup, 9.5 at four);
  // many are runs, where a workgroup without a leader is launched for nothing
  // (4,096 tokens in runs of 256: 30.1 / 15.0 / 12.5 / 10.5 us at 1 / 4 / 8 / 16;
  // 4,096 single ones 40.8 / 37.1 / 41.2 / 44.1; 512 in runs 8.3 / 7.7 / 7.6 / 7.7).
  a.chunk = n_tokens <= 256 ? 1 : n_tokens <= 1024 ? 4 : 16;
  const uint32_t y = std::min((2 * g.kvh + kAppendWaves - 1) / kAppendWaves, 65535u);
  const dim3 grid((n_tokens + a.chunk - 1) / a.chunk, y);
#define VK_APPEND(T, F)                                                                     \
  hipLaunchKernelGGL((q8_append_kernel<T, F>), grid, dim3(64 * kAppendWaves), 0, hs(stream), a)
  VK_Q8_DISPATCH(pool, VK_APPEND);
#undef VK_APPEND
  VK_LAUNCHED("q8_append_kernel");
  return 0;
}

int vapi_kv_q8_gather(const vapi_kv_q8_pool* pool, uint32_t layer, const uint32_t* block_table,
                      uint32_t n_table, uint32_t len_k, void* k_out, void* v_out,
                      vapi_stream_t stream) {
  if (int rc = check_q8_pool(pool, layer, "vapi_kv_q8_gather")) return rc;
  if (len_k > (uint64_t)n_table * pool->block_size)
    VK_FAIL(VAPI_KV_EINVAL, "vapi_kv_q8_gather: len_k %u exceeds %u blocks of %u", len_k, n_table,
            pool->block_size);
  if (len_k == 0 || (!k_out && !v_out)) return 0;
  if (!block_table) VK_FAIL(VAPI_KV_EINVAL, "vapi_kv_q8_gather: null block table");
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15)
    VK_FAIL(VAPI_KV_EINVAL, "vapi_kv_q8_gather: k_out and v_out must be 16-byte aligned");
  const Q8Geom g = q8_geom(pool);
  const Q8Ptrs p = q8_ptrs(pool, layer);
  Q8GatherArgs a;
  a.src[0] = p.k, a.src[1] = p.v;
  a.scale[0] = p.ks, a.scale[1] = p.vs;
  a.out[0] = (char*)k_out, a.out[1] = (char*)v_out;
  a.table = block_table;
  a.n_table = n_table;
  a.num_blocks = g.num_blocks;
  a.bs_shift = log2_of(g.block_size);
  a.upr = FastDiv(g.d / 16);
  a.kvh = FastDiv(g.kvh);
  a.blk = g.blk, a.head = g.head, a.tok = g.tok, a.sblk = g.sblk;
  a.total = (uint64_t)len_k * g.kvh * (g.d / 16);
  if (a.total >= 0x7FFFFFFFull)  // FastDiv's range
    VK_FAIL(VAPI_KV_EUNSUP, "vapi_kv_q8_gather: %u keys in one call", len_k);
  const dim3 grid((uint32_t)((a.total + 255) / 256), k_out && v_out ? 2 : 1);
  const int first = k_out ? 0 : 1;
#define VK_GATHER(T, F) \
  hipLaunchKernelGGL((q8_gather_kernel<T, F>), grid, dim3(256), 0, hs(stream), a, first)
  VK_Q8_DISPATCH(pool, VK_GATHER);
#undef VK_GATHER
  VK_LAUNCHED("q8_gather_kernel");
  return 0;
}

}  // extern "C"
