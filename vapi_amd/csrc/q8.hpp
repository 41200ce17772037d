// 8-bit pools: geometry, the two formats, and scales that are powers of two.
//
// A scale is 2^e, so every operation here but the final rounding to a code is
// exact: x / s is a multiplication by 2^-e, c * s fits the rows' 16-bit type
// (e4m3 has 4 significant bits, int8 7; the scale's range is cut so that the
// smallest code times the smallest scale is still a value of that type and the
// largest times the largest does not overflow it).
#pragma once

#include "attn_common.hpp"

namespace vk {

constexpr uint32_t kQ8MaxBlockSize = 256;

struct Q8Geom {
  uint32_t num_blocks, block_size, kvh, d;
  uint64_t blk, head;  // strides in codes (bytes) between blocks and kv heads
  uint32_t tok;        // and between tokens of a block
  uint32_t sblk;       // f32 scales between blocks
};

inline Q8Geom q8_geom(const vapi_kv_q8_pool* p) {
  Q8Geom g;
  g.num_blocks = p->num_blocks;
  g.block_size = p->block_size;
  g.kvh = p->num_kv_heads;
  g.d = p->head_dim;
  g.blk = (uint64_t)p->block_size * p->num_kv_heads * p->head_dim;
  const bool hnd = p->layout == VAPI_KV_LAYOUT_HND;
  g.head = hnd ? (uint64_t)p->block_size * p->head_dim : p->head_dim;
  g.tok = hnd ? p->head_dim : p->num_kv_heads * p->head_dim;
  g.sblk = p->scale_block_stride;
  return g;
}

struct Q8Ptrs {
  char *k, *v;
  float *ks, *vs;
};
inline Q8Ptrs q8_ptrs(const vapi_kv_q8_pool* p, uint32_t layer) {
  const uint64_t c = (uint64_t)layer * p->layer_stride_bytes;
  const uint64_t s = (uint64_t)layer * p->scale_layer_stride_bytes;
  return Q8Ptrs{(char*)p->k + c, (char*)p->v + c, (float*)((char*)p->k_scale + s),
                (float*)((char*)p->v_scale + s)};
}

// Checks a descriptor and a layer of it; 0 or an error code with a message.
int check_q8_pool(const vapi_kv_q8_pool* p, uint32_t layer, const char* who);

// ---- formats ------------------------------------------------------------------

// The rows' type T and format F fix the range of a row element (`kBig`: larger
// ones, and infinities, are taken as it) and the smallest scale.
template <typename T, int F>
struct Q8Range;
template <>
struct Q8Range<bf16_t, VAPI_KV_Q8_E4M3> {
  static constexpr float kBig = 1.875f * 0x1p127f, kMinScale = 0x1p-117f;
};
template <>
struct Q8Range<f16_t, VAPI_KV_Q8_E4M3> {
  static constexpr float kBig = 1.875f * 0x1p15f, kMinScale = 0x1p-15f;
};
template <>
struct Q8Range<bf16_t, VAPI_KV_Q8_INT8> {
  static constexpr float kBig = 1.984375f * 0x1p127f, kMinScale = 0x1p-126f;
};
template <>
struct Q8Range<f16_t, VAPI_KV_Q8_INT8> {
  static constexpr float kBig = 1.984375f * 0x1p15f, kMinScale = 0x1p-24f;
};

// A row element as it is stored: NaN as 0, magnitudes up to kBig. (Tests of
// the bits, which hold whatever the compiler assumes of NaN.)
template <typename T, int F>
__device__ __forceinline__ float q8_finite(T x) {
  const float f = to_f32(x);
  const uint32_t mag = __float_as_uint(f) & 0x7fffffffu;
  const float big = Q8Range<T, F>::kBig;
  if (mag > 0x7f800000u) return 0.f;
  return mag > __float_as_uint(big) ? copysignf(big, f) : f;
}

// The bits of kBig in T: magnitudes up to it are stored as they are.
template <typename T, int F>
__device__ __forceinline__ uint32_t q8_big_bits() {
  return from_f32<T>(Q8Range<T, F>::kBig).x;
}

// The least power of two s >= kMinScale with amax / s <= 448 (e4m3), < 128
// (int8); 0 for amax = 0. amax = m 2^E with m in [1, 2): s = 2^(E - 8), or
// 2^(E - 7) where m > 1.75; 2^(E - 6) for int8. Works on the bits of amax;
// subnormal ones give kMinScale.
template <typename T, int F>
__device__ __forceinline__ float q8_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int32_t e = (int32_t)(u >> 23);
  if constexpr (F == VAPI_KV_Q8_E4M3) e = e - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  else e = e - 6;
  const float s = __uint_as_float((uint32_t)max(e, 1) << 23);
  return u == 0 ? 0.f : fmaxf(s, Q8Range<T, F>::kMinScale);
}

// 1 / s for a scale (0 for none, and for what is no scale: NaN, infinities,
// negative or subnormal values a foreign pool may hold).
__device__ __forceinline__ float q8_inverse(float s) {
  const uint32_t e = __float_as_uint(s) >> 23;  // the sign counts: negative ones are past 254
  return e >= 1 && e <= 253 ? __uint_as_float((254u - e) << 23) : 0.f;
}

// Four values already divided by the scale, as codes (to nearest, ties to
// even) in one dword.
template <int F>
__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d) {
  if constexpr (F == VAPI_KV_Q8_E4M3) {
    auto lim = [](float x) { return fminf(fmaxf(x, -448.f), 448.f); };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(lim(a), lim(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(lim(c), lim(d), w, true);
    return (uint32_t)w;
  } else {
    auto one = [](float x) {
      return (uint32_t)(int32_t)fminf(fmaxf(__builtin_rintf(x), -127.f), 127.f) & 0xffu;
    };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
  }
}

// The same where no value needs a limit: magnitudes up to 448, below 127.5.
// (Adding 1.5 2^23 rounds to a whole number, ties to even, in the low bits.)
template <int F>
__device__ __forceinline__ uint32_t q8_pack4_within(float a, float b, float c, float d) {
  if constexpr (F == VAPI_KV_Q8_E4M3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    constexpr float kRound = 12582912.f;
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(b + kRound),
                                              __float_as_uint(a + kRound), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(d + kRound),
                                              __float_as_uint(c + kRound), 0x04000c0cu);
    return lo | hi;
  }
}

// The four codes of a dword as numbers.
template <int F>
__device__ __forceinline__ void q8_unpack4(uint32_t w, float (&x)[4]) {
  if constexpr (F == VAPI_KV_Q8_E4M3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int32_t)(int8_t)(w >> (8 * i));
  }
}

// The four codes of a dword times 2^e `scale`, as two dwords of T (exact).
// e4m3 has one instruction for two codes with their scale.
template <typename T, int F, bool kScaled>
__device__ __forceinline__ uint2 q8_expand4(uint32_t w, float scale) {
  if constexpr (F == VAPI_KV_Q8_E4M3) {
    const float s = kScaled ? scale : 1.f;
    if constexpr (std::is_same_v<T, bf16_t>) {
      return make_uint2(
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false)),
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true)));
    } else {
      return make_uint2(
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false)),
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true)));
    }
  } else {
    float x[4];
    q8_unpack4<F>(w, x);
    if constexpr (kScaled) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= scale;
    }
    return make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
  }
}

}  // namespace vk
