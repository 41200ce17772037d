// The decode stream over an 8-bit pool: steps of codes and scales, attended as they
// are expanded (the launches are in attn_q8.hip and attn_q8_shared.hip).
#pragma once

#include "attn_decode.hpp"
#include "q8.hpp"

namespace vk {

struct Q8Scales {
  const float *k, *v;  // the layer's
  uint32_t sblk;
};

// Streaming loads where a line is read by one wave only. Parts of one group
// read the same codes side by side (as the 16-bit stream's), and rows of whole
// tokens ([token, head, d]) that are not whole lines share them with the next
// heads' (12 x 2,047 keys, 32 kv heads of 96: 67.0 us streaming, 55.7 cached;
// 64 x 256-8,192 keys at head_dim 128, HND: 76.2 and 83.0).
inline bool q8_read_once(const AttnArgs& a) {
  return a.kv_parts.d == 1 && (a.tok_e == a.hd || a.hd % 128 == 0);
}

// Keys per step: 16 KiB of codes at head_dim 128 and 256.
template <int D>
constexpr int q8_step_keys() { return D == 256 ? 32 : 64; }

template <int D, int kKeys = q8_step_keys<D>()>
struct Q8Step {
  static constexpr int KS = kKeys, NT = KS / 16;
  uint4 k[NT][D / 64];
  uint32_t v[NT][4][D / 64];
  float ks[NT], vs[NT];
};

// Q of the segment's heads as MFMA operands: chunk c holds d = 64 (c / 2) +
// 16 g + 8 (c % 2) .. +7 of lane (col, g).
template <typename T, int D, bool kPad>
__device__ __forceinline__ void q8_load_q(uint4* qs, const AttnArgs& a, const DecodePos& p,
                                          uint32_t lane, uint32_t col, uint32_t g) {
  asm volatile("" : "+v"(lane), "+v"(col), "+v"(g));  // see flush_piece
  const uint32_t h = col < vhead_count(a, p.kh) ? col : 0;
  const uint32_t hd = kPad ? a.hd : (uint32_t)D;
  const T* qrow = (const T*)a.q + ((uint64_t)p.q0 * a.num_heads + vhead_base(a, p.kh) + h) * hd;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    const uint32_t d = 64 * (c / 2) + 16 * g + 8 * (c % 2);
    uint4 x = !kPad || d < hd ? *(const uint4*)(qrow + d) : make_uint4(0u, 0u, 0u, 0u);
    x.x ^= a.q_sign, x.y ^= a.q_sign, x.z ^= a.q_sign, x.w ^= a.q_sign;
    qs[c * 64 + lane] = x;
  }
}

// Codes and scales of the step at p.key0. Every load stays inside a block the
// table names: tiles past the row's last key re-read the tile that holds it and
// keys past it read that key (masked out of the softmax).
template <int D, bool kPad, bool kNt, int KS>
__device__ __forceinline__ void q8_load(Q8Step<D, KS>& st, const AttnArgs& a, const Q8Scales& sc,
                                        const uint32_t* __restrict__ table, const DecodePos& p,
                                        uint32_t col, uint32_t g) {
  using ConstU32 = const __attribute__((address_space(4))) uint32_t;
  using ConstF32 = const __attribute__((address_space(4))) float;
  ConstU32* tab = (ConstU32*)(table + (uint64_t)p.seq * a.max_blocks);
  const uint32_t kh = a.kv_parts.div(p.kh);
  const int32_t last = p.len_k - 1;
#pragma unroll
  for (int tt = 0; tt < KS / 16; ++tt) {
    const int32_t ts = min(p.key0 + 16 * tt, last & ~15);
    const int32_t lim = last - ts;
    const uint32_t blk = min(tab[min((uint32_t)ts >> a.bs_shift, a.max_blocks - 1)], a.last_blk);
    const uint64_t tile = (uint64_t)blk * a.blk_e + kh * a.head_e +
                          (uint64_t)((uint32_t)ts & (a.block_size - 1)) * a.tok_e;
    const uint64_t si = (uint64_t)blk * sc.sblk + kh;
    st.ks[tt] = ((ConstF32*)sc.k)[si];
    st.vs[tt] = ((ConstF32*)sc.v)[si];
    // Every load is unconditional (one under a branch makes the compiler wait
    // for the whole prefetch). Pieces past head_dim repeat the row's last: K's
    // meet zeros of Q, V's make output columns that are not stored (codes are
    // finite).
    const char* kp = a.k + tile + (uint32_t)min((int32_t)col, lim) * a.tok_e;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint32_t d = 64 * c + 16 * g;
      st.k[tt][c] = load_kv<kNt>((const uint4*)(kp + (kPad ? min(d, a.hd - 16) : d)));
    }
    const char* vp = a.v + tile;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const char* row = vp + (uint32_t)min((int32_t)(4 * g + i), lim) * a.tok_e;
      if constexpr (D == 64) {
        const uint32_t d = 4 * col;
        st.v[tt][i][0] = load_kv<kNt>((const uint32_t*)(row + (kPad ? min(d, a.hd - 4) : d)));
      } else {
#pragma unroll
        for (int h = 0; h < D / 128; ++h) {
          const uint32_t d = v_d<D>(col, 8 * h);
          const uint2 w = load_kv<kNt>((const uint2*)(row + (kPad ? min(d, a.hd - 8) : d)));
          st.v[tt][i][2 * h] = w.x, st.v[tt][i][2 * h + 1] = w.y;
        }
      }
    }
  }
}

// One step of the online softmax for 16 query columns (attend_qk and attend_pv
// of the 16-bit kernels, with the tiles' scales). P is rounded to T, whose matrix
// cores multiply it: off by at most half a step, 2^-8 of itself in bf16 and 2^-11
// in f16, which is what V and the output have too; sums and maxima are f32.
// kWhole: maxima are whole numbers, so that where a range of keys begins, which the
// stream's measured shares move from call to call, changes no rounding of P (of
// 64 x 256-8,192 keys 0.03% of the outputs differed between calls, 45% without;
// 74.5 us either way).
// kSinks: keys between the sinks and the window weigh 0, whatever their V and its scale
// hold (st is changed).
template <typename T, int F, int D, int KS, bool kWhole, bool kSinks>
__device__ __forceinline__ void q8_attend(Q8Step<D, KS>& st, const uint4 (&qf)[D / 32],
                                          floatx4 (&o)[D / 16], float& m_run, float& l_run,
                                          float scale_log2, int32_t key0, int32_t lo,
                                          int32_t len_k, int32_t sinks, uint32_t g) {
  constexpr int NT = KS / 16, DPL = D / 16;
  if (kSinks && key0 < lo) {
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
      const int32_t k0 = key0 + 16 * tt;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!row_sees<kSinks>(k0 + 4 * (int32_t)g + i, lo, len_k, sinks))
#pragma unroll
          for (int w = 0; w < D / 64; ++w) st.v[tt][i][w] = 0u;
      // (A tile lies in one block: one that holds a visible key has its scale.)
      if (k0 >= sinks && k0 + 15 < lo) st.vs[tt] = 1.f;
    }
  }
  float s[4 * NT];
  float mx = -INFINITY;
#pragma unroll
  for (int tt = 0; tt < NT; ++tt) {
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 w = st.k[tt][c];
      const uint2 a0 = q8_expand4<T, F, false>(w.x, 1.f), a1 = q8_expand4<T, F, false>(w.y, 1.f);
      const uint2 b0 = q8_expand4<T, F, false>(w.z, 1.f), b1 = q8_expand4<T, F, false>(w.w, 1.f);
      acc = mfma16x16x32<T>(make_uint4(a0.x, a0.y, a1.x, a1.y), qf[2 * c], acc);
      acc = mfma16x16x32<T>(make_uint4(b0.x, b0.y, b1.x, b1.y), qf[2 * c + 1], acc);
    }
    const float by = st.ks[tt] * scale_log2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t key = key0 + 16 * tt + 4 * (int32_t)g + i;
      s[4 * tt + i] = row_sees<kSinks>(key, lo, len_k, sinks) ? acc[i] * by : -INFINITY;
    }
    mx = max_nc(mx, max_nc(max_nc(s[4 * tt], s[4 * tt + 1]), max_nc(s[4 * tt + 2], s[4 * tt + 3])));
  }
  rescale_rows<D, DPL, kWhole>(mx, o, m_run, l_run);
  // int8 codes in bf16: the V scale on P (exact: bf16 has f32's exponents).
  constexpr bool kScaleP = F == VAPI_KV_Q8_INT8 && std::is_same_v<T, bf16_t>;
#pragma unroll
  for (int hh = 0; hh < NT / 2; ++hh) {
    float p[8], ps = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = fast_exp2(s[8 * hh + j] - m_run);
      ps += p[j];
      if constexpr (kScaleP) p[j] *= st.vs[2 * hh + j / 4];
    }
    l_run += ps;
    const uint4 pf = pack8<T>(p);
    VRow<DPL> rows[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int w = 0; w < D / 64; ++w) {
        const uint2 x = q8_expand4<T, F, !kScaleP>(st.v[2 * hh + j / 4][j % 4][w],
                                                   st.vs[2 * hh + j / 4]);
        rows[j].w[2 * w] = x.x, rows[j].w[2 * w + 1] = x.y;
      }
#pragma unroll
    for (int k = 0; k < DPL; ++k) o[k] = mfma16x16x32<T>(vcol<DPL>(rows, k), pf, o[k]);
  }
}

// The stream of workgroup `bid` of `nwg`: decode_stream_body's plan and pieces over 8-bit
// steps, P: batch + 1 words of LDS. (The plan is
// written out here, without the fused append: what changes there changes here.)
template <typename T, int F, int D, bool kPad, bool kNt, bool kSinks, bool kShared>
__device__ __forceinline__ void q8_stream_body(const AttnArgs& a, const Q8Scales& sc,
                                               const uint32_t* __restrict__ cu_q,
                                               const uint32_t* __restrict__ cu_k,
                                               const uint32_t* __restrict__ table, uint32_t* P,
                                               uint32_t bid, uint32_t nwg) {
  constexpr int DPL = D / 16, KS = Q8Step<D>::KS;
  __shared__ uint32_t wave_tot[kDecodeWavesPerWG];
  __shared__ uint4 q_lds[kDecodeWavesPerWG][D / 32 * 64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t B = a.batch;
  const uint32_t n_parts = a.plan_parts, kvh_plan = a.kvh / n_parts;
  const uint32_t t_entry = (uint32_t)__builtin_amdgcn_s_memrealtime();
  {
    constexpr uint32_t NT = 64 * kDecodeWavesPerWG;
    const uint32_t per = (B + NT - 1) / NT;
    const uint32_t b0 = min(tid * per, B), b1 = min(b0 + per, B);
    uint32_t sum = 0;
    for (uint32_t s = b0; s < b1; ++s)
      sum += decode_steps<KS, kSinks, kShared>(a, cu_q, cu_k, s) * kvh_plan;
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(inc, o);
      if (lane >= (uint32_t)o) inc += y;
    }
    if (lane == 63) wave_tot[wave] = inc;
    __syncthreads();
    uint32_t run = inc - sum;
    for (uint32_t w = 0; w < wave; ++w) run += wave_tot[w];
    for (uint32_t s = b0; s < b1; ++s) {
      P[s] = run;
      run += decode_steps<KS, kSinks, kShared>(a, cu_q, cu_k, s) * kvh_plan;
    }
    if (tid == NT - 1) P[B] = run;
    __syncthreads();
  }
  const uint32_t S = __builtin_amdgcn_readfirstlane(P[B]);
  float w[kGroups];
  load_shares(a, nwg, w);
  uint32_t bounds[kGroups + 1];
  group_bounds(w, S, bounds);
  const uint32_t x = bid % kGroups;
  const uint32_t j = (bid / kGroups) * kDecodeWavesPerWG + wave;
  const uint32_t len = bounds[x + 1] - bounds[x];
  const uint32_t nr = min(group_waves(nwg, x) / n_parts, len);
  const uint32_t jr = j / n_parts, part = j - jr * n_parts;
  uint32_t r = jr;
#pragma unroll
  for (uint32_t y = 0; y + 1 < kGroups; ++y)
    r += y < x ? min(group_waves(nwg, y) / n_parts, bounds[y + 1] - bounds[y]) : 0u;
  uint32_t* stat = a.bal + kBalStats + kStatWords * (bid * kDecodeWavesPerWG + wave);
  if (jr >= nr) {
    if (lane == 0) *(uint4*)stat = make_uint4(0u, t_entry, t_entry, 0u);
    return;
  }
  const uint32_t t_begin = bounds[x] + (uint32_t)(((uint64_t)jr * len) / nr);
  const uint32_t t_end = bounds[x] + (uint32_t)(((uint64_t)(jr + 1) * len) / nr);

  uint32_t t = t_begin;
  DecodePos pos =
      locate<KS, kSinks, kShared>(a, cu_q, cu_k, P, nullptr, t, kvh_plan, n_parts, part);
  uint4* qs = q_lds[wave];
  q8_load_q<T, D, kPad>(qs, a, pos, lane, col, g);
  bool piece_first = pos.seg_first;
  float m_run = kNegBig, l_run = 0.f;
  floatx4 o[DPL];
#pragma unroll
  for (int k = 0; k < DPL; ++k) o[k] = floatx4{0.f, 0.f, 0.f, 0.f};
  Q8Step<D> stA, stB;
  q8_load<D, kPad, kNt, KS>(stA, a, sc, table, pos, col, g);

  auto step = [&](Q8Step<D>& cur, Q8Step<D>& next) -> bool {
    const bool more = t + 1 < t_end;
    const bool seg_ends = pos.key0 + KS >= pos.len_k;
    const bool same_piece = more && !seg_ends;
    // (The last step's loads point at one cached row, as in the 16-bit stream.)
    DecodePos nxt = pos;
    if (same_piece) {
      nxt.key0 = next_step<kSinks, KS>(pos.key0, pos.lo, pos.sinks);
      nxt.seg_first = false;
    } else if (more) {
      nxt = next_segment<KS, kSinks, kShared>(a, cu_q, cu_k, P, nullptr, pos, n_parts);
    } else {
      nxt.seq = 0;
      nxt.key0 = 0;
      nxt.len_k = 1;
    }
    q8_load<D, kPad, kNt, KS>(next, a, sc, table, nxt, col, g);
    uint4 qf[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) qf[c] = qs[c * 64 + lane];
    q8_attend<T, F, D, KS, true, kSinks>(cur, qf, o, m_run, l_run, a.scale_log2, pos.key0, pos.lo,
                                         pos.len_k, pos.sinks, g);
    if (!same_piece) {
      const uint32_t seg = pos.seq * a.kvh + pos.kh;
      if (lane == 0) {
        if (piece_first) a.seg_ranges[2 * seg] = r;
        if (seg_ends) a.seg_ranges[2 * seg + 1] = r;
      }
      flush_piece<T, D, kPad>(a, pos, piece_first && seg_ends && !(kShared && pos.shared),
                              stream_slot(n_parts, r, seg), o, m_run, l_run, col, g);
      if (!more) return false;
      m_run = kNegBig;
      l_run = 0.f;
#pragma unroll
      for (int k = 0; k < DPL; ++k) o[k] = floatx4{0.f, 0.f, 0.f, 0.f};
      q8_load_q<T, D, kPad>(qs, a, nxt, lane, col, g);
      piece_first = nxt.seg_first;
    }
    pos = nxt;
    ++t;
    return true;
  };
  while (step(stA, stB) && step(stB, stA)) {
  }
  const uint32_t t_done = (uint32_t)__builtin_amdgcn_s_memrealtime();
  if (lane == 0) *(uint4*)stat = make_uint4(t_end - t_begin, t_entry, t_done, 0u);
}

}  // namespace vk
