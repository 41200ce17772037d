// Paged attention over 8-bit pools.
//
// Decode rows run the persistent stream of attn_decode.hpp (its plan, shares,
// pieces and merge) with a step of its own: half the bytes per key, so a step
// is twice as many keys and a wave again keeps 16 KiB of K and V in flight.
// Codes go from HBM into registers as they are and become 16-bit MFMA operands
// there; nothing is staged in LDS.
//  * S^T = K Q^T: a lane loads 16 codes of one key row, d = 64 c + 16 g .. +15,
//    which are the 8 + 8 values of two MFMAs' k-group g (Q is laid out to
//    match). Codes enter unscaled: the tile's K scale multiplies the f32
//    scores.
//  * O^T += V^T P^T: a lane loads the D / 16 codes of each of its keys that
//    the 16-bit kernel loads as values, and expands them with the tile's V
//    scale (e4m3: v_cvt_scalef32_pk, two codes and their scale at once; int8 in
//    f16: an f32 product before the conversion; int8 in bf16: the scale goes to
//    P instead, a power of two that moves bf16's exponent only).
// A 16-key tile lies in one block, so its two scales are wave-uniform.
//
// Prefill rows: the codes of the listed sequences are expanded once into the
// workspace as a 16-bit pool, which the 16-bit prefill kernels then read. A
// chunk of 512 queries uses each expanded value 2,048 times (4 query heads a kv
// head); the expansion moves 5 bytes a code (1 in, 2 out, 2 back in).
#include <algorithm>

#include "attn_q8.hpp"
#include "attn_shared.hpp"

namespace vk {

template <typename T, int F, int D, bool kPad, bool kNt, bool kSinks>
__global__ __launch_bounds__(64 * kDecodeWavesPerWG, kDecodeWGsPerCU) void q8_decode_stream(
    AttnArgs a, Q8Scales sc, const uint32_t* __restrict__ cu_q, const uint32_t* __restrict__ cu_k,
    const uint32_t* __restrict__ table) {
  extern __shared__ uint32_t P[];
  q8_stream_body<T, F, D, kPad, kNt, kSinks, false>(a, sc, cu_q, cu_k, table, P, blockIdx.x,
                                                    gridDim.x);
}

// ---- short contexts ------------------------------------------------------------

// Few short rows: paged_decode_small's scheme (a workgroup of 8 waves, 4 at
// head_dim 256, per (sequence, kv head), or n_split of them; steps of 32 keys in
// turn; (m, l, o) joined through LDS in wave order; a split's partials merged by
// the second launch of the 16-bit kernel) over 8-bit steps.
template <int D>
constexpr int q8_small_waves() { return D == 256 ? 4 : 8; }
constexpr uint32_t kQ8SmallPad = 4;  // floats between rows of O in LDS (bank conflicts)

template <typename T, int F, int D, bool kPad, bool kSplit, bool kSinks>
__global__ __launch_bounds__(64 * q8_small_waves<D>(), 1) void q8_decode_small(
    AttnArgs a, Q8Scales sc, const uint32_t* __restrict__ cu_q, const uint32_t* __restrict__ cu_k,
    const uint32_t* __restrict__ table, uint32_t n_split_arg) {
  constexpr int W = q8_small_waves<D>(), DPL = D / 16, KS = 32;
  const uint32_t n_split = kSplit ? n_split_arg : 1u;
  extern __shared__ __attribute__((aligned(16))) float o_lds[];  // [W][group][D + pad]
  __shared__ float2 ml_lds[W][16];
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int32_t wave = (int32_t)__builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t seg = blockIdx.x / n_split, split = blockIdx.x - seg * n_split;
  DecodePos p;
  p.seq = seg / a.kvh;
  p.kh = seg - p.seq * a.kvh;
  p.q0 = cu_q[p.seq];
  p.len_k = (int32_t)(cu_k[p.seq + 1] - cu_k[p.seq]);
  if (cu_q[p.seq + 1] - p.q0 != 1 || p.len_k <= 0) return;
  p.lo = a.wl >= 0 ? max(0, p.len_k - 1 - a.wl) : 0;
  p.fuse = 0, p.seg_first = 0;
  const KeySteps<kSinks> ks(p.lo, p.len_k - 1, a.sinks, KS);
  int32_t at = ks.start, end = ks.last + KS;  // positions of steps
  if constexpr (kSplit) {
    const uint32_t steps = (uint32_t)(end - at) / KS;
    end = at + KS * (int32_t)((split + 1) * steps / n_split);
    at += KS * (int32_t)(split * steps / n_split);
  }
  at += KS * wave;
  p.key0 = ks.key(at);
  float m_run = kNegBig, l_run = 0.f;
  floatx4 o[DPL];
#pragma unroll
  for (int k = 0; k < DPL; ++k) o[k] = floatx4{0.f, 0.f, 0.f, 0.f};
  const uint32_t count = vhead_count(a, p.kh), h0 = vhead_base(a, p.kh);
  const uint32_t hd = kPad ? a.hd : (uint32_t)D;
  if (at < end) {
    Q8Step<D, KS> stA, stB;
    q8_load<D, kPad, true, KS>(stA, a, sc, table, p, col, g);
    const T* qrow =
        (const T*)a.q + ((uint64_t)p.q0 * a.num_heads + h0 + (col < count ? col : 0)) * hd;
    uint4 qf[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint32_t d = 64 * (c / 2) + 16 * g + 8 * (c % 2);
      const uint32_t keep = !kPad || d < hd ? 0xFFFFFFFFu : 0u;
      const uint4 x = *(const uint4*)(qrow + (kPad ? min(d, hd - 8) : d));
      qf[c] = make_uint4((x.x ^ a.q_sign) & keep, (x.y ^ a.q_sign) & keep,
                         (x.z ^ a.q_sign) & keep, (x.w ^ a.q_sign) & keep);
    }
    // The next step on its way while one is computed (a wave's last repeats it).
    auto step = [&](Q8Step<D, KS>& cur, Q8Step<D, KS>& next) __attribute__((always_inline)) {
      const int32_t s0 = p.key0;
      const bool more = at + KS * W < end;
      if (more) at += KS * W, p.key0 = ks.key(at);
      q8_load<D, kPad, true, KS>(next, a, sc, table, p, col, g);
      q8_attend<T, F, D, KS, false, kSinks>(cur, qf, o, m_run, l_run, a.scale_log2, s0, p.lo, p.len_k,
                                      a.sinks, g);
      return more;
    };
    while (step(stA, stB) && step(stB, stA)) {
    }
  }
  constexpr uint32_t S = D + kQ8SmallPad;
  const float l_tot = wave_sum_g(l_run);
  if (g == 0) ml_lds[wave][col] = make_float2(m_run, l_tot);
  if (col < count) {
    float* row = o_lds + ((uint32_t)wave * a.group + col) * S;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < DPL; k += 4)
        *(float4*)(row + v_d<D>(4 * g + i, k)) =
            make_float4(o[k][i], o[k + 1][i], o[k + 2][i], o[k + 3][i]);
  }
  __syncthreads();
  for (uint32_t e = 4 * tid; e < count * D; e += 4 * 64 * W) {
    const uint32_t c = e / D, d = e % D;
    if (kPad && d >= hd) continue;
    float M = kNegBig, L = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, ml_lds[w][c].x);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = fast_exp2(ml_lds[w][c].x - M);
      const float4 y = *(const float4*)(o_lds + ((uint32_t)w * a.group + c) * S + d);
      L += ml_lds[w][c].y * f;
      x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
    }
    if constexpr (kSplit) {
      const uint64_t slot = (uint64_t)blockIdx.x * a.group + c;
      *(float4*)(a.ws_o + slot * D + d) = x;
      if (d == 0) *(float2*)(a.ws_ml + slot * 2) = make_float2(M, L);
    } else {
      const float inv = L > 0.f ? 1.f / L : 0.f;
      T* dst = (T*)a.out + ((uint64_t)p.q0 * a.num_heads + h0 + c) * hd + d;
      *(uint2*)dst = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
    }
  }
}

// ---- prefill: codes expanded into the workspace ----------------------------------

// One block and kv head of a listed sequence: K and V codes to values of T in
// an HND pool whose blocks are (list entry, block of the sequence).
template <typename T, int F>
__global__ __launch_bounds__(256) void q8_expand_kernel(AttnArgs a, Q8Scales sc, T* k_out,
                                                        T* v_out, uint32_t* table_out,
                                                        uint32_t mb) {
  const uint32_t li = blockIdx.x / mb, j = blockIdx.x - li * mb, h = blockIdx.y;
  const uint32_t seq = a.pf_seqs ? a.pf_seqs[li] : li;
  if (seq >= a.batch) return;
  const uint32_t len_q = a.cu_q[seq + 1] - a.cu_q[seq];
  const uint32_t len_k = a.cu_k[seq + 1] - a.cu_k[seq];
  if (len_q < a.pf_min_q || (int32_t)len_k <= 0 || j * a.block_size >= len_k) return;
  // Keys that a left window hides from every query: the prefill reads whole
  // steps of 32 keys, those of the sinks and from the first visible one.
  if (a.wl >= 0 && j * a.block_size >= (((uint32_t)a.sinks + 63) & ~63u) &&
      (int64_t)(j + 1) * a.block_size <= (((int64_t)len_k - len_q - a.wl) & ~(int64_t)63))
    return;
  const uint32_t to = li * mb + j;
  if (h == 0 && threadIdx.x == 0) table_out[(uint64_t)seq * mb + j] = to;
  const uint32_t blk =
      min(a.table[(uint64_t)seq * a.max_blocks + min(j, a.max_blocks - 1)], a.last_blk);
  const uint32_t upr = a.hd / 16, units = a.block_size * upr;
  const float s[2] = {sc.k[(uint64_t)blk * sc.sblk + h], sc.v[(uint64_t)blk * sc.sblk + h]};
  const uint64_t src = blk * a.blk_e + h * a.head_e;
  const uint64_t dst = ((uint64_t)to * gridDim.y + h) * a.block_size * a.hd;
  for (uint32_t i = threadIdx.x; i < 2 * units; i += 256) {
    const bool v = i >= units;
    const uint32_t u = v ? i - units : i;
    const uint32_t off = u / upr, c = u - off * upr;
    const uint4 w = *(const uint4*)((v ? a.v : a.k) + src + (uint64_t)off * a.tok_e + 16 * c);
    const float sv = s[v];
    const uint2 p0 = q8_expand4<T, F, true>(w.x, sv), p1 = q8_expand4<T, F, true>(w.y, sv);
    const uint2 p2 = q8_expand4<T, F, true>(w.z, sv), p3 = q8_expand4<T, F, true>(w.w, sv);
    uint4* out = (uint4*)((v ? v_out : k_out) + dst) + 2 * u;
    out[0] = make_uint4(p0.x, p0.y, p1.x, p1.y);
    out[1] = make_uint4(p2.x, p2.y, p3.x, p3.y);
  }
}

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
static uint32_t q8_dim(uint32_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }
// Virtual kv heads per kv head (attention.hip's rule): ceil(G / 16), 0 past 16.
static uint32_t q8_parts(uint32_t G) {
  const uint32_t n = (G + 15) / 16;
  return n <= 16 ? n : 0;
}

// The workspace of a call with prefill rows past the decode's: a table
// [batch][mb] and the expanded K and V of n_pf sequences of mb blocks.
struct Q8ExpandWs {
  size_t table, k, v, total;
};
static Q8ExpandWs q8_expand_ws(const vapi_kv_q8_pool* p, uint32_t batch, uint32_t n_pf,
                               uint32_t max_k) {
  const size_t mb = ((size_t)max_k + p->block_size - 1) / p->block_size;
  const size_t buf = up256((size_t)n_pf * mb * p->block_size * p->num_kv_heads * p->head_dim * 2);
  Q8ExpandWs w;
  w.table = 0;
  w.k = up256((size_t)batch * mb * sizeof(uint32_t));
  w.v = w.k + buf;
  w.total = w.v + buf;
  return w;
}

static size_t q8_decode_ws(const vapi_kv_q8_pool* p, uint32_t batch, uint32_t num_heads) {
  const uint32_t G = num_heads / p->num_kv_heads, n = q8_parts(G);
  return n ? decode_workspace_bytes(batch, p->num_kv_heads * n, (G + n - 1) / n,
                                    q8_dim(p->head_dim), decode_num_waves())
           : 0;
}

// What a call refuses for its sizes alone: 0 or an error code with a message.
// pf_n: sequences that the prefill covers.
static int q8_check_sizes(const vapi_kv_q8_pool* p, uint32_t num_heads, uint32_t pf_n,
                          uint32_t max_q, uint32_t max_k, const char* who) {
  if (num_heads == 0 || num_heads % p->num_kv_heads)
    VK_FAIL(VAPI_KV_EINVAL, "%s: %u query heads is not a multiple of %u kv heads", who, num_heads,
            p->num_kv_heads);
  const uint32_t G = num_heads / p->num_kv_heads;
  if (!q8_parts(G) || num_heads > 65535)
    VK_FAIL(VAPI_KV_EUNSUP, "%s: %u query heads for %u kv heads", who, num_heads, p->num_kv_heads);
  const uint64_t mb = ((uint64_t)max_k + p->block_size - 1) / p->block_size;
  if (pf_n && (pf_n > 65535 || prefill_grid(pf_n, p->num_kv_heads, G, max_q,
                                            q8_dim(p->head_dim)) > 0xFFFFFFFFull ||
               pf_n * mb > 0xFFFFFFull))
    VK_FAIL(VAPI_KV_EUNSUP, "%s: prefill batch too large for one launch", who);
  return 0;
}

template <typename T, int F, int D>
static void launch_q8_stream_d(const AttnArgs& c, const Q8Scales& sc, uint32_t nwg, size_t lds,
                               hipStream_t s) {
#define VK_Q8S(PAD, NT)                                                                     \
  hipLaunchKernelGGL((c.sinks ? q8_decode_stream<T, F, D, PAD, NT, true>                    \
                              : q8_decode_stream<T, F, D, PAD, NT, false>),                 \
                     dim3(nwg), dim3(64 * kDecodeWavesPerWG), lds, s, c, sc, c.cu_q,        \
                     c.cu_k, c.table)
  const bool pad = c.hd != D, once = q8_read_once(c);
  if (pad && once) VK_Q8S(true, true);
  else if (pad) VK_Q8S(true, false);
  else if (once) VK_Q8S(false, true);
  else VK_Q8S(false, false);
#undef VK_Q8S
}

template <typename T, int F>
static void launch_q8_decode(const AttnArgs& a, const Q8Scales& sc, void* workspace, uint32_t D,
                             hipStream_t s) {
  const uint32_t nwg = a.num_waves / kDecodeWavesPerWG;
  const uint32_t most = decode_max_plan_seqs();
  for (uint32_t b0 = 0; b0 < a.batch; b0 += most) {
    AttnArgs c = a;
    c.batch = std::min(most, a.batch - b0);
    c.cu_q = a.cu_q + b0;
    c.cu_k = a.cu_k + b0;
    c.table = a.table + (uint64_t)b0 * a.max_blocks;
    decode_bind(c, workspace, D);
    const size_t lds = (c.batch + 1) * sizeof(uint32_t);
    if (D == 256) launch_q8_stream_d<T, F, 256>(c, sc, nwg, lds, s);
    else if (D == 128) launch_q8_stream_d<T, F, 128>(c, sc, nwg, lds, s);
    else launch_q8_stream_d<T, F, 64>(c, sc, nwg, lds, s);
    launch_decode_merge(c, nwg, D, std::is_same_v<T, bf16_t>, s,
                        decode_merge_slices(c.group, D));
  }
}

// Whether a call takes the short-context kernel, and into how many workgroups a
// row's keys go, by the bytes of K codes a row has (the host's bound). Measured, 32
// q / 8 kv heads, e4m3, us a call, stream / one workgroup / shares of 32 KiB: 1 x
// 100 keys 12.6 / 9.3 / 9.1, 1 x 700 13.8 / 9.6 / 11.4, 1 x 1,337 14.2 / 13.4 /
// 11.4, 1 x 8,191 17.5 / 60.1 / 12.5, 4 x 2,000 15.0 / 19.6 / 12.6, 16 x 700 16.9 /
// 11.5 / 13.1, 16 x 2,000 23.2 / 22.3 / 19.6, 32 x 300 17.2 / 9.6 / 9.2, 32 x 700
// 20.9 / 13.3 / 13.3 (the first two columns of short rows are the host's time for
// one launch, 9 us, and two, 11). Only the longest row is known here and a share
// of a long one ends after the balanced stream does, hence the largest share.
constexpr uint64_t kQ8SmallWgs = 256;              // workgroups at once, one per CU
constexpr uint64_t kQ8SmallUnsplit = 112ull << 10;  // whole rows up to this
constexpr uint64_t kQ8SmallShare = 32ull << 10;     // else into shares of at least this
constexpr uint64_t kQ8SmallMaxBytes = 128ull << 10;
static size_t q8_small_lds(uint32_t group, uint32_t D) {
  return (size_t)(D == 256 ? 4 : 8) * group * (D + kQ8SmallPad) * sizeof(float);
}
static SmallPlan q8_small_plan(const AttnArgs& a, uint32_t D, uint32_t max_k, size_t part_bytes) {
  const uint64_t seg = (uint64_t)a.batch * a.kvh;
  if (seg > kQ8SmallWgs || q8_small_lds(a.group, D) > 56 * 1024) return {false, 1};
  const int32_t wl = row_window(a.wl, a.sinks);
  const uint64_t span = wl >= 0 ? std::min<uint64_t>(max_k, (uint64_t)wl + 32) : max_k;
  const uint64_t bytes = span * D;
  uint64_t n = 1;
  if (bytes > kQ8SmallUnsplit)
    n = std::max<uint64_t>(
        std::min<uint64_t>(kQ8SmallWgs / seg, (bytes + kQ8SmallShare - 1) / kQ8SmallShare), 1);
  n = std::min<uint64_t>(n, 32);
  while (n > 1 && seg * n * a.group * (D + 2) * sizeof(float) > part_bytes) --n;
  return {bytes <= n * kQ8SmallMaxBytes, (uint32_t)n};
}

template <typename T, int F, int D, bool kPad>
static void launch_q8_small_d(const AttnArgs& a, const Q8Scales& sc, uint32_t n_split,
                              hipStream_t s) {
  const dim3 grid(a.batch * a.kvh * n_split), block(64 * q8_small_waves<D>());
  const size_t lds = q8_small_lds(a.group, D);
  if (n_split > 1)
    hipLaunchKernelGGL((a.sinks ? q8_decode_small<T, F, D, kPad, true, true>
                                : q8_decode_small<T, F, D, kPad, true, false>),
                       grid, block, lds, s, a, sc, a.cu_q, a.cu_k, a.table, n_split);
  else
    hipLaunchKernelGGL((a.sinks ? q8_decode_small<T, F, D, kPad, false, true>
                                : q8_decode_small<T, F, D, kPad, false, false>),
                       grid, block, lds, s, a, sc, a.cu_q, a.cu_k, a.table, 1u);
}
template <typename T, int F>
static void launch_q8_small(const AttnArgs& a_in, const Q8Scales& sc, uint32_t D, uint32_t n_split,
                            void* part, hipStream_t s) {
  AttnArgs a = a_in;
  a.ws_o = (float*)part;
  a.ws_ml = (float*)part + (uint64_t)a.batch * a.kvh * n_split * a.group * D;
  const bool pad = a.hd != D;
  if (D == 256 && pad) launch_q8_small_d<T, F, 256, true>(a, sc, n_split, s);
  else if (D == 256) launch_q8_small_d<T, F, 256, false>(a, sc, n_split, s);
  else if (D == 128 && pad) launch_q8_small_d<T, F, 128, true>(a, sc, n_split, s);
  else if (D == 128) launch_q8_small_d<T, F, 128, false>(a, sc, n_split, s);
  else if (pad) launch_q8_small_d<T, F, 64, true>(a, sc, n_split, s);
  else launch_q8_small_d<T, F, 64, false>(a, sc, n_split, s);
  if (n_split > 1)
    launch_decode_small_merge(a, D, std::is_same_v<T, bf16_t>, n_split, s);
}

template <typename T, int F>
static void launch_q8_expand(const AttnArgs& a, const Q8Scales& sc, char* ws, const Q8ExpandWs& w,
                             uint32_t mb, uint32_t kvh, hipStream_t s) {
  hipLaunchKernelGGL((q8_expand_kernel<T, F>), dim3(a.pf_seqs_n * mb, kvh), dim3(256), 0, s, a,
                     sc, (T*)(ws + w.k), (T*)(ws + w.v), (uint32_t*)(ws + w.table), mb);
}

}  // namespace vk

using namespace vk;

static int q8_attention(const vapi_kv_q8_pool* pool, uint32_t layer, const void* q, void* out,
                        const uint32_t* cu_seqlens_q, const uint32_t* cu_seqlens_k,
                        const uint32_t* block_table, uint32_t batch, uint32_t max_blocks,
                        uint32_t max_seqlen_q, uint32_t max_seqlen_k, uint32_t num_heads,
                        float scale, int32_t window_left, int32_t window_right, uint32_t sinks,
                        uint32_t flags, const uint32_t* prefill_seqs, uint32_t n_prefill,
                        const vapi_kv_prefixes* prefixes, void* workspace, size_t workspace_bytes,
                        vapi_stream_t stream);

extern "C" {

size_t vapi_kv_q8_attention_workspace_size(const vapi_kv_q8_pool* pool, uint32_t batch,
                                           uint32_t n_prefill, uint32_t num_heads,
                                           uint32_t max_seqlen_q, uint32_t max_seqlen_k) {
  const char* who = "vapi_kv_q8_attention_workspace_size";
  n_prefill = max_seqlen_q > 1 ? std::min(n_prefill, batch) : 0;
  max_seqlen_k = std::max(max_seqlen_k, 1u);
  if (check_q8_pool(pool, 0, who) || batch == 0 ||
      q8_check_sizes(pool, num_heads, n_prefill, max_seqlen_q, max_seqlen_k, who))
    return 0;
  size_t need = std::max(up256(q8_decode_ws(pool, batch, num_heads)), (size_t)256);
  if (n_prefill)
    need += q8_expand_ws(pool, batch, n_prefill, max_seqlen_k).total +
            prefill_split_bytes(n_prefill, pool->num_kv_heads, num_heads / pool->num_kv_heads,
                                q8_dim(pool->head_dim), max_seqlen_q, max_seqlen_k);
  return need;
}

int vapi_kv_q8_attention(const vapi_kv_q8_pool* pool, uint32_t layer, const void* q, void* out,
                         const uint32_t* cu_seqlens_q, const uint32_t* cu_seqlens_k,
                         const uint32_t* block_table, uint32_t batch, uint32_t max_blocks,
                         uint32_t max_seqlen_q, uint32_t max_seqlen_k, uint32_t num_heads,
                         float scale, int32_t window_left, int32_t window_right, uint32_t flags,
                         const uint32_t* prefill_seqs, uint32_t n_prefill, void* workspace,
                         size_t workspace_bytes, vapi_stream_t stream) {
  return q8_attention(pool, layer, q, out, cu_seqlens_q, cu_seqlens_k, block_table, batch,
                      max_blocks, max_seqlen_q, max_seqlen_k, num_heads, scale, window_left,
                      window_right, 0, flags, prefill_seqs, n_prefill, nullptr, workspace,
                      workspace_bytes, stream);
}

int vapi_kv_q8_attention_sinks(const vapi_kv_q8_pool* pool, uint32_t layer, const void* q,
                               void* out, const uint32_t* cu_seqlens_q,
                               const uint32_t* cu_seqlens_k, const uint32_t* block_table,
                               uint32_t batch, uint32_t max_blocks, uint32_t max_seqlen_q,
                               uint32_t max_seqlen_k, uint32_t num_heads, float scale,
                               int32_t window_left, int32_t window_right, uint32_t sinks,
                               uint32_t flags, const uint32_t* prefill_seqs, uint32_t n_prefill,
                               void* workspace, size_t workspace_bytes, vapi_stream_t stream) {
  return q8_attention(pool, layer, q, out, cu_seqlens_q, cu_seqlens_k, block_table, batch,
                      max_blocks, max_seqlen_q, max_seqlen_k, num_heads, scale, window_left,
                      window_right, sinks, flags, prefill_seqs, n_prefill, nullptr, workspace,
                      workspace_bytes, stream);
}

size_t vapi_kv_q8_attention_shared_workspace_size(const vapi_kv_q8_pool* pool, uint32_t batch,
                                                  uint32_t n_prefill, uint32_t num_heads,
                                                  uint32_t max_seqlen_q, uint32_t max_seqlen_k,
                                                  const vapi_kv_prefixes* prefixes) {
  const char* who = "vapi_kv_q8_attention_shared_workspace_size";
  n_prefill = max_seqlen_q > 1 ? std::min(n_prefill, batch) : 0;
  max_seqlen_k = std::max(max_seqlen_k, 1u);
  if (check_q8_pool(pool, 0, who) || batch == 0 ||
      q8_check_sizes(pool, num_heads, n_prefill, max_seqlen_q, max_seqlen_k, who) ||
      shared_check(prefixes, batch, pool->num_kv_heads, num_heads / pool->num_kv_heads,
                   q8_dim(pool->head_dim), n_prefill, max_seqlen_q, max_seqlen_k, who))
    return 0;
  const uint32_t kvh = pool->num_kv_heads;
  return std::max(up256(q8_decode_ws(pool, batch, num_heads)), (size_t)256) +
         shared_workspace_bytes(prefixes, batch, kvh, num_heads / kvh, q8_dim(pool->head_dim),
                                n_prefill, max_seqlen_q);
}

int vapi_kv_q8_attention_shared(const vapi_kv_q8_pool* pool, uint32_t layer, const void* q,
                                void* out, const uint32_t* cu_seqlens_q,
                                const uint32_t* cu_seqlens_k, const uint32_t* block_table,
                                uint32_t batch, uint32_t max_blocks, uint32_t max_seqlen_q,
                                uint32_t max_seqlen_k, uint32_t num_heads, float scale,
                                int32_t window_left, int32_t window_right, uint32_t sinks,
                                uint32_t flags, const uint32_t* prefill_seqs, uint32_t n_prefill,
                                const vapi_kv_prefixes* prefixes, void* workspace,
                                size_t workspace_bytes, vapi_stream_t stream) {
  if (!prefixes) VK_FAIL(VAPI_KV_EINVAL, "vapi_kv_q8_attention_shared: null prefixes");
  return q8_attention(pool, layer, q, out, cu_seqlens_q, cu_seqlens_k, block_table, batch,
                      max_blocks, max_seqlen_q, max_seqlen_k, num_heads, scale, window_left,
                      window_right, sinks, flags, prefill_seqs, n_prefill, prefixes, workspace,
                      workspace_bytes, stream);
}

}  // extern "C"

static int q8_attention(const vapi_kv_q8_pool* pool, uint32_t layer, const void* q, void* out,
                        const uint32_t* cu_seqlens_q, const uint32_t* cu_seqlens_k,
                        const uint32_t* block_table, uint32_t batch, uint32_t max_blocks,
                        uint32_t max_seqlen_q, uint32_t max_seqlen_k, uint32_t num_heads,
                        float scale, int32_t window_left, int32_t window_right, uint32_t sinks,
                        uint32_t flags, const uint32_t* prefill_seqs, uint32_t n_prefill,
                        const vapi_kv_prefixes* prefixes, void* workspace, size_t workspace_bytes,
                        vapi_stream_t stream) {
  const char* who = "vapi_kv_q8_attention";
  if (int rc = check_q8_pool(pool, layer, who)) return rc;
  if (num_heads == 0 || num_heads % pool->num_kv_heads)
    VK_FAIL(VAPI_KV_EINVAL, "%s: %u query heads is not a multiple of %u kv heads", who, num_heads,
            pool->num_kv_heads);
  if (n_prefill > batch)
    VK_FAIL(VAPI_KV_EINVAL, "%s: %u prefill sequences in a batch of %u", who, n_prefill, batch);
  if (n_prefill && !prefill_seqs) VK_FAIL(VAPI_KV_EINVAL, "%s: null prefill_seqs", who);
  if (flags & ~(uint32_t)(VAPI_ATTN_DETERMINISTIC | VAPI_ATTN_NO_DECODE_ROWS))
    VK_FAIL(VAPI_KV_EINVAL, "%s: unknown flags 0x%x", who, flags);
  if (batch == 0 || max_seqlen_q == 0) return 0;
  max_seqlen_k = std::max(max_seqlen_k, 1u);  // rows without keys are written all the same
  if (!q || !out || !cu_seqlens_q || !cu_seqlens_k || !block_table)
    VK_FAIL(VAPI_KV_EINVAL, "%s: null device pointer", who);
  if (((uintptr_t)q | (uintptr_t)out) & 15)
    VK_FAIL(VAPI_KV_EINVAL, "%s: q and out must be 16-byte aligned", who);
  if (pool->num_blocks == 0)
    VK_FAIL(VAPI_KV_EINVAL, "%s: keys to attend over in an empty pool", who);
  if (max_blocks == 0) VK_FAIL(VAPI_KV_EINVAL, "%s: block table width 0", who);
  const uint32_t G = num_heads / pool->num_kv_heads, parts = q8_parts(G);
  const uint32_t D = q8_dim(pool->head_dim);
  const bool prefill = max_seqlen_q > 1;
  const bool skip_decode = prefill && (flags & VAPI_ATTN_NO_DECODE_ROWS);
  const bool listed = prefill_seqs && !skip_decode;
  const uint32_t pf_n = !prefill ? 0 : listed ? n_prefill : batch;
  if (int rc = q8_check_sizes(pool, num_heads, pf_n, max_seqlen_q, max_seqlen_k, who)) return rc;
  const uint64_t mb = ((uint64_t)max_seqlen_k + pool->block_size - 1) / pool->block_size;
  const size_t dec_ws =
      skip_decode && !prefixes ? 0 : q8_decode_ws(pool, batch, num_heads);
  const size_t off = std::max(up256(dec_ws), (size_t)256);
  const Q8ExpandWs w = pf_n ? q8_expand_ws(pool, batch, pf_n, max_seqlen_k) : Q8ExpandWs{0, 0, 0, 0};
  size_t need = pf_n ? off + w.total : dec_ws;
  if (prefixes) {
    if (int rc = shared_check(prefixes, batch, pool->num_kv_heads, G, D, pf_n, max_seqlen_q,
                              max_seqlen_k, who))
      return rc;
    need = off + shared_workspace_bytes(prefixes, batch, pool->num_kv_heads, G, D, pf_n,
                                        max_seqlen_q);
  }
  if (workspace_bytes < need || (need && !workspace))
    VK_FAIL(VAPI_KV_ESPACE, "%s: workspace %zu bytes < %zu", who, workspace_bytes, need);

  const Q8Geom g = q8_geom(pool);
  const Q8Ptrs p = q8_ptrs(pool, layer);
  AttnArgs a{};
  a.k = p.k;
  a.v = p.v;
  a.q = (const char*)q;
  a.out = (char*)out;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.table = block_table;
  a.num_slots = g.num_blocks * g.block_size;
  a.last_blk = g.num_blocks - 1;
  a.blk_e = g.blk;
  a.head_e = g.head;
  a.tok_e = g.tok;
  a.max_blocks = max_blocks;
  a.batch = batch;
  a.num_heads = num_heads;
  a.kvh = g.kvh;
  a.group = G;
  a.block_size = g.block_size;
  while ((1u << a.bs_shift) < g.block_size) ++a.bs_shift;
  a.num_waves = decode_num_waves();
  a.scale = scale;
  a.scale_log2 = fmaxf(fabsf(scale) * kLog2e, 1e-30f);
  a.q_sign = scale < 0.f ? 0x80008000u : 0u;
  a.wl = window_arg(window_left);
  a.wr = window_arg(window_right);
  a.sinks = sinks_arg(sinks, a.wl);
  a.deterministic = (flags & VAPI_ATTN_DETERMINISTIC) ? 1u : 0u;
  a.pf_min_q = skip_decode ? 1 : 2;
  a.pf_seqs = listed ? prefill_seqs : nullptr;
  a.pf_seqs_n = pf_n;
  a.pf_order = kPfListOrder;
  a.kv_parts = FastDiv(1);
  a.plan_parts = 1;
  a.g_real = G;
  a.hd = g.d;
  const Q8Scales sc{p.ks, p.vs, g.sblk};
  const hipStream_t s = hs(stream);
  const bool bf16 = pool->dtype == VAPI_KV_BF16, e4m3 = pool->format == VAPI_KV_Q8_E4M3;
#define VK_Q8(FN, ...)                                                  \
  do {                                                                  \
    if (bf16 && e4m3) FN<bf16_t, VAPI_KV_Q8_E4M3>(__VA_ARGS__);         \
    else if (bf16) FN<bf16_t, VAPI_KV_Q8_INT8>(__VA_ARGS__);            \
    else if (e4m3) FN<f16_t, VAPI_KV_Q8_E4M3>(__VA_ARGS__);             \
    else FN<f16_t, VAPI_KV_Q8_INT8>(__VA_ARGS__);                       \
  } while (0)
  AttnArgs dec = a;
  if (parts > 1) {
    dec.kvh = a.kvh * parts;
    dec.group = (G + parts - 1) / parts;
    dec.kv_parts = FastDiv(parts);
    dec.plan_parts = parts;
  } else if (a.sinks) {
    // 24 rows behind a window of 1,000 keys, 32 kv heads of 96: 315 MB read and 60.9 us
    // a head at a time, 161 MB (150 are needed) and 51-53 four at a time.
    dec.plan_parts = line_heads(a, a.hd);
  }
  if (prefixes) {
    dec.shared = prefixes->start;
    decode_bind(dec, workspace, D);
    SharedArgs sh = shared_args(prefixes, dec, D, pf_n, (char*)workspace + off);
    sh.ks = p.ks, sh.vs = p.vs, sh.sblk = g.sblk;
    launch_q8_shared(dec, sh, D, bf16, e4m3, !skip_decode, s);
    VK_LAUNCHED(who);
    return 0;
  }
  if (!skip_decode) {
    // (The partials of a split lie past the balance block, as the stream's.)
    const SmallPlan small = q8_small_plan(dec, D, max_seqlen_k, dec_ws - kDecodeBalanceBytes);
    if (small.ok)
      VK_Q8(launch_q8_small, dec, sc, D, small.n_split, (char*)workspace + kDecodeBalanceBytes, s);
    else
      VK_Q8(launch_q8_decode, dec, sc, workspace, D, s);
  }
  if (pf_n) {
    char* ws = (char*)workspace + off;
    VK_Q8(launch_q8_expand, a, sc, ws, w, (uint32_t)mb, g.kvh, s);
    AttnArgs f = a;  // the expanded pool: HND blocks of the same size, its own table
    f.k = ws + w.k;
    f.v = ws + w.v;
    f.table = (const uint32_t*)(ws + w.table);
    f.max_blocks = (uint32_t)mb;
    f.last_blk = (uint32_t)(pf_n * mb - 1);
    f.tok_e = g.d;
    f.head_e = (uint64_t)g.block_size * g.d;
    f.blk_e = f.head_e * g.kvh;
    const size_t used = off + w.total;
    launch_prefill(f, max_seqlen_q, max_seqlen_k, D, bf16,
                   workspace_bytes > used ? (char*)workspace + used : nullptr,
                   workspace_bytes > used ? workspace_bytes - used : 0, s);
  }
#undef VK_Q8
  VK_LAUNCHED(who);
  return 0;
}
