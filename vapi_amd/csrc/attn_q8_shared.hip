// Attention over shared prefixes of an 8-bit pool: the 8-bit decode stream beside tiles
// that expand the nodes' codes on their way into LDS (attn_shared.hpp).
#include "attn_q8.hpp"
#include "attn_shared.hpp"

namespace vk {

// paged_shared_stream over codes, one padded variant for all head dims of a D. 32
// sequences over 5,008 shared keys (e4m3, 32 kv heads of 128) 45.7 us and the merge 5.7,
// 138 MB at 3.0 TB/s; 220 without sharing.
template <typename T, int F, int D, bool kNt>
__global__ __launch_bounds__(kShThreads, D == 256 ? 1 : 2) void q8_shared_stream(AttnArgs a,
                                                                                 SharedArgs sh,
                                                                                 uint32_t nwg) {
  static_assert(kShThreads == 64 * kDecodeWavesPerWG, "one workgroup size");
  extern __shared__ uint32_t plan[];
  if (blockIdx.x < nwg) {
    const Q8Scales sc{sh.ks, sh.vs, sh.sblk};
    q8_stream_body<T, F, D, true, kNt, true, true>(a, sc, a.cu_q, a.cu_k, a.table, plan, blockIdx.x,
                                                   nwg);
  } else {
    sh_range<T, D, true, F>(a, sh, plan, blockIdx.x - nwg);
  }
}

template <typename T, int F>
static void launch_q8_shared_stream(const AttnArgs& a, const SharedArgs& sh, uint32_t D,
                                    uint32_t nwg, uint32_t ranges, hipStream_t s) {
  const size_t lds = shared_lds(a, sh, nwg, ranges);
  const bool once = q8_read_once(a);
#define VK_Q8H(DD)                                                          \
  hipLaunchKernelGGL((once ? q8_shared_stream<T, F, DD, true>               \
                           : q8_shared_stream<T, F, DD, false>),            \
                     dim3(nwg + ranges), dim3(kShThreads), lds, s, a, sh, nwg)
  if (D == 256) VK_Q8H(256);
  else if (D == 128) VK_Q8H(128);
  else VK_Q8H(64);
#undef VK_Q8H
}

void launch_q8_shared(const AttnArgs& a, const SharedArgs& sh, uint32_t head_dim, bool bf16,
                      bool e4m3, bool decode, hipStream_t s) {
  const uint32_t nwg = decode ? a.num_waves / kDecodeWavesPerWG : 0;
  auto launch = [&](uint32_t streams, uint32_t ranges) {
    if (bf16 && e4m3)
      launch_q8_shared_stream<bf16_t, VAPI_KV_Q8_E4M3>(a, sh, head_dim, streams, ranges, s);
    else if (bf16)
      launch_q8_shared_stream<bf16_t, VAPI_KV_Q8_INT8>(a, sh, head_dim, streams, ranges, s);
    else if (e4m3)
      launch_q8_shared_stream<f16_t, VAPI_KV_Q8_E4M3>(a, sh, head_dim, streams, ranges, s);
    else
      launch_q8_shared_stream<f16_t, VAPI_KV_Q8_INT8>(a, sh, head_dim, streams, ranges, s);
  };
  if (head_dim == 256 && decode) {  // one workgroup to a CU: one kind after the other
    launch(nwg, 0);
    launch(0, sh.ranges);
  } else {
    launch(nwg, sh.ranges);
  }
  launch_shared_merge(a, sh, head_dim, bf16, decode, s);
}

}  // namespace vk
