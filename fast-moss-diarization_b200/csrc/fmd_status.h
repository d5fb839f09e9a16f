// What a status word that the kernels set means, in words. Host only, no CUDA, so that it
// is tested without a GPU.
#ifndef FMD_STATUS_H
#define FMD_STATUS_H

#include <string>

#include "../../include/fmd_decoder.h"

namespace fmd {

// `site` (TimeoutSite, fmd_common.cuh): the kernel whose wait gave up, or 0.
inline std::string device_status_text(int status, int site) {
  static const char* const kSites[] = {"?", "k_gemv", "k_lm_head", "k_attn_decode_tma", "k_attn_prefill_tc",
                                       "k_gemm_tc", "k_layer_tail", "k_wait_probe", "k_proj_tc", "k_cache_decode",
                                       "k_cache_chunk"};
  constexpr int kNumSites = (int)(sizeof(kSites) / sizeof(kSites[0]));
  const std::string number = " (status " + std::to_string(status) + ")";
  switch (status) {
    case FMD_EIO: return "a greedy pick found no finite logit (non-finite activations)";
    case FMD_EINVAL: return "a slot or page of the KV cache was out of range on the device" + number;
    case FMD_EOVERFLOW: return "a position lay behind the KV cache's pages of its slot on the device" + number;
    case FMD_ETIMEDOUT:
      return std::string("a bounded device-side wait gave up in ") +
             (site >= 1 && site < kNumSites ? kSites[site] : "?") + number;
    default: return "an unknown status word" + number;
  }
}

// Why a step was not run as planned: `cache_error` is empty, or what CUDA said to the launch of
// a cache operator.
inline std::string refusal_text(const std::string& cache_error) {
  return cache_error.empty() ? "a decode projection was not launched (no packed weight tiles or no valid K split)"
                             : "a cache operator was not launched: " + cache_error;
}

}  // namespace fmd

#endif  // FMD_STATUS_H
