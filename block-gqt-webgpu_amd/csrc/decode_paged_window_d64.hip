// Fused decode instances over pages behind a window: structured layouts and FP16 K at d=64.
#include "decode_fast_kernel.h"

namespace bgtq {

hipError_t launch_decode_paged_window_d64(const DecodeParams &p, const FastLayout &fl, int nn, int sg, hipStream_t stream) {
  return launch_family_d64<kKindPagedWindow>(p, fl, nn, sg, stream);
}

}  // namespace bgtq
