// Fused decode instances over pages: structured layouts and FP16 K at d=128.
#include "decode_fast_kernel.h"

namespace bgtq {

hipError_t launch_decode_paged_d128(const DecodeParams &p, const FastLayout &fl, int nn, int sg, hipStream_t stream) {
  return launch_family_d128<kKindPaged>(p, fl, nn, sg, stream);
}

}  // namespace bgtq
