// Fused decode instances over pages behind a window: any packed layout at d=128.
#include "decode_fast_kernel.h"

namespace bgtq {

hipError_t launch_decode_paged_window_any128(const DecodeParams &p, const FastLayout &fl, hipStream_t stream) {
  return launch_family_any<kKindPagedWindow, 128>(p, fl, stream);
}

}  // namespace bgtq
