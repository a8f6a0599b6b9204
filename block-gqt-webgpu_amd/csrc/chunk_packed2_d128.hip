// Chunk attention instances: packed K of norm stride 2 at d=128.
#include "chunk_kernel.h"

namespace bgtq {

hipError_t launch_chunk_packed2_d128(const ChunkParams &p, bool bf16, hipStream_t stream) { return launch_k<128, 1>(p, bf16, stream); }

}  // namespace bgtq
