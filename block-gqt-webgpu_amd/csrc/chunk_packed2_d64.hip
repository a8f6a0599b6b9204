// Chunk attention instances: packed K of norm stride 2 at d=64.
#include "chunk_kernel.h"

namespace bgtq {

hipError_t launch_chunk_packed2_d64(const ChunkParams &p, bool bf16, hipStream_t stream) { return launch_k<64, 1>(p, bf16, stream); }

}  // namespace bgtq
