// Chunk attention instances: packed K of any norm stride at d=64.
#include "chunk_kernel.h"

namespace bgtq {

hipError_t launch_chunk_packed_d64(const ChunkParams &p, bool bf16, hipStream_t stream) { return launch_k<64, 2>(p, bf16, stream); }

}  // namespace bgtq
