// Chunk attention, narrow units and rebuilt rows: instances for packed K of norm stride 2 at d=64.
#include "chunk_rows.h"

namespace bgtq {

hipError_t launch_chunk_packed2_d64(const ChunkParams &p, bool bf16, int items, hipStream_t stream) {
  return launch_k<64, 1>(p, bf16, items, stream);
}

}  // namespace bgtq
