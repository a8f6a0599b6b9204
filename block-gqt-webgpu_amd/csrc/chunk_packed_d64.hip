// Chunk attention, narrow units and rebuilt rows: instances for packed K of any norm stride at d=64.
#include "chunk_rows.h"

namespace bgtq {

hipError_t launch_chunk_packed_d64(const ChunkParams &p, bool bf16, int items, hipStream_t stream) {
  return launch_k<64, 2>(p, bf16, items, stream);
}

}  // namespace bgtq
