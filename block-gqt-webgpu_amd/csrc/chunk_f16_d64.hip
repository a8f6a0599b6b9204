// Chunk attention, narrow units and rebuilt rows: instances for FP16 K at d=64.
#include "chunk_rows.h"

namespace bgtq {

hipError_t launch_chunk_f16_d64(const ChunkParams &p, bool bf16, int items, hipStream_t stream) {
  return launch_k<64, 0>(p, bf16, items, stream);
}

}  // namespace bgtq
