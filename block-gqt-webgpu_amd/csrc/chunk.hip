// Attention of chunks over the paged cache: the launch (the kernel is in
// chunk_kernel.h, its instances in translation units of their own).
#include "chunk.h"

namespace bgtq {

hipError_t launch_chunk_f16_d64(const ChunkParams &p, bool bf16, hipStream_t stream);
hipError_t launch_chunk_f16_d128(const ChunkParams &p, bool bf16, hipStream_t stream);
hipError_t launch_chunk_packed2_d64(const ChunkParams &p, bool bf16, hipStream_t stream);
hipError_t launch_chunk_packed2_d128(const ChunkParams &p, bool bf16, hipStream_t stream);
hipError_t launch_chunk_packed_d64(const ChunkParams &p, bool bf16, hipStream_t stream);
hipError_t launch_chunk_packed_d128(const ChunkParams &p, bool bf16, hipStream_t stream);

int64_t chunk_items(const ChunkParams &p) {
  const int64_t units = (p.tokens * p.group / kChunkColumns + p.sequences) * p.kv_heads;
  return units + (chunk_splits(p.max_length) ? p.target : 0);
}

hipError_t launch_chunk(const ChunkParams &p, int dim, bool bf16, hipStream_t stream) {
  if (!p.packed) return dim == 64 ? launch_chunk_f16_d64(p, bf16, stream) : launch_chunk_f16_d128(p, bf16, stream);
  bool two = true;
  for (int h = 0; h < p.kv_heads; ++h) two &= p.head[h].norm_stride == 2;
  if (two) return dim == 64 ? launch_chunk_packed2_d64(p, bf16, stream) : launch_chunk_packed2_d128(p, bf16, stream);
  return dim == 64 ? launch_chunk_packed_d64(p, bf16, stream) : launch_chunk_packed_d128(p, bf16, stream);
}

}  // namespace bgtq
