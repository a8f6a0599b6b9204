// Attention of chunks over the paged cache: what a call launches.
#include <algorithm>

#include "chunk.h"

namespace bgtq {

hipError_t launch_chunk_f16_d64(const ChunkParams &p, bool bf16, int items, hipStream_t stream);
hipError_t launch_chunk_f16_d128(const ChunkParams &p, bool bf16, int items, hipStream_t stream);
hipError_t launch_chunk_packed2_d64(const ChunkParams &p, bool bf16, int items, hipStream_t stream);
hipError_t launch_chunk_packed2_d128(const ChunkParams &p, bool bf16, int items, hipStream_t stream);
hipError_t launch_chunk_packed_d64(const ChunkParams &p, bool bf16, int items, hipStream_t stream);
hipError_t launch_chunk_packed_d128(const ChunkParams &p, bool bf16, int items, hipStream_t stream);
hipError_t launch_chunk_wide(const ChunkParams &p, int dim, bool bf16, int items, hipStream_t stream);
hipError_t launch_chunk_merge(const ChunkParams &p, int dim, bool bf16, int tile, int slots, hipStream_t stream);

ChunkPlan plan_chunks(const ChunkParams &p, int dim, bool packed, bool q8, bool bf16, int cus) {
  ChunkPlan c{};
  c.split = packed && !bf16;
  const int64_t columns = p.tokens * p.group, S = p.sequences, H = p.kv_heads;
  const int64_t blocks = (p.max_length + kChunkKeys - 1) / kChunkKeys;
  // (units that cost no more than the least item are never split: find_item)
  const bool narrow_splits = kChunkSetup + kChunkNarrow * blocks > kChunkLeastNarrow, wide_splits = kChunkSetup + kChunkWide * blocks > kChunkLeast;
  c.narrow_aim = cus;
  const bool all_narrow = columns <= kChunkSmall;
  // (as many workgroups as units and splits can be: those without an item are ahead of the rebuilding ones)
  const int64_t narrow_units = (S + (all_narrow ? columns / 32 : 0)) * H;
  const int64_t narrow_blocks = p.window ? std::min(blocks, ((int64_t)p.window + 34 + p.sinks) / kChunkKeys + 3) : blocks;
  const int64_t most_splits = std::max<int64_t>(1, (kChunkSetup + kChunkNarrow * narrow_blocks + kChunkLeastNarrow - 1) / kChunkLeastNarrow);
  c.narrow_items = std::min(narrow_units + (narrow_splits ? c.narrow_aim : 0), narrow_units * most_splits);
  const int64_t narrow_bytes = narrow_splits ? 2 * (int64_t)c.narrow_aim * 32 * (dim + 2) * 4 : 0;
  c.part_bytes = narrow_bytes;
  c.wide_sequences = all_narrow ? 0 : std::min<int64_t>(S, columns / 33);
  if (!c.wide_sequences) return c;
  c.wide_columns = 32 * chunk_wide_waves(dim, c.split);
  c.wide_aim = chunk_wide_residents(dim, c.split) * cus;
  c.group = S;
  if (packed || q8) {
    const int64_t rows = blocks * kChunkKeys, bytes = rows * H * dim * (c.split ? 6 : 4);
    // (a group is of sequences, wide or not)
    if (c.wide_sequences * bytes > kChunkRebuiltBytes) c.group = std::max<int64_t>(1, kChunkRebuiltBytes / bytes);
    const int64_t most = std::min(c.group, c.wide_sequences);
    c.rebuilt_rows = most * rows;
    c.rebuilt_bytes = most * bytes;
    if (packed) c.turned_bytes = columns * H * (dim * (c.split ? 4 : 2) + 4);
  }
  const int64_t units = (columns / c.wide_columns + std::min(c.group, c.wide_sequences)) * H;
  c.two_rounds = wide_splits && c.group <= 64 && units * (kChunkSetup + kChunkWide * blocks) > (int64_t)kChunkLong * c.wide_aim;
  c.wide_items = units + (wide_splits ? (c.two_rounds + 1) * c.wide_aim : 0);
  const int64_t slot_columns = std::min<int64_t>(c.wide_columns, (columns + 31) / 32 * 32);
  c.slots = wide_splits ? 2 * c.wide_aim : 0;
  c.part_bytes = std::max(narrow_bytes, c.slots * slot_columns * (dim + 2) * 4);
  return c;
}

hipError_t launch_chunks(const ChunkParams &params, const ChunkPlan &plan, int dim, bool bf16, int cus, hipStream_t stream) {
  ChunkParams p = params;
  bool two = true;
  for (int h = 0; h < p.kv_heads && p.packed; ++h) two &= p.head[h].norm_stride == 2;
  // Narrow items and, behind them, workgroups that rotate queries and rebuild rows.
  auto rows = [&](int64_t narrow, bool rotate, bool rebuild) -> hipError_t {
    p.narrow_items = (int32_t)narrow;
    p.rotate_items = 0;
    if (rotate && p.packed) {
      const int64_t tiles = (p.tokens * p.group + 31) / 32 * p.kv_heads;
      p.rotate_items = (int32_t)std::min<int64_t>((tiles + kChunkWaves - 1) / kChunkWaves, cus);
    }
    p.aim = plan.narrow_aim;
    p.slot_columns = 32;
    p.all_narrow = !plan.wide_sequences;
    const int items = (int)narrow + p.rotate_items + (rebuild ? (cus + p.kv_heads - 1) / p.kv_heads * p.kv_heads : 0);
    if (!p.packed) return dim == 64 ? launch_chunk_f16_d64(p, bf16, items, stream) : launch_chunk_f16_d128(p, bf16, items, stream);
    if (two) return dim == 64 ? launch_chunk_packed2_d64(p, bf16, items, stream) : launch_chunk_packed2_d128(p, bf16, items, stream);
    return dim == 64 ? launch_chunk_packed_d64(p, bf16, items, stream) : launch_chunk_packed_d128(p, bf16, items, stream);
  };
  auto wide = [&]() -> hipError_t {
    p.aim = plan.wide_aim;
    p.two_rounds = plan.two_rounds;
    p.slot_columns = (int32_t)std::min<int64_t>(plan.wide_columns, (p.tokens * p.group + 31) / 32 * 32);
    if (hipError_t e = launch_chunk_wide(p, dim, bf16, (int)plan.wide_items, stream)) return e;
    return plan.slots ? launch_chunk_merge(p, dim, bf16, plan.wide_columns, (int)std::min(plan.slots, plan.wide_items), stream) : hipSuccess;
  };
  if (!plan.wide_sequences) return rows(plan.narrow_items, false, false);
  const bool rebuild = plan.rebuilt_rows > 0;
  if (plan.group >= p.sequences) {
    if (hipError_t e = rows(plan.narrow_items, true, rebuild)) return e;
    return wide();
  }
  if (hipError_t e = rows(plan.narrow_items, true, false)) return e;
  for (int64_t s = 0; s < params.sequences; s += plan.group) {
    p.offsets = params.offsets + s;
    p.lengths = params.lengths + s;
    p.page_table = params.page_table + s * p.page_table_stride;
    p.ahead = (int32_t)s;
    p.sequences = (int32_t)std::min<int64_t>(plan.group, params.sequences - s);
    if (hipError_t e = rows(0, false, true)) return e;
    if (hipError_t e = wide()) return e;
  }
  return hipSuccess;
}

}  // namespace bgtq
