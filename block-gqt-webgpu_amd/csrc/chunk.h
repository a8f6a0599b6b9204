// Attention of chunks of new tokens over the paged cache: launch parameters
// (chunk_kernel.h has the kernel, chunk_*.hip its instances).
#pragma once

#include "bgtq_internal.h"

namespace bgtq {

constexpr int kChunkWaves = 8;                   // of a workgroup
constexpr int kChunkColumns = 32 * kChunkWaves;  // query columns (row x head of a KV head's group) of a tile
constexpr int kChunkKeys = 64;                   // tokens of a block
// Workgroups that share a compute unit: a launch aims at as many items as the chip holds.
constexpr int chunk_residents(int dim) { return dim == 64 ? 2 : 1; }
// Costs of a unit, in eighths of a wide block: its set-up, a block of a wide
// unit, one of a narrow unit (at most 32 columns: the waves share its blocks);
// the least cost of an item where a unit is split.
constexpr int kChunkSetup = 16, kChunkWide = 8, kChunkNarrow = 3, kChunkLeast = 48;
constexpr int kChunkMostSplits = 64;

struct ChunkParams {
  const int32_t *offsets;
  const uint32_t *lengths;
  const int32_t *page_table;
  int64_t page_table_stride;
  int32_t sequences, heads, kv_heads, group;  // query heads; KV heads; query heads per KV head
  int64_t tokens;
  int32_t max_length, page_shift, table_pages, pages;
  const uint16_t *q;
  uint16_t *out;
  int64_t q_row, q_head, out_row, out_head;  // elements
  float c;                                   // scale * log2(e)
  int32_t window, sinks;                     // window 0: all tokens up to the query's
  // The pool (bgtq_pages).
  const uint8_t *packed;
  int64_t packed_page, packed_head;  // bytes
  const uint16_t *norms;
  int64_t norms_page, norms_head;  // elements
  const uint16_t *k;
  int64_t k_page, k_head;
  const uint8_t *v;
  int64_t v_page, v_head;  // bytes
  const uint16_t *v_scales;
  int64_t vs_page, vs_head;
  const DevTables *tables[kMaxKvHeads];
  PagedWriteParams::Head head[kMaxKvHeads];
  uint32_t off_rot_q[kMaxKvHeads];
  // Items: units' splits; `target` of them are aimed at, a split unit's leave
  // partials in slots of slot_columns columns.
  int32_t target, slot_columns;
  uint32_t *counters;
  float *part;
};

// Bytes of a slot's partial results: (o[dim], m, l) of each column.
inline int64_t chunk_slot_bytes(int dim, int columns) { return (int64_t)columns * (dim + 2) * 4; }
// Whether a unit of so many tokens may cost more than the least item, and is then split where there are few.
constexpr bool chunk_splits(int64_t max_length) {
  return kChunkSetup + kChunkWide * ((max_length + kChunkKeys - 1) / kChunkKeys) > kChunkLeast;
}
// Items that a launch's grid has room for: its units, and as many again as it
// aims at where units are split (the items of split units number at most 2 target).
int64_t chunk_items(const ChunkParams &p);
hipError_t launch_chunk(const ChunkParams &p, int dim, bool bf16, hipStream_t stream);

}  // namespace bgtq
