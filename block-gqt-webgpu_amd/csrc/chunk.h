// Attention of chunks of new tokens over the paged cache (bgtq_paged_prefill,
// src/model/decoder.ts:46-56 with rows > 1, over pages): launch parameters.
//
// A sequence's chunk has rows x G query columns per KV head. Narrow ones (at
// most 32, and all of a small call) are attended straight from the pages (chunk_rows.h); the rows that wide
// ones see are rebuilt once, in the same launch, and attended in a second one
// (chunk_wide.hip), which reads FP16 pages as they lie. Units (a sequence, a KV
// head, a tile of columns) are cut along their tokens into items where there are
// few, whose partials are merged in their order: narrow units' by the last item
// to end, wide ones' in a third launch.
#pragma once

#include "bgtq_internal.h"

namespace bgtq {

constexpr int kChunkWaves = 8;                   // of a workgroup for narrow units
constexpr int kChunkKeys = 64;                   // tokens of a block
// Wide units: waves of a workgroup, waves per SIMD by their registers, workgroups per compute unit.
// (Eight waves instead of four share a block's DMAs and barrier, in coarser units: d=64 by single
// products 326 -> 316 us of 2048 rows behind 32768 tokens, d=128 65 -> 67 us of 2 x 1000 behind a window.)
constexpr int chunk_wide_waves(int dim, bool split) { return (dim == 128) == split ? 8 : 4; }
constexpr int chunk_wide_waves_per_simd(int dim, bool split) { return dim == 64 ? split ? 3 : 4 : 2; }
constexpr int chunk_wide_residents(int dim, bool split) {
  return 4 * chunk_wide_waves_per_simd(dim, split) / chunk_wide_waves(dim, split);
}
// Costs of a unit, in eighths of a wide block: its set-up, a block of a wide
// unit, one of a narrow unit; the least cost of a wide and of a narrow item where a unit is split.
constexpr int kChunkSetup = 16, kChunkWide = 8, kChunkNarrow = 3, kChunkLeast = 48, kChunkLeastNarrow = 32;
// A second round of wide items costs this much more; none is made of calls whose items may cost kChunkLong at most.
constexpr int kChunkRound = 64, kChunkLong = 384;
constexpr int kChunkMostSplits = 64;
// Calls of at most this many columns attend all units as narrow ones, in tiles of 32, in their one launch.
constexpr int kChunkSmall = 512;
// Bytes of rebuilt rows: sequences that take more are attended in groups, one that does alone.
constexpr int64_t kChunkRebuiltBytes = (int64_t)1 << 30;

struct ChunkParams {
  const int32_t *offsets;
  const uint32_t *lengths;
  const int32_t *page_table;
  int64_t page_table_stride;
  int32_t sequences, kv_heads, group;  // KV heads; query heads per KV head
  int32_t ahead;                       // sequences of the call before these (their offsets lie before)
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
  // Items: units' splits; `aim` of them are aimed at, a split unit's leave
  // partials in slots of slot_columns columns. narrow_items: the workgroups of
  // the first launch that attend.
  int32_t aim, slot_columns, narrow_items, rotate_items, all_narrow, two_rounds;
  uint32_t *counters;
  float *part;
  // Rebuilt rows, [KV head][row][dim]: K (and its low parts), V; null: pages are read as they lie.
  uint16_t *rebuilt_k, *rebuilt_lo, *rebuilt_v;
  int64_t rebuilt_head;  // rows of a KV head
  // Packed K: the queries in the code domain, [row][head][dim] (BF16 rows' FP16
  // values; FP16 rows': high parts, then low ones), and their powers of two.
  uint16_t *turned;
  int32_t *turned_exp;
};

// What a call launches, from what the host knows.
struct ChunkPlan {
  bool split;               // K and q as pairs of FP16 values
  int64_t wide_sequences;   // that may be wide at most
  int64_t narrow_items;     // first launch: attending workgroups
  int32_t narrow_aim, wide_aim, wide_columns, two_rounds;
  int64_t group, wide_items;  // sequences of a group; items of its launch at most
  int64_t slots;              // of its split units at most
  int64_t part_bytes, rebuilt_rows, rebuilt_bytes, turned_bytes;  // rows of a KV head; of all operands
};
ChunkPlan plan_chunks(const ChunkParams &p, int dim, bool packed, bool q8, bool bf16, int cus);
hipError_t launch_chunks(const ChunkParams &p, const ChunkPlan &plan, int dim, bool bf16, int cus, hipStream_t stream);

}  // namespace bgtq
