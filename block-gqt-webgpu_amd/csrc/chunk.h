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
// us of calls that differ by more than two runs of one do (A: 13 sequences of 3 KV heads, 301 new rows among
// single ones; B, C: 16 of five new rows behind up to 4099 tokens, 14 / 2 heads of layout B, d=64, BF16 and FP16
// rows; D: the same on 16 / 4 heads of d=128; E: on the calibration's 9 / 3 heads; F: 8 of 36 rows, as B):
//   set-up 4 / 16 / 32:              B 32.2 / 32.1 / 34.3, C 36.5 / 36.5 / 38.6
//   a narrow block 2 / 3 / 6:        A 72.5 / 70.2 / 72.8, D 35.1 / 32.5 / 32.4, E 25.0 / 22.7 / 21.3, B 32.2 / 32.1 / 34.5
//   least of a wide item 24 / 48 / 96: B 33.5 / 32.1 / 37.5, C 36.8 / 36.5 / 43.6, F 33.1 / 37.2 / 44.6
//   of a narrow one 16 / 24 / 32 / 48: A 73.3 / 73.4 / 70.2 / 73.4, E 21.2 / 21.4 / 22.7 / 25.4, D 32.8 / 32.4 / 32.5 / 35.6
constexpr int kChunkSetup = 16, kChunkWide = 8, kChunkNarrow = 3, kChunkLeast = 48, kChunkLeastNarrow = 32;
// A second round of wide items costs this much more (0 / 64 / no second round: A 71.3 / 70.2 / 70.9 us, 2048 rows behind
// 30720 tokens on 14 / 2 heads of d=64 in FP16 pages 309.8 / 309.6 / 319.7); none is made of calls whose items may cost kChunkLong at
// most, which leaves their workgroups the search for it (A 71.4 us with 0).
constexpr int kChunkRound = 64, kChunkLong = 384;
// (A bound on a merge's chain, which the shares hardly meet: 16, 32 and 128 within 1% but for 4 x 36 rows behind 8156
// tokens, as F, 37.2 us with 16, 35.0 with 64.)
constexpr int kChunkMostSplits = 64;
// Calls of at most this many columns attend all units as narrow ones, in tiles of 32, in their one launch. us, 64 / 256 /
// 512 / 1024 / 2048: 32 single tokens (224 columns, up to 32768 tokens) 62.8 / 53.9 / 53.8 / 53.8 / 54.5, D (320) 43.3 / 43.0 /
// 32.5 / 32.9 / 32.8, 2 x 36 rows of B's heads (504) 32.6 / 32.6 / 23.5 / 24.0 / 23.2, 2 x 1000 rows of 8 heads of d=128 behind a window (2000) 65.3 / 66.2 / 65.9
// / 66.1 / 94.9. From 512 to 1024 the narrow way is the faster one too in B (560: 32.1 / 21.0), C (36.5 / 23.4), 4 x 36 rows (1008: 35.0 /
// 26.5) and 74 single tokens (518, all of which find no wide unit in two launches: 67.3 / 55.6).
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
