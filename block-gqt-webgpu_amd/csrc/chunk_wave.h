// Attention of chunks over the paged cache (bgtq_paged_prefill): which item of
// work a workgroup has, and a wave's part in one: 32 query columns against
// blocks of K and V rows in LDS. chunk_rows.h and chunk_wide.hip have the kernels.
//
// The products, the softmax and its lazy rescale are prompt.hip's: S^T = K Q^T
// in 32x32x16 products leaves a lane one query's logits, and probabilities in
// FP16, carried times 2^11, are the next product's operand as they lie.
#pragma once

#include <type_traits>

#include "chunk.h"
#include "encode_row.h"
#include "gfx950_common.h"

namespace bgtq {
namespace {

using namespace gfx;
using row_enc::f16_bits_to_f32;
using row_enc::wave_sync;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLazy = 4.0f;    // growth of a maximum (log2) that O is not rescaled for
constexpr float kShift = 11.0f;  // probabilities are carried times 2^11

__device__ __forceinline__ f32x16 product(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), half2));
}
template <bool BF>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
  else return pack2(a, b);
}
// A K value's pair: high part rounded to nearest, low part times 2^11, so that it keeps 11 bits however small the value is
// (as it is, it would end at 2^-24: of rows of a scale of 2^-12 a pair had 13 bits in all). |x| at most 65504.
constexpr float kLowUp = 2048.0f;
__device__ __forceinline__ void split2_up(float x0, float x1, uint32_t &hi, uint32_t &lo) {
  hi = pack2(x0, x1);
  const half2 h = __builtin_bit_cast(half2, hi);
  lo = pack2(__builtin_fmaf(-(float)h[0], kLowUp, x0 * kLowUp), __builtin_fmaf(-(float)h[1], kLowUp, x1 * kLowUp));
}
__device__ __forceinline__ float add2(uint32_t pair, float c) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2, pair), half2{(_Float16)1.0f, (_Float16)1.0f}, c, false);
}
// c, or NaN where the pair holds an infinity or a NaN (times 0 either is NaN).
__device__ __forceinline__ float odd2(uint32_t pair, float c) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2, pair), half2{(_Float16)0.0f, (_Float16)0.0f}, c, false);
}
// XOR of a row's 16-byte piece indexes (prompt.hip).
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  return D == 64 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
}
__device__ __forceinline__ void in_place(f32x16 &o) { asm volatile("" : "+v"(o)); }
__device__ __forceinline__ float half_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
constexpr uint32_t kInf16 = 0x7c00u, kOne16 = 0x3c00u;
__device__ __forceinline__ uint32_t finite16(uint32_t w) {
  return ((w & 0x7fffu) >= kInf16 ? 0u : w & 0xffffu) | ((w >> 16 & 0x7fffu) >= kInf16 ? 0u : w & 0xffff0000u);
}
// The values of one kind (0 NaN, 1 infinity, 2 minus infinity) as 1, the others as 0.
__device__ __forceinline__ uint32_t of_kind16(uint32_t w, int kind) {
  auto is = [&](uint32_t x) { return kind == 0 ? (x & 0x7fffu) > kInf16 : x == (kind == 1 ? kInf16 : kInf16 | 0x8000u); };
  return (is(w & 0xffffu) ? kOne16 : 0u) | (is(w >> 16) ? kOne16 << 16 : 0u);
}

// A pointer of the wave's in scalar registers (left to the compiler, a DMA's descriptor became a loop over lanes).
template <typename T>
__device__ __forceinline__ const T *scalar(const T *ptr) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(ptr);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32));
  return reinterpret_cast<const T *>((uintptr_t)lo | (uintptr_t)hi << 32);
}

// The tokens that a tile's rows, at positions first .. last, see something of, in
// blocks of B: all up to the last; behind a window the sinks' blocks, then
// those from the first position's window on. at(i): the i-th block's first token.
struct Blocks {
  int sunk, skipped, count;
  template <int B>
  __device__ __forceinline__ static Blocks of(int first, int last, int window, int sinks) {
    Blocks r{0, 0, last < 0 ? 0 : last / B + 1};
    if (window) {
      r.sunk = min((sinks + B - 1) / B, r.count);
      r.skipped = max(0, max(0, first - window + 1) / B - r.sunk);
      r.count = max(0, r.count - r.skipped);
    }
    return r;
  }
  template <int B>
  __device__ __forceinline__ int at(int i) const { return (i >= sunk ? i + skipped : i) * B; }
};

// A workgroup's item: split `split` of `splits` of a unit. rows: the chunk's; splits 0: nothing.
struct Item {
  int64_t begin;               // the chunk's first row of q
  int seq, rows, n, tile, kv;  // n: the sequence's tokens
  int split, splits, slot0;    // slot0: its unit's first slot
  int64_t base;                // the sequence's first row among the rebuilt ones
};

// The units of a launch: all of them, as narrow ones; the narrow ones (beside the rebuilding
// of the wide ones' K and V); the wide ones.
enum { kAllUnits, kNarrowUnits, kWideUnits };

// The largest value of the lanes up to and with this one, none negative.
__device__ __forceinline__ int wave_prefix_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return v;
}
// A sequence's units and what each costs; a lane per sequence.
struct SequencePlan {
  int begin, rows, n, units;
  bool wide;
  float cost;
};
// What the offsets of the sequences ahead of a group's come to.
__device__ __forceinline__ int offset_ahead(const ChunkParams &p) {
  int most = 0;
  for (int i = (int)(threadIdx.x & 63) - p.ahead; i < 0; i += 64) most = max(most, min(p.offsets[i], (int)p.tokens));
  return __builtin_amdgcn_readlane(wave_prefix_max(most), 63);
}
// The offsets count as no less than those before them (`before`: the sequences' ahead of these 64), so that
// whatever they hold, the chunks are `tokens` rows at most, which the host's counts go by.
__device__ __forceinline__ SequencePlan plan_of(const ChunkParams &p, int s, int which, int tile, int &before) {
  auto offset = [&](int i) { return min(max(p.offsets[i], 0), (int)p.tokens); };
  const bool real = s < p.sequences;
  const int begin = max(before, wave_prefix_max(offset(min(s, p.sequences)))), end = max(begin, offset(min(s + 1, p.sequences)));
  before = __builtin_amdgcn_readlane(end, 63);
  const int rows = real ? end - begin : 0;
  const int n = (int)min(p.lengths[min(s, p.sequences - 1)], (uint32_t)p.max_length);
  const int64_t columns = (int64_t)rows * p.group;
  const bool wide = columns > 32, mine = which == kAllUnits || wide == (which == kWideUnits);
  const int tiles = mine ? (int)((columns + tile - 1) / tile) : 0;
  // The longest tile's blocks: at most the tokens', and behind a window what its rows see.
  int blocks = (n + kChunkKeys - 1) / kChunkKeys;
  if (p.window) {
    const int64_t seen = (int64_t)p.window + min(rows, tile / p.group + 2) + p.sinks;
    blocks = (int)min((int64_t)blocks, seen / kChunkKeys + 3);
  }
  return {begin, rows, n, tiles * p.kv_heads, wide,
          (float)(kChunkSetup + (wide && which != kAllUnits ? kChunkWide : kChunkNarrow) * (int64_t)blocks)};
}
__device__ __forceinline__ int splits_of(const SequencePlan &q, float share) {
  // (the thousandth: a quotient that is whole stays so through the reciprocal)
  return q.units ? max(1, min((int)ceilf(q.cost * __builtin_amdgcn_rcpf(share) - 1e-3f), kChunkMostSplits)) : 0;
}
__device__ __forceinline__ float wave_sum_f(float v) {
  auto turned = [](float x, auto by) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(by)::value, 0xf, 0xf, false)); };
  v += turned(v, std::integral_constant<int, 0x128>{});
  v += turned(v, std::integral_constant<int, 0x124>{});
  v += turned(v, std::integral_constant<int, 0x122>{});
  v += turned(v, std::integral_constant<int, 0x121>{});
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  // (the lanes' orders differ: one's sum for all)
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(half_sum(v))));
}
// Rows that a wide sequence's tokens take among the rebuilt ones: whole blocks.
__device__ __forceinline__ int rebuilt_rows(const SequencePlan &q) { return q.wide ? (q.n + kChunkKeys - 1) / kChunkKeys * kChunkKeys : 0; }

// Which item grid x stands for. Every workgroup finds the same plan from all
// offsets and lengths, 64 sequences at a time: a sequence's units cost its
// longest tile's blocks; an item's share t of cost is the sum's by `aim`, at
// least kChunkLeast, and a sequence's units are split into ceil(cost / t). Of up to
// 64 sequences t is raised until the items are at most `aim`, or as few as
// there are units. Where units hardly outnumber the workgroups the GPU holds, whole
// splits leave some of those idle (224 units on 1024: 4 each, 896): wide units
// then take two rounds of items, of a share t2, where 2 t2 is less. Items of split units
// number at most 2 sum / t <= 2 aim: their partials' slots. BY_SLOT: the item
// that has slot `item`.
template <bool BY_SLOT = false>
__device__ __forceinline__ Item find_item(const ChunkParams &p, int item, int which, int tile, int aim) {
  const int lane = threadIdx.x & 63;
  float all = 0.0f;
  SequencePlan q{};
  const int ahead = offset_ahead(p);
  int before = ahead;
  for (int s0 = 0; s0 < p.sequences; s0 += 64) {
    q = plan_of(p, s0 + lane, which, tile, before);
    all += wave_sum_f((float)q.units * q.cost);
  }
  const float least = which == kWideUnits ? kChunkLeast : kChunkLeastNarrow;
  float share = fmaxf(least, ceilf(all / (float)aim));
  if (p.sequences <= 64) {
    const float units = (float)wave_sum(q.units);
    // The share from t on that makes at most `target` items, or one of each unit (negative: more).
    auto fit = [&](float t, float target) {
      for (int k = 0;; ++k) {
        const float items = (float)wave_sum(splits_of(q, t) * q.units);
        if (items <= fmaxf(target, units)) return t;
        if (k == 3) return -t;
        t = fmaxf(t + 1.0f, ceilf(t * items / target));
      }
    };
    share = fabsf(fit(share, (float)aim));
    if (which == kWideUnits && p.two_rounds) {
      const float half = fit(fmaxf(least, ceilf(all / (float)(2 * aim))), (float)(2 * aim));
      if (half > 0.0f && 2.0f * half + kChunkRound < share) share = half;
    }
  }
  int first = 0, slots = 0;
  int64_t base = 0;
  before = ahead;
  for (int s0 = 0; s0 < p.sequences; s0 += 64) {
    if (p.sequences > 64) q = plan_of(p, s0 + lane, which, tile, before);
    const int splits = splits_of(q, share), items = BY_SLOT && splits < 2 ? 0 : splits * q.units, rebuilt = rebuilt_rows(q);
    const int end = first + wave_prefix(items), slot_end = slots + wave_prefix(splits > 1 ? items : 0);
    const int base_end = wave_prefix(rebuilt);  // (64 sequences of at most 2^24 tokens)
    const uint64_t here = __builtin_amdgcn_ballot_w64(item >= end - items && item < end);
    if (here) {
      const int at = __builtin_ctzll(here);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
      Item r;
      r.begin = of(q.begin);
      r.seq = s0 + at;
      r.rows = of(q.rows);
      r.n = of(q.n);
      r.splits = of(splits);
      const int local = item - (of(end) - of(items)), unit = local / r.splits;
      r.split = local - unit * r.splits;
      const int tiles = of(q.units) / p.kv_heads, back = unit / p.kv_heads;
      r.tile = tiles - 1 - back;  // the longest histories first
      r.kv = unit - back * p.kv_heads;
      r.slot0 = r.splits > 1 ? of(slot_end) - of(items) + unit * r.splits : 0;
      r.base = base + (uint32_t)(of(base_end) - of(rebuilt));
      return r;
    }
    first = __builtin_amdgcn_readlane(end, 63);
    slots = __builtin_amdgcn_readlane(slot_end, 63);
    base += (uint32_t)__builtin_amdgcn_readlane(base_end, 63);
  }
  return Item{};
}

// An item's columns: the tile's rows x heads, row-major.
struct Columns {
  int col0, count, before, first, last;  // before: the first row's position (negative: such rows see nothing); the tile's first and last
  __device__ __forceinline__ Columns(const Item &it, int G, int tile) {
    const int64_t columns = (int64_t)it.rows * G;
    col0 = it.tile * tile;  // (rows x G below 2^31: checked on the host)
    count = (int)min(columns - col0, (int64_t)tile);
    before = it.n - it.rows;
    first = before + col0 / G;
    last = before + (col0 + count - 1) / G;
  }
};

// Column c's row of out.
__device__ __forceinline__ uint16_t *out_of(const ChunkParams &p, const Item &it, const Columns &cs, int c) {
  const int j = cs.col0 + c, row = j / p.group;
  return p.out + (it.begin + row) * p.out_row + (it.kv * p.group + (j - row * p.group)) * p.out_head;
}
__device__ __forceinline__ float inverse_sum(float sum) { return sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum; }  // (a NaN stays one)

// A split unit's partial: o in pieces of four dimensions, [piece][column], then (m, l) of each column. POLICY
// kPolicySc1: for a reader in the same launch, which may run on another XCD.
template <int D, int POLICY>
struct Partial {
  __amdgpu_buffer_rsrc_t r;
  int SC;
  __device__ __forceinline__ Partial(const ChunkParams &p, const Item &it, int split) {
    SC = p.slot_columns;
    const uint32_t slot_bytes = (uint32_t)SC * (D + 2) * 4;
    r = rsrc(reinterpret_cast<uint8_t *>(p.part) + (int64_t)(it.slot0 + split) * slot_bytes, slot_bytes);
  }
  __device__ __forceinline__ void put(int piece, int column, f32x4 o) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), r, (piece * SC + column) * 16, 0, POLICY);
  }
  __device__ __forceinline__ void put(int column, float m, float l) const {
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, r, D * SC * 4 + column * 8, 0, POLICY);
  }
  __device__ __forceinline__ u32x4 o(int piece, int column) const { return __builtin_amdgcn_raw_buffer_load_b128(r, (piece * SC + column) * 16, 0, POLICY); }
  __device__ __forceinline__ u32x2 ml(int column) const { return __builtin_amdgcn_raw_buffer_load_b64(r, D * SC * 4 + column * 8, 0, POLICY); }
};
// Four dimensions of a column, final or a split unit's partial for the same launch.
template <int D, bool BF>
__device__ __forceinline__ void store_piece(const ChunkParams &p, const Item &it, const Columns &cs, int piece, int c, f32x4 o, float m, float l) {
  if (it.splits == 1) {
    const float inv = inverse_sum(l);
    *reinterpret_cast<u32x2 *>(out_of(p, it, cs, c) + 4 * piece) = u32x2{pack_out<BF>(o[0] * inv, o[1] * inv), pack_out<BF>(o[2] * inv, o[3] * inv)};
  } else {
    const Partial<D, kPolicySc1> to(p, it, it.split);
    to.put(piece, c, o);
    if (piece == 0) to.put(c, m, l);
  }
}

constexpr int kStageRow = 20, kStageBytes = 32 * kStageRow * 4;  // of a wave
// A wave's 32 columns: lane (h, q) = (lane / 32, lane % 32) has query q's part.
// SPLIT: K and q as pairs of FP16 values.
template <int D, bool SPLIT, bool BF>
struct Wave {
  static constexpr int QS = D / 16, MT = D / 32;  // 16-dimension steps of QK, 32-dimension tiles of O
  u32x4 qh[QS], ql[SPLIT ? QS : 1];               // positions 16 s + 8 h + 0..7, scaled by a power of two
  f32x16 O[MT];
  float m, l;  // log2 domain; this lane's part of the sum
  float cl;    // a product's factor: scale log2(e) over the powers of two
  int pos;     // this lane's query's position
  int window, sinks;
  uint32_t lane_at;  // this lane's bytes in a tile of K rows, and 65536 times those in one of V rows

  // Column c's row of the chunk and head (past the tile's: its last column's).
  __device__ __forceinline__ static void column(const ChunkParams &p, const Item &it, const Columns &cs, int c, int &row, int &head) {
    const int j = cs.col0 + min(c, cs.count - 1);
    row = j / p.group;
    head = it.kv * p.group + (j - row * p.group);
  }
  // Eight values of a row of q as FP32.
  __device__ __forceinline__ static void load8(const uint16_t *src, float (&x)[8]) {
    const u32x4 w = *reinterpret_cast<const u32x4 *>(src);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t u = k & 1 ? w[k >> 1] >> 16 : w[k >> 1] & 0xffffu;
      x[k] = BF ? __uint_as_float(u << 16) : f16_bits_to_f32((uint16_t)u);
    }
  }
  // The queries' FP16 operands from this lane's values; the power of two they are scaled by.
  __device__ __forceinline__ int split_queries(const float (&x)[QS][8]) {
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < QS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[s][e]));
    const int eq = split_exp(half_max(top));
    const float up = __builtin_ldexpf(1.0f, eq);
#pragma unroll
    for (int s = 0; s < QS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (SPLIT) {
          uint32_t hi, lo;
          split2(x[s][2 * e] * up, x[s][2 * e + 1] * up, hi, lo);
          qh[s][e] = hi;
          ql[s][e] = lo;
        } else {
          qh[s][e] = pack2(x[s][2 * e] * up, x[s][2 * e + 1] * up);
        }
      }
    return eq;
  }
  // Nothing seen yet. eq: the queries' power of two; K rows in the code domain (`coded`) carry the books', 2^(cent_exp - 14).
  __device__ __forceinline__ void begin(const ChunkParams &p, const Item &it, int eq, bool coded) {
    window = p.window, sinks = p.sinks;
    const int lane = threadIdx.x & 63, h = lane >> 5, qc = lane & 31, vr = 4 * h + ((lane & 15) >> 2);
    const int piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    lane_at = (uint32_t)(qc * (2 * D) + ((h ^ swizzle<D>(qc)) * 16)) |
              (uint32_t)(vr * (2 * D) + ((piece ^ swizzle<D>(vr)) * 16) + (lane & 1) * 8) << 16;
    // (it meets masked logits: not 0)
    cl = fmaxf(__builtin_ldexpf(p.c, -eq - (coded ? p.head[it.kv].cent_exp - 14 : 0)), 0x1p-126f);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) O[t][i] = 0.0f;
    m = -INFINITY, l = 0.0f;
  }
  // The queries as they are.
  __device__ __forceinline__ void load_plain(const ChunkParams &p, const Item &it, const Columns &cs, int first_column) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    int row, head;
    column(p, it, cs, first_column + (lane & 31), row, head);
    pos = cs.before + row;
    float x[QS][8];
#pragma unroll
    for (int s = 0; s < QS; ++s) load8(p.q + (it.begin + row) * p.q_row + head * p.q_head + 16 * s + 8 * h, x[s]);
    begin(p, it, split_queries(x), false);
  }
  // The queries that rotate_queries left (chunk_rows.h).
  __device__ __forceinline__ void load_turned(const ChunkParams &p, const Item &it, const Columns &cs, int first_column) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    int row, head;
    column(p, it, cs, first_column + (lane & 31), row, head);
    pos = cs.before + row;
    const int64_t at = (it.begin + row) * (p.kv_heads * p.group) + head;
    const uint16_t *src = p.turned + at * (SPLIT ? 2 * D : D) + 8 * h;
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      qh[s] = *reinterpret_cast<const u32x4 *>(src + 16 * s);
      if constexpr (SPLIT) ql[s] = *reinterpret_cast<const u32x4 *>(src + D + 16 * s);
    }
    begin(p, it, p.turned_exp[at], true);
  }
  // 16 columns of queries (lane (gq, c): column c, dimensions 32 s + 8 gq on) as a product's operand, in `b`; what they are to be scaled down by.
  __device__ __forceinline__ static float operand16(const ChunkParams &p, const Item &it, const Columns &cs, int first_column, u32x4 (&b)[D / 32]) {
    const int lane = threadIdx.x & 63, gq = lane >> 4;
    int row, head;
    column(p, it, cs, first_column + (lane & 15), row, head);
    const uint16_t *src = p.q + (it.begin + row) * p.q_row + head * p.q_head + 8 * gq;
    float y[D / 32][8], top = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      load8(src + 32 * s, y[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[s][e]));
    }
    const int e0 = split_exp(col_max(top));
    const float up = __builtin_ldexpf(1.0f, e0);
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) b[s][e] = pack2(y[s][2 * e] * up, y[s][2 * e + 1] * up);  // (16-bit values: exact)
    return __builtin_ldexpf(1.0f, -e0);
  }
  // The rotation's operands of positions 16 t .. 16 t + 15.
  __device__ __forceinline__ static void rotation16(const ChunkParams &p, int kv, int t, u32x4 (&r)[D / 32][2]) {
    const u32x4 *op = reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint8_t *>(p.tables[kv]) + p.off_rot_q[kv]) + 2 * (threadIdx.x & 63);
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) r[s][e] = op[(t * (D / 32) + s) * 128 + e];
  }
  __device__ __forceinline__ static f32x4 rotate16(const u32x4 (&r)[D / 32][2], const u32x4 (&b)[D / 32]) {
    f32x4 a{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      a = mfma(__builtin_bit_cast(half8, r[s][0]), __builtin_bit_cast(half8, b[s]), a);
      a = mfma(__builtin_bit_cast(half8, r[s][1]), __builtin_bit_cast(half8, b[s]), a);
    }
    return a;
  }
  // The queries into the code domain of their KV head, R q. SHARED: all waves have the same columns, each rotates 16 of the
  // positions (stage: 32 rows of D + 4 floats of the workgroup); else a wave its own
  // columns, 16 positions at a time (stage: 32 rows of kStageRow floats of its own). Their power of two.
  template <bool SHARED>
  __device__ __forceinline__ int load_rotated(const ChunkParams &p, const Item &it, const Columns &cs, int first_column, float *stage) {
    constexpr int KS = D / 32;
    const int lane = threadIdx.x & 63, h = lane >> 5, qc = lane & 31, gq = lane >> 4, c16 = lane & 15;
    int row, head;
    column(p, it, cs, first_column + qc, row, head);
    pos = cs.before + row;
    float x[QS][8];
    u32x4 b[2][KS], r[KS][2];
    float down[2];
    if constexpr (SHARED) {
      static_assert(QS <= kChunkWaves, "a wave per 16 positions");
      const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
      if (wave < QS) {
        rotation16(p, it.kv, wave, r);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          down[half] = operand16(p, it, cs, first_column + 16 * half, b[half]);
          *reinterpret_cast<f32x4 *>(stage + (16 * half + c16) * (D + 4) + 16 * wave + 4 * gq) = rotate16(r, b[half]) * down[half];
        }
      }
      lds_barrier();
#pragma unroll
      for (int s = 0; s < QS; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4 v = *reinterpret_cast<const f32x4 *>(stage + qc * (D + 4) + 16 * s + 8 * h + 4 * e);
#pragma unroll
          for (int k = 0; k < 4; ++k) x[s][4 * e + k] = v[k];
        }
    } else {
      rotation16(p, it.kv, 0, r);
#pragma unroll
      for (int half = 0; half < 2; ++half) down[half] = operand16(p, it, cs, first_column + 16 * half, b[half]);
#pragma unroll
      for (int t = 0; t < QS; ++t) {
        f32x4 a[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) a[half] = rotate16(r, b[half]);
        if (t + 1 < QS) rotation16(p, it.kv, t + 1, r);
        __builtin_amdgcn_sched_barrier(0);  // (the operands of all positions at once spilled)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          *reinterpret_cast<f32x4 *>(stage + (16 * half + c16) * kStageRow + 4 * gq) = a[half] * down[half];
        wave_sync();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4 v = *reinterpret_cast<const f32x4 *>(stage + qc * kStageRow + 8 * h + 4 * e);
#pragma unroll
          for (int k = 0; k < 4; ++k) x[t][4 * e + k] = v[k];
        }
        wave_sync();
      }
    }
    return split_queries(x);
  }

  // S += K Q^T of the NB x 32 K rows at LDS offset `at`; low: the queries' low parts too.
  template <int NB>
  __device__ __forceinline__ void qk(uint8_t *smem, uint32_t at, f32x16 (&S)[NB], bool low) const {
    uint32_t k_at = lane_at;
    if constexpr (D == 64) asm volatile("" : "+v"(k_at));  // (parted here: each held across the loop, one was spilled, and its reload waited for the DMAs)
    k_at &= 0xffffu;
#pragma unroll
    for (int s = 0; s < QS; ++s)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const u32x4 a = *reinterpret_cast<const u32x4 *>(smem + ((at + k_at) ^ (32u * s)) + 64 * D * b);
        S[b] = product(a, qh[s], S[b]);
        if constexpr (SPLIT)
          if (low) S[b] = product(a, ql[s], S[b]);
      }
  }
  // S of K's low parts, which are held times 2^11, to be added to.
  template <int NB>
  __device__ __forceinline__ static void low_parts(f32x16 (&S)[NB]) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[b][i] *= 1.0f / kLowUp;
  }
  // What the queries of positions lo .. hi see of the block of B tokens from t0 on: 0 nothing, 1 a part, 2 all.
  __device__ __forceinline__ int sight(int t0, int B, int lo, int hi) const {
    if (t0 > hi) return 0;
    if (window && t0 + B - 1 <= lo - window && t0 >= sinks) return 0;
    return t0 + B - 1 <= lo && (!window || t0 > hi - window) ? 2 : 1;
  }
  // Whether this lane's query sees token 4 h + k of a block from t0 on (bit k), of those in `there`.
  __device__ __forceinline__ uint64_t seen_bits(int t0, uint64_t there) const {
    auto below = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : ~(~0ull << n); };  // bits 0 .. n - 1
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // (made here: what is held across the loop spills)
    const int h = lane >> 5, d = pos - t0 - 4 * h;
    uint64_t bits = below(d + 1);
    if (window) bits &= ~below(d + 1 - window) | below(sinks - t0 - 4 * h);
    return bits & (there >> (4 * h));
  }
  // The softmax of S (masked: to the seen tokens) into P, O rescaled where a maximum grew.
  template <int NB>
  __device__ __forceinline__ void softmax(f32x16 (&S)[NB], uint32_t (&P)[8 * NB], bool masked, uint64_t seen) {
    if (masked) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint32_t w = (uint32_t)(seen >> (32 * b));
#pragma unroll
        for (int i = 0; i < 16; ++i) S[b][i] = w >> (8 * (i >> 2) + (i & 3)) & 1u ? S[b][i] : -INFINITY;
      }
    }
    float top = S[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, S[b][i]);
    top = half_max(top) * cl;
    if (__builtin_amdgcn_ballot_w64(top > m + kLazy)) {  // (also the first block: m = -inf)
      const float mn = fmaxf(m, top), a = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= a;
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          O[t][i] *= a;
          in_place(O[t]);
        }
    }
    const float mu = (m == -INFINITY ? 0.0f : m) - kShift;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[b][i], cl, -mu));
#pragma unroll
    for (int e = 0; e < 8 * NB; ++e) {
      P[e] = pack2(S[e >> 3][2 * (e & 7)], S[e >> 3][2 * (e & 7) + 1]);
      l = add2(P[e], l);
    }
  }
  // O^T += V^T P^T of the V rows at LDS offset `at`; odd: of their finite values.
  template <int NB, bool MAYBE_ODD>
  __device__ __forceinline__ void pv(uint8_t *smem, uint32_t at, const uint32_t (&P)[8 * NB], bool odd) {
    constexpr int STEP = 16 * 2 * D;  // bytes of a step's rows
    uint32_t v_at = lane_at;
    if constexpr (D == 64) asm volatile("" : "+v"(v_at));
    v_at = lds_at(smem) + at + (v_at >> 16);
    uint32_t va[MT], va8[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      va[t] = v_at ^ (64u * t);
      va8[t] = ((v_at ^ 32u) + 16 * D) ^ (64u * t);  // (swizzle(vr + 8) = swizzle(vr) ^ 2)
    }
    u32x2 v[2][MT][2];
    ds_read_tr16<MT, 0>(va, va8, v[0]);
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s) {
      const u32x4 pf{P[4 * s], P[4 * s + 1], P[4 * s + 2], P[4 * s + 3]};
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        u32x4 a{v[s & 1][t][0][0], v[s & 1][t][0][1], v[s & 1][t][1][0], v[s & 1][t][1][1]};
        if (MAYBE_ODD && odd) {
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = finite16(a[e]);
        }
        O[t] = product(a, pf, O[t]);
      }
      if (s == 0) ds_read_tr16<MT, STEP>(va, va8, v[1]);
      if constexpr (NB == 2) {
        if (s == 1) ds_read_tr16<MT, 2 * STEP>(va, va8, v[0]);
        if (s == 2) ds_read_tr16<MT, 3 * STEP>(va, va8, v[1]);
      }
    }
  }
  // V of dimension 32 t + (rare & 31), tokens 16 s + 8 (e / 2) + 4 (rare / 32) + 2 (e % 2) + 0, 1 in word e.
  __device__ __forceinline__ static u32x4 v_column(const uint8_t *smem, uint32_t at, int rare, int s, int t) {
    const int h = rare >> 5, qc = rare & 31;
    u32x4 a;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = 0;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 16 * s + 8 * (e >> 1) + 4 * h + 2 * (e & 1) + x;
        const uint8_t *from = smem + at + r * (2 * D) + (((4 * t + (qc >> 3)) ^ swizzle<D>(r)) * 16) + 2 * (qc & 7);
        a[e] |= (uint32_t)*reinterpret_cast<const uint16_t *>(from) << (16 * x);
      }
    }
    return a;
  }
  // Some queries see a part of the rows only, and some rows hold infinities
  // or NaNs: what is seen of those is added to O by itself, and the products
  // take the finite values.
  template <int NB>
  __device__ __forceinline__ void add_odd(const uint8_t *smem, uint32_t at, uint64_t seen) {
    int rare = threadIdx.x & 63;
    asm volatile("" : "+v"(rare));  // (this branch's addresses are not held across the loop)
#pragma clang loop unroll(disable)
    for (int kind = 0; kind < 3; ++kind) {
      const float value = kind == 0 ? __builtin_nanf("") : kind == 1 ? INFINITY : -INFINITY;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f32x16 n;
#pragma unroll
        for (int i = 0; i < 16; ++i) n[i] = 0.0f;
#pragma clang loop unroll(disable)
        for (int s = 0; s < 2 * NB; ++s) {
          u32x4 a = v_column(smem, at, rare, s, t), sees;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = 16 * s + 8 * (e >> 1) + 2 * (e & 1);
            a[e] = of_kind16(a[e], kind);
            sees[e] = (seen >> k & 1u ? kOne16 : 0u) | (seen >> (k + 1) & 1u ? kOne16 << 16 : 0u);
          }
          n = product(a, sees, n);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          O[t][i] = n[i] > 0.0f ? O[t][i] + value : O[t][i];
          in_place(O[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // The item's results, of this wave's columns first_column on (below `stored` of the tile's): to out, or, of a split
  // unit, as a partial (Partial).
  __device__ __forceinline__ void store(const ChunkParams &p, const Item &it, const Columns &cs, int first_column, int stored) {
    const int lane = threadIdx.x & 63, h = lane >> 5, mine = first_column + (lane & 31);
    l = half_sum(l);
    if (mine >= stored) return;
    if (it.splits == 1) {
      const float inv = inverse_sum(l);
      uint16_t *out = out_of(p, it, cs, mine);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<u32x2 *>(out + 32 * t + 8 * g + 4 * h) =
              u32x2{pack_out<BF>(O[t][4 * g] * inv, O[t][4 * g + 1] * inv), pack_out<BF>(O[t][4 * g + 2] * inv, O[t][4 * g + 3] * inv)};
      return;
    }
    const Partial<D, kCached> to(p, it, it.split);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        to.put(8 * t + 2 * g + h, mine, f32x4{O[t][4 * g], O[t][4 * g + 1], O[t][4 * g + 2], O[t][4 * g + 3]});
    if (h == 0) to.put(mine, m, l);
  }
};

// Pieces e0, e0 + step, ... below e1 of a unit's columns, merged from its items' partials in their order.
template <int D, bool BF, bool COHERENT>
__device__ __forceinline__ void merge_pieces(const ChunkParams &p, const Item &it, const Columns &cs, int e0, int e1, int step) {
  for (int e = e0; e < e1; e += step) {
    const int piece = e / cs.count, c = e - piece * cs.count;
    float M = -INFINITY, sum = 0.0f;
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int N = COHERENT ? 8 : 4, kPolicy = COHERENT ? kPolicySc1 : kCached;  // splits whose loads are in flight together
    for (int s0 = 0; s0 < it.splits; s0 += N) {
      u32x2 ml[N];
      f32x4 x[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const Partial<D, kPolicy> from(p, it, min(s0 + k, it.splits - 1));
        ml[k] = from.ml(c);
        x[k] = __builtin_bit_cast(f32x4, from.o(piece, c));
      }
      float top = M;
#pragma unroll
      for (int k = 0; k < N; ++k) top = s0 + k < it.splits ? fmaxf(top, __uint_as_float(ml[k][0])) : top;
      const float a = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - top);
      M = top;
      sum *= a;
      o *= a;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float mk = __uint_as_float(ml[k][0]);
        const bool live = s0 + k < it.splits;
        const float w = mk == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mk - M);  // (a state that saw nothing is all zeros)
        sum = live ? __builtin_fmaf(__uint_as_float(ml[k][1]), w, sum) : sum;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = live ? __builtin_fmaf(x[k][d], w, o[d]) : o[d];
      }
    }
    const float inv = inverse_sum(sum);
    *reinterpret_cast<u32x2 *>(out_of(p, it, cs, c) + 4 * piece) = u32x2{pack_out<BF>(o[0] * inv, o[1] * inv), pack_out<BF>(o[2] * inv, o[3] * inv)};
  }
}

}  // namespace
}  // namespace bgtq
