// Attention of chunks of new tokens over the paged cache (bgtq_paged_prefill):
// sequence s brings the rows offsets[s] .. offsets[s+1] - 1 of q, its last ones, and row
// i of c sees the tokens up to its own position lengths[s] - c + i (src/model/decoder.ts:46-56
// with rows > 1, over pages).
//
// Work. A unit is a sequence, a KV head and a tile of 256 query columns (the
// chunk's rows x the G heads of the KV head, row-major): the heads of a group
// share what is rebuilt of K and V. Units are cut along their tokens into
// items where there are few (find_item), a workgroup of eight waves each; the
// last item of a unit to end merges its partials in their order, so results do not
// depend on who is last.
//
// K is rebuilt in the code domain: k = R^T cs, so q . k = (R q) . cs. A
// workgroup rotates its queries once, and K's row is c_j s_g(j), one table
// lookup and one product a value, rounded to FP16 (c scaled by the books'
// largest power of two: |c| <= 1, so a finite scale's row is finite, and rows
// whose scale is a normal FP16 number lose nothing against their largest
// value). BF16 rows multiply it as it is; FP16 rows carry three bits more and
// take K and q as pairs of FP16 values (three products). 8-bit V becomes its
// FP16 values. Each thread makes eight consecutive values of a row, of both,
// from codes that it loaded a block ahead, and writes them to LDS.
//
// Wide units (more than 32 columns): a wave has 32 columns, the eight share
// blocks of 64 tokens, two buffers, one barrier a block. Narrow units: all
// waves have the same columns and blocks of 32 tokens of their own, rebuilt by
// the wave alone without barriers; their results are joined at the end.
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

constexpr int kThreads = 64 * kChunkWaves;
constexpr float kLazy = 4.0f;    // growth of a maximum (log2) that O is not rescaled for
constexpr float kShift = 11.0f;  // probabilities are carried times 2^11

// LDS: the books (as paged_rows.hip's: a byte code's at book * 1056 + 8, a
// nibble code's 16 behind them at book * 96 + 4: an offset's low five bits are the
// bit-field extract's width), the flags, then the buffers.
constexpr int kByteBook = 1056, kNibbleBook = 96, kNibbleBooks = 8 * kByteBook, kBookBytes = kNibbleBooks + 8 * kNibbleBook;
template <int D, int KF, bool SPLIT>
struct ChunkLds {
  static constexpr int TILE = kChunkKeys * D * 2;          // bytes of a block of K or V
  static constexpr int BUFFER = (SPLIT ? 3 : 2) * TILE;    // K, V (K's low parts)
  static constexpr int BOOKS = KF ? kBookBytes : 0;
  static constexpr int FLAGS = BOOKS, BUFFERS = BOOKS + 256;  // (row pieces are XORed into addresses: whole 256 bytes)
  static constexpr int JOIN = 4 * 64 * (D / 2 + 2) * 4;    // four waves' states of a narrow unit
  static constexpr int STAGE = kChunkWaves * 16 * (D + 4) * 4;  // rotated queries, 16 columns a wave
  static constexpr int PRIVATE = kChunkWaves * 32 * D * 2;
  static constexpr int most(int a, int b) { return a > b ? a : b; }
  static constexpr int BYTES = BUFFERS + most(most(2 * BUFFER, PRIVATE), most(JOIN, STAGE));
};

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
__device__ __forceinline__ float add2(uint32_t pair, float c) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2, pair), half2{(_Float16)1.0f, (_Float16)1.0f}, c, false);
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
  int64_t begin;              // the chunk's first row of q
  int seq, rows, n, tile, kv;  // n: the sequence's tokens
  int split, splits, slot0;   // slot0: its unit's first slot
};

// Which item grid x stands for. Every workgroup finds the same plan from all
// offsets and lengths, a lane per sequence, 64 at a time: a sequence's units
// cost its longest tile's blocks; an item's share t of cost is the sum's by p.target, at
// least kChunkLeast, and a sequence's units are split into ceil(cost / t). Of up to
// 64 sequences t is raised until the items are at most p.target, or as few as
// there are units. Items of split units number at most 2 sum / t <= 2 p.target.
struct SequencePlan {
  int64_t begin;
  int rows, n, units;
  float cost;
};
template <int D>
__device__ __forceinline__ SequencePlan plan_of(const ChunkParams &p, int s) {
  auto offset = [&](int i) {
    const int64_t o = p.offsets[i];
    return o < 0 ? 0 : o > p.tokens ? p.tokens : o;
  };
  const bool real = s < p.sequences;
  const int64_t begin = offset(min(s, p.sequences)), end = offset(min(s + 1, p.sequences));
  const int rows = real && end > begin ? (int)(end - begin) : 0;
  const int n = (int)min(p.lengths[min(s, p.sequences - 1)], (uint32_t)p.max_length);
  const int64_t columns = (int64_t)rows * p.group;
  const int tiles = (int)((columns + kChunkColumns - 1) / kChunkColumns);
  // The longest tile's blocks: at most the tokens', and behind a window what its rows see.
  int blocks = (n + kChunkKeys - 1) / kChunkKeys;
  if (p.window) {
    const int64_t seen = (int64_t)p.window + min(rows, kChunkColumns / p.group + 2) + p.sinks;
    blocks = (int)min((int64_t)blocks, seen / kChunkKeys + 3);
  }
  return {begin, rows, n, tiles * p.kv_heads,
          (float)(kChunkSetup + (columns > 32 ? kChunkWide : kChunkNarrow) * (int64_t)blocks)};
}
__device__ __forceinline__ int splits_of(const SequencePlan &q, float share) {
  // (the thousandth: a quotient that is whole stays so through the reciprocal)
  return q.units ? max(1, min((int)ceilf(q.cost * __builtin_amdgcn_rcpf(share) - 1e-3f), kChunkMostSplits)) : 0;
}
__device__ __forceinline__ float wave_sum_f(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}
template <int D>
__device__ __forceinline__ Item find_item(const ChunkParams &p, int item) {
  const int lane = threadIdx.x & 63;
  const float target = (float)p.target;
  float all = 0.0f;
  SequencePlan q{};
  for (int s0 = 0; s0 < p.sequences; s0 += 64) {
    q = plan_of<D>(p, s0 + lane);
    all += wave_sum_f((float)q.units * q.cost);
  }
  float share = fmaxf((float)kChunkLeast, ceilf(all / target));
  if (p.sequences <= 64) {
    for (int k = 0; k < 3; ++k) {
      const int n = splits_of(q, share);
      const float items = (float)wave_sum(n * q.units), units = (float)wave_sum(q.units);
      if (items <= fmaxf(target, units)) break;
      share = fmaxf(share + 1.0f, ceilf(share * items / target));
    }
  }
  int first = 0, slots = 0;
  for (int s0 = 0; s0 < p.sequences; s0 += 64) {
    if (p.sequences > 64) q = plan_of<D>(p, s0 + lane);
    const int splits = splits_of(q, share), items = splits * q.units;
    const int end = first + wave_prefix(items), slot_end = slots + wave_prefix(splits > 1 ? items : 0);
    const uint64_t here = __builtin_amdgcn_ballot_w64(item >= end - items && item < end);
    if (here) {
      const int at = __builtin_ctzll(here);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
      Item r;
      r.begin = (int64_t)(uint32_t)of((int)(uint32_t)q.begin);
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
      return r;
    }
    first = __builtin_amdgcn_readlane(end, 63);
    slots = __builtin_amdgcn_readlane(slot_end, 63);
  }
  return {0, 0, 0, 0, 0, 0, 0, 0, 0};
}

// KF: 0 FP16 K, 1 packed K of norm stride 2, 2 of any. BF: q and out are BF16.
template <int D, int KF, bool Q8, bool BF>
__global__ __launch_bounds__(kThreads, 2) void chunk_kernel(ChunkParams p) {
  constexpr bool SPLIT = KF != 0 && !BF;  // K and q as pairs of FP16 values
  using L = ChunkLds<D, KF, SPLIT>;
  constexpr int O8 = D / 8;                     // eighths of a row, a thread each
  constexpr int QS = D / 16;                    // 16-dimension steps of QK
  constexpr int MT = D / 32;                    // 32-dimension tiles of O
  constexpr int TILE = L::TILE;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t *const bufs = smem + L::BUFFERS;
  int *const flags = reinterpret_cast<int *>(smem + L::FLAGS);  // [hole, odd][buffer], then the last arrival's
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, qc = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item it = find_item<D>(p, blockIdx.x);
  if (it.splits == 0) return;  // uniform for the workgroup
  const int G = p.group, kv = it.kv;
  const int64_t columns = (int64_t)it.rows * G;
  const int col0 = it.tile * kChunkColumns;  // (rows x G below 2^31: checked on the host)
  const int ncol = (int)min(columns - col0, (int64_t)kChunkColumns);
  const bool narrow = columns <= 32;
  // This lane's column: its row of the chunk, head and position (past the unit's: its last column's, not stored).
  const int mine = (narrow ? 0 : 32 * wave) + qc;
  const int cj = col0 + min(mine, ncol - 1), row = cj / G, head = kv * G + (cj - row * G);
  const int before = it.n - it.rows;  // the first row's position (negative: such rows see nothing)
  const int pos = before + row;
  const int tile_first = before + col0 / G, tile_last = before + (col0 + ncol - 1) / G;

  // ---- this thread's eighth of K rows: where its codes lie ----
  const auto &H = p.head[kv];
  const int RB = H.row_bytes, NS = H.norm_stride;
  const int oct = tid % O8;
  uint32_t ext[8], tbo[8], sel[4];
  int k_off0 = 0, k_off1 = 0, g_lo = 0;
  float ce = 1.0f;  // the books' power of two
  if constexpr (KF != 0) {
    const BGTQ_GLOBAL uint8_t *Tb = reinterpret_cast<const BGTQ_GLOBAL uint8_t *>(to_global(p.tables[kv]));
    const BGTQ_GLOBAL uint32_t *gd = reinterpret_cast<const BGTQ_GLOBAL uint32_t *>(Tb + H.off_gdesc) + 8 * oct;
    uint32_t d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = gd[e];
    const int k0 = (int)(d[0] & 255u), k1 = (int)(d[4] & 255u);
    k_off0 = min(k0, RB - 4), k_off1 = min(k1, RB - 4);
    g_lo = (int)(d[0] >> 16 & 7u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t book = d[e] >> 12 & 15u;
      tbo[e] = d[e] >> 11 & 1u ? kNibbleBooks + book * kNibbleBook + 4 : book * kByteBook + 8;
      ext[e] = 8 * ((d[e] & 255u) - (uint32_t)(e < 4 ? k_off0 : k_off1)) + (d[e] >> 8 & 7u);
    }
    // A value pair's scales, picked from the four of groups g_lo .. g_lo + 3 (two words).
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a = (d[2 * k] >> 16 & 7u) - g_lo, b = (d[2 * k + 1] >> 16 & 7u) - g_lo;
      sel[k] = (2 * a) | (2 * a + 1) << 8 | (2 * b) << 16 | (2 * b + 1) << 24;
    }
    // cent_exp: max |c| 2^cent_exp lies in (2^13, 2^14].
    ce = __builtin_ldexpf(1.0f, H.cent_exp - 14);
    const BGTQ_GLOBAL float *books = reinterpret_cast<const BGTQ_GLOBAL float *>(Tb + H.off_books);
    for (int b = 0; b < H.books; ++b)
      for (int c = tid; c < H.max_centroids; c += kThreads) {
        const float x = books[b * H.max_centroids + c] * ce;
        const uint32_t w = SPLIT ? __float_as_uint(x) : pack2(x, x);
        *reinterpret_cast<uint32_t *>(smem + b * kByteBook + 8 + 4 * c) = w;
        if (c < 16) *reinterpret_cast<uint32_t *>(smem + kNibbleBooks + b * kNibbleBook + 4 + 4 * c) = w;
      }
  }
  if (tid < 8) flags[tid] = -1;

  // ---- queries: lane (h, q) holds positions 16 s + 8 h + 0..7 of column q, scaled by a power of two ----
  u32x4 qh[QS], ql[SPLIT ? QS : 1];
  float cl;  // a product's factor: scale log2(e) over the powers of two
  {
    const uint16_t *base = p.q + it.begin * p.q_row;
    // Eight values of a row of q as FP32.
    auto load8 = [&](const uint16_t *src, float (&x)[8]) {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(src);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t u = k & 1 ? w[k >> 1] >> 16 : w[k >> 1] & 0xffffu;
        x[k] = BF ? __uint_as_float(u << 16) : f16_bits_to_f32((uint16_t)u);
      }
    };
    float x[QS][8];
    if constexpr (KF == 0) {
#pragma unroll
      for (int s = 0; s < QS; ++s) load8(base + row * p.q_row + head * p.q_head + 16 * s + 8 * h, x[s]);
    } else {
      // R q on the matrix cores, 16 columns at a time, through LDS.
      constexpr int KS = D / 32, NT = D / 16;
      const u32x4 *op = reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint8_t *>(p.tables[kv]) + p.off_rot_q[kv]);
      float *const stage = reinterpret_cast<float *>(bufs) + wave * 16 * (D + 4);
      const int gq = lane >> 4, c16 = lane & 15;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int j = col0 + min((narrow ? 0 : 32 * wave) + 16 * half + c16, ncol - 1), r = j / G, hd = kv * G + (j - r * G);
        float y[KS][8], top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          load8(base + r * p.q_row + hd * p.q_head + 32 * s + 8 * gq, y[s]);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[s][e]));
        }
        const int e0 = split_exp(col_max(top));
        const float up = __builtin_ldexpf(1.0f, e0), down = __builtin_ldexpf(1.0f, -e0);
        u32x4 b[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) b[s][e] = pack2(y[s][2 * e] * up, y[s][2 * e + 1] * up);  // (16-bit values: exact)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          f32x4 a{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int o = ((t * KS + s) * 64 + lane) * 2;
            a = mfma(__builtin_bit_cast(half8, op[o]), __builtin_bit_cast(half8, b[s]), a);
            a = mfma(__builtin_bit_cast(half8, op[o + 1]), __builtin_bit_cast(half8, b[s]), a);
          }
          *reinterpret_cast<f32x4 *>(stage + c16 * (D + 4) + 16 * t + 4 * gq) = a * down;
        }
        wave_sync();
        if ((qc >> 4) == half) {
#pragma unroll
          for (int s = 0; s < QS; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const f32x4 v = *reinterpret_cast<const f32x4 *>(stage + (qc & 15) * (D + 4) + 16 * s + 8 * h + 4 * e);
#pragma unroll
              for (int k = 0; k < 4; ++k) x[s][4 * e + k] = v[k];
            }
        }
        wave_sync();
      }
    }
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
    cl = fmaxf(__builtin_ldexpf(p.c, -eq - (KF != 0 ? H.cent_exp - 14 : 0)), 0x1p-126f);  // (it meets masked logits: not 0)
  }

  f32x16 O[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[t][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;  // log2 domain; this lane's part of the sum

  // ---- rows of K and V: loaded, then rebuilt ----
  const uint8_t *const pk = KF ? p.packed + kv * p.packed_head : reinterpret_cast<const uint8_t *>(p.k + kv * p.k_head);
  const uint16_t *const pn = KF ? p.norms + kv * p.norms_head : nullptr;
  const uint8_t *const pv = p.v + kv * p.v_head;
  const uint16_t *const ps = Q8 ? p.v_scales + kv * p.vs_head : nullptr;
  const int32_t *const table = p.page_table + (int64_t)it.seq * p.page_table_stride;
  // A token's page: -1 past the sequence's, -2 where the table names none of the pool's.
  auto page_of = [&](int t) -> int {
    const int pg = table[min(t >> p.page_shift, p.table_pages - 1)];
    return t >= it.n ? -1 : (uint32_t)pg < (uint32_t)p.pages ? pg : -2;
  };
  struct KRow {
    uint32_t w[KF ? 2 : 4];
    uint32_t s[KF == 1 ? 1 : KF == 2 ? 4 : 1];
    int page;
  };
  struct VRow {
    uint32_t w[Q8 ? 2 : 4], s;
    int page;
  };
  auto load_k = [&](int t, int page, KRow &x) {
    const int64_t pg = max(page, 0);
    const int at = page < 0 ? 0 : t & ((1 << p.page_shift) - 1);
    x.page = page;
    if constexpr (KF == 0) {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(pk + (pg * p.k_page + (int64_t)at * D + 8 * oct) * 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) x.w[e] = w[e];
    } else {
      const uint8_t *src = pk + pg * p.packed_page + (int64_t)at * RB;
      __builtin_memcpy(&x.w[0], src + k_off0, 4);
      __builtin_memcpy(&x.w[1], src + k_off1, 4);
      const uint16_t *ns = pn + pg * p.norms_page + (int64_t)at * NS;
      if constexpr (KF == 1) x.s[0] = *reinterpret_cast<const uint32_t *>(ns);
      else
#pragma unroll
        for (int k = 0; k < 4; ++k) x.s[k] = ns[min(g_lo + k, NS - 1)];
    }
  };
  auto load_v = [&](int t, int page, VRow &x) {
    const int64_t pg = max(page, 0);
    const int at = page < 0 ? 0 : t & ((1 << p.page_shift) - 1);
    x.page = page;
    const uint8_t *src = pv + pg * p.v_page + ((int64_t)at * D + 8 * oct) * (Q8 ? 1 : 2);
    if constexpr (Q8) {
      const u32x2 w = *reinterpret_cast<const u32x2 *>(src);
      x.w[0] = w[0], x.w[1] = w[1];
      x.s = ps[pg * p.vs_page + at];
    } else {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(src);
#pragma unroll
      for (int e = 0; e < 4; ++e) x.w[e] = w[e];
    }
  };
  // Eight values of a K row; lo: what FP16 leaves of them.
  auto make_k = [&](const KRow &x, u32x4 &hi, u32x4 &lo) {
    if constexpr (KF == 0) {
      hi = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
    } else {
      uint32_t s01, s23 = 0;
      if constexpr (KF == 1) {
        s01 = g_lo ? x.s[0] >> 16 : x.s[0];
      } else {
        s01 = x.s[0] | x.s[1] << 16;
        s23 = x.s[2] | x.s[3] << 16;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t w = x.w[k >> 1];
        const uint32_t ca = __builtin_amdgcn_ubfe(w, ext[2 * k], tbo[2 * k]), cb = __builtin_amdgcn_ubfe(w, ext[2 * k + 1], tbo[2 * k + 1]);
        const uint32_t a = *reinterpret_cast<const uint32_t *>(smem + tbo[2 * k] + 4 * ca);
        const uint32_t b = *reinterpret_cast<const uint32_t *>(smem + tbo[2 * k + 1] + 4 * cb);
        const half2 s = __builtin_bit_cast(half2, __builtin_amdgcn_perm(s23, s01, sel[k]));
        if constexpr (SPLIT) {
          uint32_t u, v;
          split2(__uint_as_float(a) * (float)s[0], __uint_as_float(b) * (float)s[1], u, v);
          hi[k] = u;
          lo[k] = v;
        } else {
          const uint32_t c = (a & 0xffffu) | (b & 0xffff0000u);
          hi[k] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2, c) * s);
        }
      }
    }
    if (x.page < 0) {
      hi = u32x4{0u, 0u, 0u, 0u};
      if constexpr (SPLIT) lo = hi;
    }
  };
  // Eight FP16 values of a V row, zeros where there is none; odd: one of them is an infinity or a NaN.
  auto make_v = [&](const VRow &x, bool &odd) -> u32x4 {
    u32x4 v;
    if constexpr (Q8) {
      const half2 s = __builtin_bit_cast(half2, x.s | x.s << 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // c as 1024 + (c + 128) - 1152, exact
        const uint32_t u = __builtin_amdgcn_perm(0x64646464u, x.w[k >> 1] ^ 0x80808080u, k & 1 ? 0x04030402u : 0x04010400u);
        v[k] = __builtin_bit_cast(uint32_t, (__builtin_bit_cast(half2, u) - half2{(_Float16)1152.0f, (_Float16)1152.0f}) * s);
      }
    } else {
      v = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
    }
    if (x.page < 0) v = u32x4{0u, 0u, 0u, 0u};
    // (an infinity or a NaN times 0 is NaN)
    const half2 zero{(_Float16)0.0f, (_Float16)0.0f};
    float z = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) z = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2, v[k]), zero, z, false);
    odd = z != 0.0f;
    return v;
  };

  // ---- one block of NB x 32 tokens from t0 on for this wave's queries ----
  const uint32_t lds0 = lds_at(smem);
  const int vr = 4 * h + ((lane & 15) >> 2), v_piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t k_at = (uint32_t)(qc * (2 * D) + ((h ^ swizzle<D>(qc)) * 16));
  const uint32_t v_at = (uint32_t)(vr * (2 * D) + ((v_piece ^ swizzle<D>(vr)) * 16) + (lane & 1) * 8);
  const uint32_t v_at8 = (uint32_t)((vr + 8) * (2 * D) + ((v_piece ^ swizzle<D>(vr + 8)) * 16) + (lane & 1) * 8);
  // S += K Q^T of the K rows at LDS offset `at`: the operands' product, or the queries' low parts too.
  auto qk = [&](auto nb_tag, uint32_t at, f32x16 *S, bool low) {
    constexpr int NB = decltype(nb_tag)::value;
#pragma unroll
    for (int s = 0; s < QS; ++s)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const u32x4 a = *reinterpret_cast<const u32x4 *>(smem + ((at + k_at) ^ (32u * s)) + 64 * D * b);
        S[b] = product(a, qh[s], S[b]);
        if constexpr (SPLIT)
          if (low) S[b] = product(a, ql[s], S[b]);
      }
  };
  // Whether this lane's query sees token 4 h + k of a block from t0 on (bit k), of those in `there`.
  auto seen_bits = [&](int t0, uint64_t there) -> uint64_t {
    auto below = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : ~(~0ull << n); };  // bits 0 .. n - 1
    const int d = pos - t0 - 4 * h;
    uint64_t bits = below(d + 1);
    if (p.window) bits &= ~below(d + 1 - p.window) | below(p.sinks - t0 - 4 * h);
    return bits & (there >> (4 * h));
  };
  // The softmax of S (masked: to the seen tokens) into P, O rescaled where a maximum grew.
  auto softmax = [&](auto nb_tag, f32x16 *S, uint32_t *P, bool masked, uint64_t seen) {
    constexpr int NB = decltype(nb_tag)::value;
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
  };
  // O^T += V^T P^T of the V rows at LDS offset `at`. odd: some are seen by some queries only, and
  // hold infinities or NaNs: the products take the finite values, and what is
  // seen of the others is added by itself.
  auto pv_product = [&](auto nb_tag, uint32_t at, const uint32_t *P, bool odd, uint64_t seen) {
    constexpr int NB = decltype(nb_tag)::value, STEP = 16 * 2 * D;  // bytes of a step's rows
    if (!odd) {
      uint32_t va[MT], va8[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        va[t] = (lds0 + at + v_at) ^ (64u * t);
        va8[t] = (lds0 + at + v_at8) ^ (64u * t);
      }
      u32x2 v[2][MT][2];
      ds_read_tr16<MT, 0>(va, va8, v[0]);
#pragma unroll
      for (int s = 0; s < 2 * NB; ++s) {
        const u32x4 pf{P[4 * s], P[4 * s + 1], P[4 * s + 2], P[4 * s + 3]};
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const u32x2 a = v[s & 1][t][0], b = v[s & 1][t][1];
          O[t] = product(u32x4{a[0], a[1], b[0], b[1]}, pf, O[t]);
        }
        if (s == 0) ds_read_tr16<MT, STEP>(va, va8, v[1]);
        if constexpr (NB == 2) {
          if (s == 1) ds_read_tr16<MT, 2 * STEP>(va, va8, v[0]);
          if (s == 2) ds_read_tr16<MT, 3 * STEP>(va, va8, v[1]);
        }
      }
      return;
    }
    int rare = lane;
    asm volatile("" : "+v"(rare));  // (the rare branch's addresses are not held across the loop)
    const int h = rare >> 5, qc = rare & 31;
    // V of dimension 32 t + qc, tokens 16 s + 8 (e / 2) + 4 h + 2 (e % 2) + 0, 1 in word e.
    auto column = [&](int s, int t) {
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
    };
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        u32x4 a = column(s, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = finite16(a[e]);
        O[t] = product(a, u32x4{P[4 * s], P[4 * s + 1], P[4 * s + 2], P[4 * s + 3]}, O[t]);
      }
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
          u32x4 a = column(s, t), sees;
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
      }
    }
  };
  // What a wave's queries, at positions lo .. hi, see of the block of B tokens from t0 on: 0 nothing, 1 a part, 2 all.
  auto sight = [&](int t0, int B, int lo, int hi) -> int {
    if (t0 > hi) return 0;
    if (p.window && t0 + B - 1 <= lo - p.window && t0 >= p.sinks) return 0;
    return t0 + B - 1 <= lo && (!p.window || t0 > hi - p.window) ? 2 : 1;
  };

  int columns_out = ncol;
  if (!narrow) {
    // ---- wide ----
    constexpr int PASSES = kChunkKeys * O8 / kThreads, STRIDE = kThreads / O8;
    const Blocks bl = Blocks::of<kChunkKeys>(tile_first, min(tile_last, it.n - 1), p.window, p.sinks);
    const int b0 = (int)((int64_t)bl.count * it.split / it.splits), b1 = (int)((int64_t)bl.count * (it.split + 1) / it.splits);
    const int key = tid / O8;
    KRow kr[PASSES];
    VRow vw[PASSES];
    int pages[PASSES];  // of the block after the loaded one
    auto look_up = [&](int i) {
#pragma unroll
      for (int k = 0; k < PASSES; ++k) pages[k] = page_of(bl.at<kChunkKeys>(i) + key + STRIDE * k);
    };
    auto load = [&](int i) {
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        const int t = bl.at<kChunkKeys>(i) + key + STRIDE * k;
        load_k(t, pages[k], kr[k]);
        load_v(t, pages[k], vw[k]);
      }
    };
    // Block i's rows from the loaded codes into its buffer; its flags: i where a token has no page, or V an infinity or a NaN.
    auto rebuild = [&](int i) {
      uint8_t *const buf = bufs + (i & 1) * L::BUFFER;
      bool hole = false, odd = false;
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        const int r = key + STRIDE * k, at = r * (2 * D) + ((oct ^ swizzle<D>(r)) * 16);
        u32x4 hi, lo{};
        make_k(kr[k], hi, lo);
        *reinterpret_cast<u32x4 *>(buf + at) = hi;
        if constexpr (SPLIT) *reinterpret_cast<u32x4 *>(buf + 2 * TILE + at) = lo;
        bool o;
        *reinterpret_cast<u32x4 *>(buf + TILE + at) = make_v(vw[k], o);
        odd |= o;
        hole |= kr[k].page == -2;
      }
      if (__builtin_amdgcn_ballot_w64(hole) && lane == 0) flags[i & 1] = i;
      if (__builtin_amdgcn_ballot_w64(odd) && lane == 0) flags[2 + (i & 1)] = i;
    };
    // This wave's columns' positions; a wave past the unit's columns only rebuilds.
    const bool any = 32 * wave < ncol;
    const int w_lo = before + (col0 + min(32 * wave, ncol - 1)) / G, w_hi = before + (col0 + min(32 * wave + 31, ncol - 1)) / G;
    if (b0 < b1) {
      look_up(b0);
      load(b0);
      look_up(min(b0 + 1, b1 - 1));
    }
    __syncthreads();  // the books, and the queries' staging done with
    if (b0 < b1) {
      rebuild(b0);
      if (b0 + 1 < b1) {
        load(b0 + 1);
        look_up(min(b0 + 2, b1 - 1));
      }
    }
    for (int i = b0; i < b1; ++i) {
      lds_barrier();  // block i is whole, and everyone is done with the other buffer
      const bool hole = flags[i & 1] == i, odd = flags[2 + (i & 1)] == i;
      if (i + 1 < b1) {
        rebuild(i + 1);
        if (i + 2 < b1) {
          load(i + 2);
          look_up(min(i + 3, b1 - 1));
        }
      }
      const int t0 = bl.at<kChunkKeys>(i);
      const int part = any ? sight(t0, kChunkKeys, w_lo, w_hi) : 0;
      if (part == 0) continue;
      const uint32_t buf = L::BUFFERS + (uint32_t)(i & 1) * L::BUFFER;
      f32x16 S[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) S[b][e] = 0.0f;
      constexpr std::integral_constant<int, 2> two{};
      qk(two, buf, S, true);
      if constexpr (SPLIT) qk(two, buf + 2 * TILE, S, false);
      const bool masked = part == 1 || hole;
      uint64_t seen = ~0ull;
      if (masked) {
        uint64_t there = ~0ull;
        if (hole) {
          const int pg = page_of(t0 + lane);
          there = __builtin_amdgcn_ballot_w64(pg >= 0);
        }
        seen = seen_bits(t0, there);
      }
      uint32_t P[16];
      softmax(two, S, P, masked, seen);
      pv_product(two, buf + TILE, P, masked && odd, seen);
    }
  } else {
    // ---- narrow: this wave's own blocks of 32 tokens ----
    constexpr int B = 32, PASSES = B * O8 / 64, STRIDE = 64 / O8;
    const Blocks bl = Blocks::of<B>(tile_first, min(tile_last, it.n - 1), p.window, p.sinks);
    const int per = (bl.count + kChunkWaves - 1) / kChunkWaves;  // rounds of the eight waves, shared by the splits
    const int r0 = (int)((int64_t)per * it.split / it.splits), r1 = (int)((int64_t)per * (it.split + 1) / it.splits);
    const int key = lane / O8;
    const int first = r0 * kChunkWaves + wave, end = min(r1 * kChunkWaves, bl.count);
    const uint32_t own = L::BUFFERS + (uint32_t)wave * B * D * 2;
    KRow kr[PASSES];
    VRow vw[PASSES];
    int pages[PASSES];
    auto look_up = [&](int i) {
#pragma unroll
      for (int k = 0; k < PASSES; ++k) pages[k] = page_of(bl.at<B>(i) + key + STRIDE * k);
    };
    auto tokens = [&](int i, int k) { return bl.at<B>(i) + key + STRIDE * k; };
    if (first < end) {
      look_up(first);
#pragma unroll
      for (int k = 0; k < PASSES; ++k) load_k(tokens(first, k), pages[k], kr[k]);
#pragma unroll
      for (int k = 0; k < PASSES; ++k) load_v(tokens(first, k), pages[k], vw[k]);
      look_up(min(first + kChunkWaves, end - 1));
    }
    __syncthreads();  // the books, and the queries' staging done with
    for (int i = first; i < end; i += kChunkWaves) {
      const int t0 = bl.at<B>(i), next = min(i + kChunkWaves, end - 1);
      constexpr std::integral_constant<int, 1> one{};
      auto put = [&](int k, u32x4 x) {
        const int r = key + STRIDE * k;
        *reinterpret_cast<u32x4 *>(smem + own + r * (2 * D) + ((oct ^ swizzle<D>(r)) * 16)) = x;
      };
      f32x16 S[1];
#pragma unroll
      for (int e = 0; e < 16; ++e) S[0][e] = 0.0f;
      u32x4 lo[SPLIT ? PASSES : 1];
      bool hole = false;
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        u32x4 hi;
        make_k(kr[k], hi, lo[SPLIT ? k : 0]);
        put(k, hi);
        hole |= kr[k].page == -2;
      }
      // The next block's codes, from the pages looked up a block ago; its pages stay for its V.
      int next_pages[PASSES];
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        next_pages[k] = pages[k];
        load_k(tokens(next, k), pages[k], kr[k]);
      }
      wave_sync();
      qk(one, own, S, true);
      if constexpr (SPLIT) {
        wave_sync();
#pragma unroll
        for (int k = 0; k < PASSES; ++k) put(k, lo[k]);
        wave_sync();
        qk(one, own, S, false);
      }
      const bool holes = __builtin_amdgcn_ballot_w64(hole) != 0;
      const bool masked = holes || sight(t0, B, tile_first, tile_last) != 2;
      uint64_t seen = ~0ull;
      if (masked) {
        uint64_t there = ~0ull;
        if (holes) there = __builtin_amdgcn_ballot_w64(page_of(t0 + qc) >= 0);
        seen = seen_bits(t0, there);
      }
      uint32_t P[8];
      softmax(one, S, P, masked, seen);
      wave_sync();
      bool odd = false;
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        bool o;
        put(k, make_v(vw[k], o));
        odd |= o;
      }
#pragma unroll
      for (int k = 0; k < PASSES; ++k) load_v(tokens(next, k), next_pages[k], vw[k]);
      look_up(min(next + kChunkWaves, end - 1));
      wave_sync();
      pv_product(one, own, P, masked && __builtin_amdgcn_ballot_w64(odd) != 0, seen);
      wave_sync();
    }
    // The waves' states of the same columns, halved three times; wave 0 ends with the sum.
    float *const join = reinterpret_cast<float *>(bufs);
    constexpr int STATE = D / 2 + 2;  // floats of a lane
#pragma unroll
    for (int half = kChunkWaves / 2; half >= 1; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
        float *to = join + (wave - half) * 64 * STATE + lane;
        to[0] = m;
        to[64] = l;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) to[64 * (2 + 16 * t + i)] = O[t][i];
      }
      __syncthreads();
      if (wave < half) {
        const float *from = join + wave * 64 * STATE + lane;
        const float m2 = from[0], l2 = from[64];
        const float mn = fmaxf(m, m2);
        const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn), b = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m2 - mn);
        // (a state that saw nothing is all zeros)
        m = mn;
        l = l * a + l2 * b;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) O[t][i] = O[t][i] * a + from[64 * (2 + 16 * t + i)] * b;
      }
    }
    if (wave != 0) columns_out = 0;
  }

  // ---- results ----
  l = half_sum(l);
  const bool stored = mine < columns_out;
  if (it.splits == 1) {
    if (!stored) return;
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (a NaN stays one)
    uint16_t *out = p.out + (it.begin + row) * p.out_row + head * p.out_head;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<u32x2 *>(out + 32 * t + 8 * g + 4 * h) =
            u32x2{pack_out<BF>(O[t][4 * g] * inv, O[t][4 * g + 1] * inv), pack_out<BF>(O[t][4 * g + 2] * inv, O[t][4 * g + 3] * inv)};
    return;
  }
  // A split's partial: o in pieces of four dimensions, [piece][column], then (m, l) of each column; stores and
  // loads at the device's coherent level, since the merging workgroup may run on another XCD.
  const int SC = p.slot_columns;
  const uint32_t slot_bytes = (uint32_t)SC * (D + 2) * 4;
  uint8_t *const part = reinterpret_cast<uint8_t *>(p.part);
  if (stored) {
    const __amdgpu_buffer_rsrc_t r = rsrc(part + (int64_t)(it.slot0 + it.split) * slot_bytes, slot_bytes);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        __builtin_amdgcn_raw_buffer_store_b128(
            __builtin_bit_cast(u32x4, (f32x4{O[t][4 * g], O[t][4 * g + 1], O[t][4 * g + 2], O[t][4 * g + 3]})), r,
            (int)(((8 * t + 2 * g + h) * SC + mine) * 16), 0, kPolicySc1);
    if (h == 0)
      __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, r, (int)(D * SC * 4 + mine * 8), 0, kPolicySc1);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  uint32_t *const counter = p.counters + it.slot0;
  if (tid == 0)
    flags[4] = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(it.splits - 1);
  __syncthreads();
  if (!flags[4]) return;
  for (int e = tid; e < ncol * (D / 4); e += kThreads) {
    const int piece = e / ncol, c = e - piece * ncol;
    auto slot = [&](int s) { return rsrc(part + (int64_t)(it.slot0 + s) * slot_bytes, slot_bytes); };
    float M = -INFINITY, sum = 0.0f;
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int N = 8;  // splits whose loads are in flight together
    for (int s0 = 0; s0 < it.splits; s0 += N) {
      u32x2 ml[N];
      f32x4 x[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const __amdgpu_buffer_rsrc_t r = slot(min(s0 + k, it.splits - 1));
        ml[k] = coherent_load2(r, (uint32_t)(D * SC * 4 + c * 8));
        x[k] = coherent_load4(r, (uint32_t)((piece * SC + c) * 16));
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
        const bool live = s0 + k < it.splits && mk != -INFINITY;
        const float w = live ? __builtin_amdgcn_exp2f(mk - M) : 0.0f;
        sum = live ? __builtin_fmaf(__uint_as_float(ml[k][1]), w, sum) : sum;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = live ? __builtin_fmaf(x[k][d], w, o[d]) : o[d];
      }
    }
    const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
    const int j = col0 + c, r = j / G;
    uint16_t *out = p.out + (it.begin + r) * p.out_row + (kv * G + (j - r * G)) * p.out_head;
    *reinterpret_cast<u32x2 *>(out + 4 * piece) = u32x2{pack_out<BF>(o[0] * inv, o[1] * inv), pack_out<BF>(o[2] * inv, o[3] * inv)};
  }
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int D, int KF, bool Q8, bool BF>
hipError_t launch_one(const ChunkParams &p, hipStream_t stream) {
  constexpr int lds = ChunkLds<D, KF, KF != 0 && !BF>::BYTES;
  static_assert(lds <= kLdsLimit, "LDS of one workgroup");
  static const hipError_t allowed =
      hipFuncSetAttribute((const void *)chunk_kernel<D, KF, Q8, BF>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (allowed != hipSuccess) {
    (void)hipGetLastError();
    return allowed;
  }
  hipLaunchKernelGGL((chunk_kernel<D, KF, Q8, BF>), dim3((unsigned)chunk_items(p)), dim3(kThreads), lds, stream, p);
  return hipGetLastError();
}
template <int D, int KF>
hipError_t launch_k(const ChunkParams &p, bool bf16, hipStream_t stream) {
  if (p.v_scales) return bf16 ? launch_one<D, KF, true, true>(p, stream) : launch_one<D, KF, true, false>(p, stream);
  return bf16 ? launch_one<D, KF, false, true>(p, stream) : launch_one<D, KF, false, false>(p, stream);
}

}  // namespace
}  // namespace bgtq
