// Causal attention over whole prompts packed one after another
// (bgtq_prompt_attention): FP16 or BF16 rows, grouped heads, one pass over the
// keys with a running maximum and sum (src/model/attention.wgsl:13-39 computes
// the same in three passes with materialised scores).
//
// A workgroup takes kWaves x 32 query rows of one sequence and head, a wave 32
// of them as the columns of 32x32x16 products. S^T = K Q^T leaves lane (h, q) =
// (lane / 32, lane % 32) with query q's logits of the keys 8 (i / 4) + 4 h + i % 4
// in registers i: a query's maximum and sum are taken in registers and over
// one lane swap, its rescale factor is a lane's own, and the probabilities,
// rounded to the rows' type, are the B operand of O^T += V^T P^T as they lie
// (the product's 16 slots hold the keys in that order on both sides). V^T is
// read from LDS by the transposing reads. Blocks of kKeys keys go HBM -> LDS by
// DMA, 16-byte pieces XOR-swizzled by row, into two buffers: one barrier per
// block, the next block in flight under the current one's products.
//
// The running maximum is raised only when a block's exceeds it by more than 8
// (FP16 4) in the log2 domain, so most blocks skip the rescale of O. FP16
// probabilities are carried times 2^11, which the division by their sum takes
// out: at most 2^15 then, and those of 2^-25 of the maximum and up keep all
// their bits, where many small ones beside a large one whose V is small are the
// output (below, they are subnormal, off by 2^-36 of the maximum at most).
// 8192 tokens of d=128 in FP16 276 us with a threshold of 4, 301 with 1.
//
// Probabilities in the rows' type, and their sum of the same rounded values,
// leave the outputs 1.3 times as far from 64 bits as results that are rounded
// once (11 mixed prompts BF16 2.1e-3 and 1.6e-3 of their norm, FP16 2.6e-4 and
// 2.0e-4). A high and a low part of each in two products reach the latter, and
// take 128 us for 94, 8192 tokens of d=128 427 for 283: the rows carry no more bits.
//
// Measured (several boxes): 11 prompts of 568 to 2777 tokens, 14 / 2 heads of d=64,
// 85 to 92 us (700 to 760 TFLOP/s), one of 8192 tokens, 16 / 4 heads of d=128, 258 to 268 us
// (1025 to 1065 TFLOP/s; a bf16 product of 8192^3 reaches 1249). A wave's block is 512 cycles of products and
// 870 of softmax at d=64 (1024 at d=128), of which 512 are exponentials (a quarter
// of the vector rate): the vector unit bounds d=64 (70% busy), the matrix cores
// d=128 (52%), and what the waves of a SIMD do not overlap of the two. A step's V
// arrives behind the step before's products, waited for where it is read (one
// prompt of 8192 tokens 1.2% slower than with each read waited for at its use).
// Nothing splits the keys: a tile's history is one workgroup's chain, and few
// tiles and heads leave compute units idle (4096 tokens on 4 heads of d=128 88 us,
// where their products take 14).
// At d=64 the 128 registers of four waves per SIMD leave 16 or 32 bytes of scratch
// to the branch for V rows with infinities or NaNs, none to the others.
#include <type_traits>

#include "bgtq_internal.h"
#include "gfx950_common.h"

namespace bgtq {
namespace {

using namespace gfx;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = kPromptThreads, kWaves = kThreads / 64;
constexpr int kRows = 32 * kWaves;  // query rows of a workgroup
constexpr int kKeys = 64;           // keys of a block
// Growth of a maximum (log2) that O is not rescaled for, and the power of two
// that probabilities are carried times.
template <bool BF>
constexpr float kLazy = BF ? 8.0f : 4.0f;
template <bool BF>
constexpr float kShift = BF ? 0.0f : 11.0f;

struct PromptParams {
  const int32_t *offsets;
  int32_t sequences, heads, group;  // query heads; per KV head
  int64_t tokens;
  const uint16_t *q, *k, *v;
  uint16_t *out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;  // elements
  float c;  // scale * log2(e)
};

// XOR of a row's 16-byte piece indexes: 16 rows' reads of one piece (K) and
// four rows' reads of four neighbouring pieces (V) use every bank once.
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  return D == 64 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
}

template <bool BF>
__device__ __forceinline__ f32x16 product(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// Two values rounded to nearest even, packed.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), half2));
}

// c plus the two values of a pair.
template <bool BF>
__device__ __forceinline__ float add2(uint32_t pair, float c) {
  if constexpr (BF)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), bf16x2{(__bf16)1.0f, (__bf16)1.0f}, c, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2, pair), half2{(_Float16)1.0f, (_Float16)1.0f}, c, false);
}

// Infinities and NaNs among pairs of 16-bit values: the pair's magnitudes
// (their order is the integers'), and the values of one kind (0 NaN, 1
// infinity, 2 minus infinity) as 1, the others as 0; `finite`: the others kept.
template <bool BF>
struct Odd {
  static constexpr uint32_t kInf = BF ? 0x7f80u : 0x7c00u, kOne = BF ? 0x3f80u : 0x3c00u;
  static __device__ __forceinline__ uint32_t finite(uint32_t w) {
    return ((w & 0x7fffu) >= kInf ? 0u : w & 0xffffu) | ((w >> 16 & 0x7fffu) >= kInf ? 0u : w & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t of_kind(uint32_t w, int kind) {
    auto is = [&](uint32_t x) {
      return kind == 0 ? (x & 0x7fffu) > kInf : x == (kind == 1 ? kInf : kInf | 0x8000u);
    };
    return (is(w & 0xffffu) ? kOne : 0u) | (is(w >> 16) ? kOne << 16 : 0u);
  }
};

// Ties an accumulator to its registers. After each element's update under a
// branch: without it the update builds a second copy of the accumulator, and
// every block of keys moves it there and back (64 moves at d=64).
__device__ __forceinline__ void in_place(f32x16 &o) { asm volatile("" : "+v"(o)); }

// The other half's value of a query's pair of lanes.
__device__ __forceinline__ float half_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The sequence and its tile of kRows rows that grid slot `slot` stands for.
// Workgroups start in the order of their slots, and a tile's work is its
// history: the longest histories of all sequences come first, or a long
// sequence's would be left running alone at the end (11 prompts of 568 to 2777
// tokens 92 us, sequence by sequence 100). Tiles i of all the sequences that have
// one make level i; with C(i) the tiles of levels i and up, the slot's level
// is the last one with C(i) > slot, found bit by bit, a lane per sequence.
// More than 64 sequences: sequence by sequence, sequence s owning the slots from
// offsets[s] / kRows + s on, at least as many as it has tiles; the last
// sequence that starts at or before the slot is found 64 candidates at a time.
// Every wave finds the place by itself.
struct Place {
  int64_t begin;
  int len, tile;  // tile < 0: nothing to do
};
__device__ __forceinline__ Place find_place(const PromptParams &p, int64_t slot) {
  const int lane = threadIdx.x & 63;
  auto offset = [&](int s) {
    const int64_t o = p.offsets[s];
    return o < 0 ? 0 : o > p.tokens ? p.tokens : o;
  };
  if (p.sequences <= 64) {
    const int64_t begin = offset(min(lane, p.sequences)), end = offset(min(lane + 1, p.sequences));
    const int len = end > begin ? (int)(end - begin) : 0, tiles = (int)(((int64_t)len + kRows - 1) / kRows);
    auto tiles_from = [&](int level) { return wave_sum(max(tiles - level, 0)); };
    int level = 0, below = 0;  // below: C(level + 1)
    for (int bit = 1 << (31 - __builtin_clz((int)(p.tokens / kRows) + 1)); bit; bit >>= 1) {
      const int c = __builtin_amdgcn_readfirstlane(tiles_from(level + bit));
      if (c > slot) level += bit;
      else below = c;
    }
    const bool here = tiles > level;
    const uint64_t row = __builtin_amdgcn_ballot_w64(here);
    const int rank = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(row >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)row, 0u));
    const uint64_t mine = __builtin_amdgcn_ballot_w64(here && rank == (int)slot - below);
    if (mine == 0) return {0, 0, -1};
    const int at = __builtin_ctzll(mine);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)begin, at);
    return {(int64_t)lo, __builtin_amdgcn_readlane(len, at), level};
  }
  int lo = 0, n = p.sequences;
  for (;;) {
    const int step = (n + 63) / 64, at = lane * step;
    const int s = lo + (at < n ? at : 0);
    const int hits = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at < n && offset(s) / kRows + s <= slot));
    if (hits == 0) return {0, 0, -1};
    lo += (hits - 1) * step;
    n = min(step, n - (hits - 1) * step);
    if (step == 1) break;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int64_t begin = offset(lo), end = offset(lo + 1);
  Place r{begin, end > begin ? (int)(end - begin) : 0, 0};
  const int64_t local = slot - (begin / kRows + lo), tiles = (r.len + kRows - 1) / kRows;
  r.tile = local < tiles ? (int)(tiles - 1 - local) : -1;  // the longest histories first
  return r;
}

template <int D, bool BF>
__global__ __launch_bounds__(kThreads, D == 64 ? 4 : 2) void prompt_kernel(PromptParams p) {
  constexpr int PR = D / 8;                      // 16-byte pieces per row
  constexpr int QS = D / 16;                     // 16-dimension steps of QK
  constexpr int MT = D / 32;                     // 32-dimension tiles of O
  constexpr int BLOCK = kKeys * D * 2;           // bytes of a block of K or V
  constexpr int DMAS = BLOCK / 1024 / kWaves;    // DMAs per wave and operand
  __shared__ __align__(16) uint8_t smem[4 * BLOCK];  // K, V of block 0; K, V of block 1
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, qc = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t slot = blockIdx.x / (uint32_t)p.heads;
  const int head = (int)(blockIdx.x - slot * (uint32_t)p.heads), kv = head / p.group;
  const Place at = find_place(p, slot);
  if (at.tile < 0) return;  // uniform for the workgroup
  const int q0 = at.tile * kRows, row0 = q0 + 32 * wave;  // the workgroup's, this wave's first query
  const int qi = row0 + qc;                               // this lane's query
  const int n_blocks = (min(q0 + kRows, at.len) + kKeys - 1) / kKeys;

  const uint16_t *k_base = p.k + at.begin * p.k_row + kv * p.k_head;
  const uint16_t *v_base = p.v + at.begin * p.v_row + kv * p.v_head;
  // Block j's rows inside the sequence; the others arrive as zeros.
  auto issue = [&](int j) {
    const int rest = min(kKeys, at.len - j * kKeys);
    uint8_t *buf = smem + (j & 1) * 2 * BLOCK;
    const __amdgpu_buffer_rsrc_t rk = rsrc(k_base + (int64_t)j * kKeys * p.k_row, (uint32_t)(((rest - 1) * p.k_row + D) * 2));
    const __amdgpu_buffer_rsrc_t rv = rsrc(v_base + (int64_t)j * kKeys * p.v_row, (uint32_t)(((rest - 1) * p.v_row + D) * 2));
#pragma unroll
    for (int i = 0; i < DMAS; ++i) {
      const int piece = (wave * DMAS + i) * 64 + lane, r = piece / PR, c = (piece % PR) ^ swizzle<D>(r);
      dma16(rk, buf + (wave * DMAS + i) * 1024, (uint32_t)(r * (int)p.k_row * 2 + c * 16), 0);
      dma16(rv, buf + BLOCK + (wave * DMAS + i) * 1024, (uint32_t)(r * (int)p.v_row * 2 + c * 16), 0);
    }
  };
  // Q: lane (h, q) holds dimensions 16 s + 8 h + 0..7 of query q (past the
  // sequence: its last row's, not stored).
  u32x4 qf[QS];
  {
    const uint16_t *row = p.q + (at.begin + min(qi, at.len - 1)) * p.q_row + head * p.q_head;
#pragma unroll
    for (int s = 0; s < QS; ++s) qf[s] = *reinterpret_cast<const u32x4 *>(row + 16 * s + 8 * h);
    // Waited for here: left to the loop, the wait would take the next block's DMAs with it.
#pragma unroll
    for (int s = 0; s < QS; ++s) asm volatile("" : "+v"(qf[s]));
  }
  issue(0);
  f32x16 O[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[t][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;  // log2 domain; this lane's part of the sum

  // LDS addresses of this lane in a block: K, piece h of row qc (step s: ^ 32 s,
  // rows 32 on: + 64 D); V, its part of rows 4 h + (lane % 16) / 4 (tile t: ^ 64 t)
  // and 8 rows on. The swizzle of a row depends on its lane's part alone.
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void *)smem;
  const uint32_t k_at = (uint32_t)(qc * (2 * D) + ((h ^ swizzle<D>(qc)) * 16));
  const int vr = 4 * h + ((lane & 15) >> 2);
  const int v_piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_at = (uint32_t)(vr * (2 * D) + ((v_piece ^ swizzle<D>(vr)) * 16) + (lane & 1) * 8);
  const uint32_t v_at8 = (uint32_t)((vr + 8) * (2 * D) + ((v_piece ^ swizzle<D>(vr + 8)) * 16) + (lane & 1) * 8);

  // Every wave meets every block's barrier and loads its part of every block.
  auto arrive = [&](int j) {
    wait_vm<0>();   // this wave's part of block j has landed (and every earlier load)
    lds_barrier();  // everyone's has, and everyone is done with the other buffer
    if (j + 1 < n_blocks) issue(j + 1);
  };
  // d=128: the two waves of a SIMD issue their softmax ahead of each other's
  // products, which need an issue slot every 32 cycles only (one prompt of 8192
  // tokens 257 us; without 276, products first 288). d=64's four waves fill the
  // vector unit without (11 prompts 87 us, 89 with).
  auto softmax_first = [](int on) {
    if constexpr (D == 128) {
      __builtin_amdgcn_sched_barrier(0);
      if (on) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Block j's keys for this wave's queries; DIAGONAL: some queries see only a part of them.
  auto attend = [&](auto diagonal_tag, int j) {
    constexpr bool DIAGONAL = decltype(diagonal_tag)::value;
    const uint32_t buf = (uint32_t)(j & 1) * 2 * BLOCK;
    f32x16 S[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[b][i] = 0.0f;
#pragma unroll
    for (int s = 0; s < QS; ++s)
#pragma unroll
      for (int b = 0; b < 2; ++b) {  // A operand: key 32 b + qc
        const u32x4 a = *reinterpret_cast<const u32x4 *>(smem + ((buf + k_at) ^ (32u * s)) + 64 * D * b);
        S[b] = product<BF>(a, qf[s], S[b]);
      }
    if constexpr (DIAGONAL) {
      const int d = qi - j * kKeys - 4 * h;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) S[b][i] = 32 * b + 8 * (i >> 2) + (i & 3) <= d ? S[b][i] : -INFINITY;
    }
    softmax_first(1);
    float top = S[0][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, S[0][i]);
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, S[1][i]);
    top = half_max(top) * p.c;
    if (__builtin_amdgcn_ballot_w64(top > m + kLazy<BF>)) {  // (also the first block: m = -inf)
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
    const float mu = (m == -INFINITY ? 0.0f : m) - kShift<BF>;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[b][i], p.c, -mu));
    // The probabilities rounded to the rows' type; the sum is theirs, so a
    // query with one key's whole weight gets that key's V exactly.
    uint32_t P[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      P[e] = pack2<BF>(S[e >> 3][2 * (e & 7)], S[e >> 3][2 * (e & 7) + 1]);
      l = add2<BF>(P[e], l);
    }
    softmax_first(0);
    // O^T += V^T P^T, 16 keys a step, the next step's V on its way meanwhile.
    uint32_t va[MT], va8[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      va[t] = (lds0 + buf + BLOCK + v_at) ^ (64u * t);
      va8[t] = (lds0 + buf + BLOCK + v_at8) ^ (64u * t);
    }
    // A key that a query does not see has probability 0, but 0 times an
    // infinity or a NaN of its V row is not 0: such a block's products take
    // the finite values, and what is seen of the others is added by itself.
    bool plain = true;
    if constexpr (DIAGONAL) {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 most{0, 0};
#pragma unroll
      for (int i = 0; i < PR; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(smem + buf + BLOCK + (64 * i + lane) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
      }
      plain = __builtin_amdgcn_ballot_w64(most[0] >= Odd<BF>::kInf || most[1] >= Odd<BF>::kInf) == 0;
    }
    if (!DIAGONAL || plain) {
      constexpr int STEP = 16 * 2 * D;  // bytes of a step's rows
      u32x2 v[2][MT][2];
      ds_read_tr16<MT, 0>(va, va8, v[0]);
#pragma unroll
      for (int s = 0; s < kKeys / 16; ++s) {
        const u32x4 pf{P[4 * s], P[4 * s + 1], P[4 * s + 2], P[4 * s + 3]};
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const u32x2 a = v[s & 1][t][0], b = v[s & 1][t][1];
          O[t] = product<BF>(u32x4{a[0], a[1], b[0], b[1]}, pf, O[t]);
        }
        if (s == 0) ds_read_tr16<MT, STEP>(va, va8, v[1]);
        if (s == 1) ds_read_tr16<MT, 2 * STEP>(va, va8, v[0]);
        if (s == 2) ds_read_tr16<MT, 3 * STEP>(va, va8, v[1]);
      }
    } else {
      const int d = qi - j * kKeys - 4 * h;
      // V of dimension 32 t + qc, keys 16 s + 8 (e / 2) + 4 h + 2 (e % 2) + 0, 1 in word e.
      auto column = [&](int s, int t) {
        u32x4 a;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = 0;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int r = 16 * s + 8 * (e >> 1) + 4 * h + 2 * (e & 1) + x;
            const uint8_t *at = smem + buf + BLOCK + r * (2 * D) + (((4 * t + (qc >> 3)) ^ swizzle<D>(r)) * 16) + 2 * (qc & 7);
            a[e] |= (uint32_t)*reinterpret_cast<const uint16_t *>(at) << (16 * x);
          }
        }
        return a;
      };
#pragma unroll
      for (int s = 0; s < kKeys / 16; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          u32x4 a = column(s, t);
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = Odd<BF>::finite(a[e]);
          O[t] = product<BF>(a, u32x4{P[4 * s], P[4 * s + 1], P[4 * s + 2], P[4 * s + 3]}, O[t]);
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
          for (int s = 0; s < kKeys / 16; ++s) {
            u32x4 a = column(s, t), seen;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = 16 * s + 8 * (e >> 1) + 2 * (e & 1);
              a[e] = Odd<BF>::of_kind(a[e], kind);
              seen[e] = (k <= d ? Odd<BF>::kOne : 0u) | (k + 1 <= d ? Odd<BF>::kOne << 16 : 0u);
            }
            n = product<BF>(a, seen, n);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            O[t][i] = n[i] > 0.0f ? O[t][i] + value : O[t][i];
            in_place(O[t]);
          }
        }
      }
    }
  };
  // One block holds the wave's diagonal (32 rows lie within one); those after
  // it hold no key that its queries see. Loops of their own, so that the full
  // blocks' carries none of the diagonal's code.
  const int jd = row0 / kKeys;
  int j = 0;
  for (; j < min(jd, n_blocks); ++j) {
    arrive(j);
    attend(std::false_type{}, j);
  }
  if (j < n_blocks) {
    arrive(j);
    attend(std::true_type{}, j);
    ++j;
  }
  for (; j < n_blocks; ++j) arrive(j);
  l = half_sum(l);
  if (qi >= at.len) return;
  const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (a NaN stays one)
  uint16_t *out = p.out + (at.begin + qi) * p.out_row + head * p.out_head;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<u32x2 *>(out + 32 * t + 8 * g + 4 * h) =
          u32x2{pack2<BF>(O[t][4 * g] * inv, O[t][4 * g + 1] * inv), pack2<BF>(O[t][4 * g + 2] * inv, O[t][4 * g + 3] * inv)};
}

template <int D, bool BF>
hipError_t launch_d(const PromptParams &p, int64_t wgs, hipStream_t stream) {
  hipLaunchKernelGGL((prompt_kernel<D, BF>), dim3((unsigned)wgs), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

int64_t prompt_workgroups(const bgtq_prompt_desc &d) { return (d.tokens / kRows + d.sequences) * d.q_heads; }

hipError_t launch_prompt_attention(const bgtq_prompt_desc &d, hipStream_t stream) {
  PromptParams p{};
  p.offsets = d.offsets;
  p.sequences = d.sequences;
  p.heads = d.q_heads;
  p.group = d.q_heads / d.kv_heads;
  p.tokens = d.tokens;
  p.q = static_cast<const uint16_t *>(d.q);
  p.k = static_cast<const uint16_t *>(d.k);
  p.v = static_cast<const uint16_t *>(d.v);
  p.out = static_cast<uint16_t *>(d.out);
  p.q_row = d.q_row_stride, p.q_head = d.q_head_stride;
  p.k_row = d.k_row_stride, p.k_head = d.k_head_stride;
  p.v_row = d.v_row_stride, p.v_head = d.v_head_stride;
  p.out_row = d.out_row_stride, p.out_head = d.out_head_stride;
  p.c = (d.scale > 0.0f ? d.scale : (float)(1.0 / __builtin_sqrt((double)d.dim))) * kLog2e;
  const int64_t wgs = prompt_workgroups(d);
  if (d.dim == 64)
    return d.dtype == BGTQ_DTYPE_BF16 ? launch_d<64, true>(p, wgs, stream) : launch_d<64, false>(p, wgs, stream);
  return d.dtype == BGTQ_DTYPE_BF16 ? launch_d<128, true>(p, wgs, stream) : launch_d<128, false>(p, wgs, stream);
}

}  // namespace bgtq
