// Rows of the paged cache as the chunk attention multiplies them, and the
// kernel for what a wave does with blocks of its own: narrow units (at most 32
// query columns) of bgtq_paged_prefill, and the rows of wide ones rebuilt once.
//
// K is rebuilt in the code domain: k = R^T cs, so q . k = (R q) . cs. The
// queries are rotated once, and K's row is c_j s_g(j), one table lookup and one
// product a value, rounded to FP16 (c scaled by the books' largest power of two:
// |c| <= 1, so a finite scale's row is finite, and rows whose scale is a
// normal FP16 number lose nothing against their largest value). BF16 queries
// multiply it as it is; FP16 ones carry three bits more and take K and q as
// pairs of FP16 values (three products), K's low part times 2^11: products with
// it come first and are scaled down before the others are added, 32 multiplies a
// block of the wide kernel (13 sequences of the calibration heads, 301 new rows:
// 68.4 -> 69.4 us). 8-bit V becomes its FP16 values.
//
// A wave takes 32 tokens at a time, which lie in one page (so its address is
// the wave's), a lane eight consecutive values of PASSES rows. Narrow units: the
// eight waves of a workgroup have the same columns and blocks of their own,
// without barriers, K and then V of a block through 32 rows of LDS, the next
// block's codes on their way meanwhile; their states are joined at the end. FP16
// rows come by DMA (loaded into registers a round of eight blocks took 7 us).
//
// What bounds it: one workgroup of eight waves per compute unit (201 to 256
// registers and 142 KB of LDS at d=128), so a chain of set-up, two or three rounds of
// blocks, join and merge. 16 sequences of five new rows on 16 / 4 heads of d=128,
// up to 4099 tokens in FP16 pages: 20.2 us (3.6 TB/s), of which 5 the launch and finding
// the item, 4 the queries, 8 the rounds, 2 the join, 1 the merge. The rebuilding of a
// call's wide rows is bound by what it writes: 2 x 3048 seen tokens x 8 heads of
// d=128 (25 MB) 11 us behind the first 5.
#pragma once

#include "chunk_wave.h"

namespace bgtq {
namespace {

constexpr int kThreads = 64 * kChunkWaves;

// LDS: the books (as paged_rows.hip's: a byte code's at book * 1056 + 8, a
// nibble code's 16 behind them at book * 96 + 4: an offset's low five bits are the
// bit-field extract's width), a flag, then the waves' rows.
constexpr int kByteBook = 1056, kNibbleBook = 96, kNibbleBooks = 8 * kByteBook, kBookBytes = kNibbleBooks + 8 * kNibbleBook;
constexpr int most_of(int a, int b) { return a > b ? a : b; }
template <int D, int KF>
struct RowsLds {
  static constexpr int BOOKS = KF ? kBookBytes : 0;
  static constexpr int FLAG = BOOKS, ROWS = BOOKS + 256;  // (row pieces are XORed into addresses: whole 256 bytes)
  static constexpr int HALF = 32 * D * 2;                 // 32 rows
  static constexpr int OWN = KF ? HALF : 2 * HALF;        // a wave's rows: K then V; FP16 K: K, V
  static constexpr int STATE = D / 8 * 64 * 16;           // a wave's O; (m, l) of its columns lie behind all of them
  static constexpr int JOIN = kChunkWaves * (STATE + 32 * 8);
  static constexpr int STAGE = most_of(32 * (D + 4) * 4, kChunkWaves * kStageBytes);  // rotated queries
  static constexpr int BYTES = ROWS + most_of(most_of(kChunkWaves * OWN, JOIN), STAGE);
};

// The lane's eighths of 32 rows of KV head kv. KF: 0 FP16 K, 1 packed of norm stride 2, 2 packed of any.
template <int D, int KF, bool Q8, bool SPLIT>
struct Rows {
  static constexpr int O8 = D / 8, PASSES = 32 * O8 / 64, STRIDE = 64 / O8;
  static constexpr int NW = KF ? 2 : 4, NS_ = KF == 2 ? 4 : 1, VW = Q8 ? 2 : 4;
  const uint8_t *smem;
  const uint8_t *pk, *pv;
  const uint16_t *pn, *ps;
  int64_t k_page, n_page, v_page, s_page;  // bytes, elements, bytes, elements
  int rb, ns, oct, key;                    // row bytes, norm stride; this lane's eighth, its first row
  uint32_t ext[8], tbo[8], sel[4];
  int k_off0, k_off1, n_off;
  bool upper;  // KF 1: the eighth begins in group 1
  uint32_t kw[PASSES][NW], kn[PASSES][NS_], vw[PASSES][VW], vn[PASSES];

  __device__ __forceinline__ Rows(const ChunkParams &p, int kv, const uint8_t *lds) : smem(lds) {
    const int lane = threadIdx.x & 63;
    oct = lane % O8, key = lane / O8;
    const auto &H = p.head[kv];
    rb = KF ? H.row_bytes : 2 * D, ns = H.norm_stride;
    pk = KF ? p.packed + kv * p.packed_head : reinterpret_cast<const uint8_t *>(p.k + kv * p.k_head);
    k_page = KF ? p.packed_page : 2 * p.k_page;
    pn = KF ? p.norms + kv * p.norms_head : nullptr;
    n_page = p.norms_page;
    pv = p.v + kv * p.v_head;
    v_page = p.v_page;
    ps = Q8 ? p.v_scales + kv * p.vs_head : nullptr;
    s_page = p.vs_page;
    k_off0 = k_off1 = n_off = 0;
    upper = false;
    if constexpr (KF != 0) {
      const BGTQ_GLOBAL uint8_t *Tb = reinterpret_cast<const BGTQ_GLOBAL uint8_t *>(to_global(p.tables[kv]));
      const BGTQ_GLOBAL uint32_t *gd = reinterpret_cast<const BGTQ_GLOBAL uint32_t *>(Tb + H.off_gdesc) + 8 * oct;
      uint32_t d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = gd[e];
      // Codes 0..3 lie in the word at byte k_off0, 4..7 in the one at k_off1 (not past the row's end).
      k_off0 = min((int)(d[0] & 255u), rb - 4), k_off1 = min((int)(d[4] & 255u), rb - 4);
      const int g_lo = (int)(d[0] >> 16 & 7u);
      n_off = KF == 2 ? g_lo : 0;
      upper = KF == 1 && g_lo != 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t book = d[e] >> 12 & 15u;
        tbo[e] = d[e] >> 11 & 1u ? kNibbleBooks + book * kNibbleBook + 4 : book * kByteBook + 8;
        ext[e] = 8 * ((d[e] & 255u) - (uint32_t)(e < 4 ? k_off0 : k_off1)) + (d[e] >> 8 & 7u);
      }
      // A value pair's scales, picked from those of groups g_lo .. g_lo + 3 (two words).
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t a = (d[2 * k] >> 16 & 7u) - g_lo, b = (d[2 * k + 1] >> 16 & 7u) - g_lo;
        sel[k] = (2 * a) | (2 * a + 1) << 8 | (2 * b) << 16 | (2 * b + 1) << 24;
      }
    }
  }
  // The books to LDS (all threads; the caller's barrier follows).
  __device__ __forceinline__ static void books(const ChunkParams &p, int kv, uint8_t *lds) {
    if constexpr (KF != 0) {
      const auto &H = p.head[kv];
      const BGTQ_GLOBAL float *from = reinterpret_cast<const BGTQ_GLOBAL float *>(
          reinterpret_cast<const BGTQ_GLOBAL uint8_t *>(to_global(p.tables[kv])) + H.off_books);
      // cent_exp: max |c| 2^cent_exp lies in (2^13, 2^14].
      const float ce = __builtin_ldexpf(1.0f, H.cent_exp - 14);
      for (int b = 0; b < H.books; ++b)
        for (int c = threadIdx.x; c < H.max_centroids; c += kThreads) {
          const float x = from[b * H.max_centroids + c] * ce;
          const uint32_t w = SPLIT ? __float_as_uint(x) : pack2(x, x);
          *reinterpret_cast<uint32_t *>(lds + b * kByteBook + 8 + 4 * c) = w;
          if (c < 16) *reinterpret_cast<uint32_t *>(lds + kNibbleBooks + b * kNibbleBook + 4 + 4 * c) = w;
        }
    }
  }
  // Byte of this lane's eighth of pass k's row in 32 rows of LDS, pieces XORed by row.
  __device__ __forceinline__ uint32_t place(int k) const {
    const uint32_t first = (uint32_t)(key * (2 * D) + ((oct ^ swizzle<D>(key)) * 16));
    // (swizzle(key + STRIDE k) = swizzle(key) ^ 2 (k % 2) at d=64, ^ k % 4 at d=128)
    return (first ^ (D == 64 ? 32u * (k & 1) : 16u * (k & 3))) + (uint32_t)(STRIDE * k * 2 * D);
  }
  // The codes of the 32 rows from row `at` of page `page` (the wave's) on. A pass's rows are added to the
  // wave's base, so that the lane's offsets are the same for all passes (held for each, they took up to 64 registers).
  __device__ __forceinline__ void load_k(int page, int at) {
    const uint8_t *src = scalar(pk + (int64_t)page * k_page + (int64_t)at * rb);
    const uint16_t *n = KF ? scalar(pn + (int64_t)page * n_page + (int64_t)at * ns) : nullptr;
#pragma unroll
    for (int k = 0; k < PASSES; ++k) {
      const uint8_t *row = src + STRIDE * k * rb;
      const uint16_t *scales = KF ? n + STRIDE * k * ns : nullptr;
      if constexpr (KF == 0) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(row + (uint32_t)(key * (2 * D) + 16 * oct));
#pragma unroll
        for (int e = 0; e < 4; ++e) kw[k][e] = w[e];
      } else {
        __builtin_memcpy(&kw[k][0], row + (uint32_t)(key * rb + k_off0), 4);
        __builtin_memcpy(&kw[k][1], row + (uint32_t)(key * rb + k_off1), 4);
        if constexpr (KF == 1) kn[k][0] = *reinterpret_cast<const uint32_t *>(scales + (uint32_t)(2 * key));
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) kn[k][e] = scales[(uint32_t)(key * ns + min(n_off + e, ns - 1))];
      }
    }
  }
  __device__ __forceinline__ void load_v(int page, int at) {
    const uint8_t *src = scalar(pv + (int64_t)page * v_page + (int64_t)at * (Q8 ? D : 2 * D));
    const uint16_t *s = Q8 ? scalar(ps + (int64_t)page * s_page + at) : nullptr;
#pragma unroll
    for (int k = 0; k < PASSES; ++k) {
      const uint8_t *row = src + STRIDE * k * (Q8 ? D : 2 * D);
      if constexpr (Q8) {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(row + (uint32_t)(key * D + 8 * oct));
        vw[k][0] = w[0], vw[k][1] = w[1];
        vn[k] = (s + STRIDE * k)[(uint32_t)key];
      } else {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(row + (uint32_t)(key * (2 * D) + 16 * oct));
#pragma unroll
        for (int e = 0; e < 4; ++e) vw[k][e] = w[e];
        vn[k] = 0;
      }
    }
  }
  // Eight values of pass k's K row; lo: what FP16 leaves of them, times 2^11.
  __device__ __forceinline__ void make_k(int k, u32x4 &hi, u32x4 &lo) const {
    if constexpr (KF == 0) {
      hi = u32x4{kw[k][0], kw[k][1], kw[k][NW - 2], kw[k][NW - 1]};
    } else {
      uint32_t s01, s23 = 0;
      if constexpr (KF == 1) {
        s01 = upper ? kn[k][0] >> 16 : kn[k][0];
      } else {
        s01 = kn[k][0] | kn[k][NS_ - 3] << 16;
        s23 = kn[k][NS_ - 2] | kn[k][NS_ - 1] << 16;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = kw[k][j >> 1];
        const uint32_t ca = __builtin_amdgcn_ubfe(w, ext[2 * j], tbo[2 * j]), cb = __builtin_amdgcn_ubfe(w, ext[2 * j + 1], tbo[2 * j + 1]);
        const uint32_t a = *reinterpret_cast<const uint32_t *>(smem + tbo[2 * j] + 4 * ca);
        const uint32_t b = *reinterpret_cast<const uint32_t *>(smem + tbo[2 * j + 1] + 4 * cb);
        const half2 s = __builtin_bit_cast(half2, __builtin_amdgcn_perm(s23, s01, sel[j]));
        if constexpr (SPLIT) {
          uint32_t u, v;
          split2_up(__uint_as_float(a) * (float)s[0], __uint_as_float(b) * (float)s[1], u, v);
          hi[j] = u;
          lo[j] = v;
        } else {
          const uint32_t c = (a & 0xffffu) | (b & 0xffff0000u);
          hi[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2, c) * s);
        }
      }
    }
  }
  // Eight FP16 values of pass k's V row, zeros from row `rest` on; odd: NaN where one of them is an infinity or a NaN.
  __device__ __forceinline__ u32x4 make_v(int k, int rest, float &odd) const {
    u32x4 v;
    if constexpr (Q8) {
      const half2 s = __builtin_bit_cast(half2, vn[k] | vn[k] << 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // c as 1024 + (c + 128) - 1152, exact
        const uint32_t u = __builtin_amdgcn_perm(0x64646464u, vw[k][j >> 1] ^ 0x80808080u, j & 1 ? 0x04030402u : 0x04010400u);
        v[j] = __builtin_bit_cast(uint32_t, (__builtin_bit_cast(half2, u) - half2{(_Float16)1152.0f, (_Float16)1152.0f}) * s);
      }
    } else {
      v = u32x4{vw[k][0], vw[k][1], vw[k][VW - 2], vw[k][VW - 1]};
    }
    if (key + STRIDE * k >= rest) v = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 4; ++j) odd = odd2(v[j], odd);
    return v;
  }
};

// Two passes' lookups at a time: the scheduler would start them all and spill.
__device__ __forceinline__ void few_passes(int k) {
  if (k & 1) __builtin_amdgcn_sched_barrier(0);
}

// The page of a sequence's tokens t .. (a wave's): -1 where the table names none of the pool's.
__device__ __forceinline__ int chunk_page(const ChunkParams &p, int seq, int t) {
  typedef const __attribute__((address_space(4))) int32_t const_i32;
  const int32_t *row = p.page_table + (int64_t)seq * p.page_table_stride;
  const int pg = reinterpret_cast<const_i32 *>(reinterpret_cast<uintptr_t>(row))[min(t >> p.page_shift, p.table_pages - 1)];
  return (uint32_t)pg < (uint32_t)p.pages ? pg : -1;
}

template <int D, int KF, bool Q8, bool BF>
__device__ __forceinline__ void narrow_item(const ChunkParams &p, uint8_t *smem) {
  constexpr bool SPLIT = KF != 0 && !BF;
  using L = RowsLds<D, KF>;
  using W = Wave<D, SPLIT, BF>;
  using R = Rows<D, KF, Q8, SPLIT>;
  constexpr int B = 32, QS = D / 16, MT = D / 32, PASSES = R::PASSES;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item it = find_item(p, blockIdx.x, p.all_narrow ? kAllUnits : kNarrowUnits, 32, p.aim);
  if (it.splits == 0) return;  // uniform for the workgroup
  const Columns cs(it, p.group, 32);
  R rows(p, it.kv, smem);
  uint8_t *const area = smem + L::ROWS;
  const uint32_t own = L::ROWS + (uint32_t)wave * L::OWN;
  const Blocks bl = Blocks::of<B>(cs.first, min(cs.last, it.n - 1), p.window, p.sinks);
  const int per = (bl.count + kChunkWaves - 1) / kChunkWaves;  // rounds of the eight waves, shared by the splits
  const int r0 = (int)((int64_t)per * it.split / it.splits), r1 = (int)((int64_t)per * (it.split + 1) / it.splits);
  const int first = r0 * kChunkWaves + wave, end = min(r1 * kChunkWaves, bl.count);
  const int in_page = (1 << p.page_shift) - 1;
  auto token = [&](int i) { return bl.at<B>(min(i, end - 1)); };
  // FP16 rows go to LDS by DMA: K of the next block behind this one's product, V behind its own.
  constexpr int DMAS = 32 * D * 2 / 1024, PR = D / 8;
  constexpr bool DK = KF == 0, DV = DK && !Q8;
  const uint32_t own_v = own + (DK ? L::HALF : 0);
  auto dma = [&](const uint8_t *src, uint32_t to, int rest) {  // (rows from `rest` on arrive as zeros)
    const __amdgpu_buffer_rsrc_t r = rsrc(scalar(src), (uint32_t)__builtin_amdgcn_readfirstlane(max(0, min(32, rest))) * 2 * D);
#pragma unroll
    for (int k = 0; k < DMAS; ++k) {
      const int piece = k * 64 + lane, row = piece / PR, c = (piece % PR) ^ swizzle<D>(row);
      dma16(r, smem + to + k * 1024, (uint32_t)(row * (2 * D) + c * 16), 0);
    }
  };
  auto load_k = [&](int page, int t) {
    const int at = t & in_page;
    if constexpr (DK) dma(rows.pk + (int64_t)max(page, 0) * rows.k_page + (int64_t)at * (2 * D), own, page < 0 ? 0 : it.n - t);
    else rows.load_k(max(page, 0), at);
  };
  auto load_v = [&](int page, int t) {
    const int at = t & in_page;
    if constexpr (DV) dma(rows.pv + (int64_t)max(page, 0) * rows.v_page + (int64_t)at * (2 * D), own_v, page < 0 ? 0 : it.n - t);
    else rows.load_v(max(page, 0), at);
  };
  int page = -1, page1 = -1;
  if (first < end) {
    page = chunk_page(p, it.seq, token(first));
    page1 = chunk_page(p, it.seq, token(first + kChunkWaves));
    if constexpr (!DK) {
      load_k(page, token(first));
      load_v(page, token(first));
    }
  }
  R::books(p, it.kv, smem);
  W w;
  if constexpr (KF != 0) {
    w.begin(p, it, w.template load_rotated<true>(p, it, cs, 0, reinterpret_cast<float *>(area)), true);
    lds_barrier();  // the books, and the queries' staging done with
  } else {
    if (first < end) {
      load_k(page, token(first));
      __builtin_amdgcn_sched_barrier(0);
      load_v(page, token(first));
      __builtin_amdgcn_sched_barrier(0);
    }
    w.load_plain(p, it, cs, 0);
    // (waited for here: the loop's counts are of its own loads)
#pragma unroll
    for (int s = 0; s < QS; ++s) asm volatile("" : "+v"(w.qh[s]));
  }
  for (int i = first; i < end; i += kChunkWaves) {
    const int t0 = bl.at<B>(i), t1 = token(i + kChunkWaves);
    const int page2 = chunk_page(p, it.seq, token(i + 2 * kChunkWaves));
    auto put = [&](uint32_t to, int k, u32x4 x) { *reinterpret_cast<u32x4 *>(smem + to + rows.place(k)) = x; };
    f32x16 S[1];
#pragma unroll
    for (int e = 0; e < 16; ++e) S[0][e] = 0.0f;
    if constexpr (DK) {
      wait_vm<DV ? DMAS : 0>();  // K has landed; FP16 V may be on its way
      w.qk(smem, own, S, true);
      wait_lds();
      __builtin_amdgcn_sched_barrier(0);
      load_k(page1, t1);
      __builtin_amdgcn_sched_barrier(0);
    } else {
      u32x4 later[SPLIT ? PASSES : 1];  // (the low parts first: their products are scaled down)
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        u32x4 hi, lo;
        rows.make_k(k, hi, lo);
        if constexpr (SPLIT) later[k] = hi;
        put(own, k, SPLIT ? lo : hi);
        few_passes(k);
      }
      load_k(page1, t1);  // the next block's codes
      wave_sync();
      if constexpr (SPLIT) {
        w.qk(smem, own, S, false);
        w.low_parts(S);
        wave_sync();
#pragma unroll
        for (int k = 0; k < PASSES; ++k) put(own, k, later[k]);
        wave_sync();
      }
      w.qk(smem, own, S, true);
    }
    // (a block without a page is seen by nobody)
    const bool masked = page < 0 || w.sight(t0, B, cs.first, cs.last) != 2;
    const uint64_t seen = masked ? w.seen_bits(t0, page < 0 ? 0ull : ~0ull) : ~0ull;
    uint32_t P[8];
    w.softmax(S, P, masked, seen);
    float odd = 0.0f;
    if constexpr (DV) {
      wait_vm<DMAS>();  // V has landed; the next K may be on its way
      if (masked) {
#pragma unroll
        for (int k = 0; k < DMAS; ++k) {
          const u32x4 v = *reinterpret_cast<const u32x4 *>(smem + own_v + (64 * k + lane) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd = odd2(v[e], odd);
        }
      }
    } else {
      const int rest = page < 0 ? 0 : it.n - t0;
      wave_sync();
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        put(own_v, k, rows.make_v(k, rest, odd));
        few_passes(k);
      }
      if constexpr (!DK) load_v(page1, t1);
      wave_sync();
    }
    if (masked && __builtin_amdgcn_ballot_w64(odd != 0.0f) != 0) {
      w.template add_odd<1>(smem, own_v, seen);
      // (the rows are this wave's own: their infinities and NaNs become zeros)
      wave_sync();
#pragma clang loop unroll(disable)
      for (int k = 0; k < 32 * D * 2 / 1024; ++k) {
        u32x4 &v = *reinterpret_cast<u32x4 *>(smem + own_v + (64 * k + lane) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = finite16(v[e]);
      }
      wave_sync();
    }
    w.template pv<1, false>(smem, own_v, P, false);
    if constexpr (DK) {
      wait_lds();
      __builtin_amdgcn_sched_barrier(0);
      load_v(page1, t1);
      __builtin_amdgcn_sched_barrier(0);
    } else {
      wave_sync();
    }
    page = page1;
    page1 = page2;
  }
  if constexpr (DK) wait_vm<0>();  // (the last block's loads, once more, are still on their way to LDS)
  // The waves' states of the same columns, summed by all threads: four dimensions of a column each.
  constexpr int STATE = L::STATE;
  w.l = half_sum(w.l);
  __syncthreads();
  if ((lane & 31) < cs.count) {
    u32x4 *const to = reinterpret_cast<u32x4 *>(area + wave * STATE) + lane;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        to[(4 * t + g) * 64] = __builtin_bit_cast(u32x4, (f32x4{w.O[t][4 * g], w.O[t][4 * g + 1], w.O[t][4 * g + 2], w.O[t][4 * g + 3]}));
    if (lane < 32) *reinterpret_cast<u32x2 *>(area + kChunkWaves * STATE + (wave * 32 + lane) * 8) = u32x2{__float_as_uint(w.m), __float_as_uint(w.l)};
  }
  __syncthreads();
  for (int e = tid; e < cs.count * (D / 4); e += kThreads) {
    const int piece = e / cs.count, c = e - piece * cs.count;
    float m[kChunkWaves], l[kChunkWaves], M = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kChunkWaves; ++k) {
      const u32x2 ml = *reinterpret_cast<const u32x2 *>(area + kChunkWaves * STATE + (k * 32 + c) * 8);
      m[k] = __uint_as_float(ml[0]), l[k] = __uint_as_float(ml[1]);
      M = fmaxf(M, m[k]);
    }
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < kChunkWaves; ++k) {
      // (a state that saw nothing is all zeros)
      const float a = m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[k] - M);
      const f32x4 x = *(reinterpret_cast<const f32x4 *>(area + k * STATE) + (piece >> 1) * 64 + 32 * (piece & 1) + c);
      sum = __builtin_fmaf(l[k], a, sum);
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] = __builtin_fmaf(x[d], a, o[d]);
    }
    store_piece<D, BF>(p, it, cs, piece, c, o, M, sum);
  }
  if (it.splits == 1) return;
  // The last item of the unit to arrive merges.
  int *const flag = reinterpret_cast<int *>(smem + L::FLAG);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  uint32_t *const counter = p.counters + it.slot0;
  if (tid == 0) *flag = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(it.splits - 1);
  __syncthreads();
  if (!*flag) return;
  merge_pieces<D, BF, true>(p, it, cs, tid, cs.count * (D / 4), kThreads);
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The wide sequences' rows that their chunks see something of, rebuilt: KV
// head `wg` % kv_heads, every wave blocks of 32 tokens. Rows behind a
// sequence's tokens, up to a whole block of 64, become zeros.
template <int D, int KF, bool Q8, bool BF>
__device__ __forceinline__ void rebuild_rows(const ChunkParams &p, uint8_t *smem, int wg, int wgs) {
  constexpr bool SPLIT = KF != 0 && !BF;
  using R = Rows<D, KF, Q8, SPLIT>;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv = wg % p.kv_heads;
  R rows(p, kv, smem);
  const int64_t stride = (int64_t)(wgs / p.kv_heads) * kChunkWaves;
  int64_t base = 0, at = (int64_t)(wg / p.kv_heads) * kChunkWaves + wave;  // blocks before these sequences; this wave's next
  R::books(p, kv, smem);
  lds_barrier();
  int before = offset_ahead(p);
  for (int s0 = 0; s0 < p.sequences; s0 += 64) {
    const SequencePlan q = plan_of(p, s0 + lane, kWideUnits, 32, before);
    const int count = rebuilt_rows(q) / 32, end = wave_prefix(count), all = __builtin_amdgcn_readlane(end, 63);
    for (; at < base + all; at += stride) {
      const int local = (int)(at - base);
      const int i = __builtin_ctzll(__builtin_amdgcn_ballot_w64(local < end));
      const int n = __builtin_amdgcn_readlane(q.n, i), c = __builtin_amdgcn_readlane(q.rows, i);
      const int t0 = 32 * (local - (__builtin_amdgcn_readlane(end, i) - __builtin_amdgcn_readlane(count, i)));
      if (p.window && t0 / kChunkKeys * kChunkKeys + kChunkKeys - 1 <= n - c - p.window && t0 / kChunkKeys * kChunkKeys >= p.sinks) continue;
      const int page = chunk_page(p, s0 + i, t0), from = t0 & ((1 << p.page_shift) - 1), rest = page < 0 ? 0 : n - t0;
      rows.load_k(max(page, 0), from);
      rows.load_v(max(page, 0), from);
      const int64_t row0 = kv * p.rebuilt_head + (base + local) * 32;
#pragma unroll
      for (int k = 0; k < R::PASSES; ++k) {
        const int64_t to = (row0 + R::STRIDE * k) * D + (uint32_t)(rows.key * D + 8 * rows.oct);
        u32x4 hi, lo{};
        float odd = 0.0f;
        rows.make_k(k, hi, lo);
        *reinterpret_cast<u32x4 *>(p.rebuilt_k + to) = hi;
        if constexpr (SPLIT) *reinterpret_cast<u32x4 *>(p.rebuilt_lo + to) = lo;
        *reinterpret_cast<u32x4 *>(p.rebuilt_v + to) = rows.make_v(k, rest, odd);
        few_passes(k);
      }
    }
    base += all;
  }
}

// The queries of all rows into the code domain, as wide units multiply them:
// a wave 32 columns of a KV head at a time, tiles wg * 8 + wave on.
template <int D, bool BF>
__device__ __forceinline__ void rotate_queries(const ChunkParams &p, uint8_t *smem, int wg, int wgs) {
  using W = Wave<D, !BF, BF>;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (int)((p.tokens * p.group + 31) / 32) * p.kv_heads;
  for (int tile = wg * kChunkWaves + wave; tile < tiles; tile += wgs * kChunkWaves) {
    Item it{};
    it.kv = tile % p.kv_heads, it.rows = (int)p.tokens, it.tile = tile / p.kv_heads;
    const Columns cs(it, p.group, 32);
    W w;
    const int eq = w.template load_rotated<false>(p, it, cs, 0, reinterpret_cast<float *>(smem + wave * kStageBytes));
    int row, head;
    W::column(p, it, cs, lane & 31, row, head);
    const int64_t at = (int64_t)row * (p.kv_heads * p.group) + head;
    uint16_t *to = p.turned + at * (BF ? D : 2 * D) + 8 * h;
    if ((lane & 31) < cs.count) {
#pragma unroll
      for (int s = 0; s < W::QS; ++s) {
        *reinterpret_cast<u32x4 *>(to + 16 * s) = w.qh[s];
        if constexpr (!BF) *reinterpret_cast<u32x4 *>(to + D + 16 * s) = w.ql[s];
      }
      if (h == 0) p.turned_exp[at] = eq;
    }
  }
}

// Grid: p.narrow_items items, then p.rotate_items workgroups that rotate the
// queries of wide units, then those that rebuild rows.
template <int D, int KF, bool Q8, bool BF>
__global__ __launch_bounds__(kThreads, 2) void chunk_rows_kernel(ChunkParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  int wg = (int)blockIdx.x - p.narrow_items;
  if (wg < 0) {
    narrow_item<D, KF, Q8, BF>(p, smem);
    return;
  }
  if constexpr (KF != 0) {
    if (wg < p.rotate_items) {
      rotate_queries<D, BF>(p, smem, wg, p.rotate_items);
      return;
    }
    wg -= p.rotate_items;
  }
  if constexpr (KF != 0 || Q8) rebuild_rows<D, KF, Q8, BF>(p, smem, wg, (int)gridDim.x - p.narrow_items - p.rotate_items);
}

template <int D, int KF, bool Q8, bool BF>
hipError_t launch_one(const ChunkParams &p, int items, hipStream_t stream) {
  constexpr int lds = RowsLds<D, KF>::BYTES;
  static_assert(lds <= kLdsLimit, "LDS of one workgroup");
  static const hipError_t allowed =
      hipFuncSetAttribute((const void *)chunk_rows_kernel<D, KF, Q8, BF>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (allowed != hipSuccess) {
    (void)hipGetLastError();
    return allowed;
  }
  hipLaunchKernelGGL((chunk_rows_kernel<D, KF, Q8, BF>), dim3((unsigned)items), dim3(kThreads), lds, stream, p);
  return hipGetLastError();
}
template <int D, int KF>
hipError_t launch_k(const ChunkParams &p, bool bf16, int items, hipStream_t stream) {
  if (p.v_scales) return bf16 ? launch_one<D, KF, true, true>(p, items, stream) : launch_one<D, KF, true, false>(p, items, stream);
  return bf16 ? launch_one<D, KF, false, true>(p, items, stream) : launch_one<D, KF, false, false>(p, items, stream);
}

}  // namespace
}  // namespace bgtq
