// Rows of K and V into and out of a pool of pages (bgtq_paged_write,
// bgtq_paged_read).
//
// Write. Packed K of few rows: a wave per row and head (encode_row.h, the
// arithmetic of encode_wave.hip); of many, encode_tile.hip's paged kernel. V
// (and FP16 K): D / 8 lanes per row, eight values each, so a row is one
// coalesced access and its maximum takes three or four lane rotations.
// 8-bit V: s = max|v| / 127 rounded up to FP16 and c = v / s rounded to the
// nearest integer, ties to even. v and s have 11 significant bits, so a
// quotient that is no tie lies at least 2^-12 from every tie: the correctly
// rounded FP32 quotient decides as the exact one does. That quotient is
// fma(fma(-q, s, v), r, q) with r the row's correctly rounded 1 / s and q = v r
// (Markstein), three instructions a value instead of a division.
//
// Read. k = Rp^T cs, with cs_j = c_j s_g(j) the row in the code domain and
// Rp[j][i] the rotation with its columns in the model's order of dimensions
// (src/reference/production_math.py:27-31), 16 rows to a 16x16x32 f16 product
// with both operands split into FP16 hi and lo parts (three products, 2^-22
// relative). A lane rebuilds the eight consecutive positions that it feeds the
// product and ends with four consecutive dimensions of its row. The rotation
// stays in registers: all of it at d=64, the columns of one wave of four at
// d=128, whose waves exchange their rebuilt rows through LDS.
#include <hip/hip_fp16.h>

#include "bgtq_internal.h"
#include "encode_row.h"
#include "gfx950_common.h"

namespace bgtq {
namespace {

using namespace gfx;
using row_enc::f16_bits_to_f32;
using row_enc::f32_to_f16_bits;

constexpr int kWaves = 4, kThreads = 64 * kWaves;

__device__ __forceinline__ float load_one(const void *src, int dtype, int64_t at) {
  if (dtype == BGTQ_DTYPE_F32) return static_cast<const float *>(src)[at];
  const uint16_t u = static_cast<const uint16_t *>(src)[at];
  return dtype == BGTQ_DTYPE_F16 ? f16_bits_to_f32(u) : __uint_as_float((uint32_t)u << 16);
}

__device__ __forceinline__ uint32_t f32_to_bf16_bits(float v) {
  const uint32_t u = __float_as_uint(v);
  return (u & 0x7fffffffu) > 0x7f800000u ? (u >> 16) | 0x40u : (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// Whether rows at base with these strides (elements of dtype) allow 16-byte pieces.
__device__ __forceinline__ bool aligned16(const void *base, int dtype, int64_t s0, int64_t s1) {
  const int64_t e = dtype == BGTQ_DTYPE_F32 ? 4 : 2;
  return ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)(s0 * e) | (uintptr_t)(s1 * e)) & 15) == 0;
}

// Eight values from element `at` on as FP16 bits (FP32 and BF16 rounded).
__device__ __forceinline__ void load8_half(const void *src, int dtype, bool vec, int64_t at, uint16_t (&h)[8]) {
  if (!vec) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      h[k] = dtype == BGTQ_DTYPE_F16 ? static_cast<const uint16_t *>(src)[at + k] : f32_to_f16_bits(load_one(src, dtype, at + k));
    return;
  }
  if (dtype == BGTQ_DTYPE_F32) {
    const f32x4 *p = reinterpret_cast<const f32x4 *>(static_cast<const float *>(src) + at);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      h[k] = f32_to_f16_bits(a[k]);
      h[4 + k] = f32_to_f16_bits(b[k]);
    }
    return;
  }
  const u32x4 w = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(src) + at);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    h[2 * k] = (uint16_t)(w[k] & 0xffffu);
    h[2 * k + 1] = (uint16_t)(w[k] >> 16);
  }
  if (dtype == BGTQ_DTYPE_BF16) {
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = f32_to_f16_bits(__uint_as_float((uint32_t)h[k] << 16));
  }
}

// Maximum over the L = 8 or 16 lanes that share a row.
template <int L>
__device__ __forceinline__ int lanes_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false));   // quad_perm: lanes 1 0 3 2
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false));   // quad_perm: lanes 2 3 0 1
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));  // row_half_mirror
  if (L == 16) v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false));  // rotation by 8
  return v;
}

// Rows first, first + step, ... (row i of head h is row i * heads + h): V, or
// FP16 K (of_k), of the call to the pool.
template <int D, bool of_k>
__device__ __forceinline__ void write_rows(const PagedWriteParams &p, int64_t first, int64_t step) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x & 63, sub = lane % L;
  const void *src = of_k ? p.k : p.v;
  const int dtype = of_k ? p.k_dtype : p.v_dtype;
  const int64_t rs = of_k ? p.k_row_stride : p.v_row_stride, hs = of_k ? p.k_head_stride : p.v_head_stride;
  const bool q8 = !of_k && p.v_scales != nullptr, vec = aligned16(src, dtype, rs, hs);
  const int64_t n = p.slots.rows * p.kv_heads;
  for (int64_t r = first; r < n; r += step) {
    const int64_t row = r / p.kv_heads;
    const int head = (int)(r - row * p.kv_heads);
    int64_t page;
    int at;
    const bool kept = p.slots.find(row, page, at);
    uint16_t h[8];
    load8_half(src, dtype, vec, row * rs + head * hs + 8 * sub, h);
    if (!kept) continue;  // (the lanes of a row agree)
    if (!q8) {
      uint16_t *dst = of_k ? p.k_f16 + page * p.kp_page_stride + head * p.kp_head_stride
                           : static_cast<uint16_t *>(p.v_pool) + page * p.vp_page_stride + head * p.vp_head_stride;
      u32x4 w;
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = (uint32_t)h[2 * k] | (uint32_t)h[2 * k + 1] << 16;
      *reinterpret_cast<u32x4 *>(dst + (int64_t)at * D + 8 * sub) = w;
      continue;
    }
    int top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, (int)(h[k] & 0x7fffu));  // FP16 magnitudes order as their bits do
    top = lanes_max<L>(top);
    // s: rounded to nearest, then up where 127 s would fall short of the maximum.
    const float most = f16_bits_to_f32((uint16_t)top);
    uint16_t s = f32_to_f16_bits(most / 127.0f);
    if (f16_bits_to_f32(s) * 127.0f < most) ++s;
    const bool finite = top < 0x7c00;
    const float sf = f16_bits_to_f32(s), rcp = s ? 1.0f / sf : 0.0f;
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float x = f16_bits_to_f32(h[k]), q = x * rcp;
      const int c = finite ? (int)__builtin_rintf(__builtin_fmaf(__builtin_fmaf(-q, sf, x), rcp, q)) : 0;
      w[k >> 2] |= ((uint32_t)c & 255u) << (8 * (k & 3));
    }
    int8_t *dst = static_cast<int8_t *>(p.v_pool) + page * p.vp_page_stride + head * p.vp_head_stride;
    *reinterpret_cast<u32x2 *>(dst + (int64_t)at * D + 8 * sub) = u32x2{w[0], w[1]};
    if (sub == 0) p.v_scales[page * p.vs_page_stride + head * p.vs_head_stride + at] = finite ? s : (uint16_t)0x7e00u;
  }
}

// Grid y: with K, KV head y's packed rows (a wave per row), then one slice for
// V; without, V and (FP16 K) K.
struct WriteLds {
  int tab, scratch, stride, total;
};
template <int D>
__host__ __device__ inline WriteLds write_lds(int enc_bytes) {
  WriteLds L;
  L.tab = D * D * 4;
  L.scratch = L.tab + (enc_bytes + 1023) / 1024 * 1024;
  L.stride = row_enc::scratch_bytes(D);
  L.total = L.scratch + kWaves * L.stride;
  return L;
}

template <int D, bool WITH_K>
__global__ __launch_bounds__(kThreads) void paged_write_kernel(PagedWriteParams p) {
  constexpr int JL = row_enc::Lane<D>::JL, L8 = D / 8;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = blockIdx.y;
  if (!WITH_K || head == p.kv_heads) {
    const int64_t first = (int64_t)blockIdx.x * (kThreads / L8) + tid / L8, step = (int64_t)gridDim.x * (kThreads / L8);
    if (!WITH_K && head == 1) write_rows<D, true>(p, first, step);
    else write_rows<D, false>(p, first, step);
    return;
  }
  const DevTables *Tg = p.tables[head];
  const int enc_bytes = p.enc_bytes[head];
  const WriteLds L = write_lds<D>(enc_bytes);
  const float *rot_t = reinterpret_cast<const float *>(smem);
  const row_enc::Scratch<D> scr(smem + L.scratch + wave * L.stride);
  const int64_t nwaves = (int64_t)gridDim.x * kWaves;
  // The transposed rotation and the tables' header, LUT and books to LDS; the
  // first row's values meanwhile.
  {
    const uint8_t *tb = reinterpret_cast<const uint8_t *>(Tg);
    const __amdgpu_buffer_rsrc_t rr = rsrc(tb + p.off_rot_t[head], D * D * 4);
    for (int k = wave; k < D * D * 4 / 1024; k += kWaves) dma16(rr, smem + k * 1024, k * 1024 + lane * 16, 0);
    const __amdgpu_buffer_rsrc_t rt = rsrc(tb, enc_bytes);
    for (int k = wave; k < (enc_bytes + 1023) / 1024; k += kWaves) dma16(rt, smem + L.tab + k * 1024, k * 1024 + lane * 16, 0);
  }
  auto load_row = [&](int64_t r, float (&v)[JL]) {  // (a row past the call's reads row 0)
    const int64_t at = (r < p.slots.rows ? r : 0) * p.k_row_stride + head * p.k_head_stride + lane;
#pragma unroll
    for (int jl = 0; jl < JL; ++jl) v[jl] = f16_bits_to_f32(f32_to_f16_bits(load_one(p.k, p.k_dtype, at + 64 * jl)));
  };
  int64_t row = (int64_t)blockIdx.x * kWaves + wave;
  float xn[JL];
  load_row(row, xn);
  wait_vm<0>();
  __syncthreads();
  const DevTables *T = reinterpret_cast<const DevTables *>(smem + L.tab);
  row_enc::Lane<D> c;
  c.init(T, lane);
  const uint8_t *lut = tables_lut(T);
  const float *books = tables_books(T);
  const int RB = T->row_bytes, nib = T->nibble_dims, NS = T->norm_stride, logical = nib / 2 + D - nib;
  for (; row < p.slots.rows; row += nwaves) {
    float xnext[JL];
    load_row(row + nwaves, xnext);
    float x[JL];
#pragma unroll
    for (int jl = 0; jl < JL; ++jl) {  // head-perm order
      const int src = c.perm[jl];
      x[jl] = __shfl(xn[0], src & 63, 64);
      if (JL > 1) {
        const float hi = __shfl(xn[JL - 1], src & 63, 64);
        x[jl] = src >= 64 ? hi : x[jl];
      }
    }
    const uint16_t h = row_enc::encode_row<D>(
        T, c, x, [&](int i, int jl) { return rot_t[i * D + lane + 64 * jl]; }, lut, books, scr, lane);
    int64_t page;
    int at;
    if (p.slots.find(row, page, at)) {  // (uniform)
      uint8_t *prow = p.packed + page * p.packed_page_stride + head * p.packed_head_stride + (int64_t)at * RB;
      uint16_t *nrow = p.norms + page * p.norms_page_stride + head * p.norms_head_stride + (int64_t)at * NS;
      for (int o = lane; o < RB; o += 64) prow[o] = row_enc::packed_byte(scr.codes, o, nib, logical);
      if (lane < NS) nrow[lane] = h;
    }
    row_enc::wave_sync();  // scratch is rewritten by the next row
#pragma unroll
    for (int jl = 0; jl < JL; ++jl) xn[jl] = xnext[jl];
  }
}

// ---- read ----

// Four consecutive values of a row, from element `at` on.
__device__ __forceinline__ void store4(void *dst, int dtype, bool vec, int64_t at, f32x4 v) {
  if (dtype == BGTQ_DTYPE_F32) {
    float *o = static_cast<float *>(dst) + at;
    if (vec) {
      *reinterpret_cast<f32x4 *>(o) = v;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = v[k];
    }
    return;
  }
  uint32_t b[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) b[k] = dtype == BGTQ_DTYPE_F16 ? (uint32_t)f32_to_f16_bits(v[k]) : f32_to_bf16_bits(v[k]);
  uint16_t *o = static_cast<uint16_t *>(dst) + at;
  if (vec) {
    *reinterpret_cast<u32x2 *>(o) = u32x2{b[0] | b[1] << 16, b[2] | b[3] << 16};
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = (uint16_t)b[k];
  }
}

// Four values of a V or FP16 K row as they are stored, from element `at` of its row on.
template <bool of_k>
__device__ __forceinline__ f32x4 pool4(const PagedWriteParams &p, int head, int64_t page, int64_t at, float s) {
  f32x4 v;
  if (!of_k && p.v_scales) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(p.v_pool) + page * p.vp_page_stride +
                                                           head * p.vp_head_stride + at);
#pragma unroll
    for (int k = 0; k < 4; ++k)  // 8-bit V stands for the FP16 value nearest s c
      v[k] = f16_bits_to_f32(f32_to_f16_bits((float)(int8_t)(w >> (8 * k)) * s));
    return v;
  }
  const uint16_t *src = of_k ? p.k_f16 + page * p.kp_page_stride + head * p.kp_head_stride
                             : static_cast<const uint16_t *>(p.v_pool) + page * p.vp_page_stride + head * p.vp_head_stride;
  const u32x2 w = *reinterpret_cast<const u32x2 *>(src + at);
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = f16_bits_to_f32((uint16_t)(w[k >> 1] >> (16 * (k & 1))));
  return v;
}

// V (or FP16 K) rows of 16-row tile `tile` of head `head`: lane (gq, col) takes
// dimensions 16 t + 4 gq + 0..3 of row col.
template <int D, bool of_k>
__device__ __forceinline__ void read_plain(const PagedWriteParams &p, int64_t tile, int head, int gq, int col) {
  const int64_t row = tile * 16 + col;
  int64_t page;
  int at;
  if (row >= p.slots.rows || !p.slots.find(row, page, at)) return;
  void *dst = of_k ? p.k : p.v;
  const int dtype = of_k ? p.k_dtype : p.v_dtype;
  const int64_t rs = of_k ? p.k_row_stride : p.v_row_stride, hs = of_k ? p.k_head_stride : p.v_head_stride;
  const bool vec = aligned16(dst, dtype, rs, hs);
  const float s = !of_k && p.v_scales
                      ? f16_bits_to_f32(p.v_scales[page * p.vs_page_stride + head * p.vs_head_stride + at])
                      : 1.0f;
  f32x4 v[D / 16];
#pragma unroll
  for (int t = 0; t < D / 16; ++t) v[t] = pool4<of_k>(p, head, page, (int64_t)at * D + 16 * t + 4 * gq, s);
#pragma unroll
  for (int t = 0; t < D / 16; ++t) store4(dst, dtype, vec, row * rs + head * hs + 16 * t + 4 * gq, v[t]);
}

template <int D>
struct Read {
  static constexpr int KS = D / 32;                 // 32-position steps of the product
  static constexpr int CW = D / 64 * (D / 64);      // waves that share the output columns (1, 4)
  static constexpr int NT = D / 16 / CW;            // 16-column tiles per wave
  static constexpr int WORDS = D / 4 + 2;           // words of a staged packed row (row bytes <= D, its misalignment)
  static constexpr int ROWW = WORDS + 1;            // padded
  static constexpr int STAGE = 16 * ROWW * 4;       // staged rows of a wave
  static constexpr int NORMS = 16 * kMaxGroups * 4; // their scales, FP32
  static constexpr int XCH = CW > 1 ? 64 * (KS * 32 + 16) : 0;  // rebuilt operands of a wave (hi, lo; per lane, padded)
  static constexpr int BOOKS = 8192;                // centroid books: at most 8 of 256 (the pages' layouts)
  static constexpr int LDS = BOOKS + kWaves * (STAGE + NORMS + XCH);
};

template <int D>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(PagedWriteParams p, int64_t tiles) {
  using R = Read<D>;
  constexpr int KS = R::KS, NT = R::NT, CW = R::CW;
  __shared__ __align__(16) uint8_t smem[R::LDS];
  const int tid = threadIdx.x, lane = tid & 63, gq = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = blockIdx.y % p.kv_heads, what = blockIdx.y / p.kv_heads;  // what: 0 the first of K, V that is read
  const bool of_k = what == 0 && p.k != nullptr;
  const int64_t t0 = (int64_t)blockIdx.x * kWaves + wave, step = (int64_t)gridDim.x * kWaves;
  if (!of_k || p.k_f16) {
    if (of_k)
      for (int64_t t = t0; t < tiles; t += step) read_plain<D, true>(p, t, head, gq, col);
    else
      for (int64_t t = t0; t < tiles; t += step) read_plain<D, false>(p, t, head, gq, col);
    return;
  }
  // ---- packed K ----
  const BGTQ_GLOBAL DevTables *T = to_global(p.tables[head]);
  const int RB = T->row_bytes, NS = T->norm_stride, mc = T->max_centroids, ng = T->groups;
  const BGTQ_GLOBAL float *books = tables_books(T), *rot = tables_rot(T);
  const int book_floats = T->n_books * mc;
  uint8_t *const wv = smem + R::BOOKS + wave * (R::STAGE + R::NORMS + R::XCH);
  uint32_t *const stage = reinterpret_cast<uint32_t *>(wv);
  float *const nstage = reinterpret_cast<float *>(wv + R::STAGE);
  // The model dimension of each head-perm position, inverted: position of dimension c.
  uint8_t *const inv = smem + R::BOOKS;  // (the first wave's staging, dead before it is used)
  if (tid < D) inv[T->perm[tid]] = (uint8_t)tid;
  for (int e = tid; e < book_floats; e += kThreads) reinterpret_cast<float *>(smem)[e] = books[e];
  __syncthreads();
  // A operand: Rp^T, row (lane % 16) of column tile t = dimension 16 t + col,
  // columns the positions 32 s + 8 gq + e, times 2^14 (entries are at most 1).
  half8 rh[NT][KS], rl[NT][KS];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int i = inv[16 * ((CW > 1 ? wave : 0) * NT + t) + col];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = rot[(32 * s + 8 * gq + e) * D + i];
      split_scaled(v, 16384.0f, rh[t][s], rl[t][s]);
    }
  }
  // Per position of this lane: byte of the row, nibble shift, mask, book and group.
  uint32_t desc[KS][8];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = 32 * s + 8 * gq + e;
      const bool nib = j < T->nibble_dims;
      const uint32_t byte = nib ? j >> 1 : (T->nibble_dims >> 1) + j - T->nibble_dims;
      desc[s][e] = byte | (nib && (j & 1) ? 4u << 8 : 0u) | (nib ? 4u : 8u) << 12 | (uint32_t)T->group_of[j] << 16 |
                   (uint32_t)(T->pos_book[j] * mc) << 19;
    }
  __syncthreads();
  const bool vec = aligned16(p.k, p.k_dtype, p.k_row_stride, p.k_head_stride);
  const uint8_t *pk = p.packed + head * p.packed_head_stride;
  const uint16_t *nm = p.norms + head * p.norms_head_stride;
  // With shared columns (CW > 1) the waves of a workgroup take four tiles
  // together; each rebuilds one of them.
  const int64_t rounds = CW > 1 ? (tiles + step - 1) / step : tiles;
  for (int64_t i = CW > 1 ? 0 : t0; i < rounds; i += CW > 1 ? 1 : step) {
    const int64_t tile = CW > 1 ? i * step + t0 : i;
    const int64_t row = tile * 16 + col;
    int64_t page = 0;
    int at = 0;
    const bool kept = row < p.slots.rows && p.slots.find(row, page, at);
    // The row's bytes as whole words from the one that holds its first byte,
    // to LDS (rows that are not read: nothing, their lanes store nothing).
    const uint8_t *src = pk + page * p.packed_page_stride + (int64_t)at * RB;
    const uint32_t mis = (uint32_t)reinterpret_cast<uintptr_t>(src) & 3u;
    const uint32_t *words = reinterpret_cast<const uint32_t *>(src - mis);
    const int nw = kept ? (int)(mis + RB + 3) / 4 : 0;
    constexpr int PER = (R::WORDS + 3) / 4;
    uint32_t w[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) w[k] = gq + 4 * k < nw ? words[gq + 4 * k] : 0u;
    float nv[kMaxGroups / 4];
#pragma unroll
    for (int k = 0; k < kMaxGroups / 4; ++k)
      nv[k] = kept && gq + 4 * k < ng ? f16_bits_to_f32(nm[page * p.norms_page_stride + (int64_t)at * NS + gq + 4 * k]) : 0.0f;
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (gq + 4 * k < R::WORDS) stage[col * R::ROWW + gq + 4 * k] = w[k];
#pragma unroll
    for (int k = 0; k < kMaxGroups / 4; ++k) nstage[col * kMaxGroups + gq + 4 * k] = nv[k];
    row_enc::wave_sync();
    // cs of this lane's positions, scaled by a power of two per row into the split's range.
    float cs[KS][8], most = 0.0f;
    const uint8_t *bytes = reinterpret_cast<const uint8_t *>(stage + col * R::ROWW) + mis;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t d = desc[s][e];
        const uint32_t code = ((uint32_t)bytes[d & 255u] >> ((d >> 8) & 15u)) & ((1u << ((d >> 12) & 15u)) - 1u);
        const uint32_t c = (d >> 19) + code;
        cs[s][e] = reinterpret_cast<const float *>(smem)[c] * nstage[col * kMaxGroups + ((d >> 16) & 7u)];
        most = fmaxf(most, fabsf(cs[s][e]));
      }
    const int ex = split_exp(col_max(most));
    half8 bh[KS], bl[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) split_scaled(cs[s], __builtin_ldexpf(1.0f, ex), bh[s], bl[s]);
    const float unscale = __builtin_ldexpf(1.0f, -ex - 14);
    auto product = [&](const half8 (&h)[KS], const half8 (&l)[KS], float un, int64_t to, bool keep) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 a = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          a = mfma(rh[t][s], h[s], a);
          a = mfma(rl[t][s], h[s], a);
          a = mfma(rh[t][s], l[s], a);
        }
        const int c0 = 16 * ((CW > 1 ? wave : 0) * NT + t) + 4 * gq;
        if (keep) store4(p.k, p.k_dtype, vec, to * p.k_row_stride + head * p.k_head_stride + c0, a * un);
      }
    };
    if constexpr (CW == 1) {
      product(bh, bl, unscale, row, kept);
      row_enc::wave_sync();  // the staging is rewritten by the next tile
    } else {
      // This wave's operands per lane: hi and lo of every step, then unscale and whether the row is read.
      constexpr int LB = R::XCH / 64;
      uint8_t *mine = wv + R::STAGE + R::NORMS + lane * LB;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        *reinterpret_cast<half8 *>(mine + 32 * s) = bh[s];
        *reinterpret_cast<half8 *>(mine + 32 * s + 16) = bl[s];
      }
      *reinterpret_cast<u32x2 *>(mine + 32 * KS) = u32x2{__float_as_uint(unscale), kept ? 1u : 0u};
      __syncthreads();
#pragma unroll 1
      for (int o = 0; o < kWaves; ++o) {
        const uint8_t *theirs = smem + R::BOOKS + o * (R::STAGE + R::NORMS + R::XCH) + R::STAGE + R::NORMS + lane * LB;
        half8 oh[KS], ol[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          oh[s] = *reinterpret_cast<const half8 *>(theirs + 32 * s);
          ol[s] = *reinterpret_cast<const half8 *>(theirs + 32 * s + 16);
        }
        const u32x2 last = *reinterpret_cast<const u32x2 *>(theirs + 32 * KS);
        product(oh, ol, __uint_as_float(last[0]), (i * step + (int64_t)blockIdx.x * kWaves + o) * 16 + col, last[1] != 0u);
      }
      __syncthreads();  // the operands are rewritten by the next round
    }
  }
}

template <int D>
hipError_t launch_write_d(const PagedWriteParams &p, bool with_k, int lds, int cus, hipStream_t stream) {
  const int64_t heads = p.kv_heads, per_wg = kThreads / (D / 8);
  // About 16 waves per compute unit, as the row encoder of dense rows.
  const int64_t most = 4 * (int64_t)cus;
  if (!with_k) {
    const int64_t wgs = std::min<int64_t>((p.slots.rows * heads + per_wg - 1) / per_wg, 2 * most);
    hipLaunchKernelGGL((paged_write_kernel<D, false>), dim3((unsigned)wgs, p.k_f16 ? 2u : 1u), dim3(kThreads), 0, stream, p);
    return hipGetLastError();
  }
  static const hipError_t ok = hipFuncSetAttribute((const void *)paged_write_kernel<D, true>,
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, kLdsLimit);
  if (ok != hipSuccess) {
    (void)hipGetLastError();
    return ok;
  }
  const int64_t wgs = std::min<int64_t>((p.slots.rows + kWaves - 1) / kWaves, std::max<int64_t>(1, most / heads));
  hipLaunchKernelGGL((paged_write_kernel<D, true>), dim3((unsigned)wgs, (unsigned)heads + 1), dim3(kThreads), lds, stream, p);
  return hipGetLastError();
}

template <int D>
hipError_t launch_read_d(const PagedWriteParams &p, int cus, hipStream_t stream) {
  const int64_t tiles = (p.slots.rows + 15) / 16, slices = (int64_t)p.kv_heads * ((p.k ? 1 : 0) + (p.v ? 1 : 0));
  const int64_t wgs = std::min<int64_t>((tiles + kWaves - 1) / kWaves, std::max<int64_t>(1, 8 * (int64_t)cus / slices));
  hipLaunchKernelGGL((paged_read_kernel<D>), dim3((unsigned)wgs, (unsigned)slices), dim3(kThreads), 0, stream, p, tiles);
  return hipGetLastError();
}

}  // namespace

int paged_write_lds_bytes(int dim, int enc_bytes) {
  return dim == 64 ? write_lds<64>(enc_bytes).total : write_lds<128>(enc_bytes).total;
}

hipError_t launch_paged_write(const PagedWriteParams &p, bool with_k, int lds_bytes, int cus, hipStream_t stream) {
  return p.dim == 64 ? launch_write_d<64>(p, with_k, lds_bytes, cus, stream)
                     : launch_write_d<128>(p, with_k, lds_bytes, cus, stream);
}

hipError_t launch_paged_read(const PagedWriteParams &p, int cus, hipStream_t stream) {
  return p.dim == 64 ? launch_read_d<64>(p, cus, stream) : launch_read_d<128>(p, cus, stream);
}

}  // namespace bgtq
