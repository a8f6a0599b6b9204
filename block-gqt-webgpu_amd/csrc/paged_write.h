// Rows of V and FP16 K into a pool of pages: D / 8 lanes per row, eight values
// each, so a row is one coalesced access and its maximum takes three or four
// lane rotations. 8-bit V: s = max|v| / 127 rounded up to FP16, at most 515.5 (the
// largest whose 127-fold is an FP16 value), and c = v / s
// rounded to the nearest integer, ties to even. v and s have 11 significant
// bits, so a quotient that is no tie lies at least 2^-12 from every tie: the
// correctly rounded FP32 quotient decides as the exact one does. That quotient
// is fma(fma(-q, s, v), r, q) with r the row's correctly rounded 1 / s and q =
// v r (Markstein), three instructions a value instead of a division.
#pragma once

#include "bgtq_internal.h"
#include "encode_row.h"
#include "gfx950_common.h"

namespace bgtq {
namespace {

using namespace gfx;
using row_enc::f16_bits_to_f32;
using row_enc::f32_to_f16_bits;

__device__ __forceinline__ float load_one(const void *src, int dtype, int64_t at) {
  if (dtype == BGTQ_DTYPE_F32) return static_cast<const float *>(src)[at];
  const uint16_t u = static_cast<const uint16_t *>(src)[at];
  return dtype == BGTQ_DTYPE_F16 ? f16_bits_to_f32(u) : __uint_as_float((uint32_t)u << 16);
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

constexpr uint16_t kMaxScale = 0x6007u;  // 515.5 in FP16

// Maximum over the L = 8 or 16 lanes that share a row.
template <int L>
__device__ __forceinline__ int lanes_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false));   // quad_perm: lanes 1 0 3 2
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false));   // quad_perm: lanes 2 3 0 1
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));  // row_half_mirror
  if (L == 16) v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false));  // rotation by 8
  return v;
}

// V, or FP16 K (of_k), of the call to the pool: rows first, first + step, ...
// of KV head `only`; only < 0: of all heads, row i of head h numbered i * heads + h.
template <int D, bool of_k>
__device__ __forceinline__ void write_rows(const PagedWriteParams &p, int only, int64_t first, int64_t step) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x & 63, sub = lane % L;
  const void *src = of_k ? p.k : p.v;
  const int dtype = of_k ? p.k_dtype : p.v_dtype;
  const int64_t rs = of_k ? p.k_row_stride : p.v_row_stride, hs = of_k ? p.k_head_stride : p.v_head_stride;
  const bool q8 = !of_k && p.v_scales != nullptr, vec = aligned16(src, dtype, rs, hs);
  const int64_t n = only < 0 ? p.slots.rows * p.kv_heads : p.slots.rows;
  for (int64_t r = first; r < n; r += step) {
    const int64_t row = only < 0 ? r / p.kv_heads : r;
    const int head = only < 0 ? (int)(r - row * p.kv_heads) : only;
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
    // s: rounded to nearest, then up where 127 s would fall short of the maximum;
    // 515.5 at most (maxima of 65472 and 65504: 127 times 516 would round to an
    // infinity, and 65504 / 515.5 still rounds to 127).
    const float most = f16_bits_to_f32((uint16_t)top);
    uint16_t s = f32_to_f16_bits(most / 127.0f);
    if (f16_bits_to_f32(s) * 127.0f < most) ++s;
    s = s < kMaxScale ? s : kMaxScale;
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

}  // namespace
}  // namespace bgtq
