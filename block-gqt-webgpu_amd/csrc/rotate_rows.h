// Rows of heads normed and rotated (rotate.h), a lane per N values of a head's
// first half and the N they pair with: 16 bytes of each half, so no value
// crosses lanes but for a norm's sum over the D / (2 N) lanes of the head.
#pragma once

#include "bgtq_internal.h"
#include "encode_row.h"
#include "gfx950_common.h"
#include "rotate.h"

namespace bgtq {
namespace rot {

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct HeadRows {
  const void *src;
  void *dst;
  int32_t heads;
  int64_t src_row, src_head, dst_row, dst_head;  // elements
  const float *weight;                           // null: no norm
};

template <int DTYPE>
constexpr int kPer = DTYPE == BGTQ_DTYPE_F32 ? 4 : 8;  // values of 16 bytes

// N values from element `at` on, as FP32; vec: in one 16-byte access.
template <int DTYPE, int N>
__device__ __forceinline__ void load_values(const void *src, int64_t at, bool vec, float (&x)[N]) {
  uint32_t w[4];
  if constexpr (DTYPE == BGTQ_DTYPE_F32) {
    const uint32_t *p = static_cast<const uint32_t *>(src) + at;
    if (vec) __builtin_memcpy(w, __builtin_assume_aligned(p, 16), 16);
    else
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = p[k];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(w[k]);
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(src) + at;
    if (vec) __builtin_memcpy(w, __builtin_assume_aligned(p, 16), 16);
    else
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = (uint32_t)p[2 * k] | (uint32_t)p[2 * k + 1] << 16;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t u = k & 1 ? w[k >> 1] >> 16 : w[k >> 1] & 0xffffu;
      x[k] = DTYPE == BGTQ_DTYPE_F16 ? row_enc::f16_bits_to_f32((uint16_t)u) : __uint_as_float(u << 16);
    }
  }
}
template <int DTYPE, int N>
__device__ __forceinline__ void store_values(void *dst, int64_t at, bool vec, const float (&x)[N]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DTYPE == BGTQ_DTYPE_F32) w[k] = __float_as_uint(x[k]);
    else if constexpr (DTYPE == BGTQ_DTYPE_F16)
      w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x[2 * k], x[2 * k + 1]}), half2));
    else w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x[2 * k], x[2 * k + 1]}), bf16x2));
  }
  if constexpr (DTYPE == BGTQ_DTYPE_F32) {
    uint32_t *p = static_cast<uint32_t *>(dst) + at;
    if (vec) __builtin_memcpy(__builtin_assume_aligned(p, 16), w, 16);
    else
#pragma unroll
      for (int k = 0; k < 4; ++k) p[k] = w[k];
  } else {
    uint16_t *p = static_cast<uint16_t *>(dst) + at;
    if (vec) __builtin_memcpy(__builtin_assume_aligned(p, 16), w, 16);
    else
#pragma unroll
      for (int k = 0; k < N; ++k) p[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
  }
}

// Items first, first + step, ... of rows [row0, row0 + rows) x heads, a
// group of lanes each; `sub` is this lane's place in its group.
template <int D, int DTYPE>
__device__ __forceinline__ void rotate_items(const HeadRows &h, const Rotation &r, int64_t row0, int rows, uint32_t first,
                                             uint32_t step, int sub) {
  constexpr int N = kPer<DTYPE>, L = D / (2 * N), E = DTYPE == BGTQ_DTYPE_F32 ? 4 : 2;
  auto aligned = [](const void *p, int64_t a, int64_t b) {
    return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(a * E) | (uintptr_t)(b * E)) & 15) == 0;
  };
  const bool vin = aligned(h.src, h.src_row, h.src_head), vout = aligned(h.dst, h.dst_row, h.dst_head);
  const uint32_t n = (uint32_t)rows * (uint32_t)h.heads;
  for (uint32_t i = first; i < n; i += step) {
    const uint32_t local = i / (uint32_t)h.heads;
    const int head = (int)(i - local * (uint32_t)h.heads);
    const int64_t row = row0 + local;
    const int64_t from = row * h.src_row + head * h.src_head + N * sub;
    float a[N], b[N];
    load_values<DTYPE>(h.src, from, vin, a);
    load_values<DTYPE>(h.src, from + D / 2, vin, b);
    const float *cs;
    const bool ok = r.find(row, cs, D);
    float c[N], s[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      c[k] = cs[N * sub + k];
      s[k] = cs[D / 2 + N * sub + k];
    }
    if (h.weight) {
      double sum = 0.0;
#pragma unroll
      for (int k = 0; k < N; ++k) sum = add_square(b[k], add_square(a[k], sum));
      const float f = factor(lanes_sum<L>(sum), D, r.eps);
      // (weights loaded ahead of the loop cost 13%: 16384 rows 14.0 / 15.8 us)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        a[k] = (a[k] * f) * h.weight[N * sub + k];
        b[k] = (b[k] * f) * h.weight[D / 2 + N * sub + k];
      }
    }
    float y[N], z[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      y[k] = turn(a[k], b[k], c[k], s[k], false);
      z[k] = turn(b[k], a[k], c[k], s[k], true);
    }
    if (!ok) continue;
    const int64_t to = row * h.dst_row + head * h.dst_head + N * sub;
    store_values<DTYPE>(h.dst, to, vout, y);
    store_values<DTYPE>(h.dst, to + D / 2, vout, z);
  }
}

// The same for a dtype known at run time, shared by the TH threads of the
// workgroups `wg` of `wgs`: each takes a run of whole rows.
template <int D, int TH>
__device__ __forceinline__ void rotate_queries(const Rotation &r, int64_t rows, int64_t wg, int64_t wgs) {
  if (!r.q) return;
  const HeadRows h{r.q, r.q_out, r.q_heads, r.q_row_stride, r.q_head_stride, r.q_out_row_stride, r.q_out_head_stride, r.q_norm};
  auto go = [&](auto dtype) {
    constexpr int DT = decltype(dtype)::value, L = D / (2 * kPer<DT>);
    // (a run of rows holds at most 2^16 items of a 32-bit count, and one row any number of heads)
    const int64_t run = max((int64_t)1, min((rows + wgs - 1) / wgs, (int64_t)(65536 / r.q_heads)));
    for (int64_t row0 = wg * run; row0 < rows; row0 += wgs * run)
      rotate_items<D, DT>(h, r, row0, (int)min(run, rows - row0), threadIdx.x / L, TH / L, threadIdx.x % L);
  };
  if (r.q_dtype == BGTQ_DTYPE_F32) go(std::integral_constant<int, BGTQ_DTYPE_F32>{});
  else if (r.q_dtype == BGTQ_DTYPE_F16) go(std::integral_constant<int, BGTQ_DTYPE_F16>{});
  else go(std::integral_constant<int, BGTQ_DTYPE_BF16>{});
}

}  // namespace rot
}  // namespace bgtq
