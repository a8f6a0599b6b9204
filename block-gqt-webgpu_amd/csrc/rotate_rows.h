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
using gfx::u32x4;

struct HeadRows {
  const void *src;
  void *dst;
  int32_t heads;
  int64_t src_row, src_head, dst_row, dst_head;  // elements
  const float *weight;                           // null: no norm
};

template <int DTYPE>
constexpr int kPer = DTYPE == BGTQ_DTYPE_F32 ? 4 : 8;  // values of 16 bytes

// 16 bytes of values from element `at` on; vec: in one access.
template <int DTYPE>
__device__ __forceinline__ u32x4 load_words(const void *src, int64_t at, bool vec) {
  u32x4 w;
  if constexpr (DTYPE == BGTQ_DTYPE_F32) {
    const uint32_t *p = static_cast<const uint32_t *>(src) + at;
    if (vec) w = *reinterpret_cast<const u32x4 *>(p);
    else
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = p[k];
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(src) + at;
    if (vec) w = *reinterpret_cast<const u32x4 *>(p);
    else
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = (uint32_t)p[2 * k] | (uint32_t)p[2 * k + 1] << 16;
  }
  return w;
}
template <int DTYPE, int N>
__device__ __forceinline__ void values_of(u32x4 w, float (&x)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if constexpr (DTYPE == BGTQ_DTYPE_F32) {
      x[k] = __uint_as_float(w[k]);
    } else {
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
// group of lanes each; `sub` is this lane's place in its group. U: items whose loads are in
// flight together, where few waves share a SIMD.
template <int D, int DTYPE, int U>
__device__ __forceinline__ void rotate_items(const HeadRows &h, const Rotation &r, int64_t row0, int rows, uint32_t first,
                                             uint32_t step, int sub) {
  constexpr int N = kPer<DTYPE>, L = D / (2 * N), E = DTYPE == BGTQ_DTYPE_F32 ? 4 : 2;
  auto aligned = [](const void *p, int64_t a, int64_t b) {
    return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(a * E) | (uintptr_t)(b * E)) & 15) == 0;
  };
  const bool vin = aligned(h.src, h.src_row, h.src_head), vout = aligned(h.dst, h.dst_row, h.dst_head);
  const uint32_t n = (uint32_t)rows * (uint32_t)h.heads;
  for (uint32_t i0 = first; i0 < n; i0 += U * step) {
    int64_t row[U];
    int head[U];
    u32x4 raw[U][2];
    const float *cs[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = U == 1 ? i0 : min(i0 + u * step, n - 1), local = i / (uint32_t)h.heads;
      head[u] = (int)(i - local * (uint32_t)h.heads);
      row[u] = row0 + local;
      const int64_t from = row[u] * h.src_row + head[u] * h.src_head + N * sub;
      raw[u][0] = load_words<DTYPE>(h.src, from, vin);
      raw[u][1] = load_words<DTYPE>(h.src, from + D / 2, vin);
      ok[u] = r.find(row[u], cs[u], D) && (U == 1 || i0 + u * step < n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float a[N], b[N], c[N], s[N];
      values_of<DTYPE>(raw[u][0], a);
      values_of<DTYPE>(raw[u][1], b);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        c[k] = cs[u][N * sub + k];
        s[k] = cs[u][D / 2 + N * sub + k];
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
      if (!ok[u]) continue;
      const int64_t to = row[u] * h.dst_row + head[u] * h.dst_head + N * sub;
      store_values<DTYPE>(h.dst, to, vout, y);
      store_values<DTYPE>(h.dst, to + D / 2, vout, z);
    }
  }
}

// The same for a dtype known at run time, shared by the TH threads of the
// workgroups `wg` of `wgs`: each takes a run of whole rows.
template <int D, int TH, int U = 1>
__device__ __forceinline__ void rotate_queries(const Rotation &r, int64_t rows, int64_t wg, int64_t wgs) {
  if (!r.q) return;
  const HeadRows h{r.q, r.q_out, r.q_heads, r.q_row_stride, r.q_head_stride, r.q_out_row_stride, r.q_out_head_stride, r.q_norm};
  auto go = [&](auto dtype) {
    constexpr int DT = decltype(dtype)::value, L = D / (2 * kPer<DT>);
    // (a run of rows holds at most 2^16 items of a 32-bit count, and one row any number of heads)
    const int64_t run = max((int64_t)1, min((rows + wgs - 1) / wgs, (int64_t)(65536 / r.q_heads)));
    for (int64_t row0 = wg * run; row0 < rows; row0 += wgs * run)
      rotate_items<D, DT, U>(h, r, row0, (int)min(run, rows - row0), threadIdx.x / L, TH / L, threadIdx.x % L);
  };
  if (r.q_dtype == BGTQ_DTYPE_F32) go(std::integral_constant<int, BGTQ_DTYPE_F32>{});
  else if (r.q_dtype == BGTQ_DTYPE_F16) go(std::integral_constant<int, BGTQ_DTYPE_F16>{});
  else go(std::integral_constant<int, BGTQ_DTYPE_BF16>{});
}

}  // namespace rot
}  // namespace bgtq
