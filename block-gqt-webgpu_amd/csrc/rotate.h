// Head norms and position rotation of rows, in FP32 and one order of roundings
// wherever a row is rotated (rotate.hip, and K on its way into pages):
//   norm (weights given)  x' = fl(fl(x r) w), r = fl32(1 / sqrt(mean(x^2) + eps))
//     with the sum, the root and the quotient in 64 bits: any order of the sum
//     gives the same r but for one row in 2^27 or so, so every kernel may sum as
//     its lanes lie;
//   pairs (i, i + D / 2) with a table row's cosine c and sine s of i:
//     y1 = fma(x1, c, -fl(x2 s)), y2 = fma(x2, c, fl(x1 s)).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bgtq {

// A call without rotation: kernels take it as their template argument.
struct NoRotation {
  static constexpr bool kOn = false;
};
// The rotation table [table_rows][D]: D / 2 cosines, then as many sines. Rows
// whose position is none of the table's are left out.
struct Rotation {
  static constexpr bool kOn = true;
  const float *table;
  int64_t table_rows;
  const int64_t *positions;
  const float *q_norm, *k_norm;  // [D] weights, null: no norm
  double eps;
  // Queries of the same rows (null: none).
  const void *q;
  void *q_out;
  int32_t q_heads, q_dtype;
  int64_t q_row_stride, q_head_stride, q_out_row_stride, q_out_head_stride;  // elements

  // Row `row`'s table row, the first one where its position is none.
  __device__ __forceinline__ bool find(int64_t row, const float *&cs, int dim) const {
    const int64_t p = positions[row];
    const bool ok = p >= 0 && p < table_rows;
    cs = table + (ok ? p : 0) * dim;
    return ok;
  }
  __device__ __forceinline__ bool kept(int64_t row) const {
    const int64_t p = positions[row];
    return p >= 0 && p < table_rows;
  }
};

namespace rot {

// v of the lane that a DPP control names, added.
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xf, 0xf, false);
  return v + __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
}
// Sum over groups of N adjacent lanes (4, 8 or 16), in every lane.
template <int N>
__device__ __forceinline__ double lanes_sum(double v) {
  v = dpp_add<0xB1>(v);               // quad_perm: lanes 1 0 3 2
  v = dpp_add<0x4E>(v);               // quad_perm: lanes 2 3 0 1
  if (N >= 8) v = dpp_add<0x141>(v);  // row_half_mirror
  if (N >= 16) v = dpp_add<0x140>(v); // row_mirror
  return v;
}
// Sum over the four 16-lane rows that share a column (lane % 16).
__device__ __forceinline__ double col_sum(double v) {
  auto swap_add = [](double x, auto swap) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const auto lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)lo[0] | (uint64_t)hi[0] << 32) +
           __builtin_bit_cast(double, (uint64_t)lo[1] | (uint64_t)hi[1] << 32);
  };
  v = swap_add(v, [](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  return swap_add(v, [](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
}
// (a square of 24 bits is exact in 64: one rounding either way)
__device__ __forceinline__ double add_square(float x, double sum) { return __builtin_fma((double)x, (double)x, sum); }
// The hardware's reciprocal root, good to 2^-24 or so, and Halley's step behind it: good to 2^-52.
__device__ __forceinline__ float factor(double sum, int dim, double eps) {
  const double v = sum / (double)dim + eps, r = __builtin_amdgcn_rsq(v);
  const double e = __builtin_fma(-(v * r), r, 1.0);
  const double better = __builtin_fma(r * e, __builtin_fma(e, 0.375, 0.5), r);
  return (float)(v > 0.0 && v < (double)INFINITY ? better : r);  // (of 0 and infinity the step makes a NaN)
}
// One value of a pair: `other` with the sine's sign, + for the pair's second
// value. Its FP32 rounding is its own: left open, the compiler joins the
// multiply-add and a rounding to FP16 behind it into one instruction that
// rounds once, and rows would differ by where they are rotated.
__device__ __forceinline__ float turn(float x, float other, float c, float s, bool second) {
  const float t = other * s;
  float y = __builtin_fmaf(x, c, second ? t : -t);
  asm("" : "+v"(y));
  return y;
}

}  // namespace rot
}  // namespace bgtq
