// Head norms and position rotation of query and key rows in one pass
// (bgtq_rotate): rotate_rows.h has the arithmetic, a workgroup a run of whole
// rows, so that the heads of a row share its table row in the L1 cache; grid y
// is the queries, then the keys. Memory and the norm's chain bound many rows: 16384 of 14 + 2 heads
// of d=64 in BF16, normed (71 MB), take 12.9 to 14.3 us where they lie in the Infinity Cache (256 MB)
// from the call before, as a layer's rows do (a copy of as much 9.6), and 19.7 over eight sets of
// buffers in turn, from HBM (a copy 15.4); one row is a launch of 2.3 us.
#include "rotate_rows.h"

namespace bgtq {
namespace {

constexpr int kThreads = 256;

// (Six waves per SIMD: those 16384 rows, cached, 12.9 us; eight, with a register spilled, 13.6, the compiler's own four 14.6.)
template <int D>
__global__ __launch_bounds__(kThreads, 6) void rotate_kernel(Rotation q, Rotation k, int64_t rows) {
  if (blockIdx.y == 0) rot::rotate_queries<D, kThreads>(q, rows, blockIdx.x, gridDim.x);
  else rot::rotate_queries<D, kThreads>(k, rows, blockIdx.x, gridDim.x);
}

}  // namespace

hipError_t launch_rotate(const Rotation &q, const Rotation &k, int64_t rows, int dim, int cus, hipStream_t stream) {
  const int64_t lanes = rows * std::max(q.q ? q.q_heads : 0, k.q ? k.q_heads : 0) * (dim / 8);
  const int64_t wgs = std::max<int64_t>(1, std::min<int64_t>({rows, (lanes + kThreads - 1) / kThreads, 8 * (int64_t)cus}));
  const dim3 grid((unsigned)wgs, k.q ? 2u : 1u);
  if (dim == 64) hipLaunchKernelGGL(rotate_kernel<64>, grid, dim3(kThreads), 0, stream, q, k, rows);
  else hipLaunchKernelGGL(rotate_kernel<128>, grid, dim3(kThreads), 0, stream, q, k, rows);
  return hipGetLastError();
}

}  // namespace bgtq
