// Rows of K and V into and out of a pool of pages (bgtq_paged_write,
// bgtq_paged_read).
//
// Write. Packed K of few rows: a wave per row and head (encode_row.h, the
// arithmetic of encode_wave.hip), V in the same launch; of many,
// encode_tile.hip's paged kernel, V too. V and FP16 K: paged_write.h.
//
// Read. k = Rp^T cs, with cs_j = c_j s_g(j) the row in the code domain and
// Rp[j][i] the rotation with its columns in the model's order of dimensions
// (src/reference/production_math.py:27-31), 16 rows to a 16x16x32 f16 product
// with both operands split into FP16 hi and lo parts (three products, 2^-22
// relative). A lane rebuilds the eight consecutive positions that it feeds the
// product and ends with four consecutive dimensions of its row. The rotation's
// operands lie in LDS, once per workgroup. HBM's writes bound it: 131,072 rows x 2
// heads of layout B with 8-bit V to FP32 39.9 us (166 MB, 4.2 TB/s; a copy reaches
// 5.0); 4001 rows x 3 heads of the SmolLM2 tables 6.6 us, the chain of one tile.
// A write of one row x 3 heads takes 4.4 us, of 16,384 x 2 (tile encoder) 13.
#include <hip/hip_fp16.h>

#include <type_traits>

#include "bgtq_internal.h"
#include "encode_row.h"
#include "gfx950_common.h"
#include "paged_write.h"

namespace bgtq {
namespace {

using namespace gfx;
constexpr int kWaves = 4, kThreads = 64 * kWaves;

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
    if (!WITH_K && head == 1) write_rows<D, true>(p, -1, first, step);
    else write_rows<D, false>(p, -1, first, step);
    return;
  }
  const DevTables *Tg = p.tables[head];
  const int enc_bytes = p.heads[head].enc_bytes;
  const WriteLds L = write_lds<D>(enc_bytes);
  const float *rot_t = reinterpret_cast<const float *>(smem);
  const row_enc::Scratch<D> scr(smem + L.scratch + wave * L.stride);
  const int64_t nwaves = (int64_t)gridDim.x * kWaves;
  // The transposed rotation and the tables' header, LUT and books to LDS; the
  // first row's values meanwhile.
  {
    const uint8_t *tb = reinterpret_cast<const uint8_t *>(Tg);
    const __amdgpu_buffer_rsrc_t rr = rsrc(tb + p.heads[head].off_rot_t, D * D * 4);
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

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The rows read into: OUT is their dtype where K's and V's is the same and
// both allow vector stores, kAny where each is looked up as it is stored.
constexpr int kAny = -1;


// Rows leave in pieces of 128 bytes, eight lanes of 16 bytes to a row and
// eight rows to a store, so that every store writes whole lines (V alone to
// FP16, 262,144 rows: 10.9 us, 17.6 with 32 bytes of a row per store). Lane l
// has rows l / 8 and 8 + l / 8 of a tile's 16, kN values from dimension
// kN (l % 8) of each piece.
template <int D, int OUT>
struct Out {
  static constexpr int kN = OUT == BGTQ_DTYPE_F16 || OUT == BGTQ_DTYPE_BF16 ? 8 : 4;  // values per lane
  static constexpr int kPieces = D / (8 * kN);
};

// kN values (FP32, or FP16 pairs) to element `at` of the rows.
template <int OUT>
__device__ __forceinline__ void store_floats(void *dst, int dtype, int64_t at, const float *v) {
  if constexpr (OUT == BGTQ_DTYPE_F32) {
    *reinterpret_cast<f32x4 *>(static_cast<float *>(dst) + at) = f32x4{v[0], v[1], v[2], v[3]};
  } else if constexpr (OUT == BGTQ_DTYPE_F16 || OUT == BGTQ_DTYPE_BF16) {
    typedef typename std::conditional<OUT == BGTQ_DTYPE_F16, half2, bf16x2>::type pair;
    u32x4 o;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      o[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2 * k], v[2 * k + 1]}), pair));
    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(dst) + at) = o;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (dtype == BGTQ_DTYPE_F32) static_cast<float *>(dst)[at + k] = v[k];
      else if (dtype == BGTQ_DTYPE_F16) static_cast<_Float16 *>(dst)[at + k] = (_Float16)v[k];
      else static_cast<__bf16 *>(dst)[at + k] = (__bf16)v[k];
    }
  }
}

// The lane's parts of two V or FP16 K rows as they are stored. Loading and
// storing are apart, so that a loop issues its loads ahead of its stores: the
// memory counter is in order, and a wait for a load behind a store waits for
// the store too.
template <int D, int OUT, bool of_k>
struct Plain {
  static constexpr int N = Out<D, OUT>::kN, NP = Out<D, OUT>::kPieces;
  uint32_t w[2][NP][N / 2], scale[2];
  __device__ __forceinline__ void load(const PagedWriteParams &p, int head, const int64_t (&page)[2], const int (&at)[2], int sub) {
    const bool q8 = !of_k && p.v_scales;
    if (q8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint8_t *src = static_cast<const uint8_t *>(p.v_pool) + page[j] * p.vp_page_stride + head * p.vp_head_stride +
                             (int64_t)at[j] * D + N * sub;
#pragma unroll
        for (int c = 0; c < NP; ++c) __builtin_memcpy(w[j][c], __builtin_assume_aligned(src + 8 * N * c, N), N);
        scale[j] = p.v_scales[page[j] * p.vs_page_stride + head * p.vs_head_stride + at[j]];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint16_t *src =
            (of_k ? p.k_f16 + page[j] * p.kp_page_stride + head * p.kp_head_stride
                  : static_cast<const uint16_t *>(p.v_pool) + page[j] * p.vp_page_stride + head * p.vp_head_stride) +
            (int64_t)at[j] * D + N * sub;
#pragma unroll
        for (int c = 0; c < NP; ++c) __builtin_memcpy(w[j][c], __builtin_assume_aligned(src + 8 * N * c, 2 * N), 2 * N);
        scale[j] = 0;
      }
    }
  }
  // row0: the tile's first row; kept: bit r for its row r.
  __device__ __forceinline__ void store(const PagedWriteParams &p, int head, int64_t row0, uint32_t kept, int lane) {
    void *dst = of_k ? p.k : p.v;
    const int dtype = of_k ? p.k_dtype : p.v_dtype;
    const bool q8 = !of_k && p.v_scales;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 8 * j + (lane >> 3);
      const int64_t row = row0 + r;
      const int64_t to =
          (of_k ? row * p.k_row_stride + head * p.k_head_stride : row * p.v_row_stride + head * p.v_head_stride) + N * (lane & 7);
#pragma unroll
      for (int c = 0; c < NP; ++c) {
        uint32_t h[N / 2];
        if (q8) {
          // 8-bit V stands for the FP16 value nearest s c; c as 1024 + (c + 128) - 1152, exact.
          const half2 s = __builtin_bit_cast(half2, scale[j] | scale[j] << 16);
#pragma unroll
          for (int k = 0; k < N / 2; ++k) {
            const half2 x = __builtin_bit_cast(
                half2, __builtin_amdgcn_perm(0x64646464u, w[j][c][k >> 1] ^ 0x80808080u, k & 1 ? 0x04030402u : 0x04010400u));
            h[k] = __builtin_bit_cast(uint32_t, (x - half2{(_Float16)1152.0f, (_Float16)1152.0f}) * s);
          }
        } else {
#pragma unroll
          for (int k = 0; k < N / 2; ++k) h[k] = w[j][c][k];
        }
        if (!(kept >> r & 1u)) continue;
        if constexpr (OUT == BGTQ_DTYPE_F16) {
          *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(dst) + to + 8 * N * c) = u32x4{h[0], h[1], h[2], h[3]};
        } else {
          float v[N];
#pragma unroll
          for (int k = 0; k < N; ++k) v[k] = (float)__builtin_bit_cast(half2, h[k >> 1])[k & 1];
          store_floats<OUT>(dst, dtype, to + 8 * N * c, v);
        }
      }
    }
  }
};

// The place of row `row`: rows past the call's and slots outside the pool are
// not kept and take the pool's first row, so that no load stands under a test
// of its lane.
struct RowPlace {
  int64_t page;
  int at;
  bool kept;
};
__device__ __forceinline__ RowPlace place_of(const PagedSlots &slots, int64_t row) {
  RowPlace r;
  r.kept = slots.find(min(row, slots.rows - 1), r.page, r.at) && row < slots.rows;
  r.page = r.kept ? r.page : 0;
  r.at = r.kept ? r.at : 0;
  return r;
}

// V, and FP16 K: grid y is a head of the one, then of the other.
template <int D, int OUT>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(PagedWriteParams p, int64_t tiles) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int head = blockIdx.y % p.kv_heads;
  auto tile = [&](auto of_k, int64_t t) {
    int64_t page[2];
    int at[2];
    uint32_t kept = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const RowPlace r = place_of(p.slots, t * 16 + 8 * j + (lane >> 3));
      page[j] = r.page;
      at[j] = r.at;
      kept |= (uint32_t)r.kept << (8 * j + (lane >> 3));
    }
    Plain<D, OUT, decltype(of_k)::value> x;
    x.load(p, head, page, at, lane & 7);
    x.store(p, head, t * 16, kept, lane);
  };
  for (int64_t t = (int64_t)blockIdx.x * kWaves + wave; t < tiles; t += (int64_t)gridDim.x * kWaves) {
    if (p.k != nullptr && (int)blockIdx.y < p.kv_heads) tile(std::true_type{}, t);
    else tile(std::false_type{}, t);
  }
}

// Packed K, and V of the same rows where both are read: grid y is the head.
//
// LDS: the rotation's operands ([column tile][step][hi, lo][lane], 16 bytes
// each), the centroid books, one per kind of code that may read it (a byte
// code's at book * kByteBook + 8, a nibble code's 16 at kNibbleBooks + book *
// kNibbleBook + 4: a code's table offset then also is its bit-field extract's
// width operand, whose low 5 bits count), then per wave the staged rows and
// their scales.
constexpr int kByteBook = 1056, kNibbleBook = 96, kNibbleBooks = 8 * kByteBook, kBookBytes = kNibbleBooks + 8 * kNibbleBook;
template <int D>
struct Read {
  static constexpr int KS = D / 32, NT = D / 16;    // 32-position steps and 16-column tiles of the product
  static constexpr int W = D == 64 ? 4 : 8;         // waves: one workgroup's tables serve them all
  static constexpr int WORDS = D / 4;               // words of a packed row at most (row bytes <= D)
  static constexpr int ROWW = WORDS + 3;            // staged: two more that the last words' reads reach, odd
  static constexpr int STAGE = 16 * ROWW * 4;       // staged rows of a wave
  static constexpr int NORMW = kMaxGroups + 1;
  static constexpr int NORMS = 16 * NORMW * 4;
  static constexpr int OROW = 128 + 16;             // bytes of a row's piece on its way out, padded
  static constexpr int WAVE = (STAGE + NORMS + 15) / 16 * 16 + 16 * OROW;
  static constexpr int ROT = rot_q_bytes(D);
  static constexpr int LDS = ROT + kBookBytes + W * WAVE;
  static constexpr int WGS = D == 64 ? 3 : 1;       // per compute unit, by their LDS
};

template <int D, int OUT>
__global__ __launch_bounds__(64 * Read<D>::W, D == 64 ? 3 : 2) void paged_read_packed_kernel(PagedWriteParams p, int64_t tiles) {
  using R = Read<D>;
  constexpr int KS = R::KS, NT = R::NT, W = R::W;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t *const tabs = smem + R::ROT;
  const int tid = threadIdx.x, lane = tid & 63, gq = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = blockIdx.y;
  const int64_t t0 = (int64_t)blockIdx.x * W + wave, step = (int64_t)gridDim.x * W;
  auto place = [&](int64_t t) { return place_of(p.slots, t * 16 + col); };  // of this lane's row of tile t
  RowPlace now = place(t0), next = place(t0 + step);

  const auto &H = p.heads[head];
  const BGTQ_GLOBAL uint8_t *Tb = reinterpret_cast<const BGTQ_GLOBAL uint8_t *>(to_global(p.tables[head]));
  const int RB = H.row_bytes, NS = H.norm_stride, mc = H.max_centroids, ng = H.groups, ce = H.cent_exp;
  uint8_t *const wv = tabs + kBookBytes + wave * R::WAVE;
  uint32_t *const stage = reinterpret_cast<uint32_t *>(wv);
  float *const nstage = reinterpret_cast<float *>(wv + R::STAGE);
  uint8_t *const outs = wv + R::WAVE - 16 * R::OROW;
  const uint8_t *pk = p.packed + head * p.packed_head_stride;
  const uint16_t *nm = p.norms + head * p.norms_head_stride;
  // A row's words gq, gq + 4, ... (unaligned; the last one is read so that it
  // ends with the row and is shifted down, words past it repeat it) and scales
  // of groups gq, gq + 4 (past the groups: the last one's).
  constexpr int PER = (R::WORDS + 3) / 4;
  uint32_t w[PER], nv[kMaxGroups / 4];
  auto load_row = [&](const RowPlace &r) {
    const uint8_t *src = pk + r.page * p.packed_page_stride + (int64_t)r.at * RB;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      __builtin_memcpy(&w[k], src + min(4 * (gq + 4 * k), RB - 4), 4);
    }
    const uint16_t *ns = nm + r.page * p.norms_page_stride + (int64_t)r.at * NS;
#pragma unroll
    for (int k = 0; k < kMaxGroups / 4; ++k) nv[k] = ns[min(gq + 4 * k, ng - 1)];
  };
  load_row(now);
  {
    const __amdgpu_buffer_rsrc_t r = rsrc(reinterpret_cast<const uint8_t *>(p.tables[head]) + H.off_rot_k, R::ROT);
#pragma unroll
    for (int k = wave; k < R::ROT / 1024; k += W) dma16(r, smem + k * 1024, (k >> 1) * 2048 + lane * 32 + (k & 1) * 16, 0);
  }
  // This lane's positions 32 s + 8 gq + e (DevTables off_gdesc). Their codes
  // lie in two words of the row, e = 0..3 in the one that starts at byte
  // k0, e = 4..7 at k1. tbo: the code's table offset (and width, see above);
  // xn: its bit in the word, and above bit 5 the LDS address of its scale.
  uint32_t tbo[KS][8], xn[KS][8];
  int k0[KS], k1[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    uint32_t d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = reinterpret_cast<const BGTQ_GLOBAL uint32_t *>(Tb + H.off_gdesc)[32 * s + 8 * gq + e];
    k0[s] = (int)(d[0] & 255u);
    k1[s] = (int)(d[4] & 255u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t book = d[e] >> 12 & 15u;
      tbo[s][e] = d[e] >> 11 & 1u ? kNibbleBooks + book * kNibbleBook + 4 : book * kByteBook + 8;
      const uint32_t bit = 8 * ((d[e] & 255u) - (uint32_t)(e < 4 ? k0[s] : k1[s])) + (d[e] >> 8 & 7u);
      xn[s][e] = bit | (uint32_t)(4 * (col * R::NORMW + (int)(d[e] >> 16 & 7u))) << 5;
    }
  }
  {
    const BGTQ_GLOBAL float *books = reinterpret_cast<const BGTQ_GLOBAL float *>(Tb + H.off_books);
    for (int b = 0; b < H.books; ++b)
      for (int c = tid; c < mc; c += 64 * W) {
        const float x = books[b * mc + c];
        *reinterpret_cast<float *>(tabs + b * kByteBook + 8 + 4 * c) = x;
        if (c < 16) *reinterpret_cast<float *>(tabs + kNibbleBooks + b * kNibbleBook + 4 + 4 * c) = x;
      }
  }
  wait_vm<0>();  // the rotation's DMAs
  __syncthreads();
  float one = 1.0f;
  asm volatile("" : "+v"(one));  // (see split2_mix)
  for (int64_t tile = t0; tile < tiles; tile += step) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int o = 4 * (gq + 4 * k);
      stage[col * R::ROWW + gq + 4 * k] = w[k] >> (8 * max(0, o - max(0, RB - 4)) & 31);
    }
    // The scales times the power of two that brings the row's largest |c s|
    // to at most 2^14, in the split's range.
    float sv[kMaxGroups / 4], smax = 0.0f;
#pragma unroll
    for (int k = 0; k < kMaxGroups / 4; ++k) {
      sv[k] = f16_bits_to_f32((uint16_t)nv[k]);
      smax = fmaxf(smax, fabsf(sv[k]));
    }
    smax = col_max(smax);
    const int ex = smax > 0.0f ? ce + 126 - (int)(__float_as_uint(smax) >> 23) : 0;
#pragma unroll
    for (int k = 0; k < kMaxGroups / 4; ++k) nstage[col * R::NORMW + gq + 4 * k] = __builtin_ldexpf(sv[k], ex);
    // Loads in flight meanwhile: V, the next tile's K, the place of the one after.
    Plain<D, OUT, false> v;
    const uint32_t kept = (uint32_t)__builtin_amdgcn_ballot_w64(now.kept) & 0xffffu;
    if (p.v) {
      int64_t page[2];
      int at[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        page[j] = __shfl((int)now.page, 8 * j + (lane >> 3), 64);
        at[j] = __shfl(now.at, 8 * j + (lane >> 3), 64);
      }
      v.load(p, head, page, at, lane & 7);
    }
    load_row(next);
    const RowPlace after = place(tile + 2 * step);
    row_enc::wave_sync();
    half8 bh[KS], bl[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint32_t *w0 = stage + col * R::ROWW + (k0[s] >> 2), *w1 = stage + col * R::ROWW + (k1[s] >> 2);
      const uint32_t lo = __builtin_amdgcn_alignbyte(w0[1], w0[0], (uint32_t)k0[s]);
      const uint32_t hi = __builtin_amdgcn_alignbyte(w1[1], w1[0], (uint32_t)k1[s]);
      float cs[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t x = xn[s][e];
        asm volatile("" : "+v"(x));  // (its address is shifted out here, not held across the loop)
        const uint32_t code = __builtin_amdgcn_ubfe(e < 4 ? lo : hi, x, tbo[s][e]);
        cs[e] = *reinterpret_cast<const float *>(tabs + tbo[s][e] + 4 * code) *
                *reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(nstage) + (x >> 5));
      }
      split8_mix(cs, one, bh[s], bl[s]);
    }
    const float unscale = __builtin_ldexpf(1.0f, -ex - H.rot_exp);
    // The products of a 128-byte piece of every row, through LDS to whole lines.
    constexpr int N = Out<D, OUT>::kN, TP = 8 * N / 16;  // column tiles of a piece
#pragma unroll
    for (int c = 0; c < Out<D, OUT>::kPieces; ++c) {
#pragma unroll
      for (int tt = 0; tt < TP; ++tt) {
        f32x4 a{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const half8 *op = reinterpret_cast<const half8 *>(smem + ((c * TP + tt) * KS + s) * 2048) + lane;
          const half8 rh = op[0], rl = op[64];
          a = mfma(rh, bh[s], a);
          a = mfma(rl, bh[s], a);
          a = mfma(rh, bl[s], a);
        }
        a *= unscale;
        if constexpr (N == 4) {
          *reinterpret_cast<f32x4 *>(outs + col * R::OROW + 64 * tt + 16 * gq) = a;
        } else {
          typedef typename std::conditional<OUT == BGTQ_DTYPE_F16, half2, bf16x2>::type pair;
          *reinterpret_cast<u32x2 *>(outs + col * R::OROW + 32 * tt + 8 * gq) =
              u32x2{__builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a[0], a[1]}), pair)),
                    __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a[2], a[3]}), pair))};
        }
      }
      row_enc::wave_sync();
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = 8 * j + (lane >> 3);
        const u32x4 o = *reinterpret_cast<const u32x4 *>(outs + r * R::OROW + 16 * (lane & 7));
        if (!(kept >> r & 1u)) continue;
        const int64_t to = (tile * 16 + r) * p.k_row_stride + head * p.k_head_stride + 8 * N * c + N * (lane & 7);
        if constexpr (N == 8) {
          *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(p.k) + to) = o;
        } else {
          const f32x4 f = __builtin_bit_cast(f32x4, o);
          const float x[4] = {f[0], f[1], f[2], f[3]};
          store_floats<OUT>(p.k, p.k_dtype, to, x);
        }
      }
      row_enc::wave_sync();
    }
    if (p.v) v.store(p, head, tile * 16, kept, lane);
    row_enc::wave_sync();  // the staging is rewritten by the next tile
    now = next;
    next = after;
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

template <int D, int OUT>
hipError_t launch_read_d(const PagedWriteParams &p, int cus, hipStream_t stream) {
  const int64_t tiles = (p.slots.rows + 15) / 16;
  if (p.k && p.packed) {  // as many workgroups as are resident, so that each sets up once
    using R = Read<D>;
    static const hipError_t ok = hipFuncSetAttribute((const void *)paged_read_packed_kernel<D, OUT>,
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, kLdsLimit);
    if (ok != hipSuccess) {
      (void)hipGetLastError();
      return ok;
    }
    const int64_t wgs = std::min<int64_t>((tiles + R::W - 1) / R::W, std::max<int64_t>(1, R::WGS * (int64_t)cus / p.kv_heads));
    hipLaunchKernelGGL((paged_read_packed_kernel<D, OUT>), dim3((unsigned)wgs, (unsigned)p.kv_heads), dim3(64 * R::W), R::LDS,
                       stream, p, tiles);
  } else {
    const int64_t slices = (int64_t)p.kv_heads * ((p.k ? 1 : 0) + (p.v ? 1 : 0));
    const int64_t wgs = std::min<int64_t>((tiles + kWaves - 1) / kWaves, std::max<int64_t>(1, 8 * (int64_t)cus / slices));
    hipLaunchKernelGGL((paged_read_kernel<D, OUT>), dim3((unsigned)wgs, (unsigned)slices), dim3(kThreads), 0, stream, p, tiles);
  }
  return hipGetLastError();
}

template <int D>
hipError_t launch_read(const PagedWriteParams &p, int cus, hipStream_t stream) {
  auto vec = [](const void *base, int dtype, int64_t s0, int64_t s1) {
    const int64_t e = dtype == BGTQ_DTYPE_F32 ? 4 : 2;
    return !base || ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)(s0 * e) | (uintptr_t)(s1 * e)) & 15) == 0;
  };
  const int out = p.k ? p.k_dtype : p.v_dtype;
  if ((p.k && p.v && p.v_dtype != out) || !vec(p.k, p.k_dtype, p.k_row_stride, p.k_head_stride) ||
      !vec(p.v, p.v_dtype, p.v_row_stride, p.v_head_stride))
    return launch_read_d<D, kAny>(p, cus, stream);
  return out == BGTQ_DTYPE_F32   ? launch_read_d<D, BGTQ_DTYPE_F32>(p, cus, stream)
         : out == BGTQ_DTYPE_F16 ? launch_read_d<D, BGTQ_DTYPE_F16>(p, cus, stream)
                                 : launch_read_d<D, BGTQ_DTYPE_BF16>(p, cus, stream);
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
  return p.dim == 64 ? launch_read<64>(p, cus, stream) : launch_read<128>(p, cus, stream);
}

}  // namespace bgtq
