// Attention of chunks over the paged cache: units of more than 32 query columns.
//
// A workgroup has W waves of 32 columns each, of one KV head: the chunk's rows x
// the G heads of its group, row-major, so all of them share the blocks of 64 K
// and V rows that go HBM -> LDS by DMA into two buffers (prompt.hip), one barrier a
// block. The rows are FP16 pages as they lie, or those that chunk_rows.h
// rebuilt (contiguous, in the code domain).
//
// Measured: 2048 rows behind 30720 tokens, 14 / 2 heads of d=64 in BF16: 300 to 340 us
// of a call's 312 to 330 (the clocks differ), 690 to 780 TFLOP/s; prompt.hip reaches 715
// on d=64. A wave's block is 290 instructions, 1100 cycles of the vector unit's, beside 512
// of products: 204 us of this call at four waves per SIMD without a stall. The
// rest is set-up, partials (69 MB, read back by the merge in 22 us) and the last
// round's idle workgroups. FP16 queries on packed K issue 1024 cycles of products (hi and lo parts).
#include "chunk_wave.h"

namespace bgtq {
namespace {

// SRC: the pool's FP16 pages; rebuilt rows of FP16 K; rebuilt rows in the code domain.
enum { kPages, kRebuilt, kCoded };

template <int D, int SRC, bool BF>
struct Wide {
  static constexpr bool SPLIT = SRC == kCoded && !BF;
  static constexpr int W = chunk_wide_waves(D, SPLIT), PER_SIMD = chunk_wide_waves_per_simd(D, SPLIT);
  static constexpr int TILE = kChunkKeys * D * 2, BUFFER = (SPLIT ? 3 : 2) * TILE;  // K, V (K's low parts)
  static constexpr int LDS = 2 * BUFFER;
  static_assert(LDS <= kLdsLimit, "LDS of one workgroup");
};

template <int D, int SRC, bool BF>
__global__ __launch_bounds__((64 * Wide<D, SRC, BF>::W), (Wide<D, SRC, BF>::PER_SIMD)) void chunk_wide_kernel(ChunkParams p) {
  using X = Wide<D, SRC, BF>;
  constexpr bool SPLIT = X::SPLIT;
  constexpr int W = X::W, TILE = X::TILE, PR = D / 8, COLUMNS = 32 * W;
  constexpr int DMAS = TILE / 1024 / W;  // DMAs per wave and operand
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item it = find_item(p, blockIdx.x, kWideUnits, COLUMNS, p.aim);
  if (it.splits == 0) return;  // uniform for the workgroup
  const Columns cs(it, p.group, COLUMNS);
  const Blocks bl = Blocks::of<kChunkKeys>(cs.first, min(cs.last, it.n - 1), p.window, p.sinks);
  const int b0 = (int)((int64_t)bl.count * it.split / it.splits), b1 = (int)((int64_t)bl.count * (it.split + 1) / it.splits);
  const int kv = it.kv;
  // The table's entry of a block's half, and whether it names a page. Blocks of pages look theirs up two blocks ahead, since the
  // DMAs need them; rebuilt ones are tested before the loop, and in it only where a page is missing.
  const int32_t *const table = p.page_table + (int64_t)it.seq * p.page_table_stride;
  auto entry_of = [&](int i, int half) {
    const int t = bl.at<kChunkKeys>(min(i, b1 - 1)) + 32 * half;
    return table[min(t >> p.page_shift, p.table_pages - 1)];
  };
  auto entry = [&](int i) { return entry_of(i, lane >> 5); };
  auto in_pool = [&](int e) -> uint64_t { return __builtin_amdgcn_ballot_w64((uint32_t)e < (uint32_t)p.pages); };
  auto issue = [&](int i, int e) {  // e: the block's entries (pages)
    const int t0 = bl.at<kChunkKeys>(i);
    uint8_t *const buf = smem + (i & 1) * X::BUFFER;
    if constexpr (SRC == kPages) {
      const int in_page = (1 << p.page_shift) - 1;
      // A DMA's rows lie in one half of the block, so in one page; rows behind the sequence's, or of no page, arrive as zeros.
#pragma unroll
      for (int k = 0; k < DMAS; ++k) {
        const int d = wave * DMAS + k, piece = d * 64 + lane, r = piece / PR, c = (piece % PR) ^ swizzle<D>(r);
        const bool upper = d >= TILE / 2048;
        const int th = t0 + (upper ? 32 : 0), pg = __builtin_amdgcn_readlane(e, upper ? 32 : 0);
        const bool ok = (uint32_t)pg < (uint32_t)p.pages;
        const int in = ok ? min(32, max(0, it.n - th)) : 0;
        const int64_t at = ok ? pg : 0;
        const __amdgpu_buffer_rsrc_t rk = rsrc(scalar(p.k + kv * p.k_head + at * p.k_page + (int64_t)(th & in_page) * D), (uint32_t)__builtin_amdgcn_readfirstlane(in) * 2 * D);
        const __amdgpu_buffer_rsrc_t rv = rsrc(scalar(p.v + kv * p.v_head + at * p.v_page + (int64_t)(th & in_page) * D * 2), (uint32_t)__builtin_amdgcn_readfirstlane(in) * 2 * D);
        const uint32_t o = (uint32_t)((r & 31) * (2 * D) + c * 16);
        dma16(rk, buf + d * 1024, o, 0);
        dma16(rv, buf + TILE + d * 1024, o, 0);
      }
    } else {
      const int64_t at = (kv * p.rebuilt_head + it.base + t0) * D;
      const __amdgpu_buffer_rsrc_t rk = rsrc(scalar(p.rebuilt_k + at), TILE), rv = rsrc(scalar(p.rebuilt_v + at), TILE);
#pragma unroll
      for (int k = 0; k < DMAS; ++k) {
        const int d = wave * DMAS + k, piece = d * 64 + lane, r = piece / PR, c = (piece % PR) ^ swizzle<D>(r);
        const uint32_t o = (uint32_t)(r * (2 * D) + c * 16);
        dma16(rk, buf + d * 1024, o, 0);
        dma16(rv, buf + TILE + d * 1024, o, 0);
        if constexpr (SPLIT) dma16(rsrc(scalar(p.rebuilt_lo + at), TILE), buf + 2 * TILE + d * 1024, o, 0);
      }
    }
  };
  int e0 = 0, e1 = 0;  // the entries of block i, i + 1
  bool none_missing = true;
  if (b0 < b1) {
    if constexpr (SRC == kPages) {
      e0 = entry(b0), e1 = entry(b0 + 1);
    } else {
      bool ok = true;
#pragma unroll 4
      for (int i = b0; i < b1; i += 32) {
        const int at = i + (lane & 31);
        // (a half behind the sequence's tokens is seen by nobody, and its entry may be anything)
        ok &= (uint32_t)entry_of(at, lane >> 5) < (uint32_t)p.pages || bl.at<kChunkKeys>(min(at, b1 - 1)) + 32 * (lane >> 5) >= it.n;
      }
      none_missing = __builtin_amdgcn_ballot_w64(!ok) == 0;
    }
  }
  Wave<D, SPLIT, BF> w;
  if constexpr (SRC == kCoded) w.load_turned(p, it, cs, 32 * wave);
  else w.load_plain(p, it, cs, 32 * wave);
  // Waited for here: left to the loop, the wait would take the next block's DMAs with it.
#pragma unroll
  for (int s = 0; s < D / 16; ++s) asm volatile("" : "+v"(w.qh[s]));
  if (b0 < b1) issue(b0, e0);
  // This wave's columns' positions; a wave past the tile's columns only loads.
  const bool any = 32 * wave < cs.count;
  const int lo = cs.before + (cs.col0 + min(32 * wave, cs.count - 1)) / p.group,
            hi = cs.before + (cs.col0 + min(32 * wave + 31, cs.count - 1)) / p.group;
  // The next block: it has landed, and the one after it is on its way.
  auto arrive = [&](int i) -> uint64_t {
    wait_vm<0>();   // this wave's part of block i has landed
    lds_barrier();  // everyone's has, and everyone is done with the other buffer
    if constexpr (SRC == kPages) {
      const uint64_t there = in_pool(e0);
      e0 = e1;
      if (i + 1 < b1) {
        e1 = entry(i + 2);
        __builtin_amdgcn_sched_barrier(0);  // (ahead of the DMAs: its wait leaves them in flight)
        issue(i + 1, e0);
      }
      return there;
    }
    uint64_t there = ~0ull;
    if (!none_missing) there = in_pool(entry(i));
    if (i + 1 < b1) issue(i + 1, 0);
    return there;
  };
  auto attend = [&](auto masked_tag, int i, uint64_t there) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const uint32_t buf = (uint32_t)(i & 1) * X::BUFFER;
    f32x16 S[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) S[b][e] = 0.0f;
    if constexpr (SPLIT) {
      w.qk(smem, buf + 2 * TILE, S, false);
      w.low_parts(S);
    }
    w.qk(smem, buf, S, true);
    uint64_t seen = ~0ull;
    bool odd = false;
    if constexpr (MASKED) {
      seen = w.seen_bits(bl.at<kChunkKeys>(i), there);
      // A token that a query does not see has probability 0, but 0 times an infinity or a NaN of its V row is not 0.
      float z = 0.0f;
      int mine = lane;
      asm volatile("" : "+v"(mine));  // (not held across the loop)
#pragma unroll
      for (int k = 0; k < PR; ++k) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(smem + buf + TILE + (64 * k + mine) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) z = odd2(v[e], z);
      }
      odd = __builtin_amdgcn_ballot_w64(z != 0.0f) != 0;
    }
    uint32_t P[16];
    w.softmax(S, P, MASKED, seen);
    if (MASKED && odd) w.template add_odd<2>(smem, buf + TILE, seen);
    w.template pv<2, MASKED>(smem, buf + TILE, P, odd);
  };
  // Runs of blocks that all queries see whole in a loop of their own, which
  // carries none of the masks' code. (Entries behind the sequence's may name no page: such blocks are seen in part anyway.)
  for (int i = b0; i < b1; ++i) {
    uint64_t there;
    for (;;) {
      there = arrive(i);
      if (there != ~0ull || !any || w.sight(bl.at<kChunkKeys>(i), kChunkKeys, lo, hi) != 2) break;
      attend(std::false_type{}, i, there);
      if (++i == b1) break;
    }
    if (i < b1 && any && w.sight(bl.at<kChunkKeys>(i), kChunkKeys, lo, hi) != 0) attend(std::true_type{}, i, there);
  }
  w.store(p, it, cs, 32 * wave, cs.count);
}

// The partials of split units: a workgroup per slot, the unit's work shared by
// its slots. (The last item to arrive merging alone took 26 to 35 us behind 12 to 400
// of the items.)
template <int D, bool BF>
__global__ __launch_bounds__(256) void chunk_merge_kernel(ChunkParams p, int tile) {
  const Item it = find_item<true>(p, blockIdx.x, kWideUnits, tile, p.aim);
  if (it.splits == 0) return;
  const Columns cs(it, p.group, tile);
  const int n = cs.count * (D / 4);
  merge_pieces<D, BF, false>(p, it, cs, n * it.split / it.splits + (int)threadIdx.x, n * (it.split + 1) / it.splits, 256);
}

template <int D, int SRC, bool BF>
hipError_t launch_one(const ChunkParams &p, int items, hipStream_t stream) {
  constexpr int lds = Wide<D, SRC, BF>::LDS;
  static const hipError_t allowed =
      hipFuncSetAttribute((const void *)chunk_wide_kernel<D, SRC, BF>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (allowed != hipSuccess) {
    (void)hipGetLastError();
    return allowed;
  }
  hipLaunchKernelGGL((chunk_wide_kernel<D, SRC, BF>), dim3((unsigned)items), dim3(64 * Wide<D, SRC, BF>::W), lds, stream, p);
  return hipGetLastError();
}
template <int D>
hipError_t launch_d(const ChunkParams &p, bool bf16, int items, hipStream_t stream) {
  if (p.packed) return bf16 ? launch_one<D, kCoded, true>(p, items, stream) : launch_one<D, kCoded, false>(p, items, stream);
  if (p.rebuilt_k) return bf16 ? launch_one<D, kRebuilt, true>(p, items, stream) : launch_one<D, kRebuilt, false>(p, items, stream);
  return bf16 ? launch_one<D, kPages, true>(p, items, stream) : launch_one<D, kPages, false>(p, items, stream);
}

}  // namespace

hipError_t launch_chunk_wide(const ChunkParams &p, int dim, bool bf16, int items, hipStream_t stream) {
  return dim == 64 ? launch_d<64>(p, bf16, items, stream) : launch_d<128>(p, bf16, items, stream);
}

hipError_t launch_chunk_merge(const ChunkParams &p, int dim, bool bf16, int tile, int slots, hipStream_t stream) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)slots), dim3(256), 0, stream, p, tile);
    return hipGetLastError();
  };
  if (dim == 64) return bf16 ? go(chunk_merge_kernel<64, true>) : go(chunk_merge_kernel<64, false>);
  return bf16 ? go(chunk_merge_kernel<128, true>) : go(chunk_merge_kernel<128, false>);
}

}  // namespace bgtq
