// Attention backward, what its kernels (fa_bwd.cu, fa_window_bwd.cu) share: the tile shapes, the order of the blocks, and how
// products are issued and results stored.
#pragma once
#include "tcgen05.cuh"

namespace ixb {
namespace fab {

constexpr int BM = 128;  // query rows per tile
constexpr int BN = 128;  // keys per tile
constexpr int HD = 128;  // head dimension
constexpr int kStages = 2;  // (the issuers pick stage descriptors with two-way selects: no local-memory arrays)
constexpr int kTileBytes = 128 * HD * 2;
constexpr int kHalfBytes = kTileBytes / 2;
constexpr int NG = 2;             // groups of element-wise warps; each takes 128 / NG columns of a tile
constexpr int GC = 128 / NG;      // columns per group
constexpr int kWorkers = 128 * NG;

struct Out {
  void* ptr;
  long long sb, sh, ss;  // strides in elements
  bool wide;             // every row is a multiple of 32 bytes
};

__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, bool is_bf16) {
  if (is_bf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_pair(uint32_t w, bool is_bf16) {
  if (is_bf16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// One arrival per warp: every lane has fenced its tensor-memory accesses, the warp
// synchronises, lane 0 arrives (the barrier counts warps, not threads).
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) tc::mbar_arrive(bar);
}

// CTA order: heads in groups of `head_group` (their operands stay in L2 while the group
// runs); inside a group tile `slot` of every head before tile `slot + 1` of any.
__device__ __forceinline__ void cta_order(int index, int n_tiles, int n_bh, int head_group, int* slot, int* bh) {
  const int per_group = n_tiles * head_group;
  const int group = index / per_group;
  const int in_group = index - group * per_group;
  const int left = n_bh - group * head_group;
  const int g_heads = left < head_group ? left : head_group;
  *slot = in_group / g_heads;
  *bh = group * head_group + in_group % g_heads;
}

__device__ __forceinline__ void load_tile(unsigned char* dst, const CUtensorMap* map, uint64_t* bar, int row0,
                                          int h, int b) {
  tc::tma_load_4d(dst, map, bar, 0, row0, h, b);
  tc::tma_load_4d(dst + kHalfBytes, map, bar, 64, row0, h, b);
}

// The products are issued by a whole warp through an elected lane (see tc::product_ss).
// D = A B^T, both operands K-major tiles of 128 x 128 (8 steps of 16 along the head dimension)
__device__ __forceinline__ void issue_ss(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc) {
  tc::product_ss<kHalfBytes>(d, a_desc, b_desc, idesc);
}
// D (+)= A B with A in TMEM as 16-bit pairs (group g wrote its GC values of the reduced index
// as GC / 2 columns starting at column a + GC * g) and B a tile in MN-major form (16 rows =
// 2048 bytes a step)
__device__ __forceinline__ void issue_ts(uint32_t d, uint32_t a, uint64_t b_desc_mn, uint32_t idesc,
                                         bool accumulate) {
#pragma unroll
  for (int g = 0; g < NG; ++g)
    tc::product_ts<GC / 16>(d, a + g * GC, b_desc_mn + (uint32_t)(g * GC * 128 >> 4), idesc, (accumulate || g > 0) ? 1u : 0u);
}

// The part of it that group G's values make.
template <int G>
__device__ __forceinline__ void issue_ts_group(uint32_t d, uint32_t a, uint64_t b_desc_mn, uint32_t idesc, bool accumulate) {
  tc::product_ts<GC / 16>(d, a + G * GC, b_desc_mn + (uint32_t)(G * GC * 128 >> 4), idesc, accumulate ? 1u : 0u);
}

// GC accumulator columns of this thread's row -> 16-bit values in global memory
template <bool IS_BF16>
__device__ __forceinline__ void store_cols(uint32_t taddr, unsigned char* dst, float mult, bool live, bool wide) {
#pragma unroll
  for (int c = 0; c < GC / 32; ++c) {
    uint32_t acc[32];
    tc::tmem_ld32(taddr + c * 32, acc);
    tc::tmem_wait_ld();
    if (live) tc::store_row32<IS_BF16>(dst + c * 64, acc, mult, wide);
  }
}

}  // namespace fab
}  // namespace ixb
