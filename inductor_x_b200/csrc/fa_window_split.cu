// Windowed attention forward for few tiles of rows (the meaning of the arguments: fa_window.h): fa_window_fwd.cu gives a block a
// tile or two of them and all the keys they see, one step after the other, which leaves most SMs without work where there
// are few.  Here, as in fa_split.cu, a cluster of 1, 2, 4 or 8 blocks takes ONE tile of rows and shares its key tiles: slot s = 2 * rank +
// t of a cluster walks the steps s, s + slots, ... back from the rows' own positions, the first tokens' tile last.  At
// the end every slot leaves its row maxima, sums and 32-bit accumulators in shared memory, and the blocks of the cluster add them up
// row by row through distributed shared memory: one launch, no scratch, the same bits every time.
//
//   warp 0     TMA producer: Q, then K and V tiles; a tile of each in flight for each slot; clears what of V is behind the sequence
//   warp 1     MMA issuer, the slots in turn
//   warps 4-7  softmax of slot 0, warps 8-11 of slot 1: thread <-> row (softmax_tile)
//   all        after a cluster barrier warps 4-11 merge the rows of the tile, a warp a row
//
// Every mbarrier wait is bounded and raises a flag in `status`; the hardware barriers are reached by every warp whatever happened
// to it.
//
// Bound: latency.  When it is taken, and what it measured, stands at window_split_size.
#include <atomic>
#include <cmath>
#include "fa_window.h"
#include "ixb/fa_softmax.cuh"

namespace {

using namespace ixb;
using namespace ixb::fa;

// Registers: the block starts with kRegsLaunch a thread (all that 12 warps can have); the first
// warpgroup gives up what it does not need so that a softmax thread holds its row of 128 scores.
constexpr int kRegsLaunch = 168, kRegsIssue = 80, kRegsSoftmax = 208;
static_assert(kRegsIssue + NQ * kRegsSoftmax <= (1 + NQ) * kRegsLaunch, "setmaxnreg draws on the block's own registers");
constexpr int kMaxCluster = 8;
constexpr size_t kSmemBytes = (size_t)kTileBytes * 5 + 1024;
static_assert(NQ * BM * HD * sizeof(float) <= (size_t)kTileBytes * 5, "the accumulators take the place of the operands");

struct SplitParams {
  void* o;
  float* lse;            // [B, H, Sq], may be null
  int* status;           // may be null
  const int *q_lengths, *kv_lengths;
  long long o_stride_b, o_stride_h, o_stride_s;  // elements
  int H, HK, share, Sq, Sk;
  float scale_log2;
  int window, sinks;
  int rows_log2;         // R = 1 << rows_log2 rows of a head in a tile
  int tiles;             // tiles of rows a key head has
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(const void* local_smem, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local_smem)), "r"(rank));
  return remote;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

template <bool IS_BF16, int CLUSTER>
__global__ void __launch_bounds__(kThreads, 1)
    window_split_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const SplitParams p) {
  constexpr int kSlots = NQ * CLUSTER;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* q_smem = smem;
  unsigned char* k_smem = smem + kTileBytes;       // a tile for each slot
  unsigned char* v_smem = smem + kTileBytes * 3;

  __shared__ __align__(8) uint64_t q_full, k_full[NQ], k_empty[NQ], v_full[NQ], v_empty[NQ], v_raw, s_full[NQ], p_full[NQ], p_rest[NQ],
      pv_done[NQ], drained;
  __shared__ float m_row[NQ][BM], l_row[NQ][BM];
  __shared__ uint32_t tmem_base_slot;
  __shared__ volatile int failed;

  const int warp = __shfl_sync(kFull, (int)threadIdx.x >> 5, 0);  // known uniform to the compiler
  const int lane = threadIdx.x & 31;
  const int rank = CLUSTER > 1 ? (int)cluster_rank() : 0;

  // a tile of rows (see fa_window_fwd.cu) and the key tiles that some row of it sees: [lo, hi), and with `front` tile 0
  const int R = 1 << p.rows_log2, blocks_of_heads = (p.share + (BM >> p.rows_log2) - 1) >> (7 - p.rows_log2);
  const int item = (int)blockIdx.x / CLUSTER, bh = item / p.tiles, unit = p.tiles - 1 - (item - bh * p.tiles);  // late (long) ones first
  const int b = bh / p.HK, hk = bh - b * p.HK;
  const int q_tile = unit / blocks_of_heads, i0 = q_tile * BM, h0 = hk * p.share + ((unit - q_tile * blocks_of_heads) << (7 - p.rows_log2));
  const int q_len = p.q_lengths != nullptr ? min(max(__ldg(p.q_lengths + b), 0), p.Sq) : p.Sq;
  const int kv_len = p.kv_lengths != nullptr ? min(max(__ldg(p.kv_lengths + b), 0), p.Sk) : p.Sk;
  const int off = kv_len - q_len;  // query i stands at position off + i
  const int at_first = off + i0, at_last = off + min(i0 + R, q_len) - 1;
  const bool any = i0 < q_len && at_last >= 0;
  const int lo = any ? max(max(at_first, 0) - p.window + 1, 0) / BN : 0, hi = any ? at_last / BN + 1 : 0;
  const int front = lo > 0 && p.sinks > 0 ? 1 : 0, n_kv = hi - lo + front;
  auto key_tile = [&](int s) { return s < hi - lo ? hi - 1 - s : 0; };
  auto tiles_of = [&](int t) {
    const int s = NQ * rank + t;
    return n_kv > s ? (n_kv - s + kSlots - 1) / kSlots : 0;
  };
  const int n_t[NQ] = {tiles_of(0), tiles_of(1)};  // (n_t[0] is n_t[1] or one more)

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int t = 0; t < NQ; ++t) {
      mbar_init(&k_full[t], 1);
      mbar_init(&k_empty[t], 1);
      mbar_init(&v_full[t], 1);
      mbar_init(&v_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 128);
      mbar_init(&p_rest[t], 128);
      mbar_init(&pv_done[t], 1);
    }
    mbar_init(&v_raw, 1);
    mbar_init(&drained, 1);
    failed = 0;
    mbar_init_fence();
  }
  if (warp == 1) tc::tmem_alloc(&tmem_base_slot, kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = tmem_base_slot;

  int q_loads = 0, k_loads[NQ] = {0, 0}, v_loads[NQ] = {0, 0};  // producer: what it has asked for
  bool raw_pending = false;                                     // a copy completes v_raw, not v_full
  float m_used = -INFINITY, l = 0.f;                            // softmax warps: this thread's row
  const int t_own = (warp >> 2) - 1;                            // and the slot it belongs to
  const int row_own = (warp & 3) * 32 + lane;
  const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
  if (warp < 4) {
    tc::regs_dec<kRegsIssue>();
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer
      if (n_t[0] > 0) {
        bool good = true;
        q_loads = 1;
        if (lane == 0) {
          // rows and heads past the end of the tensor are zero-filled
          mbar_arrive_expect_tx(&q_full, kTileBytes);
          unsigned char* qd = q_smem;
          for (int g = 0; g < BM >> p.rows_log2; ++g, qd += R * 128) {
            tc::tma_load_4d(qd, &map_q, &q_full, 0, i0, h0 + g, b);
            tc::tma_load_4d(qd + kHalfBytes, &map_q, &q_full, 64, i0, h0 + g, b);
          }
        }
        for (int k = 0; k < n_t[0] && good; ++k) {
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            if (k >= n_t[t] || !good) continue;
            const int key0 = key_tile(NQ * rank + t + k * kSlots) * BN;
            good = k == 0 || __all_sync(kFull, mbar_wait(&k_empty[t], (k - 1) & 1, &failed));
            if (!good) continue;
            if (lane == 0) {
              unsigned char* kd = k_smem + t * kTileBytes;
              mbar_arrive_expect_tx(&k_full[t], kTileBytes);
              tc::tma_load_4d(kd, &map_k, &k_full[t], 0, key0, hk, b);
              tc::tma_load_4d(kd + kHalfBytes, &map_k, &k_full[t], 64, key0, hk, b);
            }
            k_loads[t] = k + 1;
          }
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            if (k >= n_t[t] || !good) continue;
            const int key0 = key_tile(NQ * rank + t + k * kSlots) * BN, live = kv_len - key0;
            good = k == 0 || __all_sync(kFull, mbar_wait(&v_empty[t], (k - 1) & 1, &failed));
            if (!good) continue;
            unsigned char* vd = v_smem + t * kTileBytes;
            const bool clear = live < BN && kv_len < p.Sk;  // the tile reaches behind the sequence, and not behind the tensor
            uint64_t* bar = clear ? &v_raw : &v_full[t];
            if (lane == 0) {
              mbar_arrive_expect_tx(bar, kTileBytes);
              tc::tma_load_4d(vd, &map_v, bar, 0, key0, hk, b);
              tc::tma_load_4d(vd + kHalfBytes, &map_v, bar, 64, key0, hk, b);
            }
            if (clear) {  // (one tile of all: the sequence's last)
              raw_pending = true;
              good = __all_sync(kFull, mbar_wait(&v_raw, 0, &failed));
              if (!good) continue;
              raw_pending = false;
              for (int at = live * 8 + lane; at < BN * 8; at += 32) {
                *reinterpret_cast<uint4*>(vd + at * 16) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(vd + kHalfBytes + at * 16) = make_uint4(0, 0, 0, 0);
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0) tc::mbar_arrive(&v_full[t]);
            }
            v_loads[t] = k + 1;
          }
        }
        if (!good && lane == 0) failed = 1;
      }
      __syncwarp();
    } else if (warp == 1 && n_t[0] > 0) {
      // -------------------------------------------------------------------- MMA issuer
      // The whole warp runs this role and an elected lane issues (see tc::product_ss).
      constexpr uint32_t idesc_qk = tc::instr_desc(BM, BN, IS_BF16 ? 1 : 0, 0, 0);
      constexpr uint32_t idesc_pv = tc::instr_desc(BM, HD, IS_BF16 ? 1 : 0, 0, 1);
      const uint32_t tmem = __shfl_sync(kFull, tmem_base, 0);
      const uint64_t q_desc = tc::smem_desc(smem_u32(q_smem), 16, 1024);
      const uint64_t k_desc = tc::smem_desc(smem_u32(k_smem), 16, 1024);
      const uint64_t v_desc = tc::smem_desc(smem_u32(v_smem), kHalfBytes, 1024);
      auto wait = [&](uint64_t* bar, int parity) {
        const bool up = __all_sync(kFull, mbar_wait(bar, parity, &failed));
        tc::fence_after_sync();
        return up;
      };
      auto issue_qk = [&](int t) {
        tc::product_ss<kHalfBytes>(tmem + kColS + t * 128, q_desc, k_desc + (uint32_t)(t * (kTileBytes >> 4)), idesc_qk);
        tc::commit_elected(&s_full[t]);
        tc::commit_elected(&k_empty[t]);
      };
      bool ok = wait(&q_full, 0);
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        if (!ok || n_t[t] == 0) continue;
        ok = wait(&k_full[t], 0);
        if (ok) issue_qk(t);
      }
      for (int k = 0; k < n_t[0] && ok; ++k) {
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
          if (!ok || k >= n_t[t]) continue;
          ok = wait(&v_full[t], k & 1) && wait(&p_full[t], k & 1);
          if (!ok) continue;
          const uint64_t vd = v_desc + (uint32_t)(t * (kTileBytes >> 4));
          const uint32_t o = tmem + kColO + t * 128, pa = tmem + kColS + t * 128;
          tc::product_ts<kSplit / 16>(o, pa, vd, idesc_pv, k > 0);
          ok = wait(&p_rest[t], k & 1);
          if (!ok) continue;
          // (16 keys of V are 2048 bytes of a 64-column box)
          tc::product_ts<(BN - kSplit) / 16>(o, pa + kSplit / 2, vd + (uint32_t)(kSplit / 16 * 2048 >> 4), idesc_pv, 1u);
          tc::commit_elected(&v_empty[t]);
          if (k + 1 < n_t[t]) {
            ok = wait(&k_full[t], (k + 1) & 1);
            if (ok) issue_qk(t);  // (P of this tile has been consumed by the MMAs just issued: they run in order)
          } else {
            tc::commit_elected(&pv_done[t]);
          }
        }
      }
      if (!ok && lane == 0) failed = 1;
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------------- softmax
    tc::regs_inc<kRegsSoftmax>();
    const uint32_t s_addr = lane_addr + kColS + t_own * 128, o_addr = lane_addr + kColO + t_own * 128;
    const int mine = t_own ? n_t[1] : n_t[0];
    const int qi = i0 + (row_own & (R - 1));
    const int at = qi < q_len ? off + qi : -1;  // (below 0: sees nothing)
    bool ok = true;
    for (int k = 0; k < mine; ++k) {
      ok = __all_sync(kFull, mbar_wait(&s_full[t_own], k & 1, &failed));
      if (!ok) break;
      tc::fence_after_sync();
      const int col0 = key_tile(NQ * rank + t_own + k * kSlots) * BN;
      WindowMask mask;
      mask.edge = col0 + BN - 1 > at_first || col0 <= at_last - p.window;
      mask.lim = at - col0;
      mask.from = col0 == 0 ? p.sinks : 0;
      mask.low = at - p.window + 1 - col0;
      softmax_tile<IS_BF16>(s_addr, o_addr, mask, k == 0, p.scale_log2, m_used, l, &p_full[t_own], &p_rest[t_own]);
    }
    if (ok && mine > 0) ok = __all_sync(kFull, mbar_wait(&pv_done[t_own], 0, &failed));  // the slot's last product
    if (!ok && lane == 0) failed = 1;
  }

  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const bool gave_up = failed != 0;  // (uniform: nobody writes it any more)
  if (gave_up) {
    // a role gave up: what the others have under way has to end before the block does
    if (threadIdx.x == 0) {
      tc::await_copies<1>(&q_full, q_loads);
      if (raw_pending) mbar_wait(&v_raw, 0);
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        tc::await_copies<1>(&k_full[t], k_loads[t]);
        tc::await_copies<1>(&v_full[t], v_loads[t]);
      }
      if (p.status != nullptr) atomicExch(p.status, 1);
    }
    if (warp == 1) tc::await_products(&drained);
    __syncthreads();
  }
  // Every product has ended and every copy has been consumed: the accumulators take the operands' place,
  // row after row, their 16-byte pieces swizzled by the row (a thread writes a row, a warp reads one).
  float4* o_smem = reinterpret_cast<float4*>(smem);
  constexpr int kPieces = HD / 4;
  constexpr int rows = BM;
  if (warp >= 4) {
    m_row[t_own][row_own] = gave_up ? -INFINITY : m_used;
    l_row[t_own][row_own] = gave_up ? 0.f : l;
    if (!gave_up && (t_own ? n_t[1] : n_t[0]) > 0) {
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tc::tmem_ld32(lane_addr + kColO + t_own * 128 + c * 32, o);
        tc::tmem_wait_ld();
        {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            o_smem[(t_own * BM + row_own) * kPieces + ((c * 8 + e) ^ lane)] =
                make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                            __uint_as_float(o[4 * e + 3]));
        }
      }
    }
  }
  tc::fence_before_sync();
  __syncwarp();
  if constexpr (CLUSTER > 1) cluster_sync_all();
  else __syncthreads();
  if (warp >= 4) {
    // several rows at a time (with more blocks a warp has fewer): one by one every row waits for its loads
    // and its two folds, 3 us for 128 rows of one block
    constexpr int kRows = CLUSTER <= 2 ? 4 : 8 / CLUSTER, kStep = 8 * CLUSTER;
    for (int r0 = rank * 8 + warp - 4; r0 < rows; r0 += kRows * kStep) {
      float w[kRows], top[kRows], total[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        // lane s: the statistics of slot s
        const int r = r0 + i * kStep;
        float m = -INFINITY, ls = 0.f;
        if (lane < kSlots && r < rows) {
          if constexpr (CLUSTER > 1) {
            m = ld_cluster_f32(map_to_rank(&m_row[lane % NQ][r], lane / NQ));
            ls = ld_cluster_f32(map_to_rank(&l_row[lane % NQ][r], lane / NQ));
          } else {
            m = m_row[lane][r];
            ls = l_row[lane][r];
          }
        }
        top[i] = m;  // (-inf: the slot saw nothing of the row, or nothing but NaN, which its sum says)
        total[i] = ls;
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const float m = top[i];
        top[i] = warp_max_fast(m);
        w[i] = m == -INFINITY ? 0.f : fast_exp2(m - top[i]);
        total[i] = warp_reduce<SumOp>(w[i] * total[i]);
      }
      float4 acc[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        float4 v[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int r = r0 + i * kStep;
          const float4* piece = &o_smem[(s % NQ * BM + r) * kPieces + (lane ^ (r & 31))];
          // (a slot without a key tile wrote nothing; every other one counts whatever it weighs, since no weight
          // makes a NaN or an infinity of it go away)
          v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (s < n_kv && r < rows) v[i] = CLUSTER > 1 ? ld_cluster_f32x4(map_to_rank(piece, s / NQ)) : *piece;
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const float ws = __shfl_sync(kFull, w[i], s);
          acc[i].x = fmaf(ws, v[i].x, acc[i].x);
          acc[i].y = fmaf(ws, v[i].y, acc[i].y);
          acc[i].z = fmaf(ws, v[i].z, acc[i].z);
          acc[i].w = fmaf(ws, v[i].w, acc[i].w);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = r0 + i * kStep;
        if (r >= rows) break;
        const int qi = i0 + (r & (R - 1)), h = h0 + (r >> p.rows_log2);
        if (qi >= p.Sq || h >= (hk + 1) * p.share) continue;
        const bool sees = qi < q_len && off + qi >= 0;  // (tiles that all other rows see whole are not masked)
        const float sum = sees ? total[i] : 0.f, inv = sum == 0.f ? 0.f : 1.f / sum;  // (a sum may be NaN)
        uint2 out = make_uint2(0, 0);
        if (sum != 0.f) {
          out.x = tc::round_pair<IS_BF16>(acc[i].x * inv, acc[i].y * inv);
          out.y = tc::round_pair<IS_BF16>(acc[i].z * inv, acc[i].w * inv);
        }
        *reinterpret_cast<uint2*>(reinterpret_cast<unsigned char*>(p.o) +
                                  2 * ((long long)b * p.o_stride_b + (long long)h * p.o_stride_h + (long long)qi * p.o_stride_s) + lane * 8) = out;
        if (lane == 0 && p.lse != nullptr)
          p.lse[((long long)b * p.H + h) * p.Sq + qi] = sum == 0.f ? -INFINITY : (top[i] + log2f(sum)) * 0.69314718055994530942f;
      }
    }
  }
  // nobody leaves while another block of the cluster reads its shared memory
  __syncwarp();
  if constexpr (CLUSTER > 1) cluster_sync_all();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem_base, kTmemCols);
  }
}

// The opt-ins of a kernel on the current device, asked for once: a property of (kernel, device).
template <bool IS_BF16, int CLUSTER>
int configure(int devid) {
  auto kern = window_split_kernel<IS_BF16, CLUSTER>;
  static std::atomic<bool> configured[64];
  std::atomic<bool>& done = configured[devid & 63];
  if (!done.load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e != cudaSuccess) return ixb_host::cuda_status(e);
    cudaFuncAttributes at;  // (as in fa_fwd.cu: the softmax warps wait for registers the block has to own)
    e = cudaFuncGetAttributes(&at, kern);
    if (e != cudaSuccess) return ixb_host::cuda_status(e);
    if (at.numRegs != kRegsLaunch) return IXB_ERR_UNSUPPORTED;
    done.store(true, std::memory_order_release);
  }
  return IXB_OK;
}

template <int CLUSTER>
cudaLaunchConfig_t launch_config(long long blocks, cudaLaunchAttribute* attr, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = CLUSTER;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER > 1 ? 1 : 0;
  return cfg;
}

template <bool IS_BF16, int CLUSTER>
int launch_split(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const SplitParams& p, long long items, cudaStream_t stream) {
  int devid = 0;
  cudaGetDevice(&devid);
  if (int st = configure<IS_BF16, CLUSTER>(devid)) return st;
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = launch_config<CLUSTER>(items * CLUSTER, &attr, stream);
  return ixb_host::cuda_status(cudaLaunchKernelEx(&cfg, window_split_kernel<IS_BF16, CLUSTER>, mq, mk, mv, p));
}

// Blocks of clusters of this size that the current device runs at a time (0: none), asked for once.
template <int CLUSTER>
int room_for(int devid) {
  static std::atomic<int> known[64];  // one more than the number
  std::atomic<int>& room = known[devid & 63];
  int n = room.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = launch_config<CLUSTER>(CLUSTER, &attr, nullptr);
    int clusters = 0;
    if (configure<true, CLUSTER>(devid) != IXB_OK ||
        cudaOccupancyMaxActiveClusters(&clusters, window_split_kernel<true, CLUSTER>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      clusters = 0;
    }
    n = 1 + clusters * CLUSTER;
    room.store(n, std::memory_order_relaxed);
  }
  return n - 1;
}
int room_for(int cluster, int devid, int sms) {
  return cluster == 1 ? sms : cluster == 2 ? room_for<2>(devid) : cluster == 4 ? room_for<4>(devid) : room_for<8>(devid);
}

}  // namespace

namespace ixb_host {

static long long tiles_of_rows(const WindowShape& a, int* rows_log2) {
  int log2 = 3;
  while (log2 < 7 && (1 << log2) < a.Sq) ++log2;
  if (rows_log2 != nullptr) *rows_log2 = log2;
  const int heads = BM >> log2;  // query heads in a tile
  return ((long long)a.Sq + BM - 1) / BM * ((a.H / a.HK + heads - 1) / heads);
}

// Times as measured on one B200 (84 shapes of 1 to 256 tiles of rows over windows of 256 to 4096 keys, within 15 %), in us:
//   fa_window_fwd.cu  4.7 + 1.41 a step of 128 keys; with more tiles than SMs 7.5 + 1.6 a step for each round over the SMs of the
//                     pairs of tiles of a key head
//   one block a tile  8.7 + 1.65 for each step of its longer slot
//   a cluster         9.7 + 1.8 for each of them, as long as all blocks run at once (a second round doubles it)
//   both of these     not less than 1.25 for each step's 64 KB an SM: 128 key heads of two rows, 4096 keys 52, fa_window_decode.cu 45
// 16 tiles, windows of 256, 1024 and 4096 keys: fa_window_fwd.cu 11.8, 20.2 and 54, one block 13.6, 18.7 and 38.5, two 12.2, 16.1 and
// 26, four 11.9, 14.7 and 19.8; 8 tiles and eight blocks 12, 12.3 and 17.3; 128 tiles 13.4, 21.9 and 56, one block 14.7, 20 and 40.5.
int window_split_size(const WindowShape& a, double* us) {
  const ixb_devinfo* dev = current_device();
  int devid = 0;
  *us = 0;
  if (dev == nullptr || cudaGetDevice(&devid) != cudaSuccess) return 0;
  const double sms = dev->sm_count, heads = (double)a.B * a.HK, tiles = (double)tiles_of_rows(a, nullptr), items = tiles * heads;
  const double reach = (double)a.window + (a.Sq < BM ? a.Sq : BM) + BM - 2, keys = reach < a.Sk ? reach : a.Sk;
  const double steps = ceil(keys / BN) + (a.sinks > 0 && a.window < a.Sk ? 1 : 0);
  const double plain = items <= sms ? 4.7 + 1.41 * steps : 7.5 + 1.6 * steps * ceil(heads * ceil(tiles / 2) / sms);
  double best = 0.95 * plain;  // (not for less than the estimates are worth)
  int cluster = 0;
  for (int c = 1; c <= kMaxCluster; c *= 2) {
    const double longer = ceil(steps / (2 * c)), chain = (c == 1 ? 1.65 : 1.8) * longer, load = 1.25 * heads * steps / sms;
    const double time = (c == 1 ? 8.7 : 9.7) + (chain > load ? chain : load);
    if (items * c > sms || !(time < best)) continue;
    const int room = room_for(c, devid, dev->sm_count);
    if (room <= 0 || items * c > room) continue;
    best = time;
    cluster = c;
  }
  *us = cluster ? best : plain;
  return cluster;
}

int window_split(int cluster, const WindowShape& a, const WindowView& q, const WindowView& k, const WindowView& v, const WindowView& o,
                 float* lse, int32_t* status, cudaStream_t stream) {
  SplitParams p;
  const long long tiles = tiles_of_rows(a, &p.rows_log2), items = tiles * a.B * a.HK;
  if (items > (1 << 27)) return IXB_ERR_SHAPE;
  CUtensorMap mq, mk, mv;
  if (int st = make_fa_map(&mq, q.ptr, a.is_bf16, a.B, a.H, a.Sq, q.strides[0], q.strides[1], q.strides[2], 1 << p.rows_log2)) return st;
  if (int st = make_fa_map(&mk, k.ptr, a.is_bf16, a.B, a.HK, a.Sk, k.strides[0], k.strides[1], k.strides[2])) return st;
  if (int st = make_fa_map(&mv, v.ptr, a.is_bf16, a.B, a.HK, a.Sk, v.strides[0], v.strides[1], v.strides[2])) return st;
  p.o = const_cast<void*>(o.ptr);
  p.lse = lse;
  p.status = status;
  p.q_lengths = a.q_lengths;
  p.kv_lengths = a.kv_lengths;
  p.o_stride_b = o.strides[0], p.o_stride_h = o.strides[1], p.o_stride_s = o.strides[2];
  p.H = a.H, p.HK = a.HK, p.share = a.H / a.HK, p.Sq = a.Sq, p.Sk = a.Sk;
  p.scale_log2 = a.scale * kLog2e;
  p.window = a.window, p.sinks = a.sinks;
  p.tiles = (int)tiles;
#define IXB_SPLIT_CASE(C) \
  if (cluster == C) return a.is_bf16 ? launch_split<true, C>(mq, mk, mv, p, items, stream) : launch_split<false, C>(mq, mk, mv, p, items, stream);
  IXB_SPLIT_CASE(1)
  IXB_SPLIT_CASE(2)
  IXB_SPLIT_CASE(4)
  IXB_SPLIT_CASE(8)
#undef IXB_SPLIT_CASE
  return IXB_ERR_UNSUPPORTED;
}

}  // namespace ixb_host
