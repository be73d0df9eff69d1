// Attention with a sliding window and first tokens that stay visible, backward, on tcgen05 tensor cores (the meaning of the
// arguments: fa_window.h).  With P = exp(S * scale - lse), dP = dO V^T, delta = rowsum(dO * O), dS = P * (dP - delta):
//   dV = P^T dO,  dK = scale * dS^T Q, both summed over the query heads that share a key head,  dQ = scale * dS K.
//   window_delta_kernel  delta[b, h, i]
//   window_dkv_kernel    an item is a key tile of a key head with the query tiles, of every head that shares it, in
//                        whose window it is; S^T and dP^T are formed and P^T and dS^T go back over them as the operands
//                        of dV and dK, which stay in tensor memory over all heads
//   window_dq_kernel     an item is a query tile of a head with the key tiles that it sees; dP has two buffers, so that the
//                        tensor core forms the scores and dP of a step while the exponentials of the one before are taken
// The first tokens are seen by all later queries, which would make one item of each key head as long as the sequence.
// What is behind the window of the first key tile is cut into items of its own, about as long as the others;
// each leaves the 32-bit sums of the first tokens' rows in scratch, and window_sinks_kernel adds them up in order.
// One owner for every sum, no atomics: the bits are the same from run to run.
//
// What lies behind a sequence's lengths may be anything.  The producers clear such rows of what meets all rows of the other
// side: Q and dO for dK and dV, K and V for dQ.  The others' only meet their own row of results, which is replaced.
//
// P and dS are rounded to the operands' 16 bits, the operands of dV, and of dK and dQ (see fa_window_fwd.cu); S, dP, delta and all sums
// have 32.  delta comes from the output as it is stored.  Gradients are 1.4 to 1.6 times as far off as the same formula in 32 bits.
//
// Every wait is bounded and raises a flag in `status`; the block leaves when its copies and products have ended.
//
// Bound: dK/dV the chain of a step, S -> P -> dV, next S (3050 cycles of which the tensor core works 2048) and items of equal
// length that do not fill the last round; dQ the exponentials and what lies between two items.  2 x 4096 tokens of 32/8 heads,
// window 1024, 4 first tokens, bf16: delta 29 us, dK/dV 252, dQ 175.  Masks inside the loop of the exponentials: 296 and 211
// (every tile pays for the selects); dQ's results and statistics by the element-wise warps 183.
#include <atomic>
#include "fa_window.h"
#include "ixb/fa_backward.cuh"

namespace {

using namespace ixb;
using namespace ixb::fab;

constexpr int kThreads = 128 + kWorkers;  // producer, issuer and scheduler; the element-wise groups
// Registers: the block starts with kRegsLaunch a thread (all that 12 warps can have)
constexpr int kRegsLaunch = 168, kRegsIssue = 80, kRegsWork = 208;
static_assert(kRegsIssue + NG * kRegsWork <= (1 + NG) * kRegsLaunch, "setmaxnreg draws on the block's own registers");
// the dQ kernel has a warpgroup more, which stores the results
constexpr int kDqThreads = kThreads + 128, kDqRegsLaunch = 128, kDqRegsIssue = 80, kDqRegsWork = 168, kDqRegsStore = 96;
static_assert(kDqRegsIssue + NG * kDqRegsWork + kDqRegsStore <= (2 + NG) * kDqRegsLaunch, "setmaxnreg draws on the block's own registers");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kCol0 = 0, kCol1 = 128, kCol2 = 256, kCol3 = 384;
constexpr int kKeyStages = 3;  // of K in the dQ kernel
constexpr size_t kDkvSmem = (size_t)kTileBytes * 6 + 1024, kDqSmem = (size_t)kTileBytes * (4 + kKeyStages) + 1024;

struct BwdParams {
  const float* lse;    // [B, H, Sq]
  const float* delta;  // [B, H, Sq]
  float* sums;         // [B * HK, 1 + chunks, 2, sinks, 128]: of dV and dK, or null without chunks
  Out dq, dk, dv;
  int* status;
  const int *q_lengths, *kv_lengths;
  int B, H, HK, share, Sq, Sk;
  float scale, scale_log2;
  int window, sinks, chunks;
};

struct Lengths {
  int q, kv, off;  // query i stands at position off + i
};
__device__ __forceinline__ Lengths lengths_of(const BwdParams& p, int b) {
  Lengths n;
  n.q = p.q_lengths != nullptr ? min(max(__ldg(p.q_lengths + b), 0), p.Sq) : p.Sq;
  n.kv = p.kv_lengths != nullptr ? min(max(__ldg(p.kv_lengths + b), 0), p.Sk) : p.Sk;
  n.off = n.kv - n.q;
  return n;
}
// the first n of 32
__device__ __forceinline__ uint32_t first_of(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// A copy of a tile of which only the first `live` rows are a sequence's: by a whole warp, which waits for it on `raw`, clears
// the other rows and completes one arrival on `full`.
__device__ __forceinline__ bool load_cleared(unsigned char* dst, const CUtensorMap* map, uint64_t* raw, int phase, uint64_t* full,
                                             int row0, int h, int b, int live, int lane, volatile int* failed, bool& pending) {
  if (lane == 0) {
    mbar_arrive_expect_tx(raw, kTileBytes);
    load_tile(dst, map, raw, row0, h, b);
  }
  pending = true;
  if (!__all_sync(kFull, mbar_wait(raw, phase, failed))) return false;
  pending = false;
  // a row is 128 bytes in each of the two boxes, whichever way its pieces are swizzled
  for (int at = live * 8 + lane; at < 128 * 8; at += 32) {
    *reinterpret_cast<uint4*>(dst + at * 16) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(dst + kHalfBytes + at * 16) = make_uint4(0, 0, 0, 0);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) tc::mbar_arrive(full);
  return true;
}

// The pending items that a running block takes over (cluster launch control), as in fa_bwd.cu.
struct Scheduler {
  uint4* answer;
  uint64_t *wanted, *full, *taken;
  __device__ __forceinline__ int take_next(int n, int lane, bool& ok, volatile int* failed) const {
    ok = ok && __all_sync(kFull, mbar_wait(&full[n & 1], (n >> 1) & 1, failed));
    if (!ok) return -1;
    const int index = __shfl_sync(kFull, tc::next_block(&answer[n & 1]), 0);
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&taken[n & 1]);
    return index;
  }
  __device__ __forceinline__ int run(int lane, volatile int* failed) const {
    int asked = 0;
    bool ok = true;
    for (int n = 0; ok; ++n) {
      ok = __all_sync(kFull, mbar_wait(wanted, n & 1, failed));
      if (ok && n > 0) ok = __all_sync(kFull, mbar_wait(&taken[(n - 1) & 1], ((n - 1) >> 1) & 1, failed));
      if (!ok) break;
      if (lane == 0) tc::request_next_block(&answer[n & 1], &full[n & 1]);
      asked = n + 1;
      ok = __all_sync(kFull, mbar_wait(&full[n & 1], (n >> 1) & 1, failed));
      if (!ok || __shfl_sync(kFull, tc::next_block(&answer[n & 1]), 0) < 0) break;
    }
    if (!ok && lane == 0) *failed = 1;
    return asked;
  }
};

// ------------------------------------------------------------------------------ delta
// A block 64 rows of a head.
template <bool IS_BF16>
__global__ void __launch_bounds__(256)
    window_delta_kernel(const unsigned char* o, const unsigned char* dout, float* delta, int H, int Sq, int blocks, long long o_sb,
                        long long o_sh, long long o_ss, long long d_sb, long long d_sh, long long d_ss) {
  // half a warp per row: 16 lanes x 16 bytes = the 128 16-bit values of a row; kRows rows of a half in flight
  constexpr int kRows = 4;
  const int lane = threadIdx.x & 31, sub = lane & 15;
  // (heads next to each other: in a projection's gradient so are their rows, 256 bytes of a row of all heads)
  const int bt = blockIdx.x / H, h = blockIdx.x - bt * H, b = bt / blocks, bh = b * H + h;
  const int row0 = (bt - b * blocks) * 64 + (threadIdx.x >> 5) * 2 * kRows + (lane >> 4);
  o += 2 * (b * o_sb + h * o_sh) + sub * 16;
  dout += 2 * (b * d_sb + h * d_sh) + sub * 16;
  uint4 a[kRows], g[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int i = row0 + 2 * k;
    a[k] = g[k] = make_uint4(0, 0, 0, 0);
    if (i >= Sq) continue;
    a[k] = ldg_stream(reinterpret_cast<const uint4*>(o + 2 * (i * o_ss)));
    g[k] = ldg_stream(reinterpret_cast<const uint4*>(dout + 2 * (i * d_ss)));
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const uint32_t aw[4] = {a[k].x, a[k].y, a[k].z, a[k].w}, gw[4] = {g[k].x, g[k].y, g[k].z, g[k].w};
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = unpack_pair(aw[e], IS_BF16), y = unpack_pair(gw[e], IS_BF16);
      s = fmaf(x.x, y.x, fmaf(x.y, y.y, s));
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) s += __shfl_xor_sync(kFull, s, off);
    if (sub == 0 && row0 + 2 * k < Sq) delta[(long long)bh * Sq + row0 + 2 * k] = s;
  }
}

// ------------------------------------------------------------------------------ dK, dV
// TMEM columns: [0,128) S^T then P^T, [128,256) dP^T then dS^T, [256,384) dV, [384,512) dK.
template <bool IS_BF16>
__global__ void __launch_bounds__(kThreads, 1)
    window_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const BwdParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* k_smem = smem;
  unsigned char* v_smem = smem + kTileBytes;
  unsigned char* q_smem = smem + 2 * kTileBytes;   // kStages tiles
  unsigned char* do_smem = smem + 4 * kTileBytes;  // kStages tiles

  __shared__ __align__(16) uint4 next_answer[2];
  __shared__ __align__(8) uint64_t next_wanted, next_full[2], next_taken[2], kv_full, kv_empty, q_full[kStages], q_empty[kStages],
      do_full[kStages], do_empty[kStages], raw_full, s_full, dp_full, p_full[NG], ds_full, acc_done, acc_empty, drained;
  // of a query tile: -lse in log2 units (-inf where nothing is seen: P = 0) and -delta
  __shared__ __align__(16) float nlse_s[kStages][BM], ndelta_s[kStages][BM];
  __shared__ uint32_t tmem_base_slot;
  __shared__ volatile int failed;

  const int warp = __shfl_sync(kFull, (int)threadIdx.x >> 5, 0);  // known uniform to the compiler
  const int lane = threadIdx.x & 31;

  const int n_kv_tiles = (p.Sk + BN - 1) / BN;
  // A work item: a key tile of a key head, and steps [from, from + n_it) of the walk over `tiles` query tiles from tile i0
  // on, head after head.
  struct Item {
    int kt0, i0, tiles, from, n_it, bh, b, hk, chunk;  // chunk: 0, or which of the first key tile's further ones
    Lengths n;
  };
  auto item_of = [&](int index) {
    Item w;
    int slot;
    cta_order(index, n_kv_tiles + p.chunks, p.B * p.HK, 8, &slot, &w.bh);
    w.b = w.bh / p.HK;
    w.hk = w.bh - w.b * p.HK;
    w.n = lengths_of(p, w.b);
    w.chunk = slot < p.chunks ? slot + 1 : 0;
    w.kt0 = w.chunk ? 0 : (slot - p.chunks) * BN;
    // queries in whose window a key of the tile is
    const int lo = max(w.kt0 - w.n.off, 0);
    const long long hi = min((long long)w.n.q - 1, (long long)min(w.kt0 + BN, w.n.kv) - 1 + p.window - 1 - w.n.off);
    w.i0 = lo / BM;
    const int end = w.kt0 < w.n.kv && hi >= lo ? (int)(hi / BM) + 1 : w.i0;  // the tile behind the last one
    w.tiles = end - w.i0;
    w.from = 0;
    w.n_it = w.tiles * p.share;
    if (w.chunk) {  // what comes behind them, cut into equal parts
      w.i0 = end;
      w.tiles = w.n.kv > 0 && w.n.q > 0 ? max((w.n.q - 1) / BM + 1 - end, 0) : 0;
      const long long all = (long long)w.tiles * p.share;
      w.from = (int)(all * (w.chunk - 1) / p.chunks);
      w.n_it = (int)(all * w.chunk / p.chunks) - w.from;
    }
    return w;
  };

  if (threadIdx.x == 0) {
    mbar_init(&next_wanted, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&next_full[s], 1);
      mbar_init(&next_taken[s], 2 + kWorkers / 32);  // producer, issuer and element-wise warps
    }
    mbar_init(&kv_full, 1);
    mbar_init(&kv_empty, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&q_full[s], 2);  // the copy and the statistics
      mbar_init(&q_empty[s], 1);
      mbar_init(&do_full[s], 1);
      mbar_init(&do_empty[s], 1);
    }
    mbar_init(&raw_full, 1);
    mbar_init(&s_full, 1);
    mbar_init(&dp_full, 1);
    for (int g = 0; g < NG; ++g) mbar_init(&p_full[g], 4);
    mbar_init(&ds_full, kWorkers / 32);
    mbar_init(&acc_done, 1);
    mbar_init(&acc_empty, kWorkers / 32);
    mbar_init(&drained, 1);
    failed = 0;
    mbar_init_fence();
  }
  if (warp == 1) tc::tmem_alloc(&tmem_base_slot, kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = tmem_base_slot;
  const Scheduler pending{next_answer, &next_wanted, next_full, next_taken};

  int kv_loads = 0, q_loads = 0, do_loads = 0, raw_loads = 0;  // producer: what it has asked for
  bool raw_pending = false;
  int asked = 0;                                               // scheduler: the same
  if (warp < 4) tc::regs_dec<kRegsIssue>();
  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    bool ok = true;
    int step = 0;  // query tiles asked for, over all items
    for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
      const Item w = item_of(index);
      if (w.n_it > 0) {
        if (kv_loads > 0) ok = __all_sync(kFull, mbar_wait(&kv_empty, (kv_loads - 1) & 1, &failed));
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&kv_full, 2 * kTileBytes);
          load_tile(k_smem, &map_k, &kv_full, w.kt0, w.hk, w.b);
          load_tile(v_smem, &map_v, &kv_full, w.kt0, w.hk, w.b);
        }
        ++kv_loads;
      }
      int head = w.tiles > 0 ? w.from / w.tiles : 0, tile = w.from - head * w.tiles;
      // the statistics of a tile are read a tile ahead, so that nothing waits for that read
      float lse_r[4], delta_r[4];
      auto read_stats = [&](int head, int tile) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int qi = (w.i0 + tile) * BM + e * 32 + lane;
          const long long at = ((long long)w.b * p.H + w.hk * p.share + head) * p.Sq + qi;
          const bool live = qi < w.n.q && w.n.off + qi >= 0;  // (any other sees nothing, and may hold anything)
          lse_r[e] = live ? p.lse[at] * -kLog2e : -INFINITY;
          delta_r[e] = live ? -p.delta[at] : 0.f;
          if (lse_r[e] == INFINITY) lse_r[e] = -INFINITY;     // (and so does a row whose log-sum-exp is -inf)
        }
      };
      if (w.n_it > 0) read_stats(head, tile);
      for (int it = 0; it < w.n_it && ok; ++it, ++step) {
        const int s = step % kStages, u = step / kStages;
        const int qt0 = (w.i0 + tile) * BM, h = w.hk * p.share + head;
        const int live = w.n.q - qt0;
        const bool clear = live < BM && w.n.q < p.Sq;  // the tile reaches behind the sequence, and not behind the tensor
        if (u > 0) ok = __all_sync(kFull, mbar_wait(&q_empty[s], (u - 1) & 1, &failed));
        if (!ok) break;
        if (!clear && lane == 0) {
          mbar_arrive_expect_tx(&q_full[s], kTileBytes);
          load_tile(q_smem + (size_t)s * kTileBytes, &map_q, &q_full[s], qt0, h, w.b);
        }
        if (clear) {
          ok = load_cleared(q_smem + (size_t)s * kTileBytes, &map_q, &raw_full, raw_loads & 1, &q_full[s], qt0, h, w.b, live, lane, &failed,
                            raw_pending);
          ++raw_loads;
          if (!ok) break;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          nlse_s[s][e * 32 + lane] = lse_r[e];
          ndelta_s[s][e * 32 + lane] = delta_r[e];
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&q_full[s]);
        q_loads = step + 1;
        if (++tile == w.tiles) {
          tile = 0;
          ++head;
        }
        if (it + 1 < w.n_it) read_stats(head, tile);
        if (u > 0) ok = __all_sync(kFull, mbar_wait(&do_empty[s], (u - 1) & 1, &failed));
        if (!ok) break;
        if (!clear && lane == 0) {
          mbar_arrive_expect_tx(&do_full[s], kTileBytes);
          load_tile(do_smem + (size_t)s * kTileBytes, &map_do, &do_full[s], qt0, h, w.b);
        }
        if (clear) {
          ok = load_cleared(do_smem + (size_t)s * kTileBytes, &map_do, &raw_full, raw_loads & 1, &do_full[s], qt0, h, w.b, live, lane, &failed,
                            raw_pending);
          ++raw_loads;
          if (!ok) break;
        }
        do_loads = step + 1;
      }
      if (lane == 0) tc::mbar_arrive(&next_wanted);
      index = pending.take_next(n, lane, ok, &failed);
    }
    if (!ok && lane == 0) failed = 1;
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc_kk = tc::instr_desc(128, 128, IS_BF16 ? 1 : 0, 0, 0);
    constexpr uint32_t idesc_mn = tc::instr_desc(128, 128, IS_BF16 ? 1 : 0, 0, 1);
    const uint64_t k_desc = tc::smem_desc(smem_u32(k_smem), 16, 1024);
    const uint64_t v_desc = tc::smem_desc(smem_u32(v_smem), 16, 1024);
    const uint64_t q_desc = tc::smem_desc(smem_u32(q_smem), 16, 1024);
    const uint64_t do_desc = tc::smem_desc(smem_u32(do_smem), 16, 1024);
    const uint64_t q_desc_mn = tc::smem_desc(smem_u32(q_smem), kHalfBytes, 1024);
    const uint64_t do_desc_mn = tc::smem_desc(smem_u32(do_smem), kHalfBytes, 1024);
    constexpr uint32_t kStep = kTileBytes >> 4;  // one stage further, in descriptor units
    const uint32_t tmem = __shfl_sync(kFull, tmem_base, 0);
    const uint32_t t_s = tmem + kCol0, t_dp = tmem + kCol1, t_dv = tmem + kCol2, t_dk = tmem + kCol3;
    auto wait = [&](uint64_t* bar, int parity) {
      const bool up = __all_sync(kFull, mbar_wait(bar, parity, &failed));
      tc::fence_after_sync();
      return up;
    };
    bool ok = true;
    int step = 0, items = 0;  // query tiles and items worked on so far
    for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
      const Item w = item_of(index);
      // S^T = K Q^T and dP^T = V dO^T of query tile `at` (over all items); the last of an item free K and V
      auto scores = [&](int at) {
        const int s = at & 1;
        if (!wait(&q_full[s], (at >> 1) & 1)) return false;
        // (the tensor core runs its MMAs in order: P^T of the tile before has been consumed when this one starts)
        issue_ss(t_s, k_desc, q_desc + s * kStep, idesc_kk);
        tc::commit_elected(&s_full);
        return true;
      };
      auto score_gradients = [&](int at, bool last) {
        const int s = at & 1;
        if (!wait(&do_full[s], (at >> 1) & 1)) return false;
        issue_ss(t_dp, v_desc, do_desc + s * kStep, idesc_kk);
        tc::commit_elected(&dp_full);
        if (last) tc::commit_elected(&kv_empty);
        return true;
      };
      if (w.n_it > 0) {
        ok = wait(&kv_full, items & 1) && scores(step) && score_gradients(step, w.n_it == 1);
        for (int it = 0; it < w.n_it && ok; ++it, ++step) {
          const int s = step & 1;
          const bool next = it + 1 < w.n_it;
          // dV += P^T dO in two parts: of the two groups, which share the ex2 unit, one is ahead; the first product
          // of an item waits until the results of the one before have left the accumulators
          ok = (it > 0 || items == 0 || wait(&acc_empty, (items - 1) & 1)) && wait(&p_full[0], step & 1);
          if (!ok) break;
          issue_ts_group<0>(t_dv, t_s, do_desc_mn + s * kStep, idesc_mn, it > 0);
          ok = wait(&p_full[1], step & 1);
          if (!ok) break;
          issue_ts_group<1>(t_dv, t_s, do_desc_mn + s * kStep, idesc_mn, true);
          tc::commit_elected(&do_empty[s]);
          if (next) ok = scores(step + 1);
          ok = ok && wait(&ds_full, step & 1);
          if (!ok) break;
          issue_ts(t_dk, t_dp, q_desc_mn + s * kStep, idesc_mn, it > 0);  // dK += dS^T Q
          tc::commit_elected(&q_empty[s]);
          if (next) ok = score_gradients(step + 1, it + 2 == w.n_it);
        }
        if (ok) tc::commit_elected(&acc_done);
        ++items;
      }
      index = pending.take_next(n, lane, ok, &failed);
    }
    if (!ok && lane == 0) failed = 1;
    __syncwarp();
  } else if (warp == 2) {
    asked = pending.run(lane, &failed);
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ element-wise work
    tc::regs_inc<kRegsWork>();
    const int g = (warp - 4) >> 2;  // group: query columns [GC g, GC g + GC) of a tile
    const int quad = warp & 3;
    const int row = quad * 32 + lane;  // key inside the tile
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_addr = lane_addr + kCol0 + GC * g;
    const uint32_t dp_addr = lane_addr + kCol1 + GC * g;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    int step = 0, items = 0;  // query tiles and items so far

    for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
      const Item w = item_of(index);
      const int kj = w.kt0 + row;
      int tile = w.tiles > 0 ? w.from % w.tiles : 0;
      for (int it = 0; it < w.n_it; ++it, ++step) {
        const int s = step & 1;
        const int qt0 = (w.i0 + tile) * BM;
        if (++tile == w.tiles) tile = 0;
        // the tile's statistics come into registers ahead of its scores: shared memory is busy with
        // the products' operands, and every read of it is slow
        float4 stat[GC / 4];
        bool up = __all_sync(kFull, mbar_wait(&q_full[s], (step >> 1) & 1, &failed));
        if (up) {
#pragma unroll
          for (int e = 0; e < GC / 4; ++e) stat[e] = *reinterpret_cast<const float4*>(&nlse_s[s][GC * g + 4 * e]);
          up = __all_sync(kFull, mbar_wait(&s_full, step & 1, &failed));
        }
        if (!up) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        // key kj is seen by the queries at positions kj .. kj + window - 1, a first token by all from its own on; a key
        // behind the sequence by none (its row of results is replaced at the end, but must not be NaN before)
        const int at0 = w.n.off + qt0;  // position of the tile's first query
        const bool edge = w.kt0 + BN - 1 > at0 || at0 + BM - 1 >= w.kt0 + p.window || w.kt0 + BN > w.n.kv;
        const int lo = kj >= w.n.kv ? 128 : kj - at0 - GC * g;
        const int hi = kj < p.sinks ? 128 : kj - at0 - GC * g + p.window;
        uint32_t raw[GC];
#pragma unroll
        for (int c = 0; c < GC / 32; ++c) tc::tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[c * 32]));
        tc::tmem_wait_ld();
        float2 pr[GC / 2];
#pragma unroll
        for (int c = 0; c < GC / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 l4 = stat[c * 8 + e / 4];
            const float2 l2[2] = {make_float2(l4.x, l4.y), make_float2(l4.z, l4.w)};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int at = c * 32 + e + 2 * u;
              const float2 a = fma2(make_float2(__uint_as_float(raw[at]), __uint_as_float(raw[at + 1])), sc2, l2[u]);
              pr[at / 2] = make_float2(fast_exp2(a.x), fast_exp2(a.y));
            }
          }
          if (edge) {  // (a branch of its own: inside the loop above it costs every tile its selects)
            const uint32_t seen = first_of(hi - c * 32) & ~first_of(lo - c * 32);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              if (!(seen >> e & 1u)) pr[c * 16 + e / 2].x = 0.f;
              if (!(seen >> (e + 1) & 1u)) pr[c * 16 + e / 2].y = 0.f;
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) pk[e] = pack_pair(pr[c * 16 + e].x, pr[c * 16 + e].y, IS_BF16);
          // all of this group's S columns are in registers: P^T goes over their first half
          tc::tmem_st16(s_addr + c * 16, pk);
        }
        tc::tmem_wait_st();
        tc::fence_before_sync();
        warp_arrive(&p_full[g], lane);
#pragma unroll
        for (int e = 0; e < GC / 4; ++e) stat[e] = *reinterpret_cast<const float4*>(&ndelta_s[s][GC * g + 4 * e]);

        if (!__all_sync(kFull, mbar_wait(&dp_full, step & 1, &failed))) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
#pragma unroll
        for (int c = 0; c < GC / 32; ++c) tc::tmem_ld32(dp_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[c * 32]));
        tc::tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < GC / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 d4 = stat[c * 8 + e / 4];
            const float2 d2[2] = {make_float2(d4.x, d4.y), make_float2(d4.z, d4.w)};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int at = c * 32 + e + 2 * u;
              const float2 x = mul2(pr[at / 2], add2(make_float2(__uint_as_float(raw[at]), __uint_as_float(raw[at + 1])), d2[u]));
              pk[e / 2 + u] = pack_pair(x.x, x.y, IS_BF16);
            }
          }
          tc::tmem_st16(dp_addr + c * 16, pk);
        }
        tc::tmem_wait_st();
        tc::fence_before_sync();
        warp_arrive(&ds_full, lane);
      }

      if (ok && w.n_it > 0) ok = mbar_wait(&acc_done, items & 1, &failed);
      ok = __all_sync(kFull, ok);
      if (ok) {
        tc::fence_after_sync();
        const bool live = kj < w.n.kv && w.n_it > 0;
        // the rows of the first tokens where they are a sum over several items
        const bool shared_sum = p.chunks > 0 && w.kt0 == 0;
        if (shared_sum) {
          float* sums = p.sums + (((long long)w.bh * (1 + p.chunks) + w.chunk) * 2 * p.sinks + row) * HD + GC * g;
          const long long of_dk = (long long)p.sinks * HD;
#pragma unroll
          for (int c = 0; c < 2 * GC / 32; ++c) {
            uint32_t acc[32];
            if (w.n_it > 0) {
              tc::tmem_ld32(lane_addr + (c < GC / 32 ? kCol2 : kCol3) + GC * g + c % (GC / 32) * 32, acc);
              tc::tmem_wait_ld();
            }
            if (row < p.sinks) {
              float* dst = sums + (c < GC / 32 ? 0 : of_dk) + c % (GC / 32) * 32;
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(dst + e) =
                    live ? make_float4(__uint_as_float(acc[e]), __uint_as_float(acc[e + 1]), __uint_as_float(acc[e + 2]), __uint_as_float(acc[e + 3]))
                         : make_float4(0.f, 0.f, 0.f, 0.f);
            }
          }
        }
        const bool mine = kj < p.Sk && w.chunk == 0 && !(shared_sum && row < p.sinks);
        unsigned char* dv_row = reinterpret_cast<unsigned char*>(p.dv.ptr) +
                                2 * ((long long)w.b * p.dv.sb + (long long)w.hk * p.dv.sh + (long long)kj * p.dv.ss) + 2 * GC * g;
        unsigned char* dk_row = reinterpret_cast<unsigned char*>(p.dk.ptr) +
                                2 * ((long long)w.b * p.dk.sb + (long long)w.hk * p.dk.sh + (long long)kj * p.dk.ss) + 2 * GC * g;
        if (w.n_it > 0) {
          store_cols<IS_BF16>(lane_addr + kCol2 + GC * g, dv_row, 1.f, mine && live, p.dv.wide);
          store_cols<IS_BF16>(lane_addr + kCol3 + GC * g, dk_row, p.scale, mine && live, p.dk.wide);
          tc::fence_before_sync();
          warp_arrive(&acc_empty, lane);
          ++items;
        }
        if (mine && !live) {
          // no query sees this key: the gradients are zero
          const uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int e = 0; e < GC / 8; ++e) {
            reinterpret_cast<uint4*>(dv_row)[e] = z;
            reinterpret_cast<uint4*>(dk_row)[e] = z;
          }
        }
      }
      __syncwarp();
      index = pending.take_next(n, lane, ok, &failed);
    }
    if (!ok) failed = 1;
  }

  tc::fence_before_sync();
  __syncthreads();
  if (failed) {  // (uniform: nobody writes it any more)
    // a role gave up: what the others have under way has to end before the block does
    if (threadIdx.x == 0) {
      tc::await_copies<1>(&kv_full, kv_loads);
      if (raw_pending) mbar_wait(&raw_full, (raw_loads - 1) & 1);
      tc::await_copies<kStages>(q_full, q_loads);
      tc::await_copies<kStages>(do_full, do_loads);
    }
    if (warp == 1) tc::await_products(&drained);
    if (warp == 2 && lane == 0) tc::await_copies<2>(next_full, asked);
    __syncthreads();
  }
  if (threadIdx.x == 0 && failed && p.status != nullptr) atomicExch(p.status, 1);
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem_base, kTmemCols);
  }
}

// The rows of the first tokens: the items' sums in order.  A thread four values of a row of dV or dK.
template <bool IS_BF16>
__global__ void __launch_bounds__(256) window_sinks_kernel(const BwdParams p) {
  const long long u = (long long)blockIdx.x * 256 + threadIdx.x;
  const int piece = (int)(u % (HD / 4)), which = (int)(u / (HD / 4) % 2);
  const long long r = u / (HD / 4) / 2;
  const int row = (int)(r % p.sinks);
  const long long bh = r / p.sinks;
  if (bh >= (long long)p.B * p.HK || row >= p.Sk) return;
  const float* at = p.sums + ((bh * (1 + p.chunks) * 2 + which) * p.sinks + row) * HD + piece * 4;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int c = 0; c <= p.chunks; ++c) {
    const float4 x = *reinterpret_cast<const float4*>(at + (long long)c * 2 * p.sinks * HD);
    sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
  }
  const Out& out = which ? p.dk : p.dv;
  const float m = which ? p.scale : 1.f;
  const long long b = bh / p.HK, hk = bh - b * p.HK;
  uint2 v;
  v.x = pack_pair(sum.x * m, sum.y * m, IS_BF16);
  v.y = pack_pair(sum.z * m, sum.w * m, IS_BF16);
  *reinterpret_cast<uint2*>(reinterpret_cast<unsigned char*>(out.ptr) + 2 * (b * out.sb + hk * out.sh + row * out.ss + piece * 4)) = v;
}

// ------------------------------------------------------------------------------ dQ
// TMEM columns: [0,128) S, [128,256) and [256,384) dP then dS of the steps in turn, [384,512) dQ.
// The results leave through four warps of their own, so that the element-wise warps go on to the next item's scores: those and
// the statistics, which the producer reads ahead, took 7100 of the 24700 cycles of an item of nine steps before.
template <bool IS_BF16>
__global__ void __launch_bounds__(kDqThreads, 1)
    window_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const BwdParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* q_smem = smem;
  unsigned char* do_smem = smem + kTileBytes;
  unsigned char* v_smem = smem + 2 * kTileBytes;  // kStages tiles
  unsigned char* k_smem = smem + 4 * kTileBytes;  // kKeyStages tiles

  __shared__ __align__(16) uint4 next_answer[2];
  __shared__ __align__(8) uint64_t next_wanted, next_full[2], next_taken[2], q_full, q_empty, do_full, do_empty, k_full[kKeyStages],
      k_empty[kKeyStages], v_full[kStages], v_empty[kStages], raw_full, s_full, s_read, dp_full[2], ds_full[2], acc_done, acc_empty, drained;
  // of the query tile: -lse in log2 units (-inf where nothing is seen: P = 0) and -delta
  __shared__ float nlse_s[BM], ndelta_s[BM];
  __shared__ uint32_t tmem_base_slot;
  __shared__ volatile int failed;

  const int warp = __shfl_sync(kFull, (int)threadIdx.x >> 5, 0);  // known uniform to the compiler
  const int lane = threadIdx.x & 31;

  const int n_q_tiles = (p.Sq + BM - 1) / BM;
  // A work item: a query tile of a head; key tile of step x: the first one, where it has first tokens and is in no row's
  // window, then those from lo on.
  struct Item {
    int qt0, b, h, hk, lo, first, n_kv;
    Lengths n;
  };
  auto item_of = [&](int index) {
    Item w;
    // the heads that share a key head next to each other: they walk the same keys
    const int group = index / p.share, per = n_q_tiles;
    const int bhk = group / per, tile = per - 1 - (group - bhk * per);
    w.b = bhk / p.HK;
    w.hk = bhk - w.b * p.HK;
    w.h = w.hk * p.share + index - group * p.share;
    w.qt0 = tile * BM;
    w.n = lengths_of(p, w.b);
    const int last = w.n.off + min(w.qt0 + BM, w.n.q) - 1, begin = max(w.n.off + w.qt0, 0);
    const bool any = w.qt0 < w.n.q && last >= 0;
    w.lo = any ? max(begin - p.window + 1, 0) / BN : 0;
    w.first = any && w.lo > 0 && p.sinks > 0 ? 1 : 0;
    w.n_kv = any ? last / BN + 1 - w.lo + w.first : 0;
    return w;
  };
  auto key_tile = [&](const Item& w, int x) { return w.first ? (x == 0 ? 0 : w.lo + x - 1) : w.lo + x; };

  if (threadIdx.x == 0) {
    mbar_init(&next_wanted, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&next_full[s], 1);
      mbar_init(&next_taken[s], 2 + kWorkers / 32 + 4);  // producer, issuer, element-wise and storing warps
      mbar_init(&dp_full[s], 1);
      mbar_init(&ds_full[s], kWorkers / 32);
    }
    mbar_init(&q_full, 2);                   // the copy and the statistics
    mbar_init(&q_empty, 1 + kWorkers / 32);  // the last product, and those who have read the statistics
    mbar_init(&do_full, 1);
    mbar_init(&do_empty, 1);
    for (int s = 0; s < kKeyStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(&raw_full, 1);
    mbar_init(&s_full, 1);
    mbar_init(&s_read, kWorkers / 32);
    mbar_init(&acc_done, 1);
    mbar_init(&acc_empty, 4);
    mbar_init(&drained, 1);
    failed = 0;
    mbar_init_fence();
  }
  if (warp == 1) tc::tmem_alloc(&tmem_base_slot, kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = tmem_base_slot;
  const Scheduler pending{next_answer, &next_wanted, next_full, next_taken};

  int q_loads = 0, do_loads = 0, k_loads = 0, v_loads = 0, raw_loads = 0;  // producer: what it has asked for
  bool raw_pending = false;
  int asked = 0;                                                           // scheduler: the same
  if (warp < 4) tc::regs_dec<kDqRegsIssue>();
  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    bool ok = true;
    for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
      const Item w = item_of(index);
      float lse_r[4], delta_r[4];
      if (w.n_kv > 0) {
        // (read before the wait, so that nothing waits for the reads)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int qi = w.qt0 + e * 32 + lane;
          const long long at = ((long long)w.b * p.H + w.h) * p.Sq + qi;
          const bool live = qi < w.n.q && w.n.off + qi >= 0;  // (any other sees nothing, and may hold anything)
          lse_r[e] = live ? p.lse[at] * -kLog2e : -INFINITY;
          delta_r[e] = live ? -p.delta[at] : 0.f;
          if (lse_r[e] == INFINITY) lse_r[e] = -INFINITY;     // (and so does a row whose log-sum-exp is -inf)
        }
        if (q_loads > 0) ok = __all_sync(kFull, mbar_wait(&q_empty, (q_loads - 1) & 1, &failed));
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full, kTileBytes);
          load_tile(q_smem, &map_q, &q_full, w.qt0, w.h, w.b);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          nlse_s[e * 32 + lane] = lse_r[e];
          ndelta_s[e * 32 + lane] = delta_r[e];
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&q_full);
        ++q_loads;
      }
      for (int x = 0; x < w.n_kv && ok; ++x) {
        const int j = key_tile(w, x), s = k_loads % kKeyStages, u = k_loads / kKeyStages, sv = v_loads & 1, uv = v_loads >> 1;
        const int live = w.n.kv - j * BN;
        const bool clear = live < BN && w.n.kv < p.Sk;  // the tile reaches behind the sequence, and not behind the tensor
        if (u > 0) ok = __all_sync(kFull, mbar_wait(&k_empty[s], (u - 1) & 1, &failed));
        if (!ok) break;
        if (!clear) {
          if (lane == 0) {
            mbar_arrive_expect_tx(&k_full[s], kTileBytes);
            load_tile(k_smem + (size_t)s * kTileBytes, &map_k, &k_full[s], j * BN, w.hk, w.b);
          }
        } else {
          ok = load_cleared(k_smem + (size_t)s * kTileBytes, &map_k, &raw_full, raw_loads & 1, &k_full[s], j * BN, w.hk, w.b, live, lane,
                            &failed, raw_pending);
          ++raw_loads;
          if (!ok) break;
        }
        ++k_loads;
        if (x == 0) {
          if (do_loads > 0) ok = __all_sync(kFull, mbar_wait(&do_empty, (do_loads - 1) & 1, &failed));
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&do_full, kTileBytes);
            load_tile(do_smem, &map_do, &do_full, w.qt0, w.h, w.b);
          }
          ++do_loads;
        }
        if (uv > 0) ok = __all_sync(kFull, mbar_wait(&v_empty[sv], (uv - 1) & 1, &failed));
        if (!ok) break;
        if (!clear) {
          if (lane == 0) {
            mbar_arrive_expect_tx(&v_full[sv], kTileBytes);
            load_tile(v_smem + (size_t)sv * kTileBytes, &map_v, &v_full[sv], j * BN, w.hk, w.b);
          }
        } else {
          ok = load_cleared(v_smem + (size_t)sv * kTileBytes, &map_v, &raw_full, raw_loads & 1, &v_full[sv], j * BN, w.hk, w.b, live, lane,
                            &failed, raw_pending);
          ++raw_loads;
          if (!ok) break;
        }
        ++v_loads;
      }
      if (lane == 0) tc::mbar_arrive(&next_wanted);
      index = pending.take_next(n, lane, ok, &failed);
    }
    if (!ok && lane == 0) failed = 1;
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc_kk = tc::instr_desc(128, 128, IS_BF16 ? 1 : 0, 0, 0);
    constexpr uint32_t idesc_mn = tc::instr_desc(128, 128, IS_BF16 ? 1 : 0, 0, 1);
    const uint64_t q_desc = tc::smem_desc(smem_u32(q_smem), 16, 1024);
    const uint64_t do_desc = tc::smem_desc(smem_u32(do_smem), 16, 1024);
    const uint64_t k_desc = tc::smem_desc(smem_u32(k_smem), 16, 1024);
    const uint64_t v_desc = tc::smem_desc(smem_u32(v_smem), 16, 1024);
    const uint64_t k_desc_mn = tc::smem_desc(smem_u32(k_smem), kHalfBytes, 1024);
    constexpr uint32_t kStep = kTileBytes >> 4;  // one stage further, in descriptor units
    const uint32_t tmem = __shfl_sync(kFull, tmem_base, 0);
    const uint32_t t_s = tmem + kCol0, t_dq = tmem + kCol3;
    auto wait = [&](uint64_t* bar, int parity) {
      const bool up = __all_sync(kFull, mbar_wait(bar, parity, &failed));
      tc::fence_after_sync();
      return up;
    };
    bool ok = true;
    int step = 0, items = 0;  // key tiles and items so far
    int k_next = 0, k_turn = 0, k_used = 0;  // stage and phase of the next K that is awaited, and the stage that is used next
    for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
      const Item w = item_of(index);
      // S = Q K^T and dP = dO V^T of step `at` (over all items); the last of an item free Q and dO
      auto scores = [&](int at, bool last) {
        // the scores of the step before are in registers: their columns can take these
        if ((at > 0 && !wait(&s_read, (at - 1) & 1)) || !wait(&k_full[k_next], k_turn)) return false;
        issue_ss(t_s, q_desc, k_desc + k_next * kStep, idesc_kk);
        tc::commit_elected(&s_full);
        if (last) tc::commit_elected(&q_empty);
        if (++k_next == kKeyStages) {
          k_next = 0;
          k_turn ^= 1;
        }
        return true;
      };
      auto score_gradients = [&](int at, bool last) {
        // (this buffer's dS, two steps ago, has been consumed by a product issued before: they run in order)
        if (!wait(&v_full[at & 1], (at >> 1) & 1)) return false;
        issue_ss(tmem + (at & 1 ? kCol2 : kCol1), do_desc, v_desc + (at & 1) * kStep, idesc_kk);
        tc::commit_elected(&dp_full[at & 1]);
        tc::commit_elected(&v_empty[at & 1]);
        if (last) tc::commit_elected(&do_empty);
        return true;
      };
      if (w.n_kv > 0) {
        ok = wait(&q_full, items & 1) && scores(step, w.n_kv == 1) && wait(&do_full, items & 1) && score_gradients(step, w.n_kv == 1);
        for (int x = 0; x < w.n_kv && ok; ++x, ++step) {
          if (x + 1 < w.n_kv) ok = scores(step + 1, x + 2 == w.n_kv) && score_gradients(step + 1, x + 2 == w.n_kv);
          // the first product of an item waits until the results of the one before have left the accumulators
          ok = ok && wait(&ds_full[step & 1], (step >> 1) & 1) && (x > 0 || items == 0 || wait(&acc_empty, (items - 1) & 1));
          if (!ok) break;
          issue_ts(t_dq, tmem + (step & 1 ? kCol2 : kCol1), k_desc_mn + k_used * kStep, idesc_mn, x > 0);  // dQ += dS K
          tc::commit_elected(&k_empty[k_used]);
          if (++k_used == kKeyStages) k_used = 0;
        }
        if (ok) tc::commit_elected(&acc_done);
        ++items;
      }
      index = pending.take_next(n, lane, ok, &failed);
    }
    if (!ok && lane == 0) failed = 1;
    __syncwarp();
  } else if (warp == 2) {
    asked = pending.run(lane, &failed);
  } else if (warp >= 4 + 4 * NG) {
    // ------------------------------------------------------------------ results
    tc::regs_dec<kDqRegsStore>();
    const int quad = warp & 3, row = quad * 32 + lane;
    const uint32_t acc_addr = tmem_base + ((uint32_t)(quad * 32) << 16) + kCol3;
    bool ok = true;
    int items = 0;
    for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
      const Item w = item_of(index);
      const int qi = w.qt0 + row;
      // a row that sees nothing, whatever its products hold (its log-sum-exp says so where its position does not)
      bool some = qi < w.n.q && w.n.off + qi >= 0;
      if (some) some = p.lse[((long long)w.b * p.H + w.h) * p.Sq + qi] != -INFINITY;
      unsigned char* dq_row = reinterpret_cast<unsigned char*>(p.dq.ptr) +
                              2 * ((long long)w.b * p.dq.sb + (long long)w.h * p.dq.sh + (long long)qi * p.dq.ss);
      if (w.n_kv > 0) {
        ok = __all_sync(kFull, mbar_wait(&acc_done, items & 1, &failed));
        if (!ok) break;
        tc::fence_after_sync();
#pragma unroll
        for (int g = 0; g < NG; ++g) store_cols<IS_BF16>(acc_addr + GC * g, dq_row + 2 * GC * g, p.scale, qi < p.Sq && some, p.dq.wide);
        tc::fence_before_sync();
        warp_arrive(&acc_empty, lane);
        ++items;
      }
      if (qi < p.Sq && !(some && w.n_kv > 0)) {
        const uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int e = 0; e < HD / 8; ++e) reinterpret_cast<uint4*>(dq_row)[e] = z;
      }
      __syncwarp();
      index = pending.take_next(n, lane, ok, &failed);
    }
    if (!ok && lane == 0) failed = 1;
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ element-wise work
    tc::regs_inc<kDqRegsWork>();
    const int g = (warp - 4) >> 2;  // group: key columns [GC g, GC g + GC) of a tile
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_addr = lane_addr + kCol0 + GC * g;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    int step = 0, items = 0;

    for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
      const Item w = item_of(index);
      const int qi = w.qt0 + row;
      const int at = qi < w.n.q ? w.n.off + qi : -1;  // (below 0: sees nothing)
      float2 nl2, ndl2;
      if (w.n_kv > 0) {
        ok = __all_sync(kFull, mbar_wait(&q_full, items & 1, &failed));
        if (!ok) break;
        nl2 = make_float2(nlse_s[row], nlse_s[row]);
        ndl2 = make_float2(ndelta_s[row], ndelta_s[row]);
        warp_arrive(&q_empty, lane);
        ++items;
      }
      const int at_first = w.n.off + w.qt0, at_last = at_first + BM - 1;
      for (int x = 0; x < w.n_kv; ++x, ++step) {
        if (!__all_sync(kFull, mbar_wait(&s_full, step & 1, &failed))) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        uint32_t raw[GC];
#pragma unroll
        for (int c = 0; c < GC / 32; ++c) tc::tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[c * 32]));
        tc::tmem_wait_ld();
        tc::fence_before_sync();
        warp_arrive(&s_read, lane);
        const int j0 = key_tile(w, x) * BN, col0 = j0 + GC * g;
        const bool edge = j0 + BN - 1 > at_first || j0 <= at_last - p.window || w.qt0 + BM > w.n.q;
        const int lim = at - col0, low = at - p.window + 1 - col0, from = (j0 == 0 ? p.sinks : 0) - GC * g;
        float2 pr[GC / 2];
#pragma unroll
        for (int e = 0; e < GC; e += 2) {
          const float2 a = fma2(make_float2(__uint_as_float(raw[e]), __uint_as_float(raw[e + 1])), sc2, nl2);
          pr[e / 2] = make_float2(fast_exp2(a.x), fast_exp2(a.y));
        }
        if (edge) {
#pragma unroll
          for (int c = 0; c < GC / 32; ++c) {
            const uint32_t seen = first_of(lim + 1 - c * 32) & ~(first_of(low - c * 32) & ~first_of(from - c * 32));
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              if (!(seen >> e & 1u)) pr[c * 16 + e / 2].x = 0.f;
              if (!(seen >> (e + 1) & 1u)) pr[c * 16 + e / 2].y = 0.f;
            }
          }
        }
        if (!__all_sync(kFull, mbar_wait(&dp_full[step & 1], (step >> 1) & 1, &failed))) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        const uint32_t dp_addr = lane_addr + (step & 1 ? kCol2 : kCol1) + GC * g;
#pragma unroll
        for (int c = 0; c < GC / 32; ++c) {
          uint32_t d[32];
          tc::tmem_ld32(dp_addr + c * 32, d);
          tc::tmem_wait_ld();
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = mul2(pr[c * 16 + e / 2], add2(make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])), ndl2));
            pk[e / 2] = pack_pair(x.x, x.y, IS_BF16);
          }
          tc::tmem_st16(dp_addr + c * 16, pk);
        }
        tc::tmem_wait_st();
        tc::fence_before_sync();
        warp_arrive(&ds_full[step & 1], lane);
      }

      __syncwarp();
      index = pending.take_next(n, lane, ok, &failed);
    }
    if (!ok && lane == 0) failed = 1;
  }

  tc::fence_before_sync();
  __syncthreads();
  if (failed) {  // (as above)
    if (threadIdx.x == 0) {
      tc::await_copies<1>(&q_full, q_loads);
      tc::await_copies<1>(&do_full, do_loads);
      if (raw_pending) mbar_wait(&raw_full, (raw_loads - 1) & 1);
      tc::await_copies<kKeyStages>(k_full, k_loads);
      tc::await_copies<kStages>(v_full, v_loads);
    }
    if (warp == 1) tc::await_products(&drained);
    if (warp == 2 && lane == 0) tc::await_copies<2>(next_full, asked);
    __syncthreads();
  }
  if (threadIdx.x == 0 && failed && p.status != nullptr) atomicExch(p.status, 1);
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem_base, kTmemCols);
  }
}

// The opt-ins of a kernel on the current device, asked for once: a property of (kernel, device).
template <class K>
int opt_in(K kern, std::atomic<bool>& done, size_t smem, int regs) {
  if (!done.load(std::memory_order_acquire)) {
    cudaFuncAttributes at;  // (as in fa_fwd.cu: setmaxnreg waits for registers the block has to own)
    cudaError_t e = cudaFuncGetAttributes(&at, kern);
    if (e != cudaSuccess) return ixb_host::cuda_status(e);
    if (at.numRegs != regs) return IXB_ERR_UNSUPPORTED;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return ixb_host::cuda_status(e);
    done.store(true, std::memory_order_release);
  }
  return IXB_OK;
}

// Items that the queries behind the first key tile's window are cut into, of as many steps as another item has, or as
// make 128 of them (each leaves sinks x 1 KB of sums); none where there are no such queries or no first tokens.
int sink_chunks(int H, int HK, int Sq, int Sk, int window, int sinks) {
  if (sinks == 0 || window >= Sk) return 0;
  const long long share = H / HK, q_tiles = ((long long)Sq + BM - 1) / BM;
  const long long behind = ((long long)Sk - window + BM - 1) / BM + 1;
  const long long all = share * (behind < q_tiles ? behind : q_tiles);
  const long long each = share * (((long long)window + 2 * BM - 2) / BM + 1);
  const long long items = (all + each - 1) / each;
  return (int)(items < 128 ? items : 128);
}
size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }
size_t delta_bytes(int B, int H, int Sq) { return round16((size_t)B * H * Sq * sizeof(float)); }

}  // namespace

extern "C" size_t ixb_window_attention_bwd_scratch_bytes(int32_t B, int32_t H, int32_t HK, int32_t Sq, int32_t Sk,
                                                         int32_t window, int32_t sinks) {
  if (B <= 0 || H <= 0 || HK <= 0 || Sq <= 0 || Sk <= 0 || window <= 0 || sinks < 0 || H % HK != 0) return 0;
  const size_t chunks = sink_chunks(H, HK, Sq, Sk, window, sinks);
  return delta_bytes(B, H, Sq) + (chunks ? (size_t)B * HK * (1 + chunks) * 2 * sinks * HD * sizeof(float) : 0);
}

extern "C" int ixb_window_attention_bwd(int dtype, const void* q, const void* k, const void* v, const void* o,
                                        const void* dout, const float* lse, void* dq, void* dk, void* dv, void* scratch,
                                        size_t scratch_bytes, int32_t B, int32_t H, int32_t HK, int32_t Sq, int32_t Sk,
                                        int32_t D, const int64_t* q_strides, const int64_t* k_strides,
                                        const int64_t* v_strides, const int64_t* o_strides, const int64_t* do_strides,
                                        const int64_t* dq_strides, const int64_t* dk_strides, const int64_t* dv_strides,
                                        const int32_t* q_lengths, const int32_t* kv_lengths, float scale, int32_t window,
                                        int32_t sinks, int32_t* status, ixb_stream stream) {
  if (int st = ixb_host::check_window_sizes(dtype, B, H, HK, Sq, Sk, D, scale, window, sinks)) return st;
  if (B == 0 || H == 0) return IXB_OK;
  if (Sq == 0 || Sk == 0) return IXB_ERR_SHAPE;
  const ixb_host::WindowView views[] = {{q, q_strides},   {k, k_strides},   {v, v_strides},   {o, o_strides}, {dout, do_strides},
                                        {dq, dq_strides}, {dk, dk_strides}, {dv, dv_strides}};
  if (int st = ixb_host::check_window_views(views, 8)) return st;
  if (lse == nullptr) return IXB_ERR_ARG;
  if (scratch == nullptr || scratch_bytes < ixb_window_attention_bwd_scratch_bytes(B, H, HK, Sq, Sk, window, sinks)) return IXB_ERR_SCRATCH;
  if (!ixb_host::aligned16(scratch)) return IXB_ERR_ALIGN;
  BwdParams p;
  p.window = window < Sk ? window : Sk;  // (a longer one is this one)
  p.sinks = sinks;
  p.chunks = sink_chunks(H, HK, Sq, Sk, window, sinks);
  const long long q_tiles = ((long long)Sq + BM - 1) / BM, kv_tiles = ((long long)Sk + BN - 1) / BN;
  const long long delta_blocks = ((long long)Sq + 63) / 64 * B * H, dkv_items = (kv_tiles + p.chunks) * B * HK, dq_items = q_tiles * B * H;
  if (delta_blocks > 0x7fffffffLL || dkv_items > 0x7fffffffLL || dq_items > 0x7fffffffLL) return IXB_ERR_SHAPE;
  const int is_bf16 = dtype == IXB_BF16;
  CUtensorMap mq, mk, mv, mdo;
  if (int st = ixb_host::make_fa_map(&mq, q, is_bf16, B, H, Sq, q_strides[0], q_strides[1], q_strides[2])) return st;
  if (int st = ixb_host::make_fa_map(&mk, k, is_bf16, B, HK, Sk, k_strides[0], k_strides[1], k_strides[2])) return st;
  if (int st = ixb_host::make_fa_map(&mv, v, is_bf16, B, HK, Sk, v_strides[0], v_strides[1], v_strides[2])) return st;
  if (int st = ixb_host::make_fa_map(&mdo, dout, is_bf16, B, H, Sq, do_strides[0], do_strides[1], do_strides[2])) return st;
  float* delta = static_cast<float*>(scratch);
  p.lse = lse;
  p.delta = delta;
  p.sums = p.chunks ? reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + delta_bytes(B, H, Sq)) : nullptr;
  p.dq = Out{dq, dq_strides[0], dq_strides[1], dq_strides[2], ixb_host::rows_aligned32(dq, dq_strides)};
  p.dk = Out{dk, dk_strides[0], dk_strides[1], dk_strides[2], ixb_host::rows_aligned32(dk, dk_strides)};
  p.dv = Out{dv, dv_strides[0], dv_strides[1], dv_strides[2], ixb_host::rows_aligned32(dv, dv_strides)};
  p.status = status;
  p.q_lengths = q_lengths;
  p.kv_lengths = kv_lengths;
  p.B = B, p.H = H, p.HK = HK, p.share = H / HK, p.Sq = Sq, p.Sk = Sk;
  p.scale = scale;
  p.scale_log2 = scale * kLog2e;

  auto kern_delta = is_bf16 ? window_delta_kernel<true> : window_delta_kernel<false>;
  auto kern_dkv = is_bf16 ? window_dkv_kernel<true> : window_dkv_kernel<false>;
  auto kern_sinks = is_bf16 ? window_sinks_kernel<true> : window_sinks_kernel<false>;
  auto kern_dq = is_bf16 ? window_dq_kernel<true> : window_dq_kernel<false>;
  static std::atomic<bool> configured[2][2][64];
  int devid = 0;
  cudaGetDevice(&devid);
  if (int st = opt_in(kern_dkv, configured[0][is_bf16][devid & 63], kDkvSmem, kRegsLaunch)) return st;
  if (int st = opt_in(kern_dq, configured[1][is_bf16][devid & 63], kDqSmem, kDqRegsLaunch)) return st;
  const cudaStream_t cs = (cudaStream_t)stream;
  kern_delta<<<(unsigned)delta_blocks, 256, 0, cs>>>(
      static_cast<const unsigned char*>(o), static_cast<const unsigned char*>(dout), delta, H, Sq, (Sq + 63) / 64,
      o_strides[0], o_strides[1], o_strides[2], do_strides[0], do_strides[1], do_strides[2]);
  kern_dkv<<<(unsigned)dkv_items, kThreads, kDkvSmem, cs>>>(mq, mk, mv, mdo, p);
  if (p.chunks) {
    const long long pieces = (long long)B * HK * sinks * 2 * (HD / 4);
    kern_sinks<<<(unsigned)((pieces + 255) / 256), 256, 0, cs>>>(p);
  }
  kern_dq<<<(unsigned)dq_items, kDqThreads, kDqSmem, cs>>>(mq, mk, mv, mdo, p);
  return ixb_host::cuda_status(cudaGetLastError());
}
