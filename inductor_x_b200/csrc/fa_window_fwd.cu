// Attention with a sliding window and first tokens that stay visible, forward, on tcgen05 tensor cores (the meaning of
// the arguments: fa_window.h).  The pipeline is that of fa_fwd.cu - TMA producer, MMA issuer, scheduler, two warpgroups
// of softmax, running blocks that take over pending items - on other work items:
//
// A tile of 128 rows is R rows of each of 128 / R neighbouring query heads that share a key head: R is 128, or the
// power of two that holds all of the call's queries where they are fewer (8 at least).  The tiles of a key
// head, those of the same rows one after the other, go two to an item, so that with an even number of
// sharing heads both tiles of an item see the very same keys and every tile of K and V serves both.
// An item walks the key tiles back from the one its last row stands in to the one its window begins in: every row sees its
// own position, so that the running maximum is near its end from the first step on and accumulators are hardly ever
// rescaled.  The first key tile, where that is not in the window but has first tokens, is the second step; up to kFront
// first tokens take copies, products and exponentials of kFront keys only.  A tile of rows leaves out steps that only the other one sees.
//
// What lies behind a sequence's length in K and V may be anything: scores of hidden keys are replaced before they are
// looked at, but a probability of 0 times a NaN is one, so the producer clears the rows of V behind the length in the
// tile that holds it.
//
// Probabilities are rounded to the operands' 16 bits, since P V is a product of 16-bit operands (32-bit ones take twice
// the time and the memory); they are at most 2^8, relative to a maximum that may be stale by so much, and the sum that divides them is
// of 32-bit values before that rounding.  The result is 1.3 to 1.4 times as far off as the same formula in 32 bits, rounded once.
//
// Bound: as fa_fwd.cu, the chain scores -> softmax -> P -> product of a step and the drain between items.  8192 tokens of 32/8
// heads, bf16, on one B200 at full clock: window 1024 132 - 137 us (fused_attention on nine unmasked steps 130 - 139), with 4 first
// tokens 140 - 147, or 138 where K and V lie as in a cache (where they took 144 as the second step of an item, they took 150 as the
// last one and 169 with all 128 keys of it), window 256 75 - 81, 2048 210 - 218; masks are 5 of it, stores 2.  Steps
// from the window's beginning on 6 % more (rows that see nothing of the first tile rescale their accumulators);
// the heads of one key head after the other instead of eight of them together 3 % more.
#include <atomic>
#include "fa_window.h"
#include "ixb/fa_softmax.cuh"

namespace {

using namespace ixb;
using namespace ixb::fa;

constexpr int kFront = 32;  // keys of a short step
constexpr int kFrontBytes = kFront * HD * 2;
constexpr int kStages = 2;  // (the issuer picks stage descriptors with two-way selects)
// Registers: as in fa_fwd.cu
constexpr int kRegsLaunch = 168, kRegsIssue = 88, kRegsSoftmax = 208;
static_assert(kRegsIssue + NQ * kRegsSoftmax <= (1 + NQ) * kRegsLaunch, "setmaxnreg draws on the block's own registers");
constexpr size_t kSmemBytes = (size_t)kTileBytes * (NQ + 2 * kStages) + 1024;

struct WinParams {
  void* o;
  float* lse;            // [B, H, Sq], may be null
  int* status;           // may be null
  const int *q_lengths, *kv_lengths;
  long long o_stride_b, o_stride_h, o_stride_s;  // elements
  int B, H, HK, share, Sq, Sk;
  float scale_log2;
  int window, sinks;
  int rows_log2;         // R = 1 << rows_log2 rows of a head in a tile
  int tiles;             // tiles of rows a key head has
  int per_item;          // of which an item takes two, or one
  int wide;
  int head_group;        // key heads whose items are dispatched together
};

template <bool IS_BF16>
__global__ void __launch_bounds__(kThreads, 1)
    fa_window_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_kf,
                         const __grid_constant__ CUtensorMap map_vf, const WinParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* q_smem = smem;
  unsigned char* k_smem = smem + kTileBytes * NQ;
  unsigned char* v_smem = smem + kTileBytes * (NQ + kStages);

  __shared__ __align__(16) uint4 next_answer[2];
  __shared__ __align__(8) uint64_t q_full, q_empty, next_wanted, next_full[2], next_taken[2], k_full[kStages],
      k_empty[kStages], v_full[kStages], v_empty[kStages], v_raw, s_full[NQ], p_full[NQ], p_rest[NQ], pv_done[NQ], drained;
  __shared__ uint32_t tmem_base_slot;
  __shared__ volatile int failed;

  const int warp = __shfl_sync(kFull, (int)threadIdx.x >> 5, 0);  // known uniform to the compiler
  const int lane = threadIdx.x & 31;

  const int R = 1 << p.rows_log2, blocks_of_heads = (p.share + (BM >> p.rows_log2) - 1) >> (7 - p.rows_log2);
  struct Item {
    int b, hk, off, q_len, kv_len;   // query i stands at position off + i
    int i0[NQ], h0[NQ];              // first row and first head of each tile (h0 < 0: no such tile)
    int lo[NQ], hi[NQ];              // key tiles of each tile's window (none: hi = 0)
    int lo_all, end, n_kv, front;    // key tiles [lo_all, end), and with `front` tile 0, which is in no window
  };
  auto item_of = [&](int index) {
    Item w;
    const int per_head = (p.tiles + p.per_item - 1) / p.per_item;
    const int group = index / (per_head * p.head_group), in_group = index - group * per_head * p.head_group;
    const int g_heads = min(p.head_group, p.B * p.HK - group * p.head_group);
    const int bh = group * p.head_group + in_group % g_heads, n = per_head - 1 - in_group / g_heads;
    w.b = bh / p.HK;
    w.hk = bh - w.b * p.HK;
    w.q_len = p.q_lengths != nullptr ? min(max(__ldg(p.q_lengths + w.b), 0), p.Sq) : p.Sq;
    w.kv_len = p.kv_lengths != nullptr ? min(max(__ldg(p.kv_lengths + w.b), 0), p.Sk) : p.Sk;
    w.off = w.kv_len - w.q_len;
    w.lo_all = 1 << 30;
    w.end = 0;
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      const int u = t < p.per_item ? p.per_item * n + t : p.tiles, i = u / blocks_of_heads;
      w.i0[t] = i * BM;  // (fewer rows a head than a tile has: all of them are in tile 0)
      w.h0[t] = u < p.tiles ? w.hk * p.share + ((u - i * blocks_of_heads) << (7 - p.rows_log2)) : -1;
      const int last = w.off + min(w.i0[t] + R, w.q_len) - 1;  // position of the tile's last row, and of its first
      const int begin = max(w.off + w.i0[t], 0);
      const bool any = u < p.tiles && w.i0[t] < w.q_len && last >= 0;
      w.lo[t] = any ? max(begin - p.window + 1, 0) / BN : 0;
      w.hi[t] = any ? last / BN + 1 : 0;
      if (any) {
        w.lo_all = min(w.lo_all, w.lo[t]);
        w.end = max(w.end, w.hi[t]);
      }
    }
    w.front = w.end > 0 && w.lo_all > 0 && p.sinks > 0 ? 1 : 0;
    w.n_kv = w.end > 0 ? w.end - w.lo_all + w.front : 0;
    return w;
  };
  // key tile of step x of an item: the first tokens' is the second
  auto key_tile = [&](const Item& w, int x) { return !w.front ? w.end - 1 - x : x == 0 ? w.end - 1 : x == 1 ? 0 : w.end - x; };

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    mbar_init(&next_wanted, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&next_full[s], 1);
      mbar_init(&next_taken[s], 2 + NQ * 4);  // producer, issuer and the softmax warps
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(&v_raw, 1);
    for (int t = 0; t < NQ; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 128);
      mbar_init(&p_rest[t], 128);
      mbar_init(&pv_done[t], 1);
    }
    mbar_init(&drained, 1);
    failed = 0;
    mbar_init_fence();
  }
  if (warp == 1) tc::tmem_alloc(&tmem_base_slot, kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = tmem_base_slot;

  // The item after item n of this block: answer n of the scheduler warp.  Taken by a whole warp.
  auto take_next = [&](int n, bool& ok) {
    ok = ok && __all_sync(kFull, mbar_wait(&next_full[n & 1], (n >> 1) & 1, &failed));
    if (!ok) return -1;
    const int index = __shfl_sync(kFull, tc::next_block(&next_answer[n & 1]), 0);
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&next_taken[n & 1]);
    return index;
  };

  int q_loads = 0, k_loads = 0, v_loads = 0, raw_loads = 0;  // producer: what it has asked for
  bool raw_pending = false;                                  // the last copy of V completes v_raw, not v_full
  int asked = 0;                                             // scheduler: the same
  if (warp < 4) {
    tc::regs_dec<kRegsIssue>();
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer
      bool ok = true;
      int step = 0;  // key tiles loaded so far, over all items
      for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
        const Item w = item_of(index);
        if (w.n_kv > 0) {
          ok = q_loads == 0 || __all_sync(kFull, mbar_wait(&q_empty, (q_loads - 1) & 1, &failed));
          if (!ok) break;
          if (lane == 0) {
            // rows and heads past the end of the tensor are zero-filled by the copy engine (a head behind the key head's own
            // is another one's: its rows are not stored)
            mbar_arrive_expect_tx(&q_full, kTileBytes * NQ);
#pragma unroll
            for (int t = 0; t < NQ; ++t) {
              unsigned char* qd = q_smem + t * kTileBytes;
              const int h0 = max(w.h0[t], 0);
              for (int g = 0; g < BM >> p.rows_log2; ++g, qd += R * 128) {
                tc::tma_load_4d(qd, &map_q, &q_full, 0, w.i0[t], h0 + g, w.b);
                tc::tma_load_4d(qd + kHalfBytes, &map_q, &q_full, 64, w.i0[t], h0 + g, w.b);
              }
            }
          }
          ++q_loads;
        }
        for (int x = 0; x < w.n_kv; ++x, ++step) {
          const int s = step & 1, u = step >> 1, j = key_tile(w, x);
          const bool brief = w.front && p.sinks <= kFront && x == 1;
          ok = u == 0 || __all_sync(kFull, mbar_wait(&k_empty[s], (u - 1) & 1, &failed));
          if (!ok) break;
          if (lane == 0) {
            // (a short step's keys are the first kFront rows of each box)
            unsigned char* kd = k_smem + (size_t)s * kTileBytes;
            const CUtensorMap* map = brief ? &map_kf : &map_k;
            mbar_arrive_expect_tx(&k_full[s], brief ? kFrontBytes : kTileBytes);
            tc::tma_load_4d(kd, map, &k_full[s], 0, j * BN, w.hk, w.b);
            tc::tma_load_4d(kd + kHalfBytes, map, &k_full[s], 64, j * BN, w.hk, w.b);
            if (x + 1 == w.n_kv) tc::mbar_arrive(&next_wanted);
          }
          k_loads = step + 1;
          ok = u == 0 || __all_sync(kFull, mbar_wait(&v_empty[s], (u - 1) & 1, &failed));
          if (!ok) break;
          unsigned char* vd = v_smem + (size_t)s * kTileBytes;
          const int live = w.kv_len - j * BN;
          // the tile reaches behind the sequence, and not behind the tensor (the first one does not, where it is in no window)
          const bool clear = live < BN && w.kv_len < p.Sk;
          uint64_t* bar = clear ? &v_raw : &v_full[s];
          if (lane == 0) {
            const CUtensorMap* map = brief ? &map_vf : &map_v;
            mbar_arrive_expect_tx(bar, brief ? kFrontBytes : kTileBytes);
            tc::tma_load_4d(vd, map, bar, 0, j * BN, w.hk, w.b);
            tc::tma_load_4d(vd + kHalfBytes, map, bar, 64, j * BN, w.hk, w.b);
          }
          if (clear) {
            raw_pending = true;
            ok = __all_sync(kFull, mbar_wait(&v_raw, raw_loads & 1, &failed));
            ++raw_loads;
            if (!ok) break;
            raw_pending = false;
            // a row is 128 bytes in each of the two boxes, whichever way its pieces are swizzled
            for (int at = live * 8 + lane; at < BN * 8; at += 32) {
              *reinterpret_cast<uint4*>(vd + at * 16) = make_uint4(0, 0, 0, 0);
              *reinterpret_cast<uint4*>(vd + kHalfBytes + at * 16) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&v_full[s]);
          }
          v_loads = step + 1;
        }
        if (ok && w.n_kv == 0 && lane == 0) tc::mbar_arrive(&next_wanted);
        __syncwarp();
        index = take_next(n, ok);
      }
      if (!ok && lane == 0) failed = 1;
    } else if (warp == 1) {
      // -------------------------------------------------------------------- MMA issuer
      // The whole warp runs this role and an elected lane issues (see tc::product_ss).
      constexpr uint32_t idesc_qk = tc::instr_desc(BM, BN, IS_BF16 ? 1 : 0, 0, 0);
      constexpr uint32_t idesc_front = tc::instr_desc(BM, kFront, IS_BF16 ? 1 : 0, 0, 0);
      constexpr uint32_t idesc_pv = tc::instr_desc(BM, HD, IS_BF16 ? 1 : 0, 0, 1);
      const uint32_t tmem = __shfl_sync(kFull, tmem_base, 0);
      const uint64_t q_desc = tc::smem_desc(smem_u32(q_smem), 16, 1024);
      const uint64_t k_desc = tc::smem_desc(smem_u32(k_smem), 16, 1024);
      const uint64_t v_desc = tc::smem_desc(smem_u32(v_smem), kHalfBytes, 1024);
      // tile t, stage s: the address field moves by whole tiles and cannot carry out of it
      auto issue_qk = [&](int t, int stage, bool brief) {
        tc::product_ss<kHalfBytes>(tmem + kColS + t * 128, q_desc + (uint32_t)(t * (kTileBytes >> 4)),
                                   k_desc + (uint32_t)(stage * (kTileBytes >> 4)), brief ? idesc_front : idesc_qk);
        tc::commit_elected(&s_full[t]);
      };
      bool ok = true;
      int step = 0;               // key tiles consumed so far, over all items
      int items = 0;              // items with keys so far
      int products[NQ] = {0, 0};  // P tiles consumed so far
      for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
        int n_kv, first[NQ], behind[NQ], last[NQ];  // window steps [first, behind) of a tile of rows, and its last one
        bool front, brief;                          // step 1 is the first tokens', and short
        {
          const Item w = item_of(index);
          n_kv = w.n_kv;
          front = w.front != 0;
          brief = front && p.sinks <= kFront;
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            auto step_of = [&](int j) { return front && j < w.end - 1 ? w.end - j : w.end - 1 - j; };
            const bool any = w.hi[t] > 0;
            first[t] = any ? step_of(w.hi[t] - 1) : n_kv;
            behind[t] = any ? step_of(w.lo[t]) + 1 : n_kv;
            last[t] = !any ? -1 : front ? max(1, behind[t] - 1) : w.lo[t] > 0 && p.sinks > 0 ? n_kv - 1 : behind[t] - 1;
          }
        }
        auto looks = [&](int t, int x) { return (x >= first[t] && x < behind[t]) || x == last[t] || (front && x == 1 && last[t] > 0); };
        bool begun[NQ] = {false, false};
        if (n_kv > 0) {
          ok = __all_sync(kFull, mbar_wait(&q_full, items & 1, &failed)) &&
               __all_sync(kFull, mbar_wait(&k_full[step & 1], (step >> 1) & 1, &failed));
          if (!ok) break;
          ++items;
          tc::fence_after_sync();
#pragma unroll
          for (int t = 0; t < NQ; ++t)
            if (looks(t, 0)) issue_qk(t, step & 1, false);  // (the last row's own tile: never the short step)
          tc::commit_elected(&k_empty[step & 1]);
          if (n_kv == 1) tc::commit_elected(&q_empty);
        }
        for (int x = 0; x < n_kv; ++x) {
          const int s = (step + x) & 1, u = (step + x) >> 1;
          const int s1 = (step + x + 1) & 1, u1 = (step + x + 1) >> 1;
          ok = __all_sync(kFull, mbar_wait(&v_full[s], u & 1, &failed));
          if (x + 1 < n_kv) ok = ok && __all_sync(kFull, mbar_wait(&k_full[s1], u1 & 1, &failed));
          if (!ok) break;
          const bool brief_now = brief && x == 1, brief_next = brief && x == 0;
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            if (looks(t, x)) {
              // O_t += P_t V_j in two parts, as in fa_fwd.cu
              ok = ok && __all_sync(kFull, mbar_wait(&p_full[t], products[t] & 1, &failed));
              if (!ok) break;
              tc::fence_after_sync();
              const uint64_t vd = v_desc + (uint32_t)(s * (kTileBytes >> 4));
              const uint32_t o = tmem + kColO + t * 128, pa = tmem + kColS + t * 128;
              if (brief_now) tc::product_ts<kFront / 16>(o, pa, vd, idesc_pv, begun[t]);
              else tc::product_ts<kSplit / 16>(o, pa, vd, idesc_pv, begun[t]);
              ok = __all_sync(kFull, mbar_wait(&p_rest[t], products[t] & 1, &failed));
              if (!ok) break;
              tc::fence_after_sync();
              // (16 keys of V are 2048 bytes of a 64-column box)
              if (!brief_now) tc::product_ts<(BN - kSplit) / 16>(o, pa + kSplit / 2, vd + (uint32_t)(kSplit / 16 * 2048 >> 4), idesc_pv, 1u);
              ++products[t];
              begun[t] = true;
              if (x == last[t]) tc::commit_elected(&pv_done[t]);
            }
            // P_t has been consumed by the MMAs just issued (the tensor core runs them in
            // order), so tile t's buffer can take the scores of the next step
            if (x + 1 < n_kv && looks(t, x + 1)) issue_qk(t, s1, brief_next);
          }
          if (!ok) break;
          tc::commit_elected(&v_empty[s]);
          if (x + 1 < n_kv) tc::commit_elected(&k_empty[s1]);
          if (x + 2 == n_kv) tc::commit_elected(&q_empty);  // the item's last scores are issued
        }
        step += n_kv;
        index = take_next(n, ok);
      }
      if (!ok && lane == 0) failed = 1;
      __syncwarp();
    } else if (warp == 2) {
      // -------------------------------------------------------------------- scheduler (as in fa_fwd.cu)
      bool ok = true;
      for (int n = 0; ok; ++n) {
        ok = __all_sync(kFull, mbar_wait(&next_wanted, n & 1, &failed));
        if (ok && n > 0) ok = __all_sync(kFull, mbar_wait(&next_taken[(n - 1) & 1], ((n - 1) >> 1) & 1, &failed));
        if (!ok) break;
        if (lane == 0) tc::request_next_block(&next_answer[n & 1], &next_full[n & 1]);
        asked = n + 1;
        ok = __all_sync(kFull, mbar_wait(&next_full[n & 1], (n >> 1) & 1, &failed));
        if (!ok || __shfl_sync(kFull, tc::next_block(&next_answer[n & 1]), 0) < 0) break;
      }
      if (!ok && lane == 0) failed = 1;
    }
  } else {
    // ----------------------------------------------------------- softmax + epilogue
    tc::regs_inc<kRegsSoftmax>();
    const int t = (warp >> 2) - 1;           // tile of rows of this warp group
    const int quad = warp & 3;               // TMEM lane quadrant this warp may touch
    const int row = quad * 32 + lane;        // row inside the tile
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_addr = lane_addr + kColS + t * 128;
    const uint32_t o_addr = lane_addr + kColO + t * 128;
    bool ok = true;
    int seen = 0;   // score tiles of this tile of rows so far, over all items
    int closed = 0; // items in which this tile of rows had work
    for (int n = 0, index = blockIdx.x; index >= 0 && ok; ++n) {
      const Item w = item_of(index);
      const int i0 = t ? w.i0[1] : w.i0[0], h0 = t ? w.h0[1] : w.h0[0], lo = t ? w.lo[1] : w.lo[0], hi = t ? w.hi[1] : w.hi[0];
      const int qi = i0 + (row & (R - 1)), h = h0 + (row >> p.rows_log2);
      const int at = qi < w.q_len ? w.off + qi : -1;  // (below 0: sees nothing)
      // every row of the tile sees all of a key tile that ends before the first row and begins in the last row's window
      const int at_first = w.off + i0, at_last = w.off + min(i0 + R, w.q_len) - 1;
      const bool brief = p.sinks <= kFront && w.front;
      float m_used = -INFINITY;  // reference maximum (scaled, log2 domain)
      float l = 0.f;             // running sum of exp2(s - m_used)
      // key tiles hi - 1 .. lo, and tile 0 where it is not among them but has first tokens: the item's step 1, or its last
      const int steps = hi - lo + (p.sinks > 0 && lo > 0 ? 1 : 0), front_step = !w.front ? hi - lo : hi == w.end ? 1 : 0;
      for (int i = 0; i < steps; ++i) {
        const bool front = i == front_step;
        const int j = hi - 1 - i + (i > front_step ? 1 : 0);
        if (!__all_sync(kFull, mbar_wait(&s_full[t], seen & 1, &failed))) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        const int col0 = front ? 0 : j * BN;
        WindowMask mask;
        mask.edge = front || col0 + BN - 1 > at_first || col0 <= at_last - p.window;
        mask.lim = at - col0;
        mask.from = col0 == 0 ? p.sinks : 0;
        mask.low = at - p.window + 1 - col0;
        if (front && brief)
          softmax_tile<IS_BF16, kFront>(s_addr, o_addr, mask, i == 0, p.scale_log2, m_used, l, &p_full[t], &p_rest[t]);
        else
          softmax_tile<IS_BF16>(s_addr, o_addr, mask, i == 0, p.scale_log2, m_used, l, &p_full[t], &p_rest[t]);
        ++seen;
      }
      if (ok && hi > 0) {
        ok = __all_sync(kFull, mbar_wait(&pv_done[t], closed & 1, &failed));  // the tile's last product
        ++closed;
      }
      if (ok && h0 >= 0) {
        tc::fence_after_sync();
        if (at < 0) l = 0.f;  // (tiles that all other rows see whole are not masked)
        const bool live = qi < p.Sq && h < (w.hk + 1) * p.share;
        unsigned char* orow = reinterpret_cast<unsigned char*>(p.o) +
                              2 * ((long long)w.b * p.o_stride_b + (long long)h * p.o_stride_h +
                                   (long long)qi * p.o_stride_s);
        if (hi > 0) {
          const float inv = 1.f / l;  // (l may be NaN)
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            tc::tmem_ld32(o_addr + c * 32, o);
            tc::tmem_wait_ld();
            if (live && l != 0.f) tc::store_row32<IS_BF16>(orow + c * 64, o, inv, p.wide != 0);
          }
        }
        if (live && l == 0.f) {  // nothing was seen
#pragma unroll
          for (int c = 0; c < HD / 8; ++c) reinterpret_cast<uint4*>(orow)[c] = make_uint4(0, 0, 0, 0);
        }
        if (live && p.lse != nullptr) {
          const float lse = l == 0.f ? -INFINITY : (m_used + log2f(l)) * 0.69314718055994530942f;  // (l may be NaN)
          p.lse[((long long)w.b * p.H + h) * p.Sq + qi] = lse;
        }
      }
      // (the next item's scores may be written meanwhile, but its first product waits for this
      // warp's probabilities, which come after the reads of O above)
      tc::fence_before_sync();
      index = take_next(n, ok);
    }
    if (!ok && lane == 0) failed = 1;
  }

  tc::fence_before_sync();
  __syncthreads();
  if (failed) {  // (uniform: nobody writes it any more)
    // a role gave up: what the others have under way has to end before the block does
    if (threadIdx.x == 0) {
      tc::await_copies<1>(&q_full, q_loads);
      tc::await_copies<kStages>(k_full, k_loads);
      if (raw_pending) mbar_wait(&v_raw, (raw_loads - 1) & 1);
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

}  // namespace

namespace ixb_host {

int window_prefill(const WindowShape& a, const WindowView& q, const WindowView& k, const WindowView& v, const WindowView& o,
                   float* lse, int32_t* status, cudaStream_t stream) {
  WinParams p;
  p.rows_log2 = 3;
  while (p.rows_log2 < 7 && (1 << p.rows_log2) < a.Sq) ++p.rows_log2;
  CUtensorMap mq, mk, mv;
  if (int st = make_fa_map(&mq, q.ptr, a.is_bf16, a.B, a.H, a.Sq, q.strides[0], q.strides[1], q.strides[2], 1 << p.rows_log2)) return st;
  if (int st = make_fa_map(&mk, k.ptr, a.is_bf16, a.B, a.HK, a.Sk, k.strides[0], k.strides[1], k.strides[2])) return st;
  if (int st = make_fa_map(&mv, v.ptr, a.is_bf16, a.B, a.HK, a.Sk, v.strides[0], v.strides[1], v.strides[2])) return st;
  CUtensorMap mkf = mk, mvf = mv;
  if (a.sinks > 0 && a.window < a.Sk) {
    if (int st = make_fa_map(&mkf, k.ptr, a.is_bf16, a.B, a.HK, a.Sk, k.strides[0], k.strides[1], k.strides[2], kFront)) return st;
    if (int st = make_fa_map(&mvf, v.ptr, a.is_bf16, a.B, a.HK, a.Sk, v.strides[0], v.strides[1], v.strides[2], kFront)) return st;
  }
  p.o = const_cast<void*>(o.ptr);
  p.lse = lse;
  p.status = status;
  p.q_lengths = a.q_lengths;
  p.kv_lengths = a.kv_lengths;
  p.o_stride_b = o.strides[0];
  p.o_stride_h = o.strides[1];
  p.o_stride_s = o.strides[2];
  p.B = a.B, p.H = a.H, p.HK = a.HK, p.share = a.H / a.HK, p.Sq = a.Sq, p.Sk = a.Sk;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.window = a.window, p.sinks = a.sinks;
  const int heads = BM >> p.rows_log2;  // query heads in a tile
  const long long tiles = (long long)((a.Sq + BM - 1) / BM) * ((p.share + heads - 1) / heads);
  // One tile an item where that leaves no SM with two: a step of one takes about two thirds of a step of both.
  // 3 x 4 key heads, 500 queries of share 3, window 600: 25.9 -> 21.7 us.
  const ixb_devinfo* dev = current_device();
  if (dev == nullptr) return IXB_ERR_CUDA;
  p.per_item = tiles * a.B * a.HK <= dev->sm_count ? 1 : NQ;
  const long long items = (tiles + p.per_item - 1) / p.per_item * a.B * a.HK;
  if (items > 0x7fffffffLL) return IXB_ERR_SHAPE;
  p.tiles = (int)tiles;
  p.head_group = 8;
  p.wide = rows_aligned32(o.ptr, o.strides) ? 1 : 0;
  auto kern = a.is_bf16 ? fa_window_fwd_kernel<true> : fa_window_fwd_kernel<false>;
  // the shared-memory opt-in is a property of (kernel, device): set once per device
  static std::atomic<bool> configured[2][64];
  int devid = 0;
  cudaGetDevice(&devid);
  std::atomic<bool>& done = configured[a.is_bf16][devid & 63];
  if (!done.load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e != cudaSuccess) return cuda_status(e);
    cudaFuncAttributes at;  // (as in fa_fwd.cu: the softmax warps wait for registers the block has to own)
    e = cudaFuncGetAttributes(&at, kern);
    if (e != cudaSuccess) return cuda_status(e);
    if (at.numRegs != kRegsLaunch) return IXB_ERR_UNSUPPORTED;
    done.store(true, std::memory_order_release);
  }
  kern<<<(unsigned)items, kThreads, kSmemBytes, stream>>>(mq, mk, mv, mkf, mvf, p);
  return cuda_status(cudaGetLastError());
}

}  // namespace ixb_host

extern "C" int ixb_window_attention(int dtype, const void* q, const void* k, const void* v, void* o, float* lse,
                                    int32_t B, int32_t H, int32_t HK, int32_t Sq, int32_t Sk, int32_t D,
                                    const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                    const int64_t* o_strides, const int32_t* q_lengths, const int32_t* kv_lengths, float scale,
                                    int32_t window, int32_t sinks, int32_t* status, ixb_stream stream) {
  if (int st = ixb_host::check_window_sizes(dtype, B, H, HK, Sq, Sk, D, scale, window, sinks)) return st;
  if (B == 0 || H == 0 || Sq == 0) return IXB_OK;
  if (Sk == 0) return IXB_ERR_SHAPE;
  const ixb_host::WindowView views[] = {{q, q_strides}, {k, k_strides}, {v, v_strides}, {o, o_strides}};
  if (int st = ixb_host::check_window_views(views, 4)) return st;
  const ixb_host::WindowShape a{dtype == IXB_BF16, B, H, HK, Sq, Sk, q_lengths, kv_lengths, scale, window < Sk ? window : Sk, sinks};
  if (ixb_host::window_decodes(a))
    return ixb_host::window_decode(a, views[0], views[1], views[2], views[3], lse, status, (cudaStream_t)stream);
  double us;
  if (const int cluster = ixb_host::window_split_size(a, &us))
    return ixb_host::window_split(cluster, a, views[0], views[1], views[2], views[3], lse, status, (cudaStream_t)stream);
  return ixb_host::window_prefill(a, views[0], views[1], views[2], views[3], lse, status, (cudaStream_t)stream);
}
