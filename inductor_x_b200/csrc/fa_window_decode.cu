// Windowed attention of a few queries over a long cache: the decoding step (the meaning of the arguments: fa_window.h).
// All that a key head's queries need is read once: a block takes the queries of every query head that shares the key head
// (queries x sharing heads, in groups of 8 or 16), and the keys are the first tokens that lie in front of the window and the
// window itself, cut into tiles of 16.  The tiles are shared over the kWarps warps of 1, 2, 4 or 8 blocks of a cluster.  A warp
// keeps its own running maximum, sum and accumulators and has its own ring of copies: nothing waits for another warp
// before the end, when the warps of a block and then the blocks of the cluster add up, row by row through distributed
// shared memory: one launch, no scratch, the same bits every time.
//
// Probabilities are rounded to the operands' 16 bits, as in fa_window_fwd.cu; maxima, sums and accumulators have 32.
//
// Bound: memory.  A key costs 512 bytes and, per row, 512 multiplications, so that warp-wide 16 x 8 x 16 products are
// enough.  They are taken with the keys (S^T = K Q^T) and the dimensions (O^T = V^T P^T) as their 16 rows and the queries as
// their 8 columns, since hardly more than 8 queries share a key.  K and V come out of shared memory as whole 16-byte
// pieces: the order of the reduced dimensions of S is free, so a lane's piece of 8 dimensions is taken for four of its pairs;
// the rows of O are free too, so a lane pairs up its pieces of two keys element by element.
// 64 sequences of up to 16384 keys, window 4096, 32/8 heads: 143 us, 6570 GB/s (a copy 6532); 8 sequences 25 us, 5.3 TB/s; one, window
// 1024, 5.5 us.  With the queries as the 16 rows the same within 3 %, and twice the accumulators: an SM takes 50 GB/s either way.
#include <atomic>
#include "fa_window.h"
#include "ixb/tcgen05.cuh"

namespace {

using namespace ixb;

constexpr int HD = 128, kTile = 16, kWarps = 4, kThreads = kWarps * 32, kStages = 3;
constexpr int kBoxBytes = kTile * 128;        // 16 keys of 64 dimensions
constexpr int kStageBytes = 4 * kBoxBytes;    // K and V
constexpr int kPitch = HD + 4;                // floats: of a row of partial sums
constexpr size_t kSmemBytes = (size_t)kWarps * kStages * kStageBytes + 1024;

struct DecodeParams {
  const unsigned char* q;
  unsigned char* o;
  float* lse;     // [B, H, Sq], may be null
  int* status;    // may be null
  const int *q_lengths, *kv_lengths;
  long long q_sb, q_sh, q_ss, o_sb, o_sh, o_ss;  // elements
  int H, HK, share, Sq, Sk, rows, groups;        // rows = share * Sq, in `groups` of 8 * NT
  float scale_log2;
  int window, sinks;
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
// d += a b: 16 rows x 16, 16 x 8
template <bool IS_BF16> __device__ __forceinline__ void product(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (IS_BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the 8 x 8 matrix of which a lane holds two neighbours of row lane / 4, the other way round
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// piece `chunk` (16 bytes of 8 dimensions) of key `key` in a box of 128-byte rows that the copy engine has swizzled
__device__ __forceinline__ uint4 piece(const unsigned char* box, int key, int chunk) {
  return *reinterpret_cast<const uint4*>(box + key * 128 + ((chunk ^ (key & 7)) << 4));
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <bool IS_BF16, int NT, int CLUSTER>
__global__ void __launch_bounds__(kThreads, 2)
    window_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const DecodeParams p) {
  constexpr int kRows = 8 * NT;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full[kWarps][kStages];
  __shared__ float m_part[kWarps][kRows], l_part[kWarps][kRows], m_block[kRows], l_block[kRows];
  __shared__ volatile int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3;
  const int rank = CLUSTER > 1 ? (int)cluster_rank() : 0;
  const int item = (int)blockIdx.x / CLUSTER, group = item % p.groups, bh = item / p.groups, b = bh / p.HK, hk = bh - b * p.HK;
  const int row0 = group * kRows;
  const int q_len = p.q_lengths != nullptr ? min(max(__ldg(p.q_lengths + b), 0), p.Sq) : p.Sq;
  const int kv_len = p.kv_lengths != nullptr ? min(max(__ldg(p.kv_lengths + b), 0), p.Sk) : p.Sk;
  const int off = kv_len - q_len;  // query i stands at position off + i
  const bool any = q_len > 0 && kv_len > 0;
  // keys [0, front) and [low, kv_len) are seen by some query
  const int low = any ? max(max(off, 0) - p.window + 1, 0) : 0, front = any ? min(p.sinks, low) : 0;
  const int front_tiles = (front + kTile - 1) / kTile, tiles = any ? front_tiles + (kv_len - low + kTile - 1) / kTile : 0;
  auto first_key = [&](int t) { return t < front_tiles ? t * kTile : low + (t - front_tiles) * kTile; };
  const int worker = rank * kWarps + warp;
  constexpr int kWorkers = CLUSTER * kWarps;
  const int mine = tiles > worker ? (tiles - worker + kWorkers - 1) / kWorkers : 0;

  if (threadIdx.x == 0) failed = 0;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], 1);
    mbar_init_fence();
  }
  __syncthreads();
  unsigned char* ring = smem + warp * kStages * kStageBytes;
  auto ask = [&](int i, int place) {  // tile i of this warp (one lane)
    unsigned char* dst = ring + place * kStageBytes;
    uint64_t* bar = &full[warp][place];
    const int key = first_key(worker + i * kWorkers);
    mbar_arrive_expect_tx(bar, kStageBytes);
    tc::tma_load_4d(dst, &map_k, bar, 0, key, hk, b);
    tc::tma_load_4d(dst + kBoxBytes, &map_k, bar, 64, key, hk, b);
    tc::tma_load_4d(dst + 2 * kBoxBytes, &map_v, bar, 0, key, hk, b);
    tc::tma_load_4d(dst + 3 * kBoxBytes, &map_v, bar, 64, key, hk, b);
  };
  if (lane == 0)
    for (int i = 0; i < kStages && i < mine; ++i) ask(i, i);

  // Q: the column n of each 8.  Piece 2c + odd of a half of 64 dimensions is two of the lane's steps of 16.
  uint32_t qf[NT][8][2];
  int at[NT][2];  // positions of the queries 2c and 2c + 1 (below 0: sees nothing)
  auto position = [&](int r) {
    const int i = r % p.Sq;
    return r < p.rows && i < q_len ? off + i : -1;
  };
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = row0 + t * 8 + n, g = r / p.Sq, i = r - g * p.Sq;
    const bool live = r < p.rows && i < q_len;
    const unsigned char* src = p.q + 2 * (b * p.q_sb + (hk * p.share + g) * p.q_sh + i * p.q_ss);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 v = live ? ldg_keep(src + 2 * (k / 2 * 64 + (2 * c + k % 2) * 8)) : make_uint4(0, 0, 0, 0);
      qf[t][2 * k][0] = v.x;
      qf[t][2 * k][1] = v.y;
      qf[t][2 * k + 1][0] = v.z;
      qf[t][2 * k + 1][1] = v.w;
    }
    at[t][0] = position(row0 + t * 8 + 2 * c);
    at[t][1] = position(row0 + t * 8 + 2 * c + 1);
  }

  // acc: product j, dimensions 8n + j and 64 + 8n + j of the queries 2c and 2c + 1
  float acc[NT][8][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][j][e] = 0.f;
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
  }
  bool ok = true;
  int s = 0, turn = 0;
  for (int i = 0; i < mine; ++i) {
    ok = __all_sync(kFull, mbar_wait(&full[warp][s], turn, &failed));
    if (!ok) break;
    const unsigned char *kb = ring + s * kStageBytes, *vb = kb + 2 * kBoxBytes;
    const int tile = worker + i * kWorkers, key0 = first_key(tile), end = tile < front_tiles ? front : kv_len;
    float sc[NT][4];  // keys n (0, 1) and n + 8 (2, 3) of the queries 2c and 2c + 1
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[t][e] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 x = piece(kb + k / 2 * kBoxBytes, n, 2 * c + k % 2), y = piece(kb + k / 2 * kBoxBytes, 8 + n, 2 * c + k % 2);
      const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        product<IS_BF16>(sc[t], a0, qf[t][2 * k][0], qf[t][2 * k][1]);
        product<IS_BF16>(sc[t], a1, qf[t][2 * k + 1][0], qf[t][2 * k + 1][1]);
      }
    }
    // what a query does not see: keys behind its own position, or between the first tokens and its window; or no key of the walk
    const bool edge = key0 + kTile > end || p.Sq > 1;
    if (edge) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + n + (e >> 1) * 8, place = at[t][e & 1];
          if (key >= end || key > place || (key <= place - p.window && key >= p.sinks)) sc[t][e] = -INFINITY;
        }
    }
    uint32_t pr[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top[2], f[2], x[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) x[h] = fmaxf(sc[t][h], sc[t][2 + h]);
#pragma unroll
      for (int o = 4; o < 32; o *= 2)
#pragma unroll
        for (int h = 0; h < 2; ++h) x[h] = fmaxf(x[h], __shfl_xor_sync(kFull, x[h], o));
      bool grow = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[h] *= p.scale_log2;  // scale > 0: scaling commutes with the maximum
        // the reference moves only when it would grow by more than 2^8 (the last division makes a stale one exact)
        top[h] = x[h] > m[t][h] + 8.f ? x[h] : m[t][h];
        f[h] = top[h] == m[t][h] ? 1.f : fast_exp2(m[t][h] - top[h]);  // (0 at first)
        grow = grow || top[h] != m[t][h];
      }
      if (__any_sync(kFull, grow)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          l[t][h] *= f[h];
          m[t][h] = top[h];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][j][e] *= f[e & 1];
      }
      const float ref[2] = {m[t][0] == -INFINITY ? 0.f : m[t][0], m[t][1] == -INFINITY ? 0.f : m[t][1]};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float a = fast_exp2(fmaf(sc[t][2 * u], p.scale_log2, -ref[0])), z = fast_exp2(fmaf(sc[t][2 * u + 1], p.scale_log2, -ref[1]));
        l[t][0] += a;
        l[t][1] += z;
        pr[t][u] = transposed(tc::round_pair<IS_BF16>(a, z));  // keys 2c, 2c + 1 (and 8 behind them) of query n
      }
    }
    // V: keys 2c, 2c + 1, 2c + 8, 2c + 9, dimensions 8n .. 8n + 7 of each half; product j takes dimension 8n + j of both
    uint4 v[2][4];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = 2 * c + (e & 1) + (e >> 1) * 8;
        v[half][e] = piece(vb + half * kBoxBytes, key, n);
        if (edge && key0 + key >= end) v[half][e] = make_uint4(0, 0, 0, 0);  // (a probability of 0 times whatever lies there)
      }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned pick = j & 1 ? 0x7632u : 0x5410u;
      uint32_t a[4];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int u = 0; u < 2; ++u) a[2 * u + half] = __byte_perm(word(v[half][2 * u], j / 2), word(v[half][2 * u + 1], j / 2), pick);
#pragma unroll
      for (int t = 0; t < NT; ++t) product<IS_BF16>(acc[t][j], a, pr[t][0], pr[t][1]);
    }
    __syncwarp();  // (the whole warp has read the tile)
    if (lane == 0 && i + kStages < mine) ask(i + kStages, s);
    if (++s == kStages) {
      s = 0;
      turn ^= 1;
    }
  }
  if (!ok) {  // what this warp has under way ends before its block leaves
    failed = 1;
    for (int i = 1; i < kStages; ++i) {
      const int other = (s + i) % kStages;
      mbar_wait(&full[warp][other], s + i < kStages ? turn : turn ^ 1);
    }
  }

  // ---- the warps' sums: the ring makes room for them
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int o = 4; o < 32; o *= 2) l[t][h] += __shfl_xor_sync(kFull, l[t][h], o);
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);  // [kWarps][kRows][kPitch], then the block's [kRows][kPitch]
  static_assert((kWarps + 1) * kRows * kPitch * sizeof(float) <= (size_t)kWarps * kStages * kStageBytes, "the partial sums take the ring's place");
  float* block_sums = sums + kWarps * kRows * kPitch;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = t * 8 + 2 * c + h;
      if (n == 0) {
        m_part[warp][r] = m[t][h];
        l_part[warp][r] = l[t][h];
      }
      float* dst = sums + (warp * kRows + r) * kPitch;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int j = 0; j < 8; j += 4)
          *reinterpret_cast<float4*>(dst + half * 64 + 8 * n + j) =
              make_float4(acc[t][j][2 * half + h], acc[t][j + 1][2 * half + h], acc[t][j + 2][2 * half + h], acc[t][j + 3][2 * half + h]);
    }
  __syncthreads();
  const int rows = min(kRows, p.rows - row0);
  auto finish = [&](int r, float4 x, float top, float total) {
    const int g = (row0 + r) / p.Sq, i = row0 + r - g * p.Sq, h = hk * p.share + g;
    const float inv = total == 0.f ? 0.f : 1.f / total;  // (a sum may be NaN)
    uint2 out;
    out.x = tc::round_pair<IS_BF16>(x.x * inv, x.y * inv);
    out.y = tc::round_pair<IS_BF16>(x.z * inv, x.w * inv);
    *reinterpret_cast<uint2*>(p.o + 2 * (b * p.o_sb + h * p.o_sh + i * p.o_ss) + lane * 8) = out;
    if (lane == 0 && p.lse != nullptr)
      p.lse[((long long)b * p.H + h) * p.Sq + i] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.69314718055994530942f;
  };
  // a warp a row, a lane four columns
  for (int r = warp; r < rows; r += kWarps) {
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_part[w][r]);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = m_part[w][r] == -INFINITY ? 0.f : fast_exp2(m_part[w][r] - top);
      const float4 y = *reinterpret_cast<const float4*>(sums + (w * kRows + r) * kPitch + lane * 4);
      total = fmaf(f, l_part[w][r], total);
      x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
    }
    if constexpr (CLUSTER == 1) {
      finish(r, x, top, total);
    } else {
      *reinterpret_cast<float4*>(block_sums + r * kPitch + lane * 4) = x;
      if (lane == 0) {
        m_block[r] = top;
        l_block[r] = total;
      }
    }
  }
  if constexpr (CLUSTER > 1) {
    __syncwarp();
    cluster_sync_all();
    for (int r = rank + warp * CLUSTER; r < rows; r += CLUSTER * kWarps) {
      float top = -INFINITY, total = 0.f, ms[CLUSTER], ls[CLUSTER];
      float4 y[CLUSTER];
#pragma unroll
      for (int k = 0; k < CLUSTER; ++k) {
        ms[k] = ld_cluster_f32(map_to_rank(&m_block[r], k));
        ls[k] = ld_cluster_f32(map_to_rank(&l_block[r], k));
        y[k] = ld_cluster_f32x4(map_to_rank(block_sums + r * kPitch + lane * 4, k));
        top = fmaxf(top, ms[k]);
      }
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < CLUSTER; ++k) {
        const float f = ms[k] == -INFINITY ? 0.f : fast_exp2(ms[k] - top);
        total = fmaf(f, ls[k], total);
        x.x = fmaf(f, y[k].x, x.x), x.y = fmaf(f, y[k].y, x.y), x.z = fmaf(f, y[k].z, x.z), x.w = fmaf(f, y[k].w, x.w);
      }
      finish(r, x, top, total);
    }
    __syncwarp();
    cluster_sync_all();  // nobody leaves while another block reads its shared memory
  }
  if (threadIdx.x == 0 && failed && p.status != nullptr) atomicExch(p.status, 1);
}

template <bool IS_BF16, int NT, int CLUSTER>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const DecodeParams& p, long long items, cudaStream_t stream) {
  auto kern = window_decode_kernel<IS_BF16, NT, CLUSTER>;
  static std::atomic<bool> configured[64];
  int devid = 0;
  cudaGetDevice(&devid);
  if (!configured[devid & 63].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e != cudaSuccess) return ixb_host::cuda_status(e);
    configured[devid & 63].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  cfg.gridDim = dim3((unsigned)(items * CLUSTER));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CLUSTER;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = CLUSTER > 1 ? 1 : 0;
  return ixb_host::cuda_status(cudaLaunchKernelEx(&cfg, kern, mk, mv, p));
}

}  // namespace

namespace ixb_host {

// Keys that the queries of a sequence see at most.
static long long keys_seen(const WindowShape& a) {
  const long long keys = (long long)a.window + a.Sq - 1 + a.sinks;
  return keys < a.Sk ? keys : a.Sk;
}
static int clusters_of(long long items, long long tiles, int sms) {
  int cluster = 1;
  while (cluster < 8 && items * cluster <= sms && tiles > kWarps * cluster) cluster *= 2;
  return cluster;
}

// Whether this kernel promises to be quicker than the other two, as measured on one B200 (35 shapes of 16 to 128 rows a key head, 8
// to 512 key heads, within 15 %): 5 us + 0.6 a tile of a warp, and not less than 1.25 for each 8 tiles an SM.
// Against fa_window_fwd.cu: 16 rows, 8 key heads, 1024 keys 6.8 and 24.2, 4096 keys 12.3 and 63; 64 rows, 64 key heads, 1024 keys 23.2
// and 24.6, 256 key heads, 2048 keys 142 and 71; 128 rows, 8 key heads, 4096 keys 23 and 62, 64 key heads, 1024 keys 44.5 and 24.9.
bool window_decodes(const WindowShape& a) {
  const long long share = a.H / a.HK, rows = share * a.Sq;
  if (rows > 256) return false;
  const ixb_devinfo* dev = current_device();
  if (dev == nullptr) return true;
  const double sms = dev->sm_count, heads = (double)a.B * a.HK, keys = (double)keys_seen(a);
  const int groups = rows <= 8 ? 1 : (int)((rows + 15) / 16);
  const long long tiles = ((long long)keys + 2 * kTile - 2) / kTile;
  const int cluster = clusters_of((long long)heads * groups, tiles, dev->sm_count);
  const double chain = 0.6 * tiles / (kWarps * cluster), load = 1.25 * heads * groups * tiles / (8 * sms);
  double other;
  window_split_size(a, &other);
  return 5 + (chain > load ? chain : load) < other;
}

int window_decode(const WindowShape& a, const WindowView& q, const WindowView& k, const WindowView& v, const WindowView& o,
                  float* lse, int32_t* status, cudaStream_t stream) {
  const ixb_devinfo* dev = current_device();
  if (dev == nullptr) return IXB_ERR_CUDA;
  CUtensorMap mk, mv;
  if (int st = make_fa_map(&mk, k.ptr, a.is_bf16, a.B, a.HK, a.Sk, k.strides[0], k.strides[1], k.strides[2], kTile)) return st;
  if (int st = make_fa_map(&mv, v.ptr, a.is_bf16, a.B, a.HK, a.Sk, v.strides[0], v.strides[1], v.strides[2], kTile)) return st;
  DecodeParams p;
  p.q = static_cast<const unsigned char*>(q.ptr);
  p.o = static_cast<unsigned char*>(const_cast<void*>(o.ptr));
  p.lse = lse;
  p.status = status;
  p.q_lengths = a.q_lengths;
  p.kv_lengths = a.kv_lengths;
  p.q_sb = q.strides[0], p.q_sh = q.strides[1], p.q_ss = q.strides[2];
  p.o_sb = o.strides[0], p.o_sh = o.strides[1], p.o_ss = o.strides[2];
  p.H = a.H, p.HK = a.HK, p.share = a.H / a.HK, p.Sq = a.Sq, p.Sk = a.Sk;
  p.rows = p.share * a.Sq;
  p.scale_log2 = a.scale * kLog2e;
  p.window = a.window, p.sinks = a.sinks;
  const int nt = p.rows <= 8 ? 1 : 2;
  p.groups = (p.rows + 8 * nt - 1) / (8 * nt);
  const long long items = (long long)a.B * a.HK * p.groups;
  if (items > (1 << 27)) return IXB_ERR_SHAPE;
  const int cluster = clusters_of(items, (keys_seen(a) + 2 * kTile - 2) / kTile, dev->sm_count);
#define IXB_DECODE_CASE(N, C) \
  if (nt == N && cluster == C) return a.is_bf16 ? launch<true, N, C>(mk, mv, p, items, stream) : launch<false, N, C>(mk, mv, p, items, stream);
  IXB_DECODE_CASE(1, 1)
  IXB_DECODE_CASE(1, 2)
  IXB_DECODE_CASE(1, 4)
  IXB_DECODE_CASE(1, 8)
  IXB_DECODE_CASE(2, 1)
  IXB_DECODE_CASE(2, 2)
  IXB_DECODE_CASE(2, 4)
  IXB_DECODE_CASE(2, 8)
#undef IXB_DECODE_CASE
  return IXB_ERR_UNSUPPORTED;
}

}  // namespace ixb_host
