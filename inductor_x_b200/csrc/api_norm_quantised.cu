// Root-mean-square norm with the residual's addition and an 8-bit output:
//   h = x (+ residual), rounded to the storage type; y = h * rsqrt(mean(h^2) + eps) * w in 32 bits;
//   scale = max |y| / 448 over the row or over each 128 values of it; q = e4m3(y / scale).
//
// A row is read once and stays in the registers of W warps, as units of 32 lanes.  A group of 128 values belongs to one
// warp (half of one for vectors of 16 bits), so that its largest magnitude takes shuffles only; the row's sum, and its
// largest magnitude where the scale is the row's, go through shared memory.
//   norm_quantised_kernel          16-byte vectors of the row, where rows and pointers allow it
//   norm_quantised_shifted_kernel  rows off a boundary: the vectors are those of memory, of which the row covers the first and
//                                  the last in part
//   norm_quantised_long_kernel     rows that no block holds, and operands that are off a boundary by different offsets: a view of
//                                  x that starts off one, since q and h start on one (16384 x 4096 bf16 with residual 327 us,
//                                  by vectors 72; 5003 x 1537 fp16 42, shifted 17)
// Bound: memory, 2 (4 with residual) + 1 (3) bytes a value in 16 bits.
#include <cuda_fp8.h>
#include <atomic>
#include <cmath>
#include "host.h"
#include "ixb/common.cuh"

namespace {

using namespace ixb;
constexpr int kGroup = 128;
constexpr float kLargest = 448.f;

struct NormParams {
  const void *x, *res, *w;  // res may be null
  unsigned char* q;
  float* scales;
  void* h_out;              // may be null
  long long rows;
  int cols, group;
  float per_col, eps;        // 1 / cols
};

// Magnitudes are compared as bits: the order of floats without a sign, and NaN above all.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
template <int WIDTH> __device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float scale_of(uint32_t top) { return __uint_as_float(top) * (1.f / kLargest); }
// What values are multiplied with whose largest magnitude is `top`.  The approximate reciprocal is 2^-23 of itself off, 2^-19 of
// a step of the 8-bit value.
__device__ __forceinline__ float factor_of(uint32_t top) {
  float inverse;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(__uint_as_float(top)));
  return kLargest * inverse;
}
// Whether that leaves the range of normal numbers (zero and infinity do).
__device__ __forceinline__ bool extreme(uint32_t top) { return top - 0x0d800000u > 0x71800000u - 0x0d800000u; }  // not in 2^[-100, 100]
// Then values and their largest magnitude come nearer to 1 first, by a power of two.
__device__ __forceinline__ float tame(uint32_t& top) {
  const float t = __uint_as_float(top);
  const float pre = t < 1.f ? 0x1p64f : 0x1p-64f;
  top = t == 0.f ? 0x7f800000u : __float_as_uint(t * pre);  // (nothing but zeros: times 448 / infinity)
  return pre;
}

// A vector as pairs.
template <class T> struct Pairs {
  static constexpr int E = Elem<T>::kVec;
  float2 v[E / 2];
  __device__ __forceinline__ void unpack(const uint4& raw) { ixb::unpack<T>(raw, reinterpret_cast<float*>(v)); }
  __device__ __forceinline__ uint4 pack() const { return ixb::pack<T>(reinterpret_cast<const float*>(v)); }
  __device__ __forceinline__ void add(const uint4& raw) {
    Pairs g;
    g.unpack(raw);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) v[e] = add2(v[e], g.v[e]);
  }
  __device__ __forceinline__ float2 squares(float2 sum) const {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) sum = fma2(v[e], v[e], sum);
    return sum;
  }
  __device__ __forceinline__ void scale(float r, const uint4& w) {
    Pairs g;
    g.unpack(w);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) v[e] = mul2(mul2(v[e], make_float2(r, r)), g.v[e]);
  }
  __device__ __forceinline__ void keep(uint32_t lives) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      if (!(lives >> e & 1u)) v[e / 2].x = 0.f;
      if (!(lives >> (e + 1) & 1u)) v[e / 2].y = 0.f;
    }
  }
  __device__ __forceinline__ uint32_t bits(int e) const { return __float_as_uint(e & 1 ? v[e / 2].y : v[e / 2].x); }
  __device__ __forceinline__ uint32_t largest(uint32_t m = 0) const {
#pragma unroll
    for (int e = 0; e < E; e += 2) m = __vimax3_u32(m, bits(e) & 0x7fffffffu, bits(e + 1) & 0x7fffffffu);
    return m;
  }
};
template <int N> __device__ __forceinline__ void store_bytes(unsigned char* q, const uint32_t (&two)[N]) {
  if constexpr (N == 4) *reinterpret_cast<uint2*>(q) = make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
  else *reinterpret_cast<uint32_t*>(q) = two[0] | two[1] << 16;
}

// Zeros in place of the elements of a vector whose bit is not set.
template <int E> __device__ __forceinline__ uint4 kept(const uint4& v, uint32_t lives) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (E == 8) w[k] &= (lives >> (2 * k) & 1u ? 0xffffu : 0u) | (lives >> (2 * k + 1) & 1u ? 0xffff0000u : 0u);
    else if (!(lives >> k & 1u)) w[k] = 0u;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// W warps a row, each U units of 32 vectors.
template <class T, int W, int U>
__global__ void __launch_bounds__(W < 8 ? 256 : W * 32) norm_quantised_kernel(const NormParams p) {
  constexpr int kRows = W < 8 ? 8 / W : 1, E = Elem<T>::kVec, kLanes = kGroup / E;
  __shared__ float sums[kRows * W];
  __shared__ uint32_t tops[kRows * W];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at = warp % W, team = warp / W;
  const long long row = (long long)blockIdx.x * kRows + team;
  const bool live = row < p.rows;
  const long long base = live ? row * p.cols : 0;
  const int cols = live ? p.cols : 0;
  const T *x = static_cast<const T*>(p.x) + base, *res = static_cast<const T*>(p.res) + base, *w = static_cast<const T*>(p.w);
  const uint4 none = make_uint4(0, 0, 0, 0);  // (what is behind the row counts as zero)
  auto col = [&](int u) { return ((at + u * W) * 32 + lane) * E; };
  uint4 raw[U], more[U];
#pragma unroll
  for (int u = 0; u < U; ++u) raw[u] = col(u) < cols ? ldg_stream(x + col(u)) : none;
  if (p.res != nullptr) {
#pragma unroll
    for (int u = 0; u < U; ++u) more[u] = col(u) < cols ? ldg_stream(res + col(u)) : none;
  }
  Pairs<T> f[U];
  float2 squares = make_float2(0.f, 0.f);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    f[u].unpack(raw[u]);
    if (p.res != nullptr) {
      f[u].add(more[u]);
      const uint4 h = f[u].pack();
      f[u].unpack(h);
      if (p.h_out != nullptr && col(u) < cols) *reinterpret_cast<uint4*>(static_cast<T*>(p.h_out) + base + col(u)) = h;
    }
    squares = f[u].squares(squares);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) raw[u] = col(u) < cols ? ldg_keep(w + col(u)) : none;
  float s = warp_reduce<SumOp>(squares.x + squares.y);
  if constexpr (W > 1) {
    if (lane == 0) sums[warp] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += sums[team * W + i];
  }
  const float r = rsqrtf(s * p.per_col + p.eps);
  auto put = [&](int u, uint32_t top) {
    float pre = 1.f;
    if (extreme(top)) pre = tame(top);
    const float by = factor_of(top);
    if (col(u) >= cols) return;
    uint32_t two[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      if (pre != 1.f) f[u].v[e] = mul2(f[u].v[e], make_float2(pre, pre));
      const float2 t = mul2(f[u].v[e], make_float2(by, by));
      two[e] = e4m3x2(t.x, t.y);
    }
    store_bytes(p.q + base + col(u), two);
  };
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    f[u].scale(r, raw[u]);
    const uint32_t mine = col(u) < cols ? f[u].largest() : 0u;  // (behind the row there are zeros, but r may be infinite)
    if (p.group == 0) {
      top = max(top, mine);
      continue;
    }
    const uint32_t m = group_max<kLanes>(mine);
    if (lane % kLanes == 0 && col(u) < cols) p.scales[row * ((p.cols + kGroup - 1) / kGroup) + col(u) / kGroup] = scale_of(m);
    put(u, m);
  }
  if (p.group != 0) return;
  top = __reduce_max_sync(kFull, top);
  if constexpr (W > 1) {
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top = max(top, tops[team * W + i]);
  }
  if (at == 0 && lane == 0 && live) p.scales[row] = scale_of(top);
#pragma unroll
  for (int u = 0; u < U; ++u) put(u, top);
}

// Rows off a boundary: the vectors are those of memory, and the row begins `shift` elements into its first one.  W warps take
// rows that all begin alike, `step` apart (rows eight apart do, whatever their length), so that what a thread holds of w, where
// its vectors are cut and which scales they take stay as they are; the next row is asked for while one is worked on.  A
// group's border lies inside the vector that begins with it, whose first elements are the group's before: the largest
// magnitudes of groups meet in shared memory.
// (The shift as a constant, one of eight loops for each: 120 us instead of 50 at 9000 x 3001; the blocks of an SM then run
// different code, more than its instruction cache holds.)
template <class T, int W, int U>
__global__ void __launch_bounds__(W < 8 ? 256 : W * 32, W <= 8 ? 4 : W == 16 ? 2 : 1) norm_quantised_shifted_kernel(const NormParams p, long long step) {
  constexpr int kTeams = W < 8 ? 8 / W : 1, E = Elem<T>::kVec, kLanes = kGroup / E, kGroups = W * U * 32 / kLanes;
  constexpr uint32_t kAll = (1u << E) - 1u;
  __shared__ float sums[2][kTeams * W];
  // of each group the largest magnitude in the vectors that begin in it, and in the one that begins with the next; where the
  // scale is the row's, the warps' largest.  (Rows use the two sets in turn: nobody writes a row's before all have read the
  // one before the last.)
  __shared__ uint2 magnitudes[kTeams][2 * kGroups];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at = warp % W, team = warp / W, groups = (p.cols + kGroup - 1) / kGroup;
  const long long first = ((long long)(blockIdx.x / 8) * kTeams + team) * 8 + blockIdx.x % 8;
  auto barrier = [&] {
    if constexpr (W > 1) team_barrier(1 + team, W * 32);
    else __syncwarp();
  };
  uint2* tops = magnitudes[team];
  for (int g = at * 32 + lane; g < 2 * kGroups; g += W * 32) tops[g] = make_uint2(0, 0);
  barrier();
  if (first >= p.rows) return;  // (a whole team)
  const int shift = off_boundary(static_cast<const T*>(p.x) + first * p.cols);
  uint32_t own[E];  // what is left of a magnitude in the group that begins with the vector
#pragma unroll
  for (int e = 0; e < E; ++e) own[e] = e < shift ? 0u : 0x7fffffffu;
  auto vector = [&](int u) { return (at + u * W) * 32 + lane; };
  uint32_t lives[U];  // which of a vector's elements are the row's, a bit each
  uint4 w[U], raw[U], more[U];
  const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int col = vector(u) * E - shift, begin = max(0, -col), end = min(E, p.cols - col);
    lives[u] = end <= begin ? 0u : ((1u << end) - 1u) & ~((1u << begin) - 1u);
  }
  auto ask = [&](long long row) {
    const T *x = static_cast<const T*>(p.x) + row * p.cols - shift, *res = static_cast<const T*>(p.res) + row * p.cols - shift;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = lives[u] != 0 ? ldg_stream(x + vector(u) * E) : none;
      if (p.res != nullptr) more[u] = lives[u] != 0 ? ldg_stream(res + vector(u) * E) : none;
    }
  };
  ask(first);
  // w from the row's first element of a vector on: two of its own vectors, or value by value where those are off a boundary
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const T* from = static_cast<const T*>(p.w) + vector(u) * E - shift;
    w[u] = none;
    if (lives[u] == 0) continue;
    if (off_boundary(static_cast<const T*>(p.w)) == 0) {
      const uint4 low = vector(u) > 0 && shift > 0 ? ldg_keep(from + shift - E) : none;
      const uint4 high = vector(u) * E < p.cols ? ldg_keep(from + shift) : none;
      w[u] = kept<E>(shift > 0 ? shift_words<T>(low, high, E - shift) : high, lives[u]);
    } else {
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = lives[u] >> e & 1u ? Elem<T>::to_f(from[e]) : 0.f;
      w[u] = pack<T>(f);
    }
  }
  int n = 0;
  for (long long row = first; row < p.rows; row += step, n ^= 1) {
    uint2* mine = tops + n * kGroups;
    Pairs<T> f[U];
    float2 squares = make_float2(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (a vector's elements of other rows count as zero)
      if (lives[u] != kAll) {
        raw[u] = kept<E>(raw[u], lives[u]);
        if (p.res != nullptr) more[u] = kept<E>(more[u], lives[u]);
      }
      f[u].unpack(raw[u]);
      if (p.res != nullptr) {
        f[u].add(more[u]);
        const uint4 h = f[u].pack();
        f[u].unpack(h);
        if (p.h_out != nullptr && lives[u] != 0) {
          T* dst = static_cast<T*>(p.h_out) + row * p.cols - shift + vector(u) * E;
          if (lives[u] == kAll) {
            *reinterpret_cast<uint4*>(dst) = h;
          } else {
            const uint32_t words[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (lives[u] >> e & 1u) {
                if constexpr (E == 8) reinterpret_cast<unsigned short*>(dst)[e] = (unsigned short)(words[e / 2] >> (e % 2 * 16));
                else reinterpret_cast<uint32_t*>(dst)[e] = words[e];
              }
          }
        }
      }
      squares = f[u].squares(squares);
    }
    if (row + step < p.rows) ask(row + step);
    float sum = warp_reduce<SumOp>(squares.x + squares.y);
    if constexpr (W > 1) {
      if (lane == 0) sums[n][warp] = sum;
      barrier();
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) sum += sums[n][team * W + i];
    }
    const float r = rsqrtf(sum * p.per_col + p.eps);
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      f[u].scale(r, w[u]);
      if (lives[u] != kAll) f[u].keep(lives[u]);  // (r may be infinite)
      if (p.group == 0) {
        top = f[u].largest(top);
        continue;
      }
      uint32_t before = 0, m = 0;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        m = __vimax3_u32(m, f[u].bits(e) & own[e], f[u].bits(e + 1) & own[e + 1]);
        before = __vimax3_u32(before, f[u].bits(e) & (own[e] ^ 0x7fffffffu), f[u].bits(e + 1) & (own[e + 1] ^ 0x7fffffffu));
      }
      const bool border = vector(u) % kLanes == 0;
      m = group_max<kLanes>(border ? m : max(m, before));
      if (border) {
        const int group = vector(u) / kLanes;
        mine[group].x = m;
        if (group > 0) mine[group - 1].y = before;
      }
    }
    if (p.group == 0) {
      top = __reduce_max_sync(kFull, top);
      if (lane == 0) mine[at].x = top;
    }
    barrier();
    if (p.group == 0) {
#pragma unroll
      for (int i = 0; i < W; ++i) top = max(top, mine[i].x);
      if (at == 0 && lane == 0) p.scales[row] = scale_of(top);
    }
    unsigned char* q = p.q + row * p.cols - shift;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = vector(u), group = v / kLanes;
      uint32_t top_low = top;  // of a vector's elements before `shift`
      if (p.group != 0) {
        const uint2 of = mine[group], of_before = mine[v % kLanes == 0 && v > 0 ? group - 1 : group];
        top = max(of.x, of.y);
        top_low = max(of_before.x, of_before.y);
        if (v % kLanes == 0 && group < groups) p.scales[row * groups + group] = scale_of(top);
      }
      if (lives[u] == 0) continue;
      uint32_t of_high = top, of_low = top_low;
      if (extreme(of_high) || extreme(of_low)) {
        const float pre = extreme(of_high) ? tame(of_high) : 1.f, pre_low = extreme(of_low) ? tame(of_low) : 1.f;
#pragma unroll
        for (int e = 0; e < E; e += 2)
          f[u].v[e / 2] = mul2(f[u].v[e / 2], make_float2(own[e] ? pre : pre_low, own[e + 1] ? pre : pre_low));
      }
      const float by = factor_of(of_high), low = factor_of(of_low);
      uint32_t two[E / 2];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 t = mul2(f[u].v[e / 2], make_float2(own[e] ? by : low, own[e + 1] ? by : low));
        two[e / 2] = e4m3x2(t.x, t.y);
      }
      if (lives[u] != kAll) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (lives[u] >> e & 1u) q[v * E + e] = (unsigned char)(two[e / 2] >> (e % 2 * 8));
      } else {
        store_bytes(q + v * E, two);
      }
    }
  }
}

// Rows that no block holds in registers: read three times, a block a row.
template <class T> __global__ void __launch_bounds__(1024) norm_quantised_long_kernel(const NormParams p) {
  __shared__ float sums[32];
  __shared__ uint32_t tops[32];
  const long long base = (long long)blockIdx.x * p.cols;
  const T *x = static_cast<const T*>(p.x) + base, *w = static_cast<const T*>(p.w);
  T* h_out = static_cast<T*>(p.h_out) + base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto value = [&](int c) {
    const float v = Elem<T>::to_f(x[c]);
    return p.res == nullptr ? v : Elem<T>::to_f(Elem<T>::from_f(v + Elem<T>::to_f(static_cast<const T*>(p.res)[base + c])));
  };
  float s = 0.f;
  for (int c = threadIdx.x; c < p.cols; c += 1024) {
    const float v = value(c);
    if (p.h_out != nullptr) h_out[c] = Elem<T>::from_f(v);
    s = fmaf(v, v, s);
  }
  s = warp_reduce<SumOp>(s);
  if (lane == 0) sums[warp] = s;
  __syncthreads();
  s = warp_reduce<SumOp>(sums[lane]);
  const float r = rsqrtf(s * p.per_col + p.eps);
  auto put = [&](int c, float pre, float by) { p.q[base + c] = (unsigned char)e4m3x2(value(c) * r * Elem<T>::to_f(w[c]) * pre * by, 0.f); };
  const int groups = (p.cols + kGroup - 1) / kGroup;
  uint32_t top = 0;
  for (int g = warp; g < groups; g += 32) {
    uint32_t m = 0;
    for (int c = g * kGroup + lane; c < min(p.cols, (g + 1) * kGroup); c += 32) m = max(m, magnitude(value(c) * r * Elem<T>::to_f(w[c])));
    if (p.group == 0) {
      top = max(top, m);
      continue;
    }
    m = __reduce_max_sync(kFull, m);
    if (lane == 0) p.scales[(long long)blockIdx.x * groups + g] = scale_of(m);
    const float pre = extreme(m) ? tame(m) : 1.f, by = factor_of(m);
    for (int c = g * kGroup + lane; c < min(p.cols, (g + 1) * kGroup); c += 32) put(c, pre, by);
  }
  if (p.group != 0) return;
  top = __reduce_max_sync(kFull, top);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  top = __reduce_max_sync(kFull, tops[lane]);
  if (threadIdx.x == 0) p.scales[blockIdx.x] = scale_of(top);
  const float pre = extreme(top) ? tame(top) : 1.f, by = factor_of(top);
  for (int c = threadIdx.x; c < p.cols; c += 1024) put(c, pre, by);
}

template <class T> int run_long(const NormParams& p, cudaStream_t stream) {
  norm_quantised_long_kernel<T><<<(unsigned)p.rows, 1024, 0, stream>>>(p);
  return ixb_host::cuda_status(cudaGetLastError());
}

template <class T, int W, int U> int launch_vectors(const NormParams& p, cudaStream_t stream) {
  constexpr int kRows = W < 8 ? 8 / W : 1;
  norm_quantised_kernel<T, W, U><<<(unsigned)((p.rows + kRows - 1) / kRows), W < 8 ? 256 : W * 32, 0, stream>>>(p);
  return ixb_host::cuda_status(cudaGetLastError());
}

template <class T, int W, int U> int launch_shifted(const NormParams& p, int sms, cudaStream_t stream) {
  constexpr int kTeams = W < 8 ? 8 / W : 1, kThreads = W < 8 ? 256 : W * 32;
  auto kern = norm_quantised_shifted_kernel<T, W, U>;
  static std::atomic<int> known[64];  // blocks an SM holds
  int devid = 0;
  cudaGetDevice(&devid);
  int blocks = known[devid & 63].load(std::memory_order_relaxed);
  if (blocks == 0) {
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kern, kThreads, 0);
    if (e != cudaSuccess || blocks < 1) return e != cudaSuccess ? ixb_host::cuda_status(e) : IXB_ERR_UNSUPPORTED;
    known[devid & 63].store(blocks, std::memory_order_relaxed);
  }
  const long long need = (p.rows + 8 * kTeams - 1) / (8 * kTeams) * 8, most = (long long)sms * blocks / 8 * 8, grid = need < most ? need : most;
  kern<<<(unsigned)grid, kThreads, 0, stream>>>(p, grid * kTeams);
  return ixb_host::cuda_status(cudaGetLastError());
}

template <class T> int run(const NormParams& p, cudaStream_t stream) {
  const ixb_devinfo* dev = ixb_host::current_device();
  if (dev == nullptr) return IXB_ERR_CUDA;
  using ixb_host::aligned16;
  const int kVec = Elem<T>::kVec;
  const bool vectors = p.cols % kVec == 0 && aligned16(p.x) && aligned16(p.res) && aligned16(p.w) && aligned16(p.h_out) &&
                       (reinterpret_cast<uintptr_t>(p.q) & (kVec - 1)) == 0;
  const uintptr_t off = reinterpret_cast<uintptr_t>(p.x) & 15u;
  auto alike = [off](const void* t) { return t == nullptr || (reinterpret_cast<uintptr_t>(t) & 15u) == off; };
  if (!vectors && !(alike(p.res) && alike(p.h_out) && (reinterpret_cast<uintptr_t>(p.q) & (kVec - 1)) == off / sizeof(T)))
    return run_long<T>(p, stream);
  // Two units of 32 vectors a warp: 16384 x 4096 bf16 with residual 79 us so, 101 with four (half the warps, more registers
  // each), 116 with one; 2048 x 2048 6.6 with two, 7.8 with one.  More only where 32 warps have to hold the row.
  const int touched = vectors ? p.cols / kVec : (p.cols + kVec - 2) / kVec + 1, units = (touched + 31) / 32;
  int warps = 1, each = 1;
  while (warps < 32 && warps * 2 < units) warps *= 2;
  while (warps * each < units) each *= 2;
#define IXB_NORM_CASE(W, U)    \
  if (warps == W && each == U) \
    return vectors ? launch_vectors<T, W, U>(p, stream) : launch_shifted<T, W, U>(p, dev->sm_count, stream);
  IXB_NORM_CASE(1, 1)
  IXB_NORM_CASE(1, 2)
  IXB_NORM_CASE(2, 2)
  IXB_NORM_CASE(4, 2)
  IXB_NORM_CASE(8, 2)
  IXB_NORM_CASE(16, 2)
  IXB_NORM_CASE(32, 2)
  IXB_NORM_CASE(32, 4)
  if constexpr (Elem<T>::kVec == 4) {
    IXB_NORM_CASE(32, 8)
  }
#undef IXB_NORM_CASE
  return run_long<T>(p, stream);
}

}  // namespace

extern "C" int ixb_rmsnorm_quantised(int dtype, const void* x, const void* res, const void* w, void* q, float* scales,
                                     void* h_out, int64_t rows, int64_t cols, int32_t group, float eps, ixb_stream stream) {
  if (rows < 0 || cols <= 0 || (group != 0 && group != kGroup)) return IXB_ERR_ARG;
  if (rows == 0) return IXB_OK;
  if (rows > 0x7fffffffLL || cols > (1 << 20)) return IXB_ERR_SHAPE;
  if (!x || !w || !q || !scales || (res == nullptr && h_out != nullptr)) return IXB_ERR_ARG;
  const NormParams p{x, res, w, static_cast<unsigned char*>(q), scales, h_out, rows, (int)cols, group, (float)(1.0 / (double)cols), eps};
  const cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case IXB_BF16: return run<bf16>(p, s);
    case IXB_F16: return run<f16>(p, s);
    case IXB_F32: return run<float>(p, s);
    default: return IXB_ERR_DTYPE;
  }
}
