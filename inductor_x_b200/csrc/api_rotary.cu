// Rotary positions with several axes: pair i of a head is turned by the angle position[axis(i)] * frequency(i).
// Sines and cosines are formed once a token, for all heads of q and k; a thread keeps those of its pairs while it walks the
// heads, and asks for its first values before it forms them.
// Bound: memory, every value read and written once.
#include <cmath>
#include "host.h"
#include "ixb/common.cuh"

namespace {

using namespace ixb;
constexpr int kMaxPairs = 128;
constexpr int kMaxTurns = 2048;  // a block's, 16 KB

struct Operand {
  const void* in;
  void* out;
  long long in_sb, in_sh, in_ss, out_sb, out_sh, out_ss;  // elements
  int heads;
};
struct RotaryParams {
  Operand x[2];
  const void* positions;
  long long pos_sa, pos_sb, pos_ss;
  int wide;        // positions of 64 bits
  int B, S, D, pairs, neighbours, inverse;
  unsigned long long turns[kMaxPairs];  // 2^-64 of a turn a position
  unsigned char axis[kMaxPairs];
};

// The turn of pair i for token (b, s).  The product of a position and a frequency in 2^-64 of a turn wraps around at whole turns
// by itself, so that a far position keeps its fraction of one; its upper half is that fraction to 2^-32.
// The parameters are read by their generic address: lanes that read different ones as constants take turns.
__device__ __forceinline__ float2 turn_of(const RotaryParams& p, int i, int b, int s) {
  unsigned long long turns;
  unsigned axis;
  asm("ld.u64 %0, [%1];" : "=l"(turns) : "l"(&p.turns[i]));
  asm("ld.u8 %0, [%1];" : "=r"(axis) : "l"(&p.axis[i]));
  const long long at = axis * p.pos_sa + b * p.pos_sb + s * p.pos_ss;
  const long long pos = p.wide ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
  const int fraction = (int)(((unsigned long long)pos * turns) >> 32);  // in [-1/2, 1/2) of a turn
  float sn, c;
  sincospif((float)fraction * 0x1p-31f, &sn, &c);
  return make_float2(c, p.inverse ? -sn : sn);
}

// The pairs of two vectors: (low[e], high[e]), or the neighbours of low and then of high.
template <class T, bool NEIGHBOURS, int N> __device__ __forceinline__ void turn_pairs(uint4& low, uint4& high, const float2 (&turn)[N]) {
  float f[N], g[N];
  unpack<T>(low, f);
  unpack<T>(high, g);
  if constexpr (NEIGHBOURS) {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      const float a = f[2 * e], c = f[2 * e + 1], d = g[2 * e], h = g[2 * e + 1];
      f[2 * e] = a * turn[e].x - c * turn[e].y;
      f[2 * e + 1] = a * turn[e].y + c * turn[e].x;
      g[2 * e] = d * turn[N / 2 + e].x - h * turn[N / 2 + e].y;
      g[2 * e + 1] = d * turn[N / 2 + e].y + h * turn[N / 2 + e].x;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float a = f[e], c = g[e];
      f[e] = a * turn[e].x - c * turn[e].y;
      g[e] = a * turn[e].y + c * turn[e].x;
    }
  }
  low = pack<T>(f);
  high = pack<T>(g);
}

// Vectors: a part is kVec pairs of a head, two vectors of it, or one of the vectors behind the pairs.  A block takes `tokens`
// tokens at a time and all heads of them, q's and then k's; a thread is a part of a token and walks heads `slots`
// apart, kAhead of them in flight.
// 2 x 8192 tokens of 32 + 8 heads, there and back: 128 threads and 5 heads in flight 109 us (94 % of a copy's rate), the same on
// 256 threads 124, 4 heads in flight on those 128, 3 or 2 190; blocks that go on to further tokens 120 - 142, with the next
// heads asked for as each is done 143 - 173 (loads and stores in turn cost more than waiting).
constexpr int kAhead = 5, kThreads = 128;
template <class T, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads, 5) rotary_vector_kernel(const __grid_constant__ RotaryParams p, int parts, int tokens, int slots, int heads_first) {
  constexpr int kVec = Elem<T>::kVec;
  extern __shared__ float2 cs[];  // [tokens][pairs]
  const int part = threadIdx.x % parts, place = threadIdx.x / parts;
  const int token = heads_first ? place / slots : place % tokens, slot = heads_first ? place % slots : place / tokens;
  const int all = p.B * p.S, heads = p.x[0].heads + p.x[1].heads, turned = p.pairs / kVec;
  const bool copies = part >= turned;
  const int lo = copies ? 2 * p.pairs + (part - turned) * kVec : NEIGHBOURS ? 2 * kVec * part : kVec * part;
  const int hi = copies ? lo : NEIGHBOURS ? lo + kVec : lo + p.pairs;
  const int first = blockIdx.x * tokens;
  const bool live = place < slots * tokens && first + token < all;
  const int b = (first + token) / p.S, s = (first + token) - b * p.S;
  const T* in[2];
  T* out[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    in[w] = static_cast<const T*>(p.x[w].in) + b * p.x[w].in_sb + s * p.x[w].in_ss;
    out[w] = static_cast<T*>(p.x[w].out) + b * p.x[w].out_sb + s * p.x[w].out_ss;
  }
  uint4 va[kAhead], vb[kAhead];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + i * slots;
      if (!live || h >= heads) continue;
      const T* from = h < p.x[0].heads ? in[0] + h * p.x[0].in_sh : in[1] + (h - p.x[0].heads) * p.x[1].in_sh;
      va[i] = ldg_stream(from + lo);
      if (!copies) vb[i] = ldg_stream(from + hi);
    }
  };
  fetch(slot);
  const int b0 = first / p.S, s0 = first - b0 * p.S;
  const unsigned per_pair = (1u << 20) / p.pairs + 1;  // (u / pairs is exact so below kMaxTurns)
  for (int u = threadIdx.x; u < tokens * p.pairs; u += kThreads) {
    const int k = (int)((u * per_pair) >> 20);
    int tb = b0, ts = s0 + k;
    while (ts >= p.S) {
      ts -= p.S;
      ++tb;
    }
    if (first + k < all) cs[u] = turn_of(p, u - k * p.pairs, tb, ts);
  }
  __syncthreads();
  if (!live) return;
  float2 turn[kVec];
  if (!copies) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) turn[e] = cs[token * p.pairs + part * kVec + e];
  }
  for (int h0 = slot; h0 < heads; h0 += kAhead * slots) {
    if (h0 > slot) fetch(h0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + i * slots;
      if (h >= heads) break;
      T* to = h < p.x[0].heads ? out[0] + h * p.x[0].out_sh : out[1] + (h - p.x[0].heads) * p.x[1].out_sh;
      uint4 low = va[i], high = vb[i];
      if (!copies) {
        turn_pairs<T, NEIGHBOURS>(low, high, turn);
        *reinterpret_cast<uint4*>(to + hi) = high;
      }
      *reinterpret_cast<uint4*>(to + lo) = low;
    }
  }
}

// Heads that are no whole vectors, or off a boundary: a block a token, pair by pair.  3 x 1369 tokens of 16 + 16 heads of 72 (36
// pairs), fp16: 19.5 us, 1.94 TB/s (heads of 80 by vectors 11.4).
template <class T> __global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float2 cs[kMaxPairs];
  const int b = blockIdx.x / p.S, s = blockIdx.x % p.S;
  for (int i = threadIdx.x; i < p.pairs; i += blockDim.x) cs[i] = turn_of(p, i, b, s);
  __syncthreads();
  for (int which = 0; which < 2; ++which) {
    const Operand& x = p.x[which];
    const T* in = static_cast<const T*>(x.in) + b * x.in_sb + s * x.in_ss;
    T* out = static_cast<T*>(x.out) + b * x.out_sb + s * x.out_ss;
    for (int u = threadIdx.x; u < x.heads * p.pairs; u += blockDim.x) {
      const int h = u / p.pairs, i = u % p.pairs, lo = p.neighbours ? 2 * i : i, hi = p.neighbours ? 2 * i + 1 : i + p.pairs;
      const float a = Elem<T>::to_f(in[h * x.in_sh + lo]), c = Elem<T>::to_f(in[h * x.in_sh + hi]);
      out[h * x.out_sh + lo] = Elem<T>::from_f(a * cs[i].x - c * cs[i].y);
      out[h * x.out_sh + hi] = Elem<T>::from_f(a * cs[i].y + c * cs[i].x);
    }
    const int rest = p.D - 2 * p.pairs;
    for (int u = threadIdx.x; u < x.heads * rest; u += blockDim.x) {
      const int h = u / rest, e = 2 * p.pairs + u % rest;
      out[h * x.out_sh + e] = in[h * x.in_sh + e];
    }
  }
}

template <class T> int run(const RotaryParams& p, cudaStream_t stream) {
  constexpr int kVec = Elem<T>::kVec;
  const int parts = p.pairs / kVec + (p.D - 2 * p.pairs) / kVec;
  bool vectors = p.pairs % kVec == 0 && p.D % kVec == 0 && parts <= 32;
  for (const Operand& x : p.x)
    vectors = vectors && (x.heads == 0 || (ixb_host::aligned16(x.in) && ixb_host::aligned16(x.out) &&
                                           ((x.in_sb | x.in_sh | x.in_ss | x.out_sb | x.out_sh | x.out_ss) & (kVec - 1)) == 0));
  const long long all = (long long)p.B * p.S;
  if (!vectors) {
    rotary_kernel<T><<<(unsigned)all, 256, 0, stream>>>(p);
    return ixb_host::cuda_status(cudaGetLastError());
  }
  const ixb_devinfo* dev = ixb_host::current_device();
  if (dev == nullptr) return IXB_ERR_CUDA;
  const int heads = p.x[0].heads + p.x[1].heads;
  // neighbouring threads take neighbouring memory: the heads of a token where they follow one another, else tokens of a head
  const Operand& x = p.x[p.x[0].heads > 0 ? 0 : 1];
  const int heads_first = x.in_sh <= x.in_ss || p.S == 1, places = kThreads / parts;
  // about kAhead heads a thread, fewer where that leaves SMs without a block (heads that do not follow one another, 32 + 8 of
  // 16384 tokens: 125 us, with at least 4 tokens a block 132, 8 140, 16 167)
  int tokens = places * kAhead / heads;
  if (tokens * p.pairs > kMaxTurns) tokens = kMaxTurns / p.pairs;
  while (tokens > 1 && (all + tokens - 1) / tokens < 2 * dev->sm_count) tokens /= 2;
  if (tokens < 1) tokens = 1;
  if (tokens > places) tokens = places;
  const int slots = places / tokens < heads ? places / tokens : heads;
  auto kern = p.neighbours ? rotary_vector_kernel<T, true> : rotary_vector_kernel<T, false>;
  kern<<<(unsigned)((all + tokens - 1) / tokens), kThreads, tokens * p.pairs * sizeof(float2), stream>>>(p, parts, tokens, slots, heads_first);
  return ixb_host::cuda_status(cudaGetLastError());
}

}  // namespace

extern "C" int ixb_axial_rotary(int dtype, const void* q, void* q_out, const int64_t* q_strides, const int64_t* q_out_strides,
                                int32_t heads, const void* k, void* k_out, const int64_t* k_strides,
                                const int64_t* k_out_strides, int32_t k_heads, const void* positions, int position_dtype,
                                const int64_t* position_strides, int32_t B, int32_t S, int32_t D, int32_t axes,
                                const int32_t* sections, const double* frequencies, int neighbours, int inverse,
                                ixb_stream stream) {
  if (B < 0 || S < 0 || heads < 0 || k_heads < 0 || D < 0 || axes < 1 || sections == nullptr || frequencies == nullptr) return IXB_ERR_ARG;
  if (dtype != IXB_BF16 && dtype != IXB_F16 && dtype != IXB_F32) return IXB_ERR_DTYPE;
  if (position_dtype != IXB_I32 && position_dtype != IXB_I64) return IXB_ERR_DTYPE;
  RotaryParams p = {};
  for (int a = 0; a < axes; ++a) {
    if (sections[a] < 0) return IXB_ERR_ARG;
    if (axes > kMaxPairs || sections[a] > kMaxPairs - p.pairs) return IXB_ERR_SHAPE;
    for (int j = 0; j < sections[a]; ++j, ++p.pairs) {
      if (!std::isfinite(frequencies[p.pairs])) return IXB_ERR_ARG;
      const long double turns = std::fabs(frequencies[p.pairs]) / 6.283185307179586476925286766559L;
      const unsigned long long part = (unsigned long long)std::ldexp(turns - std::floor(turns), 64);
      p.turns[p.pairs] = frequencies[p.pairs] < 0 ? 0 - part : part;
      p.axis[p.pairs] = (unsigned char)a;
    }
  }
  if (2 * p.pairs > D) return IXB_ERR_SHAPE;
  if (B == 0 || S == 0 || D == 0 || heads + (long long)k_heads == 0) return IXB_OK;
  // (the kernels count a token's values, and the tokens, in 32 bits)
  if ((long long)B * S > (1 << 30) || (heads + (long long)k_heads) * D > (1 << 30)) return IXB_ERR_SHAPE;
  if ((heads && (!q || !q_out || !q_strides || !q_out_strides)) || (k_heads && (!k || !k_out || !k_strides || !k_out_strides)) ||
      !positions || !position_strides)
    return IXB_ERR_ARG;
  static const int64_t none[3] = {0, 0, 0};
  if (!heads) q_strides = q_out_strides = none;
  if (!k_heads) k_strides = k_out_strides = none;
  p.x[0] = Operand{q, q_out, q_strides[0], q_strides[1], q_strides[2], q_out_strides[0], q_out_strides[1], q_out_strides[2], heads};
  p.x[1] = Operand{k, k_out, k_strides[0], k_strides[1], k_strides[2], k_out_strides[0], k_out_strides[1], k_out_strides[2], k_heads};
  p.positions = positions;
  p.pos_sa = position_strides[0], p.pos_sb = position_strides[1], p.pos_ss = position_strides[2];
  p.wide = position_dtype == IXB_I64;
  p.B = B, p.S = S, p.D = D, p.neighbours = neighbours != 0, p.inverse = inverse != 0;
  if (dtype == IXB_BF16) return run<bf16>(p, (cudaStream_t)stream);
  if (dtype == IXB_F16) return run<f16>(p, (cudaStream_t)stream);
  return run<float>(p, (cudaStream_t)stream);
}
