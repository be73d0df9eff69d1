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
  double turns[kMaxPairs];          // whole turns a position
  unsigned char axis[kMaxPairs];
};

// The turn of pair i for token (b, s): in whole turns and 64 bits until the fraction is known - 32 bits hold nothing of a far
// position's.
__device__ __forceinline__ float2 turn_of(const RotaryParams& p, int i, int b, int s) {
  const long long at = p.axis[i] * p.pos_sa + b * p.pos_sb + s * p.pos_ss;
  const double pos = p.wide ? (double)static_cast<const long long*>(p.positions)[at] : (double)static_cast<const int*>(p.positions)[at];
  const double t = pos * p.turns[i];
  float sn, c;
  sincospif(2.f * (float)(t - rint(t)), &sn, &c);
  return make_float2(c, p.inverse ? -sn : sn);
}

// Vectors: a part is kVec pairs of a head, two vectors of it, or one of the vectors behind the pairs.  A block takes `tokens`
// tokens and all heads; a thread is a part of a token and walks heads, `threads / (parts * tokens)` apart.
template <class T> __global__ void __launch_bounds__(256) rotary_vector_kernel(const __grid_constant__ RotaryParams p, int parts, int tokens, int slots,
                                                                                int heads_first) {
  constexpr int kVec = Elem<T>::kVec;
  extern __shared__ float2 cs[];  // [tokens][pairs]
  const int part = threadIdx.x % parts, place = threadIdx.x / parts;
  const int token = heads_first ? place / slots : place % tokens, slot = heads_first ? place % slots : place / tokens;
  const long long first = (long long)blockIdx.x * tokens, all = (long long)p.B * p.S;
  const bool live = place < slots * tokens && first + token < all;
  const int b = (int)((first + token) / p.S), s = (int)((first + token) % p.S);
  const int turned = p.pairs / kVec;
  const bool copies = part >= turned;
  const int lo = copies ? 2 * p.pairs + (part - turned) * kVec : p.neighbours ? 2 * kVec * part : kVec * part;
  const int hi = copies ? lo : p.neighbours ? lo + kVec : lo + p.pairs;
  uint4 va, vb;
  auto fetch = [&](int which, int h) {
    const Operand& x = p.x[which];
    const T* in = static_cast<const T*>(x.in) + b * x.in_sb + s * x.in_ss + h * x.in_sh;
    va = ldg_stream(in + lo);
    if (!copies) vb = ldg_stream(in + hi);
  };
  int which = p.x[0].heads > slot ? 0 : 1, h = slot;
  bool more = live && h < p.x[which].heads;
  if (more) fetch(which, h);
  for (int u = threadIdx.x; u < tokens * p.pairs; u += blockDim.x) {
    const int k = u / p.pairs;
    if (first + k < all) cs[u] = turn_of(p, u - k * p.pairs, (int)((first + k) / p.S), (int)((first + k) % p.S));
  }
  __syncthreads();
  float2 turn[kVec];
  if (live && !copies) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) turn[e] = cs[token * p.pairs + part * kVec + e];
  }
  while (more) {
    const Operand& x = p.x[which];
    T* out = static_cast<T*>(x.out) + b * x.out_sb + s * x.out_ss + h * x.out_sh;
    const uint4 a = va, c = vb;
    h += slots;
    if (which == 0 && h >= p.x[0].heads) {
      which = 1;
      h = slot;
    }
    more = h < p.x[which].heads;
    if (more) fetch(which, h);
    if (copies) {
      *reinterpret_cast<uint4*>(out + lo) = a;
      continue;
    }
    float f[2 * kVec], g[2 * kVec];
    unpack<T>(a, f);
    unpack<T>(c, f + kVec);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const int i = p.neighbours ? 2 * e : e, j = p.neighbours ? 2 * e + 1 : e + kVec;
      g[i] = f[i] * turn[e].x - f[j] * turn[e].y;
      g[j] = f[i] * turn[e].y + f[j] * turn[e].x;
    }
    *reinterpret_cast<uint4*>(out + lo) = pack<T>(g);
    *reinterpret_cast<uint4*>(out + hi) = pack<T>(g + kVec);
  }
}

// Heads that are no whole vectors, or off a boundary: a block a token, pair by pair.
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
  bool vectors = p.pairs % kVec == 0 && p.D % kVec == 0;
  for (const Operand& x : p.x)
    vectors = vectors && (x.heads == 0 || (ixb_host::aligned16(x.in) && ixb_host::aligned16(x.out) &&
                                           ((x.in_sb | x.in_sh | x.in_ss | x.out_sb | x.out_sh | x.out_ss) & (kVec - 1)) == 0));
  const long long all = (long long)p.B * p.S;
  if (!vectors) {
    rotary_kernel<T><<<(unsigned)all, 256, 0, stream>>>(p);
    return ixb_host::cuda_status(cudaGetLastError());
  }
  const int parts = p.pairs / kVec + (p.D - 2 * p.pairs) / kVec;
  const int heads = p.x[0].heads > p.x[1].heads ? p.x[0].heads : p.x[1].heads;
  // neighbouring threads take neighbouring memory: the heads of a token where they follow one another, else tokens of a head
  const Operand& x = p.x[p.x[0].heads > 0 ? 0 : 1];
  const int heads_first = x.in_sh <= x.in_ss || p.S == 1;
  const int places = 256 / parts;
  int slots = heads_first ? (heads < places ? heads : places) : 1, tokens = places / slots;
  if (!heads_first) {
    if (tokens > 16) tokens = 16;
    slots = places / tokens < heads ? places / tokens : heads;
  }
  if (tokens > 16) tokens = 16;
  rotary_vector_kernel<T><<<(unsigned)((all + tokens - 1) / tokens), 256, tokens * p.pairs * sizeof(float2), stream>>>(p, parts, tokens, slots,
                                                                                                                   heads_first);
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
      p.turns[p.pairs] = frequencies[p.pairs] * 0.15915494309189533577;  // 1 / (2 pi)
      p.axis[p.pairs] = (unsigned char)a;
    }
  }
  if (2 * p.pairs > D) return IXB_ERR_SHAPE;
  if (B == 0 || S == 0 || D == 0 || heads + (long long)k_heads == 0) return IXB_OK;
  if ((long long)B * S > 0x7fffffffLL) return IXB_ERR_SHAPE;
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
