// Rotary positions with several axes: pair i of a head is turned by the angle position[axis(i)] * frequency(i).
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

// a block a token
template <class T> __global__ void rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float2 cs[kMaxPairs];
  const int b = blockIdx.x / p.S, s = blockIdx.x % p.S;
  for (int i = threadIdx.x; i < p.pairs; i += blockDim.x) {
    const long long at = p.axis[i] * p.pos_sa + b * p.pos_sb + s * p.pos_ss;
    const double pos = p.wide ? (double)static_cast<const long long*>(p.positions)[at] : (double)static_cast<const int*>(p.positions)[at];
    // in whole turns and 64 bits until the fraction is known: 32 bits hold nothing of a far position's
    const double t = pos * p.turns[i];
    float sn, c;
    sincospif(2.f * (float)(t - rint(t)), &sn, &c);
    cs[i] = make_float2(c, p.inverse ? -sn : sn);
  }
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
  const unsigned grid = (unsigned)((long long)B * S);
  if (dtype == IXB_BF16) rotary_kernel<bf16><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  else if (dtype == IXB_F16) rotary_kernel<f16><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  else rotary_kernel<float><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  return ixb_host::cuda_status(cudaGetLastError());
}
