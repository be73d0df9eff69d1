// Root-mean-square norm with the residual's addition and an 8-bit output:
//   h = x (+ residual), rounded to the storage type; y = h * rsqrt(mean(h^2) + eps) * w in 32 bits;
//   scale = max |y| / 448 over the row or over each 128 values of it; q = e4m3(y / scale).
#include <cuda_fp8.h>
#include <cmath>
#include "host.h"
#include "ixb/common.cuh"

namespace {

using namespace ixb;
constexpr int kGroup = 128;
constexpr float kLargest = 448.f;

// a block a row
template <class T>
__global__ void norm_quantised_kernel(const T* x, const T* res, const T* w, unsigned char* q, float* scales, T* h_out, int cols,
                                      int group, float eps) {
  __shared__ float part[8];
  const long long row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto value = [&](int c) {
    float v = Elem<T>::to_f(x[row * cols + c]);
    if (res != nullptr) v = Elem<T>::to_f(Elem<T>::from_f(v + Elem<T>::to_f(res[row * cols + c])));
    return v;
  };
  auto fold = [&](float v, bool max) {
    v = max ? warp_reduce<MaxOp>(v) : warp_reduce<SumOp>(v);
    __syncthreads();
    if (lane == 0) part[warp] = v;
    __syncthreads();
    float t = part[0];
    for (int i = 1; i < 8; ++i) t = max ? MaxOp::combine(t, part[i]) : t + part[i];
    return t;
  };
  float s = 0.f;
  for (int c = threadIdx.x; c < cols; c += 256) {
    const float v = value(c);
    if (h_out != nullptr) h_out[row * cols + c] = Elem<T>::from_f(v);
    s = fmaf(v, v, s);
  }
  const float r = rsqrtf(fold(s, false) / cols + eps);
  auto normed = [&](int c) { return value(c) * r * Elem<T>::to_f(w[c]); };
  auto put = [&](int c, float y, float scale) {
    const float t = y / (scale > 0.f || scale != scale ? scale : 1.f);
    q[row * cols + c] = (unsigned char)__nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
  };
  if (group == 0) {
    float top = 0.f;
    for (int c = threadIdx.x; c < cols; c += 256) top = MaxOp::combine(top, fabsf(normed(c)));
    const float scale = fold(top, true) / kLargest;
    if (threadIdx.x == 0) scales[row] = scale;
    for (int c = threadIdx.x; c < cols; c += 256) put(c, normed(c), scale);
  } else {
    const int groups = (cols + kGroup - 1) / kGroup;
    for (int g = warp; g < groups; g += 8) {
      float top = 0.f;
      for (int c = g * kGroup + lane; c < min(cols, (g + 1) * kGroup); c += 32) top = MaxOp::combine(top, fabsf(normed(c)));
      const float scale = warp_reduce<MaxOp>(top) / kLargest;
      if (lane == 0) scales[row * groups + g] = scale;
      for (int c = g * kGroup + lane; c < min(cols, (g + 1) * kGroup); c += 32) put(c, normed(c), scale);
    }
  }
}

template <class T>
int run(const void* x, const void* res, const void* w, void* q, float* scales, void* h_out, int64_t rows, int64_t cols,
        int group, float eps, cudaStream_t stream) {
  norm_quantised_kernel<T><<<(unsigned)rows, 256, 0, stream>>>((const T*)x, (const T*)res, (const T*)w, (unsigned char*)q,
                                                               scales, (T*)h_out, (int)cols, group, eps);
  return ixb_host::cuda_status(cudaGetLastError());
}

}  // namespace

extern "C" int ixb_rmsnorm_quantised(int dtype, const void* x, const void* res, const void* w, void* q, float* scales,
                                     void* h_out, int64_t rows, int64_t cols, int32_t group, float eps, ixb_stream stream) {
  if (rows < 0 || cols <= 0 || (group != 0 && group != kGroup)) return IXB_ERR_ARG;
  if (rows == 0) return IXB_OK;
  if (rows > 0x7fffffffLL || cols > (1 << 20)) return IXB_ERR_SHAPE;
  if (!x || !w || !q || !scales || (res == nullptr && h_out != nullptr)) return IXB_ERR_ARG;
  const cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case IXB_BF16: return run<bf16>(x, res, w, q, scales, h_out, rows, cols, group, eps, s);
    case IXB_F16: return run<f16>(x, res, w, q, scales, h_out, rows, cols, group, eps, s);
    case IXB_F32: return run<float>(x, res, w, q, scales, h_out, rows, cols, group, eps, s);
    default: return IXB_ERR_DTYPE;
  }
}
