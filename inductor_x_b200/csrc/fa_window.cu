// Attention with a sliding window and first tokens that stay visible, forward and backward:
//   query i of sequence b stands at position p = kv_length[b] - q_length[b] + i and sees key j when
//   j <= p and (j > p - window or j < sinks), j < kv_length[b], i < q_length[b];
//   out = softmax(scale q k^T) v over what it sees, lse its log-sum-exp (no key: 0 and -inf).
// H query heads share HK key heads, H / HK neighbours each.
#include <cmath>
#include "fa_window.h"
#include "ixb/tcgen05.cuh"

namespace {

using namespace ixb;
constexpr int HD = 128;

struct View {
  const void* ptr;
  long long sb, sh, ss;  // strides in elements
};
struct WinParams {
  View q, k, v, o, dout, dq, dk, dv;
  const float* lse_in;
  float* lse;
  const int *q_lengths, *kv_lengths;  // [B], may be null
  int B, H, HK, Sq, Sk;
  float scale;
  int window, sinks;
};

template <class T> __device__ __forceinline__ float4 row4(const View& t, int b, int h, long long s, int lane) {
  const T* at = static_cast<const T*>(t.ptr) + b * t.sb + h * t.sh + s * t.ss + lane * 4;
  return make_float4(Elem<T>::to_f(at[0]), Elem<T>::to_f(at[1]), Elem<T>::to_f(at[2]), Elem<T>::to_f(at[3]));
}
template <class T> __device__ __forceinline__ void put4(const View& t, int b, int h, long long s, int lane, float4 x) {
  T* at = const_cast<T*>(static_cast<const T*>(t.ptr)) + b * t.sb + h * t.sh + s * t.ss + lane * 4;
  at[0] = Elem<T>::from_f(x.x);
  at[1] = Elem<T>::from_f(x.y);
  at[2] = Elem<T>::from_f(x.z);
  at[3] = Elem<T>::from_f(x.w);
}
__device__ __forceinline__ float dot(float4 a, float4 b) {
  return warp_reduce<SumOp>(fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, a.w * b.w))));
}
__device__ __forceinline__ float4 axpy(float a, float4 x, float4 y) {
  return make_float4(fmaf(a, x.x, y.x), fmaf(a, x.y, y.y), fmaf(a, x.z, y.z), fmaf(a, x.w, y.w));
}

struct Lengths {
  int q, kv;
};
__device__ __forceinline__ Lengths lengths_of(const WinParams& p, int b) {
  Lengths n;
  n.q = p.q_lengths ? min(max(p.q_lengths[b], 0), p.Sq) : p.Sq;
  n.kv = p.kv_lengths ? min(max(p.kv_lengths[b], 0), p.Sk) : p.Sk;
  return n;
}

// a warp a query row: dq
template <class T> __global__ void window_dq_kernel(const WinParams p, float* delta) {
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= (long long)p.B * p.H * p.Sq) return;
  const int b = (int)(row / ((long long)p.H * p.Sq)), h = (int)(row / p.Sq % p.H), i = (int)(row % p.Sq);
  const Lengths n = lengths_of(p, b);
  const int at = n.kv - n.q + i;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < n.q && at >= 0) {
    const float4 q = row4<T>(p.q, b, h, i, lane), go = row4<T>(p.dout, b, h, i, lane);
    const float dl = dot(go, row4<T>(p.o, b, h, i, lane)), lse = p.lse_in[row];
    if (lane == 0) delta[row] = dl;
    const int hk = h / (p.H / p.HK), low = max(0, at - p.window + 1);
    for (int j = 0; j <= at; ++j) {
      if (j < low && j >= p.sinks) j = low;
      const float4 k = row4<T>(p.k, b, hk, j, lane);
      const float pr = expf(dot(q, k) * p.scale - lse);
      acc = axpy(pr * (dot(go, row4<T>(p.v, b, hk, j, lane)) - dl) * p.scale, k, acc);
    }
  }
  put4<T>(p.dq, b, h, i, lane, acc);
}

// a warp a key row: dk and dv, the query heads that share it in turn
template <class T> __global__ void window_dkv_kernel(const WinParams p, const float* delta) {
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= (long long)p.B * p.HK * p.Sk) return;
  const int b = (int)(row / ((long long)p.HK * p.Sk)), hk = (int)(row / p.Sk % p.HK), j = (int)(row % p.Sk);
  const Lengths n = lengths_of(p, b);
  float4 dk = make_float4(0.f, 0.f, 0.f, 0.f), dv = dk;
  if (j < n.kv) {
    const float4 k = row4<T>(p.k, b, hk, j, lane), v = row4<T>(p.v, b, hk, j, lane);
    const int share = p.H / p.HK;
    const int first = max(0, j - (n.kv - n.q));
    const long long last = j < p.sinks ? n.q : min((long long)n.q, (long long)j + p.window - (n.kv - n.q));
    for (int h = hk * share; h < (hk + 1) * share; ++h)
      for (int i = first; i < last; ++i) {
        const long long at = ((long long)b * p.H + h) * p.Sq + i;
        const float4 q = row4<T>(p.q, b, h, i, lane), go = row4<T>(p.dout, b, h, i, lane);
        const float pr = expf(dot(q, k) * p.scale - p.lse_in[at]);
        dv = axpy(pr, go, dv);
        dk = axpy(pr * (dot(go, v) - delta[at]) * p.scale, q, dk);
      }
  }
  put4<T>(p.dk, b, hk, j, lane, dk);
  put4<T>(p.dv, b, hk, j, lane, dv);
}

View view_of(const void* ptr, const int64_t* strides) { return View{ptr, strides[0], strides[1], strides[2]}; }

}  // namespace

extern "C" size_t ixb_window_attention_scratch_bytes(int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

extern "C" int ixb_window_attention(int dtype, const void* q, const void* k, const void* v, void* o, float* lse, void*,
                                    size_t, int32_t B, int32_t H, int32_t HK, int32_t Sq, int32_t Sk, int32_t D,
                                    const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                    const int64_t* o_strides, const int32_t* q_lengths, const int32_t* kv_lengths, float scale,
                                    int32_t window, int32_t sinks, int32_t* status, ixb_stream stream) {
  if (int st = ixb_host::check_window_sizes(dtype, B, H, HK, Sq, Sk, D, scale, window, sinks)) return st;
  if (B == 0 || H == 0 || Sq == 0) return IXB_OK;
  if (Sk == 0) return IXB_ERR_SHAPE;
  const ixb_host::WindowView views[] = {{q, q_strides}, {k, k_strides}, {v, v_strides}, {o, o_strides}};
  if (int st = ixb_host::check_window_views(views, 4)) return st;
  const ixb_host::WindowShape a{dtype == IXB_BF16, B, H, HK, Sq, Sk, q_lengths, kv_lengths, scale, window < Sk ? window : Sk, sinks};
  return ixb_host::window_prefill(a, views[0], views[1], views[2], views[3], lse, status, (cudaStream_t)stream);
}

extern "C" size_t ixb_window_attention_bwd_scratch_bytes(int32_t B, int32_t H, int32_t HK, int32_t Sq, int32_t Sk,
                                                         int32_t window, int32_t sinks) {
  if (B <= 0 || H <= 0 || HK <= 0 || Sq <= 0 || Sk <= 0) return 0;
  return (size_t)B * H * Sq * sizeof(float);
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
  WinParams p = {};
  p.q = view_of(q, q_strides);
  p.k = view_of(k, k_strides);
  p.v = view_of(v, v_strides);
  p.o = view_of(o, o_strides);
  p.dout = view_of(dout, do_strides);
  p.dq = view_of(dq, dq_strides);
  p.dk = view_of(dk, dk_strides);
  p.dv = view_of(dv, dv_strides);
  p.lse_in = lse;
  p.q_lengths = q_lengths;
  p.kv_lengths = kv_lengths;
  p.B = B, p.H = H, p.HK = HK, p.Sq = Sq, p.Sk = Sk;
  p.scale = scale, p.window = window, p.sinks = sinks;
  float* delta = static_cast<float*>(scratch);
  const cudaStream_t s = (cudaStream_t)stream;
  const unsigned rows = (unsigned)(((long long)B * H * Sq + 7) / 8), keys = (unsigned)(((long long)B * HK * Sk + 7) / 8);
  if (dtype == IXB_BF16) {
    window_dq_kernel<bf16><<<rows, 256, 0, s>>>(p, delta);
    window_dkv_kernel<bf16><<<keys, 256, 0, s>>>(p, delta);
  } else {
    window_dq_kernel<f16><<<rows, 256, 0, s>>>(p, delta);
    window_dkv_kernel<f16><<<keys, 256, 0, s>>>(p, delta);
  }
  return ixb_host::cuda_status(cudaGetLastError());
}
