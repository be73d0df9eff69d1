// What the translation units of the windowed attention share: its arguments, and the checks of them.
#pragma once
#include <cmath>

#include "fa_maps.h"

namespace ixb_host {

struct WindowView {
  const void* ptr;
  const int64_t* strides;  // of the (batch, head, sequence) axes, in elements
};
// Query i of sequence b stands at p = kv_length - q_length + i and sees key j when j <= p and (j > p - window or
// j < sinks); query head h reads key head h / (H / HK).
struct WindowShape {
  int is_bf16, B, H, HK, Sq, Sk;
  const int *q_lengths, *kv_lengths;  // [B] on the device, or null: Sq and Sk
  float scale;
  int window, sinks;
};
constexpr int kMaxSinks = 128;  // all of them in the first key tile

inline int check_window_sizes(int dtype, int32_t B, int32_t H, int32_t HK, int32_t Sq, int32_t Sk, int32_t D, float scale,
                              int32_t window, int32_t sinks) {
  if (B < 0 || H < 0 || HK < 0 || Sq < 0 || Sk < 0 || window < 1 || sinks < 0 || !(scale > 0.f) || !(scale < INFINITY)) return IXB_ERR_ARG;
  if (dtype != IXB_BF16 && dtype != IXB_F16) return IXB_ERR_DTYPE;
  if (D != 128 || (HK == 0 ? H != 0 : H % HK != 0) || sinks > kMaxSinks) return IXB_ERR_SHAPE;
  return IXB_OK;
}
inline int check_window_views(const WindowView* views, int n) {
  for (int t = 0; t < n; ++t) {
    if (views[t].ptr == nullptr || views[t].strides == nullptr) return IXB_ERR_ARG;
    if (!aligned16(views[t].ptr)) return IXB_ERR_ALIGN;
    for (int i = 0; i < 3; ++i)
      if (views[t].strides[i] <= 0 || views[t].strides[i] % 8 != 0) return IXB_ERR_ALIGN;
  }
  return IXB_OK;
}

// fa_window_fwd.cu
int window_prefill(const WindowShape& a, const WindowView& q, const WindowView& k, const WindowView& v, const WindowView& o,
                   float* lse, int32_t* status, cudaStream_t stream);
// fa_window_split.cu: over how many blocks the keys of a tile of rows are shared where that is quicker (0: not, fa_window_fwd.cu), what the
// quicker of the two promises to take, and the call
int window_split_size(const WindowShape& a, double* us);
int window_split(int cluster, const WindowShape& a, const WindowView& q, const WindowView& k, const WindowView& v, const WindowView& o,
                 float* lse, int32_t* status, cudaStream_t stream);
// fa_window_decode.cu: whether it takes a call, and the call
bool window_decodes(const WindowShape& a);
int window_decode(const WindowShape& a, const WindowView& q, const WindowView& k, const WindowView& v, const WindowView& o,
                  float* lse, int32_t* status, cudaStream_t stream);

}  // namespace ixb_host
