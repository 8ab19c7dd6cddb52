// Arguments of one hga_fp8_linear call.
#pragma once

#include "hga_common.cuh"

namespace hga {

struct Fp8Linear {
  int64_t m, n, k;
  const void* x;
  int64_t x_stride;
  int x_dtype;
  const float* x_scale;
  const void* w;
  int64_t w_stride;
  const float* w_scale;
  int64_t ws_stride;
  const void* bias;
  void* out;
  int64_t out_stride;
  int out_dtype;
  void* workspace;
};

}  // namespace hga
