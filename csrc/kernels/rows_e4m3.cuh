// Rows in e4m3 with an fp32 scale for each block of 128 columns, as every kernel that writes or multiplies them sees them:
//     a = max |y| over the block, at least 2^-100;  scale = a / 448;  code = e4m3(y * (448 / a)), nearest, ties to even.
// A value that is not finite has no part in `a` and becomes the code of NaN, so its row's products are NaN.  The floor keeps 448 / a
// and a / 448 normal numbers; a block below it loses bits, not its sign or its zeros.  Scales lie block by block, [blocks, rows]: the
// rows of a tile are one run for the kernels that multiply.
#pragma once
#include "gemm_common.cuh"

#include <cuda_fp8.h>

namespace xft {

constexpr float kE4m3Top = 448.f, kE4m3Least = 7.8886090522101181e-31f;       // 2^-100

struct E4m3Scale { float scale, inv; };

// max |v| over N values that are finite.  `odd`: there is an infinity among them (a NaN needs no care: maxima pass it over, and it converts to
// its code).
template <int N>
__device__ __forceinline__ float e4m3_top(const float* v, bool& odd) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) top = fmaxf(top, fabsf(v[j]));
  odd = top > 3.4e38f;
  if (odd) {
    top = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) top = fmaxf(top, fabsf(v[j]) <= 3.4e38f ? fabsf(v[j]) : 0.f);
  }
  return top;
}
__device__ __forceinline__ E4m3Scale e4m3_scale_of(float top) { return {__fdiv_rn(top, kE4m3Top), __fdiv_rn(kE4m3Top, top)}; }
__device__ __forceinline__ E4m3Scale e4m3_scale(float top) { return e4m3_scale_of(fmaxf(top, kE4m3Least)); }
// four codes, the first in the low byte
__device__ __forceinline__ uint32_t e4m3_codes(const float* v, float inv, bool odd) {
  uint32_t q = __nv_cvt_float2_to_fp8x2(make_float2(v[0] * inv, v[1] * inv), __NV_SATFINITE, __NV_E4M3) |
               (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[2] * inv, v[3] * inv), __NV_SATFINITE, __NV_E4M3) << 16;
  if (odd) {                                                                  // the conversion saturates infinities
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!(fabsf(v[j]) <= 3.4e38f)) q = (q & ~(0xFFu << 8 * j)) | 0x7Fu << 8 * j;
  }
  return q;
}

// By size, and the launch in front of this one writes the weights: a step's kernel, which asks for weights before it waits for that launch, is
// then not started beside it.
constexpr int kRowsFormAfterCopy = -2;

// Arguments of xft_gemm_rows_e4m3 (mirrored in ops/native_e4m3.py).
struct RowsGemm {
  const void* x; const float* x_scale; const void* w; const float* w_scale;
  void* out; float* out_scale; const float* bias; const void* residual;
  const void* group_tiles; const int* num_group_tiles; const float* col_scale; int* status;
  long long x_ld, out_ld;                              // row pitch of x_scale and of out_scale
  int x_rows, ldx, w_rows, ldw, scale_ld;              // codes: pitches in bytes, multiples of 16
  int T, N, K, ldo, out_fp32, ldr, act;
  int gated, dual_off;
  int group_w_rows, max_tiles, bn;                     // grouped form: rows of a tile of the table
  int form;                                            // -1: by size; kRowsFormAfterCopy; 0: gemm_e4m3_sm100.cu, else a tile of gemm_rows_e4m3_sm100.cu
  float res_scale;
};

}  // namespace xft
