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

__device__ __forceinline__ float e4m3_top(float top, float y) {
  const float a = fabsf(y);
  return a <= 3.4e38f ? fmaxf(top, a) : top;
}
__device__ __forceinline__ E4m3Scale e4m3_scale_of(float top) { return {__fdiv_rn(top, kE4m3Top), __fdiv_rn(kE4m3Top, top)}; }
__device__ __forceinline__ E4m3Scale e4m3_scale(float top) { return e4m3_scale_of(fmaxf(top, kE4m3Least)); }
// two codes, the first in the low byte
__device__ __forceinline__ uint32_t e4m3_codes(float a, float b, float inv) {
  uint32_t v = __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
  if (!(fabsf(a) <= 3.4e38f)) v = (v & 0xFF00u) | 0x7Fu;                      // the conversion saturates infinities
  if (!(fabsf(b) <= 3.4e38f)) v = (v & 0x00FFu) | 0x7F00u;
  return v;
}

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
  int form;                                            // -1: by size; 0: gemm_e4m3_sm100.cu, else a tile of gemm_rows_e4m3_sm100.cu
  float res_scale;
};

}  // namespace xft
