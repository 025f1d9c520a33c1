// Rows on their way into e4m3 products (rows_e4m3.cuh has the form):
//     h = x + r;  y = h * rsqrt(mean(h^2) + eps) * gain;  codes and scales of y         (norm), or codes and scales of x alone
// h leaves in bf16 (the stream that goes on, rounded once, and what the norm sees), y on request (a router reads it), codes always.
//
// A row stays in registers: x and r are read once, and a block of 128 columns lies with 16 neighbouring threads of eight columns each,
// so its maximum is four shuffles and only the norm's sum crosses the block.  y is not rounded before its codes are taken.  Bound by
// bytes where rows are many, by the chain fetch, reduction, store where they are few.  us on B200: norm of 16384 x 8192 with a bf16 residual 164 (0.88 of
// the copy rate), codes alone 76 (0.82), 33 x 16384 8, one row of 4096 6.
#include "rows_e4m3.cuh"

#include <cstddef>

namespace xft {

struct RowsE4m3Params {
  const __nv_bfloat16* x; long long ldx;
  const void* r; long long ldr;                // bf16 or fp32, or null
  const float* gain; float eps;                // NORM
  int K;
  uint8_t* codes; long long ldc;
  float* scale; long long lds;                 // [K / 128, lds]
  __nv_bfloat16* h; long long ldh;             // x + r
  __nv_bfloat16* y; long long ldy;             // normalised rows, or null
};

enum { kNoResidual = 0, kResidualBf16 = 1, kResidualFp32 = 2 };

template <int NT, int CH, int RES, bool NORM>
__global__ void __launch_bounds__(NT) rows_e4m3_kernel(const RowsE4m3Params p) {
  __shared__ float s_ss[NT / 32];
  grid_dep_launch();
  grid_dep_wait();
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, nch = p.K / 8;
  uint4 v[CH];
  const uint4* x = reinterpret_cast<const uint4*>(p.x + row * p.ldx);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = tid + c * NT;
    v[c] = i < nch ? x[i] : make_uint4(0, 0, 0, 0);
  }
  auto pair = [&](int c, int j) { return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&v[c])[j]); };
  if constexpr (RES != kNoResidual) {
    float r[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = tid + c * NT;
      if (i >= nch) continue;
      if constexpr (RES == kResidualFp32) {
        const float4* from = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.r) + row * p.ldr) + 2 * i;
        const float4 a = from[0], b = from[1];
        r[c][0] = a.x; r[c][1] = a.y; r[c][2] = a.z; r[c][3] = a.w; r[c][4] = b.x; r[c][5] = b.y; r[c][6] = b.z; r[c][7] = b.w;
      } else {
        const uint4 u = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.r) + row * p.ldr)[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&u)[j]);
          r[c][2 * j] = f.x; r[c][2 * j + 1] = f.y;
        }
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = tid + c * NT;
      if (i >= nch) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = pair(c, j);
        reinterpret_cast<__nv_bfloat162*>(&v[c])[j] = __floats2bfloat162_rn(f.x + r[c][2 * j], f.y + r[c][2 * j + 1]);
      }
      reinterpret_cast<uint4*>(p.h + row * p.ldh)[i] = v[c];
    }
  }
  float inv = 1.f;
  if constexpr (NORM) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = pair(c, j);
        ss += f.x * f.x + f.y * f.y;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if constexpr (NT > 32) {
      if ((tid & 31) == 0) s_ss[tid >> 5] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int w = 0; w < NT / 32; ++w) ss += s_ss[w];
    }
    inv = rsqrtf(__fdiv_rn(ss, (float)p.K) + p.eps);
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = tid + c * NT;
    float y[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = pair(c, j);
      y[2 * j] = f.x; y[2 * j + 1] = f.y;
    }
    if constexpr (NORM) {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      if (i < nch) { a = __ldg(reinterpret_cast<const float4*>(p.gain) + 2 * i); b = __ldg(reinterpret_cast<const float4*>(p.gain) + 2 * i + 1); }
      y[0] *= a.x; y[1] *= a.y; y[2] *= a.z; y[3] *= a.w;
      y[4] *= b.x; y[5] *= b.y; y[6] *= b.z; y[7] *= b.w;
    }
    bool odd;
    float top = e4m3_top<8>(y, odd);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (i >= nch) continue;
    // The row's factor 1 / rms is in the scale alone where the block lies above the floor: it cancels in a code, whose rounding then sees one
    // rounding of the product with the gain and two of the scaling.  Below the floor, with that factor or without it, the values are
    // multiplied by it first: 448 / 2^-100 times a factor above 6e5 (eps below 2.8e-12) leaves 32 bits, and so does 448 over such a maximum.
    // So they are where the factor is no number.
    E4m3Scale s;
    float lacks = inv;                                                 // what y has still to be multiplied by
    if constexpr (!NORM) {
      s = e4m3_scale(top);
    } else if (const float a = top * inv; top >= kE4m3Least && a >= kE4m3Least && a <= 3.4e38f) {
      s = e4m3_scale_of(top);
      s.scale = __fdiv_rn(a, kE4m3Top);
    } else {
      s = e4m3_scale(a <= 3.4e38f ? a : 0.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= inv;
      odd = odd || inv > 3.4e38f;
      lacks = 1.f;
    }
    uint2 q;
    q.x = e4m3_codes(y, s.inv, odd);
    q.y = e4m3_codes(y + 4, s.inv, odd);
    reinterpret_cast<uint2*>(p.codes + row * p.ldc)[i] = q;
    if ((i & 15) == 0) p.scale[(i >> 4) * p.lds + row] = s.scale;
    if constexpr (NORM) {
      if (p.y) {
        uint4 u;
#pragma unroll
        for (int j = 0; j < 4; ++j) reinterpret_cast<__nv_bfloat162*>(&u)[j] = __floats2bfloat162_rn(y[2 * j] * lacks, y[2 * j + 1] * lacks);
        reinterpret_cast<uint4*>(p.y + row * p.ldy)[i] = u;
      }
    }
  }
}

template <int RES, bool NORM>
static int launch_rows_e4m3(const RowsE4m3Params& p, int rows, cudaStream_t st) {
  const int nch = p.K / 8;
  cudaError_t e;
#define XFT_ROWS_LAUNCH(NT, CH) e = launch_pdl(rows_e4m3_kernel<NT, CH, RES, NORM>, dim3(rows), dim3(NT), 0, st, p)
  if (nch <= 32) XFT_ROWS_LAUNCH(32, 1);
  else if (nch <= 64) XFT_ROWS_LAUNCH(64, 1);
  else if (nch <= 128) XFT_ROWS_LAUNCH(128, 1);
  else if (nch <= 256) XFT_ROWS_LAUNCH(256, 1);
  else if (nch <= 512) XFT_ROWS_LAUNCH(256, 2);
  else if (nch <= 1024) XFT_ROWS_LAUNCH(256, 4);
  else if (nch <= 2048) XFT_ROWS_LAUNCH(256, 8);
  else XFT_ROWS_LAUNCH(256, 16);
#undef XFT_ROWS_LAUNCH
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace xft

using namespace xft;

// Arguments of xft_rows_e4m3 (packed by ops/native_e4m3.py).
struct RowsArgs {
  const void* x; const void* r; const float* gain; void* codes; float* scale; void* h; void* y;
  long long ldx, ldr, ldc, lds, ldh, ldy;
  int rows, K, r_kind; float eps;                // r_kind: 0 none, 1 bf16, 2 fp32
};

// Size and field offsets of RowsArgs, for the layout check of the Python side.
extern "C" int xft_rows_args_layout(long long* out, int n) {
  const long long v[] = {sizeof(RowsArgs),         offsetof(RowsArgs, x),     offsetof(RowsArgs, r),    offsetof(RowsArgs, gain),
                         offsetof(RowsArgs, codes), offsetof(RowsArgs, scale), offsetof(RowsArgs, h),    offsetof(RowsArgs, y),
                         offsetof(RowsArgs, ldx),  offsetof(RowsArgs, ldr),   offsetof(RowsArgs, ldc),  offsetof(RowsArgs, lds),
                         offsetof(RowsArgs, ldh),  offsetof(RowsArgs, ldy),   offsetof(RowsArgs, rows), offsetof(RowsArgs, K),
                         offsetof(RowsArgs, r_kind), offsetof(RowsArgs, eps)};
  const int m = (int)(sizeof(v) / sizeof(v[0]));
  for (int i = 0; i < m && i < n; ++i) out[i] = v[i];
  return m;
}

// gain null: codes and scales of x [rows, K] (no residual).  K a multiple of 8, at most 32768; rows of x, r, h, y on 16 bytes, rows of
// codes on 8, gain on 16.
extern "C" int xft_rows_e4m3(const RowsArgs* args, cudaStream_t st) {
  const RowsArgs& a = *args;
  auto on = [](const void* q, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(q) & (bytes - 1)) == 0; };
  if (a.rows <= 0) return 0;
  if (a.K <= 0 || (a.K & 7) || a.K > 32768 || (a.ldx & 7) || (a.ldc & 7) || (a.ldh & 7) || (a.ldy & 7) || (a.ldr & (a.r_kind == 2 ? 3 : 7)) ||
      (a.r_kind && (!a.r || !a.h || !a.gain)) || !on(a.x, 16) || !on(a.r, 16) || !on(a.gain, 16) || !on(a.h, 16) || !on(a.y, 16) || !on(a.codes, 8))
    return -1;
  RowsE4m3Params p{};
  p.x = (const __nv_bfloat16*)a.x; p.ldx = a.ldx; p.r = a.r; p.ldr = a.ldr; p.gain = a.gain; p.eps = a.eps; p.K = a.K; p.codes = (uint8_t*)a.codes;
  p.ldc = a.ldc; p.scale = a.scale; p.lds = a.lds; p.h = (__nv_bfloat16*)a.h; p.ldh = a.ldh; p.y = (__nv_bfloat16*)a.y; p.ldy = a.ldy;
  if (!a.gain) return launch_rows_e4m3<kNoResidual, false>(p, a.rows, st);
  if (a.r_kind == 0) return launch_rows_e4m3<kNoResidual, true>(p, a.rows, st);
  return a.r_kind == 1 ? launch_rows_e4m3<kResidualBf16, true>(p, a.rows, st) : launch_rows_e4m3<kResidualFp32, true>(p, a.rows, st);
}
