// What stands around the products of routed experts over rows in e4m3 (rows_e4m3.cuh): the plan of rows by expert, the rows in that order,
// and the weighted sum of what the experts gave.  The products themselves are xft_gemm_rows_e4m3 over the plan's tiles.
#include "rows_e4m3.cuh"

namespace xft {

// ------------------------------------------------------------------------------------------ plan
// Pairs (token, slot) whose expert is one of [e0, e0 + E) get a row each, those of an expert one behind the other.  pos [pairs]: row or -1;
// src [row]: token; row_w [row]: weight; tiles: {expert, first row, rows, 0} of at most bn rows each; meta: {tiles, rows}.
//
// One pass counts and one places, the pairs of a warp that ask for the same expert together (one addition in shared memory for all of them).
// A cluster shares the pairs: its CTAs read each other's counts and know where their rows start.  Bound by the chain of two passes, a scan
// and a barrier; us, one CTA for all as in moe_plan_kernel / here: 24576 pairs 64 experts 37 / 12, 48 pairs 9 / 9.
struct PlanRows {
  const int* idx; const float* w; int pairs, k, e0, E, bn;
  int* pos; int* src; float* row_w; int4* tiles; int* meta; int max_tiles;
};
constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int ld_dsmem_int(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__global__ void __launch_bounds__(kPlanThreads) plan_rows_kernel(const PlanRows p, int ctas) {
  __shared__ int cnt[256], at[256], off[257], toff[257], s_sum[2][8];
  grid_dep_launch();
  grid_dep_wait();
  const int tid = threadIdx.x, lane = tid & 31, rank = blockIdx.x;
  const int per = (p.pairs + ctas - 1) / ctas, i0 = rank * per, i1 = min(i0 + per, p.pairs);
  if (tid < 256) cnt[tid] = 0;
  __syncthreads();
  int first[4];                                                        // of this thread's first four pairs: place among the CTA's of the expert
  for (int j0 = 0; i0 + j0 * kPlanThreads < i1; j0 += 4) {
    int e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + (j0 + j) * kPlanThreads + tid;
      e[j] = i < i1 ? p.idx[i] - p.e0 : -1;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + (j0 + j) * kPlanThreads + tid;
      const bool in = e[j] >= 0 && e[j] < p.E;
      const unsigned same = __match_any_sync(0xffffffffu, in ? e[j] : 256 + lane);
      const int lead = __ffs(same) - 1;
      int base = 0;
      if (in && lane == lead) base = atomicAdd(&cnt[e[j]], __popc(same));
      base = __shfl_sync(0xffffffffu, base, lead) + __popc(same & ((1u << lane) - 1));
      if (j0 == 0) first[j] = base;
      else if (in) p.pos[i] = base;
    }
  }
  __syncthreads();
  if (ctas > 1) { cluster_arrive(); cluster_wait(); }
  int total = 0, before = 0, tiles = 0;
  if (tid < 256) {
    for (int r = 0; r < ctas; ++r) {
      const int v = ctas == 1 ? cnt[tid] : ld_dsmem_int(dsmem_addr(smem_u32(&cnt[tid]), r));
      if (r < rank) before += v;
      total += v;
    }
    tiles = (total + p.bn - 1) / p.bn;
  }
  if (ctas > 1) cluster_arrive();                                      // (waited for at the end: nobody leaves while its counts are read)
  int rs = total, ts = tiles;
  if (tid < 256) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, rs, o), b = __shfl_up_sync(0xffffffffu, ts, o);
      if (lane >= o) { rs += a; ts += b; }
    }
    if (lane == 31) { s_sum[0][tid >> 5] = rs; s_sum[1][tid >> 5] = ts; }
  }
  __syncthreads();
  if (tid < 256) {
    for (int w = 0; w < tid >> 5; ++w) { rs += s_sum[0][w]; ts += s_sum[1][w]; }
    off[tid + 1] = rs;
    toff[tid + 1] = ts;
    at[tid] = rs - total + before;
    if (tid == 0) { off[0] = 0; toff[0] = 0; }
  }
  __syncthreads();
  for (int j0 = 0; i0 + j0 * kPlanThreads < i1; j0 += 4) {
    int e[4], l[4];
    float w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + (j0 + j) * kPlanThreads + tid;
      e[j] = i < i1 ? p.idx[i] - p.e0 : -1;
      w[j] = i < i1 ? p.w[i] : 0.f;
      l[j] = j0 == 0 ? first[j] : i < i1 ? p.pos[i] : 0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + (j0 + j) * kPlanThreads + tid;
      if (i >= i1) continue;
      const bool in = e[j] >= 0 && e[j] < p.E;
      const int row = in ? at[e[j]] + l[j] : -1;
      p.pos[i] = row;
      if (in) { p.src[row] = i / p.k; p.row_w[row] = w[j]; }
    }
  }
  const int nt = min(toff[p.E], p.max_tiles);
  for (int ti = rank * kPlanThreads + tid; ti < nt; ti += ctas * kPlanThreads) {
    int lo = 0, hi = p.E;                                              // the expert whose tiles hold ti: toff[lo] <= ti < toff[lo + 1]
    while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (toff[m] <= ti) lo = m; else hi = m; }
    const int row = (ti - toff[lo]) * p.bn;
    p.tiles[ti] = make_int4(lo, off[lo] + row, min(p.bn, off[lo + 1] - off[lo] - row), 0);
  }
  if (rank == 0 && tid == 0) { p.meta[0] = nt; p.meta[1] = off[p.E]; }
  if (ctas > 1) cluster_wait();
}

// ------------------------------------------------------------------------------------------ rows by expert
// Row r of the output is row src[r] of the input, codes and scales; rows from *used on are left alone.  A warp per row: bound by the bytes.
__global__ void __launch_bounds__(256) gather_e4m3_kernel(const uint8_t* __restrict__ codes, long long ldc, const float* __restrict__ scale,
                                                          long long lds, const int* __restrict__ src, const int* __restrict__ used,
                                                          uint8_t* __restrict__ out, long long ldo, float* __restrict__ out_scale,
                                                          long long ldos, int K) {
  grid_dep_launch();
  grid_dep_wait();
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= *used) return;
  const long long s = src[r];
  const uint4* from = reinterpret_cast<const uint4*>(codes + s * ldc);
  uint4* to = reinterpret_cast<uint4*>(out + (long long)r * ldo);
  const int n = (K + 15) / 16, nb = (K + 127) / 128;
  float f[2];                                                          // scales of the first 64 blocks on their way beside the codes
#pragma unroll
  for (int j = 0; j < 2; ++j) f[j] = lane + 32 * j < nb ? scale[(lane + 32 * j) * lds + s] : 0.f;
  for (int i = lane; i < n; i += 128) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) if (i + 32 * j < n) v[j] = from[i + 32 * j];
#pragma unroll
    for (int j = 0; j < 4; ++j) if (i + 32 * j < n) to[i + 32 * j] = v[j];
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) if (lane + 32 * j < nb) out_scale[(lane + 32 * j) * ldos + r] = f[j];
  for (int i = lane + 64; i < nb; i += 32) out_scale[i * ldos + r] = scale[i * lds + s];
}

// ------------------------------------------------------------------------------------------ weighted sum
// y[t] = sum_s w[t, s] rows[pos[t, s]] + add[t], in fp32 and in the order of the slots; w null: the rows carry their weights.  A thread has
// eight columns of a token, the rows of eight slots are under way together.  Bound by the bytes of the rows.
template <typename RT>
__device__ __forceinline__ void load8(const RT* p, float (&v)[8]) {
  if constexpr (sizeof(RT) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&u)[j]);
      v[2 * j] = f.x; v[2 * j + 1] = f.y;
    }
  }
}

struct SumRows {
  const void* rows; const int* pos; const float* w; int k, T, H;
  const float* add32; const __nv_bfloat16* add16;
  float* out32; __nv_bfloat16* out16;
};

template <typename RT>
__global__ void __launch_bounds__(256) sum_rows_kernel(const SumRows p) {
  grid_dep_launch();
  grid_dep_wait();
  const int per = p.H / 8;                                             // threads of a token
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x, t = at / per;
  if (t >= p.T) return;
  const int c = (int)(at - t * per) * 8;
  const RT* rows = reinterpret_cast<const RT*>(p.rows);
  float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[8][8];
  for (int s0 = 0; s0 < p.k; s0 += 8) {
    int r[8];
    float f[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      r[s] = s0 + s < p.k ? p.pos[t * p.k + s0 + s] : -1;
      f[s] = p.w && s0 + s < p.k ? p.w[t * p.k + s0 + s] : 1.f;
    }
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (r[s] >= 0) load8(rows + (size_t)r[s] * p.H + c, v[s]);
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (r[s] >= 0)
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] += f[s] * v[s][j];
  }
  if (p.add32 || p.add16) {
    if (p.add32) load8(p.add32 + t * p.H + c, v[0]);
    else load8(p.add16 + t * p.H + c, v[0]);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] += v[0][j];
  }
  if (p.out32) {
    float4* to = reinterpret_cast<float4*>(p.out32 + t * p.H + c);
    to[0] = make_float4(a[0], a[1], a[2], a[3]);
    to[1] = make_float4(a[4], a[5], a[6], a[7]);
  } else {
    uint4 u;
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<__nv_bfloat162*>(&u)[j] = __floats2bfloat162_rn(a[2 * j], a[2 * j + 1]);
    *reinterpret_cast<uint4*>(p.out16 + t * p.H + c) = u;
  }
}

}  // namespace xft

using namespace xft;

extern "C" int xft_plan_rows(const int* idx, const float* w, int T, int k, int e0, int e1, int bn, int* pos, int* src, float* row_w,
                             void* tiles, int* meta, int max_tiles, cudaStream_t st) {
  if (T <= 0) return 0;
  if (e1 <= e0 || e1 - e0 > 256 || k <= 0 || bn <= 0 || (long long)T * k > 0x7fffffffLL / 2) return -1;
  const PlanRows p{idx, w, T * k, k, e0, e1 - e0, bn, pos, src, row_w, reinterpret_cast<int4*>(tiles), meta, max_tiles};
  const int ctas = p.pairs > 2 * kPlanThreads ? 8 : 1;                 // below, the cluster's barriers take longer than the pairs
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_xft_pdl ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, plan_rows_kernel, p, ctas);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// Rows of codes on 16 bytes, and as long as K rounded up to 16.
extern "C" int xft_gather_e4m3(const void* codes, long long ldc, const float* scale, long long lds, const int* src, const int* used,
                               int max_rows, int K, void* out, long long ldo, float* out_scale, long long ldos, cudaStream_t st) {
  if (max_rows <= 0) return 0;
  if (K <= 0 || (ldc & 15) || (ldo & 15) || ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(out)) & 15)) return -1;
  const cudaError_t e = launch_pdl(gather_e4m3_kernel, dim3((max_rows + 7) / 8), dim3(256), 0, st, (const uint8_t*)codes, ldc, scale, lds, src,
                                   used, (uint8_t*)out, ldo, out_scale, ldos, K);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// rows [.., H] bf16 or fp32; add32 / add16 and out32 / out16: one of each pair, add may be null.  H a multiple of 8, everything on 16 bytes.
extern "C" int xft_sum_rows(const void* rows, int rows_fp32, const int* pos, const float* w, int k, const float* add32, const void* add16,
                            float* out32, void* out16, int T, int H, cudaStream_t st) {
  if (T <= 0) return 0;
  if (H <= 0 || (H & 7) || k <= 0 || !out32 == !out16 ||
      ((reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(add32) | reinterpret_cast<uintptr_t>(add16) |
        reinterpret_cast<uintptr_t>(out32) | reinterpret_cast<uintptr_t>(out16)) & 15))
    return -1;
  const SumRows p{rows, pos, w, k, T, H, add32, (const __nv_bfloat16*)add16, out32, (__nv_bfloat16*)out16};
  const long long threads = (long long)T * (H / 8);
  const dim3 grid((unsigned)((threads + 255) / 256));
  const cudaError_t e = rows_fp32 ? launch_pdl(sum_rows_kernel<float>, grid, dim3(256), 0, st, p)
                                  : launch_pdl(sum_rows_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
