// Attention of the nodes of trees of drafted tokens over the paged cache: a node sees the context's keys and the nodes whose bits its
// mask has.
//
//   o_i = sum_j p_ij v_j / (sum_j p_ij + exp(sink)),  p_ij = exp(scale q_i k_j - max),  j over the keys that node i sees
//
// All rows (node, query head) of one kv head read the same keys: 64 of them per CTA, 16 a warp, flash attention with
// mma.sync.m16n8k16, keys in tiles through cp.async, two in flight.  Long caches are cut into slices whose sums a second kernel joins.
// Masks matter in the last tiles alone, where the nodes' keys are.  Values of keys that no node sees (for its mask or the window) and of slots
// behind the last key count as zero: 0 x what a slot happens to hold may be NaN.
//
// This is the kernel for what tree_attention_sm100.cu does not take: blocks that are no multiple of 64, int8 caches with heads of 64 or
// 256, scales of zero or below.  Bound by the instructions around mma.sync, of one warp where few rows share a key.  us: 8 trees of 13
// nodes, 32 and 8 heads of 64, int8, 4000 keys 86 (its bytes take 5).
#include "tree_attention.cuh"
#include "mma_sync.cuh"

namespace xft {
namespace {

constexpr int kTaRows = 64, kTaThreads = 128;

__device__ __forceinline__ void ta_cp16(void* smem, const void* g, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(g), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ta_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ta_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// rows of D bf16, 16-byte pieces exchanged with the row's low bits
template <int D>
__device__ __forceinline__ __nv_bfloat16* ta_at(__nv_bfloat16* t, int row, int piece) {
  return t + row * D + ((piece ^ (row & 7)) << 3);
}

template <int D>
constexpr int kTaKeys = D == 256 ? 32 : 64;
template <int D>
constexpr int kTaSmem = (kTaRows + 4 * kTaKeys<D>) * D * 2 + 8 * kTaKeys<D> * 4;

template <int D, bool INT8>
__global__ void __launch_bounds__(kTaThreads) tree_attention_kernel(const TreeAttnArgs p) {
  constexpr int KT = kTaKeys<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __nv_bfloat16* sQ = reinterpret_cast<__nv_bfloat16*>(smem);
  __nv_bfloat16* sK = sQ + kTaRows * D;                  // two tiles
  __nv_bfloat16* sV = sK + 2 * KT * D;                   // two tiles
  float* s_scale = reinterpret_cast<float*>(sV + 2 * KT * D);          // int8: [2][keys | values][KT]
  long long* s_at = reinterpret_cast<long long*>(s_scale + 4 * KT);    // [2][KT]: where a tile's keys are, and whether they are seen
  __shared__ unsigned long long s_mask[kTaRows][kTreeWords], s_union[kTreeWords];
  __shared__ int s_pos[kTreeMaxNodes], s_first;
  grid_dep_launch();
  grid_dep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const TreeSeq s(p, b);
  int h0;
  const int heads = tree_heads(p, kvh, h0), rows = s.n * heads;
  const int n_rt = (p.max_q * p.group + kTaRows - 1) / kTaRows;
  const int row0 = (blockIdx.x % n_rt) * kTaRows, slice = blockIdx.x / n_rt;
  if (row0 >= rows) return;
  const int node0 = row0 / heads;
  if (tid < kTreeWords) s_union[tid] = 0;
  if (tid == 0) s_first = 0x7fffffff;
  __syncthreads();
  if (p.window > 0) {
    int first = 0x7fffffff;
    for (int i = tid; i < s.n; i += kTaThreads) first = min(first, s_pos[i] = p.positions[s.q0 + i]);
    atomicMin(&s_first, first);
    __syncthreads();
  }
  for (int i = tid; i < s.n * p.words; i += kTaThreads) {
    const int nd = i / p.words, w = i - nd * p.words;
    unsigned long long m = p.mask[(long long)(s.q0 + nd) * p.words + w];
    if (nd >= node0 && nd - node0 < kTaRows) s_mask[nd - node0][w] = m;
    if (p.window > 0) m = tree_within(m, 64 * w, s.n, s_pos[nd], s_pos, p.window, p.keep);
    if (m) atomicOr(&s_union[w], m);
  }
  // rows of queries, 16 bytes at a time; rows behind the last one are zero
  for (int i = tid; i < kTaRows * (D / 8); i += kTaThreads) {
    const int r = i / (D / 8), c = i % (D / 8), row = row0 + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows) v = *reinterpret_cast<const uint4*>(p.q + ((long long)(s.q0 + row / heads) * p.hq + h0 + row % heads) * D + c * 8);
    *reinterpret_cast<uint4*>(ta_at<D>(sQ, r, c)) = v;
  }
  __syncthreads();
  // tiles: those of the kept first keys, then those from the first key of the widest window
  const int end = (s.kv + KT - 1) / KT;
  int lo = 0, n_keep = 0, first_key = 0;
  if (p.window > 0) {
    first_key = tree_first(p, s, s_first);
    lo = min(first_key / KT, end);
    n_keep = min((min(p.keep, s.kv) + KT - 1) / KT, lo);
  }
  const int nt = n_keep + end - lo, per = (nt + p.nsplit - 1) / p.nsplit;
  const int t_end = min(nt, (slice + 1) * per);
  // rows of a tile's keys: twice the place in the cache, plus one where some node sees the key; below zero behind the last one
  auto locate = [&](int t, int buf) {
    if (tid >= KT) return;
    const int key = (t < n_keep ? t : t - n_keep + lo) * KT + tid;
    const bool in = key < s.kv;
    const bool seen = in && (key < s.ctx ? key >= first_key || key < p.keep : (bool)(s_union[(key - s.ctx) >> 6] >> ((key - s.ctx) & 63) & 1));
    const int block = key / p.bs;
    s_at[buf * KT + tid] = in ? 2 * (((long long)tree_block(p, b, block) * p.hkv + kvh) * p.bs + key - block * p.bs) + seen : -1;
  };
  auto fetch = [&](int t, int buf) {
    __nv_bfloat16 *dk = sK + buf * KT * D, *dv = sV + buf * KT * D;
    constexpr int per_row = INT8 ? D / 16 : D / 8;
    for (int i = tid; i < KT * per_row; i += kTaThreads) {
      const int r = i / per_row, c = i % per_row;
      const long long where = s_at[buf * KT + r], at = where < 0 ? 0 : where >> 1;
      const bool in = where >= 0, seen = in && (where & 1);
      if constexpr (INT8) {
        uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (in) raw[0] = *reinterpret_cast<const uint4*>(static_cast<const int8_t*>(p.kc) + at * D + c * 16);
        if (seen) raw[1] = *reinterpret_cast<const uint4*>(static_cast<const int8_t*>(p.vc) + at * D + c * 16);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int8_t* q = reinterpret_cast<const int8_t*>(&raw[x]);
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = gl_pack((float)q[2 * e], (float)q[2 * e + 1]);
          __nv_bfloat16* d = x ? dv : dk;
          *reinterpret_cast<uint4*>(ta_at<D>(d, r, 2 * c)) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(ta_at<D>(d, r, 2 * c + 1)) = make_uint4(w[4], w[5], w[6], w[7]);
        }
        if (c == 0) {
          s_scale[(2 * buf) * KT + r] = in ? p.ks[at] : 0.f;
          s_scale[(2 * buf + 1) * KT + r] = seen ? p.vs[at] : 0.f;
        }
      } else {
        ta_cp16(ta_at<D>(dk, r, c), static_cast<const __nv_bfloat16*>(p.kc) + at * D + c * 8, in);
        ta_cp16(ta_at<D>(dv, r, c), static_cast<const __nv_bfloat16*>(p.vc) + at * D + c * 8, seen);
      }
    }
    ta_commit();
  };
  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const int r0 = row0 + warp * 16 + (lane >> 2);
  const int nd[2] = {min(r0, rows - 1) / heads, min(r0 + 8, rows - 1) / heads};
  const int pos[2] = {p.window > 0 ? s_pos[nd[0]] : 0, p.window > 0 ? s_pos[nd[1]] : 0};
  const bool busy = row0 + warp * 16 < rows;
  if (slice * per < t_end) {
    locate(slice * per, 0);
    if (slice * per + 1 < t_end) locate(slice * per + 1, 1);
    __syncthreads();
    fetch(slice * per, 0);
  }
  for (int t = slice * per, it = 0; t < t_end; ++t, ++it) {
    const int buf = it & 1;
    if (t + 1 < t_end) { fetch(t + 1, buf ^ 1); ta_wait<1>(); } else ta_wait<0>();
    __syncthreads();
    if (busy) {
      const int k0 = (t < n_keep ? t : t - n_keep + lo) * KT;
      __nv_bfloat16 *kt = sK + buf * KT * D, *vt = sV + buf * KT * D;
      float x[KT / 8][4];
#pragma unroll
      for (int j = 0; j < KT / 8; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t a[4];
        gl_ldsm(a, ta_at<D>(sQ, warp * 16 + (lane & 15), c * 2 + (lane >> 4)));
#pragma unroll
        for (int j = 0; j < KT / 8; j += 2) {
          uint32_t w[4];
          gl_ldsm(w, ta_at<D>(kt, j * 8 + (lane & 7) + ((lane >> 4) & 1) * 8, c * 2 + ((lane >> 3) & 1)));
          gl_mma(x[j], a, w[0], w[1]);
          gl_mma(x[j + 1], a, w[2], w[3]);
        }
      }
      const bool masked = k0 + KT > s.ctx || p.window > 0;
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < KT / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kl = j * 8 + 2 * (lane & 3) + (e & 1), key = k0 + kl, half = e >> 1;
          float v = x[j][e] * p.scale;
          if (INT8) v *= s_scale[(2 * buf) * KT + kl];
          if (p.softcap > 0.f) v = p.softcap * tanhf(v / p.softcap);
          v *= kTreeLog2e;
          if (masked) {
            bool sees = key < s.ctx;
            int kpos = key;
            if (!sees && key < s.kv) {
              const int i = key - s.ctx;
              sees = s_mask[nd[half] - node0][i >> 6] >> (i & 63) & 1;
              if (p.window > 0) kpos = s_pos[i];
            }
            if (p.window > 0) sees = sees && ((long long)pos[half] - kpos < p.window || kpos < p.keep);
            if (!sees) v = -INFINITY;
          }
          x[j][e] = v;
          top[half] = fmaxf(top[half], v);
        }
      float alpha[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
        top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 2));
        const float mx = fmaxf(m[half], top[half]);
        alpha[half] = mx == -INFINITY ? 1.f : exp2f(m[half] - mx);
        m[half] = mx;
        l[half] *= alpha[half];
      }
#pragma unroll
      for (int j = 0; j < KT / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int half = e >> 1;
          float v = x[j][e] == -INFINITY ? 0.f : exp2f(x[j][e] - m[half]);
          if (INT8) {
            l[half] += v;
            v *= s_scale[(2 * buf + 1) * KT + j * 8 + 2 * (lane & 3) + (e & 1)];
          } else {                                       // the sum uses the rounded values, as the product does
            v = __bfloat162float(__float2bfloat16(v));
            l[half] += v;
          }
          x[j][e] = v;
        }
#pragma unroll
      for (int j = 0; j < D / 8; ++j) { o[j][0] *= alpha[0]; o[j][1] *= alpha[0]; o[j][2] *= alpha[1]; o[j][3] *= alpha[1]; }
#pragma unroll
      for (int c = 0; c < KT / 16; ++c) {
        const uint32_t a[4] = {gl_pack(x[2 * c][0], x[2 * c][1]), gl_pack(x[2 * c][2], x[2 * c][3]), gl_pack(x[2 * c + 1][0], x[2 * c + 1][1]),
                               gl_pack(x[2 * c + 1][2], x[2 * c + 1][3])};
#pragma unroll
        for (int j = 0; j < D / 8; j += 2) {
          uint32_t w[4];
          gl_ldsm_t(w, ta_at<D>(vt, c * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, j + (lane >> 4)));
          gl_mma(o[j], a, w[0], w[1]);
          gl_mma(o[j + 1], a, w[2], w[3]);
        }
      }
    }
    if (t + 2 < t_end) locate(t + 2, buf);
    __syncthreads();
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = r0 + 8 * half;
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
    if (row >= rows) continue;
    const int h = h0 + row % heads;
    const long long at = (long long)(s.q0 + row / heads) * p.hq + h;
    if (p.nsplit == 1) {
      float f = 1.f, sum = l[half];
      if (p.sinks) {
        const float sink = p.sinks[h] * kTreeLog2e, mx = fmaxf(m[half], sink);
        f = exp2f(m[half] - mx);
        sum = sum * f + exp2f(sink - mx);
      }
      f = l[half] == 0.f ? 0.f : f / sum;                // a row that sees nothing
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<uint32_t*>(p.out + at * D + j * 8 + 2 * (lane & 3)) = gl_pack(o[j][2 * half] * f, o[j][2 * half + 1] * f);
    } else {
      float* to = p.part_o + (at * p.nsplit + slice) * D;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(to + j * 8 + 2 * (lane & 3)) = make_float2(o[j][2 * half], o[j][2 * half + 1]);
      if ((lane & 3) == 0) *reinterpret_cast<float2*>(p.part_ml + (at * p.nsplit + slice) * 2) = make_float2(m[half], l[half]);
    }
  }
}

// Joins the slices: a warp per row, a slice's weight per lane and 4 columns of four slices at a time
template <int D>
__global__ void __launch_bounds__(128) tree_join_kernel(const TreeAttnArgs p) {
  grid_dep_launch();
  grid_dep_wait();
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row < (long long)p.cu_q[0] * p.hq || row >= (long long)min(p.T, p.cu_q[p.B]) * p.hq) return;          // of no sequence
  float2 ml[2];                                          // slices lane and lane + 32
  float mx = -INFINITY;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int s = lane + 32 * e;
    ml[e] = s < p.nsplit ? *reinterpret_cast<const float2*>(p.part_ml + (row * p.nsplit + s) * 2) : make_float2(-INFINITY, 0.f);
    mx = fmaxf(mx, ml[e].x);
  }
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const bool any = mx != -INFINITY;
  float extra = 0.f;
  if (p.sinks) {
    const float sink = p.sinks[row % p.hq] * kTreeLog2e;
    mx = fmaxf(mx, sink);
    extra = exp2f(sink - mx);
  }
  float f[2], sum = 0.f;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    f[e] = ml[e].y == 0.f ? 0.f : exp2f(ml[e].x - mx);   // (a slice without keys for this row has written no sums)
    sum += ml[e].y == 0.f ? 0.f : ml[e].y * f[e];
  }
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = any || sum != 0.f ? 1.f / (sum + extra) : 0.f;       // (a sum that is NaN: any is false where every score was)
  const float* part = p.part_o + row * p.nsplit * D;
  constexpr int C = D < 128 ? 2 : D / 32;                // columns of a lane
  float o[C] = {};
  for (int s0 = 0; s0 < p.nsplit; s0 += 4) {
    float v[4][C], w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int s = s0 + e;
      w[e] = __shfl_sync(0xffffffffu, s < 32 ? f[0] : f[1], s & 31);
      const float y = __shfl_sync(0xffffffffu, s < 32 ? ml[0].y : ml[1].y, s & 31);
      if (s >= p.nsplit || y == 0.f) {
        w[e] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) v[e][c] = 0.f;
      } else if constexpr (C == 2) {
        *reinterpret_cast<float2*>(v[e]) = *reinterpret_cast<const float2*>(part + (long long)s * D + 2 * lane);
      } else {
#pragma unroll
        for (int c = 0; c < C; c += 4)
          *reinterpret_cast<float4*>(v[e] + c) = *reinterpret_cast<const float4*>(part + (long long)s * D + c * 32 + 4 * lane);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] += w[e] * v[e][c];
  }
  __nv_bfloat16* out = p.out + row * D;
  if constexpr (C == 2) {
    *reinterpret_cast<uint32_t*>(out + 2 * lane) = gl_pack(o[0] * inv, o[1] * inv);
  } else {
#pragma unroll
    for (int c = 0; c < C; c += 4)
      *reinterpret_cast<uint2*>(out + c * 32 + 4 * lane) = make_uint2(gl_pack(o[c] * inv, o[c + 1] * inv), gl_pack(o[c + 2] * inv, o[c + 3] * inv));
  }
}

template <int D, bool INT8>
int launch(const TreeAttnArgs& a, cudaStream_t st) {
  auto k = tree_attention_kernel<D, INT8>;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kTaSmem<D>) != cudaSuccess) return 3000 + (int)cudaGetLastError();
  const int n_rt = (a.max_q * a.group + kTaRows - 1) / kTaRows;
  const cudaError_t e = launch_pdl(k, dim3(n_rt * a.nsplit, a.hkv, a.B), dim3(kTaThreads), (size_t)kTaSmem<D>, st, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace

int launch_tree_join(const TreeAttnArgs& a, cudaStream_t st) {
  auto k = a.D == 64 ? tree_join_kernel<64> : a.D == 128 ? tree_join_kernel<128> : tree_join_kernel<256>;
  const cudaError_t e = launch_pdl(k, dim3((unsigned)(((long long)a.T * a.hq + 3) / 4)), dim3(128), 0, st, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace xft

using namespace xft;

// See the file comment; `packed`: TreeAttnArgs.  Returns 0, -1 for an unsupported shape, or a CUDA error.
extern "C" int xft_tree_attention(const char* packed, cudaStream_t st) {
  TreeAttnArgs a;
  memcpy(&a, packed, sizeof(a));
  if (a.B <= 0 || a.T <= 0 || a.max_q <= 0) return 0;
  if (a.B > 65535 || a.max_q > 64 * a.words || a.words > kTreeWords || a.group < 1 || a.nsplit < 1 || a.nsplit > 64 ||
      (a.nsplit > 1 && (!a.part_o || !a.part_ml)) || (a.window > 0 && !a.positions) || a.bs < 1)
    return -1;
  int rc = -1;
  const bool i8 = a.ks != nullptr;
  if (a.form) rc = launch_tree_attention_tc(a, st);
  else if (a.D == 64) rc = i8 ? launch<64, true>(a, st) : launch<64, false>(a, st);
  else if (a.D == 128) rc = i8 ? launch<128, true>(a, st) : launch<128, false>(a, st);
  else if (a.D == 256) rc = i8 ? launch<256, true>(a, st) : launch<256, false>(a, st);
  return rc || a.nsplit == 1 ? rc : launch_tree_join(a, st);
}
