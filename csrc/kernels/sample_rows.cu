// A token per row of logits with the row's own temperature, top-k, top-p and min-p and a given uniform number u.
//
// Order a row by logit (largest first, of equal ones the lower index) and weigh w_i = exp((x_i - max) / T).  Kept are, of the first k,
// the elements with less than p of those k's mass in front of them, and of these the ones with w_i >= min_p; the token is the first
// element up to which more than u of the kept mass lies.  T <= 0: the first element.
//
// Each limit keeps a beginning of that order, so the smallest of the three masses is the mass of what all keep, and the token is the
// element of the whole row at which the running mass passes u times that.  Everything comes down to finding the place in the order
// where a count or a mass is reached; the row is never sorted.  Masses are whole numbers, 2^shift w rounded, w in 64 bits: their sums
// do not depend on an order, and with shift 45 (rows of up to 2^17; one less for each doubling) the rounding of a sum of V of them is
// below 2^-36 of it on average, so a token differs from exact arithmetic's with a probability of about 2^-36 per kept element.
//
// A place is found digit by digit of the 64-bit number (image of the logit, ~index), whose unsigned order is the row's: counts and
// masses of 2048 bins of the elements that agree with the digits so far, until one is left.
#include "ptx.cuh"

namespace xft {

struct SampleArgs {
  const void* x;             // [rows, V] fp32 or bf16
  const float* temperature;  // [rows], or null: the scalar below
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;      // [rows]
  long long* out;            // [rows]
  long long ld;              // elements between rows
  int rows, V, bf16, k0;
  float t0, p0, m0;
};

namespace {

constexpr int kSampleThreads = 1024;
constexpr int kSampleBins = 2048;
typedef unsigned long long u64;

// Unsigned order of the images is the order of the floats; NaN counts as -inf, -0 as 0
__device__ __forceinline__ float logit(float x) { return x == x ? x + 0.f : -INFINITY; }
__device__ __forceinline__ uint32_t image(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct SampleRow {
  const void* x;
  int V, bf16, shift;
  float top;
  double inv_t;
  __device__ float at(int i) const {
    return logit(bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i]) : static_cast<const float*>(x)[i]);
  }
  // 2^shift exp((x - top) / T); a top of +inf leaves its equals alone, -inf weighs nothing
  __device__ double weight(float v) const {
    if (v == top) return 1.0;
    if (v == -INFINITY || top == INFINITY) return 0.0;
    return exp((static_cast<double>(v) - static_cast<double>(top)) * inv_t);
  }
  __device__ u64 mass(float v) const { return static_cast<u64>(__double2ll_rn(ldexp(weight(v), shift))); }
};

struct SampleShared {
  unsigned cnt[kSampleBins];
  u64 mass[kSampleBins];
  u64 warp_c[32], warp_m[32];
  u64 found[4];
};

// Sum of v over the threads in front of this one and of all, in thread order
__device__ void scan(u64 v, u64* warps, u64& before, u64& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  u64 s = v;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  if (lane == 31) warps[w] = s;
  __syncthreads();
  before = s - v;
  total = 0;
  for (int i = 0; i < kSampleThreads / 32; ++i) {
    if (i < w) before += warps[i];
    total += warps[i];
  }
  __syncthreads();
}

// The place where the running count reaches `want` (by_mass false) or the running mass exceeds it; returns the mass up to and with the
// element there and its index.  `want` lies within the row's count or mass.
__device__ void place(const SampleRow& r, SampleShared& sh, bool by_mass, u64 want, u64& upto, unsigned& index) {
  const int tid = threadIdx.x;
  u64 prefix = 0, done_m = 0, done_c = 0;
  for (int bits = 0; bits < 64;) {
    const int take = min(11, 64 - bits), shift = 64 - bits - take;
    for (int i = tid; i < kSampleBins; i += kSampleThreads) { sh.cnt[i] = 0; sh.mass[i] = 0; }
    __syncthreads();
    for (int i = tid; i < r.V; i += kSampleThreads) {
      const float v = r.at(i);
      const u64 c = (u64)image(v) << 32 | (0xffffffffu - (unsigned)i);
      if (bits && (c >> (64 - bits)) != prefix) continue;
      const int bin = kSampleBins - 1 - (int)((c >> shift) & ((1u << take) - 1));         // descending order: bin 0 is the first
      atomicAdd(&sh.cnt[bin], 1u);
      const u64 m = r.mass(v);
      if (m) atomicAdd(&sh.mass[bin], m);
    }
    __syncthreads();
    // two bins a thread
    const unsigned c0 = sh.cnt[2 * tid], c1 = sh.cnt[2 * tid + 1];
    const u64 m0 = sh.mass[2 * tid], m1 = sh.mass[2 * tid + 1];
    u64 bc, bm, tc, tm;
    scan(c0 + c1, sh.warp_c, bc, tc);
    scan(m0 + m1, sh.warp_m, bm, tm);
    bc += done_c; bm += done_m;
    for (int e = 0; e < 2; ++e) {
      const unsigned c = e ? c1 : c0;
      const u64 m = e ? m1 : m0;
      const bool here = by_mass ? (bm <= want && bm + m > want) : (bc < want && bc + c >= want);
      if (here) { sh.found[0] = kSampleBins - 1 - (2 * tid + e); sh.found[1] = bm; sh.found[2] = bc; sh.found[3] = c; }
      bc += c; bm += m;
    }
    __syncthreads();
    prefix = bits ? (prefix << take | sh.found[0]) : sh.found[0];
    done_m = sh.found[1]; done_c = sh.found[2];
    bits += take;
    __syncthreads();
  }
  index = 0xffffffffu - (unsigned)(prefix & 0xffffffffu);
  upto = done_m + r.mass(r.at((int)index));
}

__global__ void __launch_bounds__(kSampleThreads) sample_rows_kernel(const SampleArgs a) {
  __shared__ SampleShared sh;
  grid_dep_launch();
  grid_dep_wait();
  const int row = blockIdx.x, tid = threadIdx.x;
  SampleRow r;
  r.x = a.bf16 ? (const void*)(static_cast<const __nv_bfloat16*>(a.x) + row * a.ld) : (const void*)(static_cast<const float*>(a.x) + row * a.ld);
  r.V = a.V; r.bf16 = a.bf16;
  r.shift = min(45, 62 - (32 - __clz(a.V)));
  u64 best = 0;                                                        // image and ~index of the first element
  for (int i = tid; i < a.V; i += kSampleThreads) best = max(best, (u64)image(r.at(i)) << 32 | (0xffffffffu - (unsigned)i));
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) sh.warp_c[tid >> 5] = best;
  __syncthreads();
  for (int i = 0; i < kSampleThreads / 32; ++i) best = max(best, sh.warp_c[i]);
  __syncthreads();
  const unsigned first = 0xffffffffu - (unsigned)best;
  r.top = r.at((int)first);
  const float t = a.temperature ? a.temperature[row] : a.t0;
  if (r.top == -INFINITY || !(t > 0.f)) {
    if (tid == 0) a.out[row] = r.top == -INFINITY ? -1 : (long long)first;
    return;
  }
  r.inv_t = 1.0 / (double)t;
  const int k = a.top_k ? a.top_k[row] : a.k0;
  const float p = a.top_p ? a.top_p[row] : a.p0, least = a.min_p ? a.min_p[row] : a.m0;
  // masses of the row and of what min-p keeps
  u64 all = 0, over = 0, before;
  for (int i = tid; i < a.V; i += kSampleThreads) {
    const float v = r.at(i);
    const double w = r.weight(v);
    const u64 m = static_cast<u64>(__double2ll_rn(ldexp(w, r.shift)));
    all += m;
    if (w >= fmin((double)least, 1.0)) over += m;
  }
  scan(all, sh.warp_c, before, all);
  scan(over, sh.warp_m, before, over);
  u64 kept = all;
  unsigned at;
  if (k > 0 && k < a.V) place(r, sh, false, k, kept, at);
  u64 some = kept;
  if (p < 1.f) {                                                       // the first element whose running mass reaches p times the mass
    const u64 want = (u64)ceil(fmax((double)p, 0.0) * (double)kept);
    place(r, sh, true, want > 0 ? want - 1 : 0, some, at);
  }
  kept = min(kept, some);
  if (least > 0.f) kept = min(kept, over);
  const float u = a.uniform[row];
  const u64 want = min((u64)(fmin(u > 0.f ? (double)u : 0.0, 1.0 - 0x1p-24) * (double)kept), kept - 1);
  place(r, sh, true, want, some, at);
  if (tid == 0) a.out[row] = at;
}

}  // namespace
}  // namespace xft

using namespace xft;

// See the file comment; `packed`: SampleArgs.  Rows without a logit above -inf give -1.
extern "C" int xft_sample_rows(const char* packed, cudaStream_t st) {
  SampleArgs a;
  memcpy(&a, packed, sizeof(a));
  if (a.rows <= 0) return 0;
  if (a.V < 1 || a.V > (1 << 24)) return -1;
  const cudaError_t e = launch_pdl(sample_rows_kernel, dim3(a.rows), dim3(kSampleThreads), 0, st, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
