// A token per row of logits with the row's own temperature, top-k, top-p and min-p and a given uniform number u.
//
// Order a row by logit (largest first, of equal ones the lower index) and weigh w_i = exp((x_i - max) / T).  Kept are, of the first k,
// the elements with less than p of those k's mass in front of them, and of these the ones with w_i >= min_p; the token is the first
// element up to which more than u of the kept mass lies.  T <= 0: the first element.
//
// Each limit keeps a beginning of that order, so the smallest of the three masses is the mass of what all keep, and the token is the
// element of the whole row at which the running mass passes u times that.  Everything comes down to finding the place in the order
// where a count or a mass is reached; the row is never sorted.  Masses are whole numbers, 2^shift w, so their sums do not depend on an
// order.  They have to be exact to far below an element's share, or another token comes out than exact arithmetic's: tokens are equal
// but for a probability of about 2^-35 per kept element.
//
// A row's read is all the traffic, so it is read once, by a cluster whose CTAs hold a slice each in shared memory:
//   1. the largest logit, over the cluster;
//   2. a histogram of 1024 bins whose edges are even in the logit, 32 a factor of two in w (counts alone, 32 per logit, where k is small
//      enough for the next step to take all of the first k): a bin's mass is its middle's weight times the sum of 2^-e, e the distance
//      from the middle, by a polynomial, from a distance that is rounded to 2^-30 and not to a logit's 2^-20 (two numbers in 32 bits
//      carry it); the sums are two 32-bit atomics (one of 64 bits is a loop: 20 times slower);
//   3. the bins' sums, exchanged over the cluster; every CTA finds the bins where the limits and the token can lie;
//   4. those bins' elements, or all up to there if that is what at most 2048 are, go to the first CTA, which sorts them, weighs them in 64
//      bits and finds the place; one more such round for each limit whose elements are too many.
// What that does not settle (a bin of more than 2048 elements, as with equal logits, a limit among weights below 2^-32, a
// largest logit above 1e38) the first
// CTA settles alone, digit by digit of the 64-bit number (image of the logit, ~index), whose unsigned order is the row's.
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

typedef unsigned long long u64;
constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 1024, kSampleList = 2048;
constexpr float kSampleEdge = kSampleBins - 1.5f;        // from here on: the elements outside the bins
constexpr int kSampleUnit = 28;                          // a weight's factor in its bin has so many bits behind the point

// Unsigned order of the images is the order of the floats; NaN counts as -inf, -0 as 0
__device__ __forceinline__ float logit(float x) { return x == x ? x + 0.f : -INFINITY; }
__device__ __forceinline__ uint32_t image(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_image(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ u64 element(float x, unsigned i) { return (u64)image(logit(x)) << 32 | (0xffffffffu - i); }

struct SampleRow {
  const void* x;
  int V, bf16, shift;
  float top;
  double inv_t;
  __device__ float at(int i) const {
    return logit(bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i]) : static_cast<const float*>(x)[i]);
  }
  // exp((x - top) / T); a top of +inf leaves its equals alone, -inf weighs nothing
  __device__ double weight(float v) const {
    if (v == top) return 1.0;
    if (v == -INFINITY || top == INFINITY) return 0.0;
    return exp((static_cast<double>(v) - static_cast<double>(top)) * inv_t);
  }
  __device__ u64 mass(double w) const { return static_cast<u64>(__double2ll_rn(ldexp(w, shift))); }
};

struct SampleLimits { int k; float p, least, u; };

struct SampleShared {
  union {
    struct { unsigned cnt[kSampleBins], lo[kSampleBins], hi[kSampleBins]; } own;       // this CTA's slice
    u64 list[kSampleList];                               // the first CTA's, once the sums have been exchanged
    u64 fine[kSampleBins];                               // place()
  };
  u64 mass[kSampleBins];                                 // of the whole row
  unsigned cnt[kSampleBins];
  u64 warps[kSampleWarps], found[4];
  float top[16];                                         // of each CTA
  unsigned first[16];
  u64 over[16];
  unsigned n_list, at;
  int what, from, to;                                    // the next round: see Round
  u64 base;
};

enum Round { kDone, kAlone, kAll, kFirst, kShare, kLeast, kPick };

// Sum of v over the threads in front of this one and of all, in thread order
__device__ void scan(u64 v, u64* warps, u64& before, u64& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  if (lane == 31) warps[w] = s;
  __syncthreads();
  before = s - v;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSampleWarps; ++i) {
    if (i < w) before += warps[i];
    total += warps[i];
  }
  __syncthreads();
}

// -- alone --------------------------------------------------------------------------------------------------------------------------
// The place where the running count reaches `want` (by_mass false) or the running mass exceeds it; returns the mass up to and with the
// element there and its index.  `want` lies within the row's count or mass.
__device__ void place(const SampleRow& r, SampleShared& sh, bool by_mass, u64 want, u64& upto, unsigned& index) {
  const int tid = threadIdx.x;
  u64 prefix = 0, done_m = 0, done_c = 0;
  for (int bits = 0; bits < 64;) {
    const int take = min(10, 64 - bits), shift = 64 - bits - take;
    for (int i = tid; i < kSampleBins; i += kSampleThreads) { sh.cnt[i] = 0; sh.fine[i] = 0; }
    __syncthreads();
    for (int i = tid; i < r.V; i += kSampleThreads) {
      const float v = r.at(i);
      const u64 c = element(v, i);
      if (bits && (c >> (64 - bits)) != prefix) continue;
      const int bin = kSampleBins - 1 - (int)((c >> shift) & ((1u << take) - 1));         // descending order: bin 0 is the first
      atomicAdd(&sh.cnt[bin], 1u);
      const u64 m = r.mass(r.weight(v));
      if (m) atomicAdd(&sh.fine[bin], m);
    }
    __syncthreads();
    const unsigned c0 = sh.cnt[2 * tid], c1 = sh.cnt[2 * tid + 1];
    const u64 m0 = sh.fine[2 * tid], m1 = sh.fine[2 * tid + 1];
    u64 bc, bm, tc, tm;
    scan(c0 + c1, sh.warps, bc, tc);
    scan(m0 + m1, sh.warps, bm, tm);
    bc += done_c; bm += done_m;
    for (int e = 0; e < 2; ++e) {
      const unsigned c = e ? c1 : c0;
      const u64 m = e ? m1 : m0;
      const bool here = by_mass ? (bm <= want && bm + m > want) : (bc < want && bc + c >= want);
      if (here) { sh.found[0] = kSampleBins - 1 - (2 * tid + e); sh.found[1] = bm; sh.found[2] = bc; }
      bc += c; bm += m;
    }
    __syncthreads();
    prefix = bits ? (prefix << take | sh.found[0]) : sh.found[0];
    done_m = sh.found[1]; done_c = sh.found[2];
    bits += take;
    __syncthreads();
  }
  index = 0xffffffffu - (unsigned)(prefix & 0xffffffffu);
  upto = done_m + r.mass(r.weight(r.at((int)index)));
}

// Mass that a share of it has to reach, and that a token's running mass has to exceed
__device__ __forceinline__ u64 reach(float p, u64 mass) { return (u64)ceil(fmax((double)p, 0.0) * (double)mass); }
__device__ __forceinline__ u64 exceed(float u, u64 mass) {
  return min((u64)(fmin(u > 0.f ? (double)u : 0.0, 1.0 - 0x1p-24) * (double)mass), mass - 1);
}

__device__ unsigned alone(const SampleRow& r, SampleShared& sh, const SampleLimits& lim) {
  u64 all = 0, over = 0, before;
  for (int i = threadIdx.x; i < r.V; i += kSampleThreads) {
    const double w = r.weight(r.at(i));
    const u64 m = r.mass(w);
    all += m;
    if (w >= fmin((double)lim.least, 1.0)) over += m;
  }
  scan(all, sh.warps, before, all);
  scan(over, sh.warps, before, over);
  u64 kept = all, some;
  unsigned at;
  if (lim.k > 0 && lim.k < r.V) place(r, sh, false, lim.k, kept, at);
  some = kept;
  if (lim.p < 1.f) {
    const u64 want = reach(lim.p, kept);
    place(r, sh, true, want > 0 ? want - 1 : 0, some, at);
  }
  kept = min(kept, some);
  if (lim.least > 0.f) kept = min(kept, over);
  place(r, sh, true, exceed(lim.u, kept), some, at);
  return at;
}

// -- the elements of a round --------------------------------------------------------------------------------------------------------
__device__ void sort_list(u64* list, int n) {
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kSampleThreads) list[i] = 0;
  __syncthreads();
  for (int run = 2; run <= size; run <<= 1)
    for (int step = run >> 1; step > 0; step >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += kSampleThreads) {
        const int a = 2 * step * (i / step) + i % step, b = a + step;
        const u64 x = list[a], y = list[b];
        if ((x < y) == ((a & run) == 0)) { list[a] = y; list[b] = x; }
      }
      __syncthreads();
    }
}

// Where the sorted list's running mass (behind `base`) first reaches `want`, or with `pass` exceeds it: place and mass up to there; the
// last element if nowhere
struct ListMasses {
  u64 m[4], c[4];                                        // of the thread's four elements, and up to and with each
  int n;
  u64 end;
  __device__ ListMasses(const SampleRow& r, SampleShared& sh, int n_, u64 base, double* w) : n(n_) {
    u64 sum = 0, before;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = threadIdx.x * 4 + e;
      w[e] = i < n ? r.weight(from_image((uint32_t)(sh.list[i] >> 32))) : 0.0;
      m[e] = i < n ? r.mass(w[e]) : 0;
      sum += m[e];
    }
    scan(sum, sh.warps, before, end);
    end += base;
    before += base;
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = before += m[e];
  }
  // (the element, mass up to and with it), the same in every thread
  template <class F>
  __device__ void first(SampleShared& sh, F test, int& at, u64& upto) const {
    if (threadIdx.x == 0) { sh.found[0] = n - 1; sh.found[1] = end; }
    __syncthreads();
#pragma unroll
    for (int e = 3; e >= 0; --e) {
      const int i = threadIdx.x * 4 + e;
      // of neighbours that both pass, the one whose predecessor does not
      if (i < n && test(i, c[e]) && !(i > 0 && test(i - 1, c[e] - m[e]))) { sh.found[0] = i; sh.found[1] = c[e]; }
    }
    __syncthreads();
    at = (int)sh.found[0];
    upto = sh.found[1];
    __syncthreads();
  }
};

// The bin of the row's running mass: the first at whose end test(mass) holds; kSampleBins if none.  `before`: mass in front of it
template <class F>
__device__ int bin_of(SampleShared& sh, const u64 (&c)[2], const u64 (&m)[2], F test, u64& before) {
  if (threadIdx.x == 0) sh.found[2] = kSampleBins;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (test(c[e]) && !(threadIdx.x + e > 0 && test(c[e] - m[e]))) { sh.found[2] = 2 * threadIdx.x + e; sh.found[3] = c[e] - m[e]; }
  __syncthreads();
  const int b = (int)sh.found[2];
  before = sh.found[3];
  __syncthreads();
  return b;
}

template <int C>
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  if (C > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
}
__device__ __forceinline__ void st_peer(const void* own, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dsmem_addr(smem_u32(own), rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void st_peer(const void* own, uint32_t rank, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dsmem_addr(smem_u32(own), rank)), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_peer(const void* own, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(dsmem_addr(smem_u32(own), rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t add_peer(const void* own, uint32_t rank, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(dsmem_addr(smem_u32(own), rank)), "r"(v) : "memory");
  return old;
}

// C CTAs a row.  HELD: the slices fit in shared memory
template <int C, bool HELD>
__global__ void __launch_bounds__(kSampleThreads) sample_rows_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) float slice[];
  __shared__ SampleShared sh;
  grid_dep_launch();
  grid_dep_wait();
  const int tid = threadIdx.x, lane = tid & 31;
  const int row = blockIdx.x / C;
  const uint32_t rank = C > 1 ? cluster_ctarank() : 0;
  SampleRow r;
  r.x = a.bf16 ? (const void*)(static_cast<const __nv_bfloat16*>(a.x) + row * a.ld) : (const void*)(static_cast<const float*>(a.x) + row * a.ld);
  r.V = a.V; r.bf16 = a.bf16;
  r.shift = min(45, 62 - (32 - __clz(a.V)));
  // the slice: groups of four that start on 16 bytes where the row's do; `skew` elements of the first group are in front of the row
  const int skew = a.bf16 ? 0 : (int)(reinterpret_cast<uintptr_t>(r.x) >> 2 & 3);
  const int groups = (a.V + skew + 3) / 4, per = (groups + C - 1) / C;
  const int g0 = min(groups, (int)rank * per), ng = min(groups, g0 + per) - g0;
  const float* xf = static_cast<const float*>(r.x) - skew;
  auto fetch = [&](int g) -> float4 {                    // group g of the row; what is not the row's is -inf
    const int i = 4 * g - skew;
    if (!a.bf16 && i >= 0 && i + 4 <= a.V) return __ldg(reinterpret_cast<const float4*>(xf + 4 * g));
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e >= 0 && i + e < a.V ? r.at(i + e) : -INFINITY;
    return make_float4(v[0], v[1], v[2], v[3]);
  };
  auto group = [&](int j) -> float4 { return HELD ? reinterpret_cast<const float4*>(slice)[j] : fetch(g0 + j); };
  float top = -INFINITY;
#pragma unroll 8
  for (int j = tid; j < ng; j += kSampleThreads) {
    const float4 v = fetch(g0 + j);
    if (HELD) reinterpret_cast<float4*>(slice)[j] = v;
    top = fmaxf(fmaxf(fmaxf(top, v.x), fmaxf(v.y, v.z)), v.w);
  }
  for (int i = tid; i < kSampleBins; i += kSampleThreads) sh.own.cnt[i] = sh.own.lo[i] = sh.own.hi[i] = 0;
  if (tid == 0) sh.n_list = 0;
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) sh.warps[tid >> 5] = __float_as_uint(top);
  __syncthreads();
  for (int i = 0; i < kSampleWarps; ++i) top = fmaxf(top, __uint_as_float((uint32_t)sh.warps[i]));
  if (tid < C) st_peer(&sh.top[rank], tid, __float_as_uint(top));
  cluster_barrier<C>();
  for (int i = 0; i < C; ++i) top = fmaxf(top, sh.top[i]);
  top += 0.f;
  r.top = top;

  const float t = a.temperature ? a.temperature[row] : a.t0;
  SampleLimits lim;
  lim.k = a.top_k ? a.top_k[row] : a.k0;
  lim.p = a.top_p ? a.top_p[row] : a.p0;
  lim.least = a.min_p ? a.min_p[row] : a.m0;
  lim.u = a.uniform[row];
  if (lim.k >= a.V) lim.k = 0;
  if (top == -INFINITY) {
    if (rank == 0 && tid == 0) a.out[row] = -1;
    return;                                              // (no CTA looks into another's memory from here on)
  }
  if (!(t > 0.f)) {                                      // the first of the largest
    unsigned first = 0xffffffffu;
    for (int j = tid; j < ng; j += kSampleThreads) {
      const float4 v = group(j);
      const int i = 4 * (g0 + j) - skew;
      if (first == 0xffffffffu)
        first = v.x == top ? i : v.y == top ? i + 1 : v.z == top ? i + 2 : v.w == top ? i + 3 : 0xffffffffu;
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.warps[tid >> 5] = first;
    __syncthreads();
    if (tid == 0) {
      for (int i = 0; i < kSampleWarps; ++i) first = min(first, (unsigned)sh.warps[i]);
      st_peer(&sh.first[rank], 0, first);
    }
    cluster_barrier<C>();
    if (rank == 0 && tid == 0) {
      for (int i = 0; i < C; ++i) first = min(first, sh.first[i]);
      a.out[row] = first;
    }
    return;
  }
  r.inv_t = 1.0 / (double)t;
  const bool counts = lim.k > 0 && lim.k <= kSampleList;           // all of the first k are sorted
  const double per_octave = 32.0 * 1.4426950408889634 * r.inv_t;
  const float kh = counts ? 32.f : (float)per_octave, kl = counts ? 0.f : (float)(per_octave - (double)kh);
  // distance from the largest in bins, and the same in every pass: rounding does not change the order of two logits
  auto distance = [&](float x) { return __fmul_rn(__fsub_rn(top, x), kh); };
  constexpr float kMagic = 12582912.f;                   // 1.5 * 2^23: what is added to it is rounded to a whole number
  auto bin_at = [&](float d) { return (int)(__float_as_uint(__fadd_rn(d, kMagic)) - 0x4b400000u); };
  u64 over = 0;
  const bool huge = top > 1e38f;                         // a difference can be above what 32 bits hold
  if (huge) {
    // settled alone
  } else if (counts) {
    for (int j = tid; j < ng; j += kSampleThreads) {
      const float4 v = group(j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d = distance((&v.x)[e]);
        if (d < kSampleEdge) atomicAdd(&sh.own.cnt[bin_at(d)], 1u);
      }
    }
  } else {
    const bool both = lim.k > 0;
    for (int j = tid; j < ng; j += kSampleThreads) {
      const float4 v = group(j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = (&v.x)[e], s = __fsub_rn(top, x), d = __fmul_rn(s, kh);
        if (d < kSampleEdge) {
          // s + low is top - x, d + rest that in bins
          const float back = __fsub_rn(s, top), low = __fadd_rn(__fsub_rn(top, __fsub_rn(s, back)), __fsub_rn(-x, back));
          const float rest = fmaf(low, kh, fmaf(s, kl, fmaf(s, kh, -d)));
          const float whole = __fadd_rn(d, kMagic), off = __fadd_rn(__fsub_rn(d, __fsub_rn(whole, kMagic)), rest);
          const int n = (int)(__float_as_uint(whole) - 0x4b400000u);
          // 2^(-off / 32) - 1, |off| <= 1/2: (ln2 / 32)^i / i! off^i
          const float q = off * fmaf(off, fmaf(off, fmaf(off, 9.17256e-9f, -1.69385098e-6f), 2.34596198e-4f), -2.16608494e-2f);
          const unsigned w = __float_as_uint(fmaf(q, (float)(1 << kSampleUnit), kMagic)) - 0x4b400000u + (1u << kSampleUnit);
          atomicAdd(&sh.own.lo[n], w & 0x3fffu);
          atomicAdd(&sh.own.hi[n], w >> 14);
          if (both) atomicAdd(&sh.own.cnt[n], 1u);
        } else {
          over += __float2uint_rn(exp2f((float)r.shift - d * (1.f / 32)));         // below 2^-31: a logit's rounding does not count
        }
      }
    }
  }
  for (int o = 16; o > 0; o >>= 1) over += __shfl_xor_sync(0xffffffffu, over, o);
  if (lane == 0) sh.warps[tid >> 5] = over;
  __syncthreads();
  if (tid < C) {
    over = 0;
    for (int i = 0; i < kSampleWarps; ++i) over += sh.warps[i];
    st_peer(&sh.over[rank], tid, over);
  }
  cluster_barrier<C>();
  // every CTA sums its share of the bins over the cluster and hands it to all
  for (int i = tid; i < kSampleBins / C; i += kSampleThreads) {
    const int n = rank * (kSampleBins / C) + i;
    unsigned cnt = 0;
    u64 w = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      cnt += ld_peer(&sh.own.cnt[n], c);
      if (!counts) w += ((u64)ld_peer(&sh.own.hi[n], c) << 14) + ld_peer(&sh.own.lo[n], c);
    }
    const u64 m = counts ? 0 : (u64)__double2ll_rn(exp2((double)r.shift - kSampleUnit - n * (1.0 / 32)) * (double)w);
    // without counts, what a bin holds at most: its weights' factors are within 1.1 % of one
    if (!counts && lim.k <= 0) cnt = (unsigned)((w + (w >> 6) + (1u << (kSampleUnit - 1))) >> kSampleUnit);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      st_peer(&sh.cnt[n], c, cnt);
      st_peer(&sh.mass[n], c, m);
    }
  }
  cluster_barrier<C>();
  // running counts and masses, two bins a thread
  u64 mass[2], upto[2], cnt[2], count[2], before, total, many;
#pragma unroll
  for (int e = 0; e < 2; ++e) { mass[e] = sh.mass[2 * tid + e]; cnt[e] = sh.cnt[2 * tid + e]; }
  scan(cnt[0] + cnt[1], sh.warps, before, many);
  count[0] = before + cnt[0]; count[1] = count[0] + cnt[1];
  scan(mass[0] + mass[1], sh.warps, before, total);
  upto[0] = before + mass[0]; upto[1] = upto[0] + mass[1];
  for (int i = 0; i < C; ++i) total += sh.over[i];
  u64 kept = total;                                      // (the first CTA's; the others know the first round only)
  // the bins in which an element that weighs `least` can be
  const float least = lim.least > 0.f ? fminf(lim.least, 1.f) : 0.f;
  const float d_least = least > 0.f ? -32.f * log2f(least) : INFINITY;
  const int n_least = d_least < kSampleEdge - 1.f ? (int)rintf(d_least) : kSampleBins;
  auto next = [&](int done) -> int4 {                    // the round behind `done`: (what, first bin, last bin), base in sh.base
    u64 base = 0;
    if (done < kFirst && lim.k > 0) {
      const int b = bin_of(sh, count, cnt, [&](u64 c) { return c >= (u64)lim.k; }, base);
      if (b == kSampleBins) return make_int4(kAlone, 0, 0, 0);
      const int in = (int)base;
      if (2 * tid <= b && b < 2 * tid + 2) sh.base = upto[b & 1] - mass[b & 1];
      __syncthreads();
      return make_int4(kFirst, b, b, in);
    }
    if (done < kShare && lim.p < 1.f) {
      const u64 want = max(reach(lim.p, kept), (u64)1);
      const int b = bin_of(sh, upto, mass, [&](u64 c) { return c >= want; }, base);
      if (b == kSampleBins) return make_int4(kAlone, 0, 0, 0);
      if (2 * tid <= b && b < 2 * tid + 2) { sh.base = upto[b & 1] - mass[b & 1]; sh.found[0] = count[b & 1]; }
      __syncthreads();
      const bool all = lim.k <= 0 && sh.found[0] <= kSampleList;
      __syncthreads();
      return all ? make_int4(kAll, 0, b, 0) : make_int4(kShare, b, b, 0);
    }
    if (done < kLeast && least > 0.f) {
      const int b = max(0, min(n_least, kSampleBins) - 1), e = min(kSampleBins - 1, n_least + 1);
      if (2 * tid <= b && b < 2 * tid + 2) sh.base = upto[b & 1] - mass[b & 1];
      if (2 * tid <= e && e < 2 * tid + 2) sh.found[0] = count[e & 1];
      __syncthreads();
      const bool all = lim.k <= 0 && !(lim.p < 1.f) && sh.found[0] <= kSampleList, idle = sh.base >= kept;
      __syncthreads();
      if (!idle && n_least == kSampleBins) return make_int4(kAlone, 0, 0, 0);
      if (!idle && all) return make_int4(kAll, 0, e, 0);
      if (!idle) return make_int4(kLeast, b, e, 0);
    }
    const u64 want = exceed(lim.u, kept);
    const int b = bin_of(sh, upto, mass, [&](u64 c) { return c > want; }, base);
    if (b == kSampleBins) return make_int4(kAlone, 0, 0, 0);
    if (2 * tid <= b && b < 2 * tid + 2) sh.base = upto[b & 1] - mass[b & 1];
    __syncthreads();
    return make_int4(kPick, b, b, 0);
  };
  int4 todo;
  if (huge) todo = make_int4(kAlone, 0, 0, 0);
  else if (counts) {
    u64 base;
    const int b = bin_of(sh, count, cnt, [&](u64 c) { return c >= (u64)lim.k; }, base);
    todo = b == kSampleBins ? make_int4(kAlone, 0, 0, 0) : make_int4(kAll, 0, b, 0);
  } else todo = next(kDone);
  while (todo.x > kAlone) {
    // the bins' elements go to the first CTA
    for (int j0 = 0; j0 < ng; j0 += kSampleThreads) {
      const int j = j0 + tid;
      float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (j < ng) v = group(j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d = distance((&v.x)[e]);
        bool in = d < kSampleEdge;
        if (in) {
          const int n = bin_at(d);
          in = n >= todo.y && n <= todo.z;
        }
        const unsigned who = __ballot_sync(0xffffffffu, in);
        if (who) {
          unsigned to = 0;
          if (lane == 0) to = add_peer(&sh.n_list, 0, __popc(who));
          to = __shfl_sync(0xffffffffu, to, 0) + __popc(who & ((1u << lane) - 1u));
          if (in && to < kSampleList) st_peer(&sh.list[to], 0, element((&v.x)[e], 4 * (g0 + j) - skew + e));
        }
      }
    }
    cluster_barrier<C>();
    if (rank == 0) {
      const int n = (int)sh.n_list;
      if (n > kSampleList || n < 1) {
        todo = make_int4(kAlone, 0, 0, 0);
      } else {
        sort_list(sh.list, n);
        const u64 base = todo.x == kAll ? 0 : sh.base;
        double w[4];
        const ListMasses l(r, sh, n, base, w);
        int at;
        u64 m;
        if (todo.x == kAll) {
          if (lim.k > 0) l.first(sh, [&](int i, u64) { return i + 1 >= lim.k; }, at, kept);
          u64 some = kept;
          if (lim.p < 1.f) {
            const u64 want = max(reach(lim.p, kept), (u64)1);
            l.first(sh, [&](int, u64 c) { return c >= want; }, at, some);
          }
          if (least > 0.f) {                             // mass of what weighs enough
            u64 mine = 0, b4, over_m;
#pragma unroll
            for (int e = 0; e < 4; ++e) mine += w[e] >= (double)least ? l.m[e] : 0;
            scan(mine, sh.warps, b4, over_m);
            some = min(some, over_m);
          }
          kept = min(kept, some);
        } else if (todo.x == kFirst) {
          l.first(sh, [&](int i, u64) { return i + 1 >= lim.k - todo.w; }, at, kept);
        } else if (todo.x == kShare) {
          const u64 want = max(reach(lim.p, kept), (u64)1);
          l.first(sh, [&](int, u64 c) { return c >= want; }, at, m);
          kept = min(kept, m);
        } else if (todo.x == kLeast) {
          u64 mine = 0, b4, over_m;
#pragma unroll
          for (int e = 0; e < 4; ++e) mine += w[e] >= (double)least ? l.m[e] : 0;
          scan(mine, sh.warps, b4, over_m);
          kept = min(kept, base + over_m);
        }
        if (todo.x == kAll || todo.x == kPick) {
          const u64 want = exceed(lim.u, kept);
          l.first(sh, [&](int, u64 c) { return c > want; }, at, m);
          if (tid == 0) a.out[row] = 0xffffffffu - (unsigned)(sh.list[at] & 0xffffffffu);
          todo = make_int4(kDone, 0, 0, 0);
        } else {
          todo = next(todo.x);
        }
      }
      __syncthreads();
      if (tid == 0) sh.n_list = 0;
      if (tid < C) {
        st_peer(&sh.what, tid, (uint32_t)todo.x);
        st_peer(&sh.from, tid, (uint32_t)todo.y);
        st_peer(&sh.to, tid, (uint32_t)todo.z);
      }
    }
    cluster_barrier<C>();
    if (rank != 0) todo = make_int4(sh.what, sh.from, sh.to, 0);
  }
  if (todo.x == kAlone && rank == 0) {
    __syncthreads();
    const unsigned at = alone(r, sh, lim);
    if (tid == 0) a.out[row] = at;
  }
}

template <int C, bool HELD>
int launch(const SampleArgs& a, cudaStream_t st) {
  auto k = sample_rows_kernel<C, HELD>;
  const int groups = (a.V + 3 + 3) / 4, bytes = HELD ? (groups + C - 1) / C * 16 : 0;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return 3000 + (int)cudaGetLastError();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * C);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_xft_pdl ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace
}  // namespace xft

using namespace xft;

// See the file comment; `packed`: SampleArgs.  Rows without a logit above -inf give -1.
extern "C" int xft_sample_rows(const char* packed, cudaStream_t st) {
  SampleArgs a;
  memcpy(&a, packed, sizeof(a));
  if (a.rows <= 0) return 0;
  if (a.V < 1 || a.V > (1 << 24) || a.rows > (1 << 27)) return -1;
  // slices of at most 19 Ki elements leave room for two CTAs per SM; few rows are cut finer
  if (a.V <= 4096) return launch<1, true>(a, st);
  if (a.V <= 19456 && a.rows >= 296) return launch<1, true>(a, st);
  if (a.V <= 8 * 45056) return launch<8, true>(a, st);
  return launch<8, false>(a, st);
}
