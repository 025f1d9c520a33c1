// A token per row of logits with the row's own temperature, top-k, top-p and min-p and a given uniform number u.
//
// Order a row by logit (largest first, of equal ones the lower index) and weigh w_i = exp((x_i - max) / T).  Kept are, of the first k,
// the elements with less than p of those k's mass in front of them, and of these the ones with w_i >= min_p; the token is the first
// element up to which more than u of the kept mass lies.  T <= 0: the first element.
//
// Each limit keeps a beginning of that order, so the smallest of the three masses is the mass of what all keep, and the token is the
// element of the whole row at which the running mass passes u times that.  Everything comes down to finding the place in the order
// where a count or a mass is reached; the row is never sorted.  Masses are whole numbers, 2^shift w, so their sums do not depend on an
// order, and shares of them are taken in whole numbers, so that equal logits share evenly.  They have to be exact to far below an element's
// share, or another token comes out than exact arithmetic's.  A weight of an element that a round gathers is one of 64 bits; the other bins'
// sums are off by up to 2^-27.4 of each weight, by the same in a bin of equal logits, less the more different ones there are.  Of 5.5 million
// rows of 1 to 2 million logits, a tenth of them with u within 10^-6 of 1, where borders are dense, 84 tokens were others than in 64 bits: those whose
// border lay within 2^-34 of the kept mass from u, and one, in a row of a million logits of few values, 2^-30.
//
// A row is read from memory by a cluster of up to 8 CTAs with a slice each, which few rows' CTAs hold in shared memory.  Many rows' read
// theirs again for the few elements of step 3, from L2 as far as it holds them (512 rows of 151936, top-p: 717 MB from HBM for 311 MB):
//   1. a histogram of each slice, 1024 bins down from about the slice's largest logit on a grid that is the same for the whole row, 16 bins
//      a factor of two in w (counts alone, 16 bins per logit, where k is small enough for step 3 to take all of the first k): a bin's mass is
//      its middle's weight times the sum of 2^e, e the distance from the middle in octaves, by a polynomial, from a distance that is
//      good to 2^-30 (two numbers in 32 bits carry it); the sums are two 32-bit atomics (one of 64 bits in shared memory is a loop: 20
//      times slower).  What weighs less than 2^-48 of the largest is left out;
//   2. the bins' sums, exchanged over the cluster; every CTA finds the bins where the limits and the token can lie;
//   3. those bins' elements, or all up to there if those are at most 2048, go to the first CTA, which sorts them, weighs them in 64
//      bits and finds the place; one more such round for each limit whose elements are too many.  A bin of more than 2048 at the place of a
//      k above 1536, of a share or of the token is cut in 1024 parts in the same way first.  The other CTAs leave before the last round.
// What that does not settle the first CTA settles alone, digit by digit of the 64-bit number (image of the logit, ~index), whose unsigned
// order is the row's: more than 2048 equal logits or nearly so at such a place; more than 2048 within 1/16 of a logit where a k of up to 1536
// ends; more than 2048 in the three bins around the weight min_p; a limit among weights that are left out; logits of which a bin is
// less than 32 bits resolve.  us: a row of 32000 equal logits 260, of 152064 1210; min-p of 0.02 to 0.1 at T = 2 to 3 over 128256
// normal logits of deviation 2.2, whose border is so crowded, 680, 64 such rows 790 (T = 1.5: 28 and 63).
//
// Bound by the serial steps of a cluster where rows are few (a row of 32000 10.7 us), by instructions and the atomics where they are many (512
// rows of 151936, top-p, 295 us, their bytes take 48: 75 instructions a logit in all, of which its place in the bins and its weight there take 27, the
// rest are the atomics, the search for the largest and two more passes for the elements of the share and of the token).
#include "ptx.cuh"

#include <type_traits>

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
constexpr int kSampleBins = 1024, kSampleList = 2048, kSampleFirst = 1536;             // counts alone up to the last (bins come whole)
constexpr float kSampleEdge = kSampleBins - 1.5f;        // from here on: the elements outside the bins
constexpr int kSamplePer = 16;                           // bins an octave, or a logit
constexpr int kSampleUnit = 27;                          // a weight's factor in its bin has so many bits behind the point

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
  int V, bf16;
  float top;
  double inv_t, unit;                                    // mass of the weight 1
  __device__ float at(int i) const {
    return logit(bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i]) : static_cast<const float*>(x)[i]);
  }
  // exp((x - top) / T); a top of +inf leaves its equals alone, -inf weighs nothing
  __device__ double weight(float v) const {
    if (v == top) return 1.0;
    if (v == -INFINITY || top == INFINITY) return 0.0;
    return exp((static_cast<double>(v) - static_cast<double>(top)) * inv_t);
  }
  __device__ u64 mass(double w) const { return __double2ull_rn(w * unit); }
};

struct SampleLimits { int k; float p, least, u; };

struct SampleShared {
  union {
    struct { unsigned cnt[kSampleBins], lo[kSampleBins], hi[kSampleBins], zoom_cnt[kSampleBins]; u64 zoom_mass[kSampleBins]; } own;        // this CTA's
                                                         // slice; the first CTA's: of one bin, cut into 1024
    u64 list[kSampleList];                               // the first CTA's, once the sums have been exchanged
    struct { unsigned lo[kSampleBins], hi[kSampleBins]; } fine;          // place()
  };
  u64 mass[kSampleBins];                                 // of the whole row
  unsigned cnt[kSampleBins];
  u64 warps[kSampleWarps], found[4], kept;
  unsigned warp_counts[kSampleWarps];
  float top[8], ref[8];                                  // of each CTA: its slice's largest logit, and where its bins begin
  u64 first[8];
  double root[kSamplePer];                               // 2^(-i / 16)
  int above;
  unsigned n_list, at;
  int what, from, to, sub;                               // the next round: see Round
  u64 base;
  u64 rest;                                              // of the bins' mass, beside the first round's elements
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

// The same of a count and a mass
__device__ void scan2(unsigned c, u64 m, SampleShared& sh, unsigned& before_c, u64& before_m, u64& total_m) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  unsigned sc = c;
  u64 sm = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned tc = __shfl_up_sync(0xffffffffu, sc, o);
    const u64 tm = __shfl_up_sync(0xffffffffu, sm, o);
    if (lane >= o) { sc += tc; sm += tm; }
  }
  if (lane == 31) { sh.warps[w] = sm; sh.warp_counts[w] = sc; }
  __syncthreads();
  before_c = sc - c; before_m = sm - m; total_m = 0;
#pragma unroll
  for (int i = 0; i < kSampleWarps; ++i) {
    if (i < w) { before_c += sh.warp_counts[i]; before_m += sh.warps[i]; }
    total_m += sh.warps[i];
  }
  __syncthreads();
}

// -- alone --------------------------------------------------------------------------------------------------------------------------
// The place where the running count reaches `want` (by_mass false) or the running mass exceeds it; returns the mass up to and with the
// element there and its index.  `want` lies within the row's count or mass.
__device__ __noinline__ void place(const SampleRow& r, SampleShared& sh, bool by_mass, u64 want, u64& upto, unsigned& index) {
  const int tid = threadIdx.x;
  u64 prefix = 0, done_m = 0, done_c = 0;
  for (int bits = 0; bits < 64;) {
    const int take = min(10, 64 - bits), shift = 64 - bits - take;
    for (int i = tid; i < kSampleBins; i += kSampleThreads) { sh.cnt[i] = 0; sh.fine.lo[i] = sh.fine.hi[i] = 0; }
    __syncthreads();
    for (int i = tid; i < r.V; i += kSampleThreads) {
      const float v = r.at(i);
      const u64 c = element(v, i);
      if (bits && (c >> (64 - bits)) != prefix) continue;
      const int bin = kSampleBins - 1 - (int)((c >> shift) & ((1u << take) - 1));         // descending order: bin 0 is the first
      atomicAdd(&sh.cnt[bin], 1u);
      const u64 m = r.mass(r.weight(v));
      if (m) {
        const unsigned add = (unsigned)m, old = atomicAdd(&sh.fine.lo[bin], add);
        const unsigned up = (unsigned)(m >> 32) + (old + add < add);
        if (up) atomicAdd(&sh.fine.hi[bin], up);
      }
    }
    __syncthreads();
    const unsigned c0 = sh.cnt[2 * tid], c1 = sh.cnt[2 * tid + 1];
    const u64 m0 = (u64)sh.fine.hi[2 * tid] << 32 | sh.fine.lo[2 * tid], m1 = (u64)sh.fine.hi[2 * tid + 1] << 32 | sh.fine.lo[2 * tid + 1];
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

// f * mass, 0 <= f < 1, in whole numbers: down, or up.  (A product in 64-bit floats is off by more than nothing where a share ends between two of
// many equal logits, and that decides which of them it is.)
__device__ u64 share(float f, u64 mass, bool up) {
  const uint32_t bits = __float_as_uint(f), e = max(bits >> 23, 1u), digits = bits >> 23 ? (bits & 0x7fffffu) | 0x800000u : bits;
  const u64 lo = mass * digits, hi = __umul64hi(mass, digits);             // f = digits 2^(e - 150)
  const int by = 150 - (int)e;                           // at least 24, and hi is below 2^24
  const u64 whole = by < 64 ? hi << (64 - by) | lo >> by : by < 128 ? hi >> (by - 64) : 0;
  const u64 rest = by < 64 ? lo << (64 - by) : by == 64 ? lo : by < 128 ? lo | hi << (128 - by) : lo | hi;
  return whole + (up && rest != 0);
}
// Mass that a share of it has to reach, and that a token's running mass has to exceed
__device__ __forceinline__ u64 reach(float p, u64 mass) { return p > 0.f ? share(p, mass, true) : 0; }
__device__ __forceinline__ u64 exceed(float u, u64 mass) { return u > 0.f ? share(fminf(u, 1.f - 0x1p-24f), mass, false) : 0; }

__device__ __noinline__ unsigned alone(const SampleRow& r, SampleShared& sh, const SampleLimits& lim) {
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
// One bitonic step between neighbours of a warp's 64 elements, 32 apart in the two registers
__device__ __forceinline__ void sort_pair(u64& x, u64& y, bool down) {
  if ((x < y) == down) { const u64 t = x; x = y; y = t; }
}
__device__ __forceinline__ void sort_steps(u64& x0, u64& x1, int i0, int run, int step) {
  if (step == 32) { sort_pair(x0, x1, (i0 & run) == 0); step = 16; }
  for (; step > 0; step >>= 1) {
    const u64 y0 = __shfl_xor_sync(0xffffffffu, x0, step), y1 = __shfl_xor_sync(0xffffffffu, x1, step);
    const bool low = (i0 & step) == 0;                   // the lower of two keeps the larger where the run goes down
    x0 = ((x0 > y0) == (low == ((i0 & run) == 0))) ? x0 : y0;
    x1 = ((x1 > y1) == (low == (((i0 + 32) & run) == 0))) ? x1 : y1;
  }
}
// Largest first; a warp sorts 64 elements in registers, only longer distances go through shared memory
__device__ void sort_list(u64* list, int n) {
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kSampleThreads) list[i] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int run = 64; run <= size; run <<= 1) {
    for (int step = run >> 1; step >= 64; step >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += kSampleThreads) {
        const int a = 2 * step * (i / step) + i % step, b = a + step;
        const u64 x = list[a], y = list[b];
        if ((x < y) == ((a & run) == 0)) { list[a] = y; list[b] = x; }
      }
      __syncthreads();
    }
    for (int i = (threadIdx.x >> 5) * 64 + lane; i < size; i += 2 * kSampleThreads) {
      u64 x0 = list[i], x1 = list[i + 32];
      if (run == 64)
        for (int r = 2; r < 64; r <<= 1) sort_steps(x0, x1, i, r, r >> 1);
      sort_steps(x0, x1, i, run, 32);
      list[i] = x0;
      list[i + 32] = x1;
    }
    __syncthreads();
  }
}

// A list of up to 128, largest first: an element's place is the number of larger ones, counted by four threads
__device__ void sort_few(u64* list, int n) {
  const int i = threadIdx.x >> 2, part = threadIdx.x & 3;
  const u64 x = i < n ? list[i] : 0;
  int at = 0;
  for (int j = part; j < n; j += 4) at += list[j] > x;
  at += __shfl_xor_sync(0xffffffffu, at, 1);
  at += __shfl_xor_sync(0xffffffffu, at, 2);
  __syncthreads();
  if (part == 0 && i < n) list[at] = x;
  __syncthreads();
}

// A sorted list's masses: E elements a thread, of one warp (lists of up to 128) or of the CTA.  Elements and masses that are asked for come
// out the same in every thread.
template <int E, bool WARP>
struct ListMasses {
  u64 m[E], c[E];                                        // of the thread's elements, and up to and with each, behind `base`
  double w[E];
  int n;
  u64 end;
  __device__ void sums(SampleShared& sh, u64 v, u64& before, u64& total) const {
    if (WARP) {
      u64 s = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, s, o);
        if ((threadIdx.x & 31) >= o) s += t;
      }
      before = s - v;
      total = __shfl_sync(0xffffffffu, s, 31);
    } else {
      scan(v, sh.warps, before, total);
    }
  }
  __device__ ListMasses(const SampleRow& r, SampleShared& sh, int n_, u64 base) : n(n_) {
    u64 sum = 0, before;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = threadIdx.x * E + e;
      w[e] = i < n ? r.weight(from_image((uint32_t)(sh.list[i] >> 32))) : 0.0;
      m[e] = i < n ? r.mass(w[e]) : 0;
      sum += m[e];
    }
    sums(sh, sum, before, end);
    end += base;
    before += base;
#pragma unroll
    for (int e = 0; e < E; ++e) c[e] = before += m[e];
  }
  __device__ u64 least(SampleShared& sh, float limit) const {            // mass of what weighs so much
    u64 sum = 0, before, total;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += w[e] >= (double)limit ? m[e] : 0;
    sums(sh, sum, before, total);
    return total;
  }
  // The first element whose place and running mass pass, and that mass; the last element if none does
  template <class F>
  __device__ void first(SampleShared& sh, F test, int& at, u64& upto) const {
    int mine = -1;
    u64 mass = 0;
#pragma unroll
    for (int e = E - 1; e >= 0; --e) {
      const int i = threadIdx.x * E + e;
      if (i < n && test(i, c[e])) { mine = i; mass = c[e]; }
    }
    if (WARP) {
      const unsigned who = __ballot_sync(0xffffffffu, mine >= 0);
      const int from = who ? __ffs(who) - 1 : 0;
      at = __shfl_sync(0xffffffffu, mine, from);
      upto = __shfl_sync(0xffffffffu, mass, from);
      if (!who) { at = n - 1; upto = end; }
    } else {
      if (threadIdx.x == 0) { sh.found[0] = n - 1; sh.found[1] = end; }
      __syncthreads();
      // of neighbours that both pass, the one whose predecessor does not
      if (mine >= 0 && (mine > threadIdx.x * E || mine == 0 || !test(mine - 1, c[0] - m[0]))) { sh.found[0] = mine; sh.found[1] = mass; }
      __syncthreads();
      at = (int)sh.found[0];
      upto = sh.found[1];
      __syncthreads();
    }
  }
};

// The bin of the row's running mass: the first at whose end test(mass) holds; kSampleBins if none.  `before`: mass in front of it
template <class T, class F>
__device__ int bin_of(SampleShared& sh, const T (&c)[2], const T (&m)[2], F test, u64& before) {
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

// Four logits at an end of the row (out of line, where it does not lengthen the loops over the others)
template <bool BF16>
__device__ __noinline__ float4 end_group(const void* x, int i, int V) {
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool in = i + e >= 0 && i + e < V;
    v[e] = !in ? -INFINITY : BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i + e]) : static_cast<const float*>(x)[i + e];
  }
  return make_float4(v[0], v[1], v[2], v[3]);
}

// C CTAs a row of fp32 or BF16 logits.  HELD: the slices fit in shared memory
template <int C, bool HELD, bool BF16>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_rows_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) float slice[];
  __shared__ SampleShared sh;
  grid_dep_launch();
  grid_dep_wait();
  const int tid = threadIdx.x, lane = tid & 31;
  const int row = blockIdx.x / C;
  const uint32_t rank = C > 1 ? cluster_ctarank() : 0;
  if (C > 1) cluster_arrive();                           // another CTA's shared memory is there from its start on: see all_here
  SampleRow r;
  r.x = BF16 ? (const void*)(static_cast<const __nv_bfloat16*>(a.x) + row * a.ld) : (const void*)(static_cast<const float*>(a.x) + row * a.ld);
  r.V = a.V; r.bf16 = BF16;
  const int shift = min(45, 63 - (32 - __clz(a.V)));     // masses of a row stay below 2^64
  const float t = a.temperature ? a.temperature[row] : a.t0;
  SampleLimits lim;
  lim.k = a.top_k ? a.top_k[row] : a.k0;
  lim.p = a.top_p ? a.top_p[row] : a.p0;
  lim.least = a.min_p ? a.min_p[row] : a.m0;
  lim.u = a.uniform[row];
  if (lim.k >= a.V) lim.k = 0;
  // the slice: groups of four that start on 16 (bf16: 8) bytes; `skew` elements of the row's first group are in front of it
  const int skew = (int)(reinterpret_cast<uintptr_t>(r.x) >> (BF16 ? 1 : 2) & 3);
  const int groups = (a.V + skew + 3) / 4, per = (groups + C - 1) / C;
  const int g0 = min(groups, (int)rank * per), ng = min(groups, g0 + per) - g0;
  const float* xf = static_cast<const float*>(r.x) - skew;
  auto fetch = [&](int g) -> float4 {                    // group g of the row; what is not the row's is -inf
    const int i = 4 * g - skew;
    const bool in = i >= 0 && i + 4 <= a.V;
    if (!BF16 && in) return __ldg(reinterpret_cast<const float4*>(xf + 4 * g));
    if (BF16 && in) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(r.x) + i));
      return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    }
    return end_group<BF16>(r.x, i, a.V);
  };
  auto group = [&](int j) -> float4 { return HELD ? reinterpret_cast<const float4*>(slice)[j] : fetch(g0 + j); };
  if (tid < kSamplePer) sh.root[tid] = exp2(tid * (-1.0 / kSamplePer));
  if (tid == 0) { sh.n_list = 0; sh.above = 0; }
  // in front of the first store to another CTA; that all have started is long known here, their slices have been read in between
  auto all_here = [&]() {
    if (C > 1) { __syncwarp(); cluster_wait(); }
  };
  auto clear = [&]() {
    for (int i = tid; i < kSampleBins; i += kSampleThreads) sh.own.cnt[i] = sh.own.lo[i] = sh.own.hi[i] = 0;
  };
  clear();
  auto cta_max = [&](float v) -> float {
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0) sh.warps[tid >> 5] = __float_as_uint(v);
    __syncthreads();
    for (int i = 0; i < kSampleWarps; ++i) v = fmaxf(v, __uint_as_float((uint32_t)sh.warps[i]));
    __syncthreads();
    return v + 0.f;
  };
  r.inv_t = 1.0 / (double)t;
  const bool greedy = !(t > 0.f), counts = lim.k > 0 && lim.k <= kSampleFirst, both = lim.k > kSampleFirst;     // counts: all of the first k are sorted
  const double per_logit = kSamplePer * 1.4426950408889634 * r.inv_t;
  float kh = counts ? (float)kSamplePer : (float)per_logit;
  const float kl = counts ? 0.f : (float)(per_logit - (double)kh);
  // place on the grid, the same in every pass and slice: rounding does not change the order of two logits
  auto grid = [&](float x) { return __fmul_rn(x, kh); };
  constexpr float kMagic = 12582912.f, kGrid = 2097152.f;          // 1.5 * 2^23: what is added to it is rounded to a whole number
  auto whole = [&](float p) { return __fsub_rn(__fadd_rn(p, kMagic), kMagic); };
  float ref = -INFINITY;                                 // where the bins begin
  bool above = false;                                    // an element was in front of them
  // distance from the middle of x's bin: in grid units x is p + rest.  Its order in a bin is that of the logits too
  auto beside = [&](float x, float p, float mid) -> float {
    const float rest = fmaf(x, kl, fmaf(x, kh, -p));
    return __fadd_rn(__fsub_rn(p, __fsub_rn(mid, kMagic)), rest);
  };
  auto part_of = [](float off) -> int { return max(0, min(kSampleBins - 1, (int)((0.5f - off) * kSampleBins))); };
  int zoom = -1;                                         // the bin whose elements alone are counted, in 1024 parts of it (`zooms`)
  auto put = [&](float x, auto zooms) {
    constexpr bool kZooms = decltype(zooms)::value;
    const float p = grid(x), d = ref - p;
    if (!(d < kSampleEdge)) return;
    const float mid = __fadd_rn(p, kMagic);
    int n = (int)(__float_as_uint(__fadd_rn(ref, kMagic)) - __float_as_uint(mid));
    if (n < 0) { above = true; return; }
    if (kZooms && n != zoom) return;
    if (!counts) {
      const float off = beside(x, p, mid);
      if (kZooms) n = part_of(off);
      // 2^(off / 16) - 1, |off| <= 1/2: (ln2 / 16)^i / i! off^i
      const float q = off * fmaf(off, fmaf(off, fmaf(off, 1.46760905e-7f, 1.35507817e-5f), 9.38384793e-4f), 4.33216988e-2f);
      const unsigned w = __float_as_uint(fmaf(q, (float)(1 << kSampleUnit), kMagic)) - 0x4b400000u + (1u << kSampleUnit);
      atomicAdd(&sh.own.lo[n], w & 0x3fffu);
      atomicAdd(&sh.own.hi[n], w >> 14);
      if (!kZooms && !both) return;
    }
    atomicAdd(&sh.own.cnt[n], 1u);
  };
  auto put4 = [&](const float4& v, auto zooms) { put(v.x, zooms); put(v.y, zooms); put(v.z, zooms); put(v.w, zooms); };
  auto max4 = [](float m, const float4& v) { return fmaxf(fmaxf(fmaxf(m, v.x), fmaxf(v.y, v.z)), v.w); };
  float top = -INFINITY;                                 // the slice's largest
  constexpr int kAhead = 4;                              // groups that a thread has under way
  auto ahead = [&](int j, float4 (&v)[kAhead]) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e)
      v[e] = j + e * kSampleThreads < ng ? group(j + e * kSampleThreads) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  };
  if (HELD) {
#pragma unroll 8
    for (int j = tid; j < ng; j += kSampleThreads) {
      const float4 v = fetch(g0 + j);
      reinterpret_cast<float4*>(slice)[j] = v;
      top = max4(top, v);
    }
  } else {
    // the bins begin well above the first groups' largest, so that the rest can be counted as it comes
    float4 v[kAhead];
    ahead(tid, v);
#pragma unroll
    for (int e = 0; e < kAhead; ++e) top = max4(top, v[e]);
    const float begin = grid(cta_max(top));
    if (!greedy && fabsf(begin) < kGrid) ref = whole(begin) + (ng > kAhead * kSampleThreads ? 256.f : 0.f);
    for (int j = tid; j < ng; j += kAhead * kSampleThreads) {
      if (j != tid) ahead(j, v);
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        top = max4(top, v[e]);
        if (ref > -INFINITY) put4(v[e], std::false_type());
      }
    }
    if (above) sh.above = 1;
  }
  top = cta_max(top);
  if (greedy) {                                          // the first of the largest
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
    all_here();
    if (tid == 0) {
      for (int i = 0; i < kSampleWarps; ++i) first = min(first, (unsigned)sh.warps[i]);
      st_peer(&sh.first[rank], 0, element(top, first));
    }
    cluster_barrier<C>();
    if (rank == 0 && tid == 0) {
      u64 best = 0;
      for (int i = 0; i < C; ++i) best = max(best, sh.first[i]);
      a.out[row] = (uint32_t)(best >> 32) == image(-INFINITY) ? -1 : (long long)(0xffffffffu - (uint32_t)best);
    }
    return;
  }
  const bool fits = fabsf(grid(top)) < kGrid;            // (a slice that does not fit has nothing to add where the row's largest does)
  if (HELD || sh.above || ref == -INFINITY) {
    if (!HELD) {
      __syncthreads();
      clear();
      __syncthreads();
    }
    ref = fits ? whole(grid(top)) : -INFINITY;
    if (fits)
      for (int j = tid; j < ng; j += kAhead * kSampleThreads) {
        float4 v[kAhead];
        ahead(j, v);
#pragma unroll
        for (int e = 0; e < kAhead; ++e) put4(v[e], std::false_type());
      }
  }
  all_here();
  if (tid < C) {
    st_peer(&sh.top[rank], tid, __float_as_uint(top));
    st_peer(&sh.ref[rank], tid, __float_as_uint(ref));
  }
  cluster_barrier<C>();
  float row_ref = -INFINITY;                             // where the row's bins begin
  for (int i = 0; i < C; ++i) { top = fmaxf(top, sh.top[i]); row_ref = fmaxf(row_ref, sh.ref[i]); }
  r.top = top;
  if (top == -INFINITY) {
    if (rank == 0 && tid == 0) a.out[row] = -1;
    return;                                              // (no CTA looks into another's memory from here on)
  }
  const bool settled = fabsf(grid(top)) < kGrid - 4.f * kSampleBins;
  // at low temperatures, whatever has weight lies within a few bins of 1 / 16 logit
  const bool sharp = !settled && !counts && t <= 1.f && fabsf(top) * kSamplePer < kGrid - 4.f * kSampleBins;
  if (sharp) { kh = kSamplePer; row_ref = whole(grid(top)); }
  const float row_top = settled ? whole(grid(top)) : 0.f;
  const int lead = settled ? (int)(row_ref - row_top) : 0;         // the largest logit's bin
  // a mass is 2^shift for what lies in the middle of that bin
  r.unit = ldexp(settled && !counts ? exp2(((double)top * per_logit - (double)row_top) * (1.0 / kSamplePer)) : 1.0, shift);
  auto lower = [&](int c) {                              // by how many bins CTA c's begin below the row's
    return (int)fminf(row_ref - sh.ref[c], 2.f * kSampleBins);
  };
  // 2^(e - n / 16)
  auto middle = [&](int n, int e) -> double {
    const double x = sh.root[n & (kSamplePer - 1)];
    return __hiloint2double(__double2hiint(x) + ((e - (n >> 4)) << 20), __double2loint(x));
  };
  // every CTA sums its share of the bins over the cluster and hands it to all; P threads a bin
  constexpr int P = C < 4 ? 1 : 4, kShareBins = kSampleBins / C;
  if (settled)
    for (int i = tid; i < kShareBins * P; i += kSampleThreads) {
      const int n = rank * kShareBins + i / P, part = i % P;
      unsigned cnt = 0;
      u64 w = 0;
#pragma unroll
      for (int c = 0; c < C / P; ++c) {
        const int from = part * (C / P) + c, by = C > 1 ? lower(from) : 0;
        if (n >= by) {
          cnt += ld_peer(&sh.own.cnt[n - by], from);
          if (!counts) w += ((u64)ld_peer(&sh.own.hi[n - by], from) << 14) + ld_peer(&sh.own.lo[n - by], from);
        }
      }
#pragma unroll
      for (int o = 1; o < P; o <<= 1) {
        cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
        w += __shfl_xor_sync(0xffffffffu, w, o);
      }
      const u64 m = counts ? 0 : __double2ull_rn(middle(n - lead, shift - kSampleUnit) * (double)w);
      // without counts, what a bin holds at most: its weights' factors are within 2.2 % of one
      if (!counts && lim.k <= 0) cnt = (unsigned)((w + (w >> 5) + (1u << (kSampleUnit - 1))) >> kSampleUnit);
#pragma unroll
      for (int c = 0; c < C / P; ++c) {
        const int to = part * (C / P) + c;
        st_peer(&sh.cnt[n], to, cnt);
        if (!counts) st_peer(&sh.mass[n], to, m);
      }
    }
  cluster_barrier<C>();
  // running counts and masses, two bins a thread
  u64 mass[2], upto[2], before, total;
  unsigned cnt[2], count[2], front;
#pragma unroll
  for (int e = 0; e < 2; ++e) { mass[e] = counts ? 0 : sh.mass[2 * tid + e]; cnt[e] = sh.cnt[2 * tid + e]; }
  scan2(cnt[0] + cnt[1], mass[0] + mass[1], sh, front, before, total);
  count[0] = front + cnt[0]; count[1] = count[0] + cnt[1];
  upto[0] = before + mass[0]; upto[1] = upto[0] + mass[1];
  u64 kept = total;                                      // (the first CTA's; the others know the first round only)
  // the bins in which an element that weighs `least` can be
  const float least = lim.least > 0.f ? fminf(lim.least, 1.f) : 0.f;
  const float d_least = least > 0.f ? (float)lead - kSamplePer * log2f(least) : INFINITY;
  const int n_least = d_least < kSampleEdge - 1.f ? (int)rintf(d_least) : kSampleBins;
  auto next = [&](int done) -> int4 {                    // the round behind `done`: (what, first bin, last bin), base in sh.base
    u64 base = 0;
    if (done < kFirst && lim.k > 0) {
      const int b = bin_of(sh, count, cnt, [&](u64 c) { return c >= (u64)lim.k; }, base);
      const int in = (int)base;
      if (2 * tid <= b && b < 2 * tid + 2) sh.base = upto[b & 1] - mass[b & 1];
      __syncthreads();
      if (b < kSampleBins) return make_int4(kFirst, b, b, in);         // (else fewer than k have weight)
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
  // the first CTA: the mass that a round's sorted list leaves, and in the last round the token
  bool first = settled && !counts;                       // (else there are no masses of bins)
  auto settle = [&](const auto& l, const int4& todo) -> u64 {
    const bool all = todo.x == kAll;
    int at;
    // in the first round the elements' own masses take the place of their bins', which are good to 2^-27 of each
    u64 some, left = sharp ? l.end : first ? sh.rest + l.end - (all ? 0 : sh.base) : kept;
    if (all && lim.k > 0) l.first(sh, [&](int i, u64) { return i + 1 >= lim.k; }, at, left);
    if (todo.x == kFirst) l.first(sh, [&](int i, u64) { return i + 1 >= lim.k - todo.w; }, at, left);
    some = left;
    if ((all || todo.x == kShare) && lim.p < 1.f) {
      const u64 want = max(reach(lim.p, left), (u64)1);
      l.first(sh, [&](int, u64 c) { return c >= want; }, at, some);
    }
    if ((all || todo.x == kLeast) && least > 0.f) some = min(some, (all ? 0 : sh.base) + l.least(sh, least));
    left = min(left, some);
    if (all || todo.x == kPick) {
      const u64 want = exceed(lim.u, left);
      l.first(sh, [&](int, u64 c) { return c > want; }, at, some);
      if (tid == 0) a.out[row] = 0xffffffffu - (unsigned)(sh.list[at] & 0xffffffffu);
    }
    return left;
  };
  int4 todo;
  if (!settled) {
    todo = sharp ? make_int4(kAll, 0, min(kSampleBins - 1, (int)(t * 500.f) + 2), 0) : make_int4(kAlone, 0, 0, 0);          // 2^-45
  } else if (counts) {
    u64 base;
    const int b = bin_of(sh, count, cnt, [&](u64 c) { return c >= (u64)lim.k; }, base);
    // fewer than k in the bins, as where most of a row is masked: what is 64 logits below the largest (48, where the bins begin above it) has no
    // weight, unless T is above 1.9: the k elements that are left out, at most 1536, weigh less than 2^-48 (2^-36) of it each, together less
    // than a third of the step between two numbers u below 1
    todo = b < kSampleBins ? make_int4(kAll, 0, b, 0) : t <= 1.9f ? make_int4(kAll, 0, kSampleBins - 1, 0) : make_int4(kAlone, 0, 0, 0);
  } else {
    todo = next(kDone);
    const u64 base = todo.x == kAll ? 0 : sh.base;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (todo.x > kAlone && 2 * tid + e == todo.z) sh.rest = kept - (upto[e] - base);
    __syncthreads();
  }
  while (todo.x > kAlone) {
    // a bin of too many elements: its 1024 parts are counted as the bins were, and the part is taken that the place lies in
    int part = -1;
    if ((todo.x == kFirst || todo.x == kShare || todo.x == kPick) && todo.y == todo.z && sh.cnt[todo.y] > kSampleList) {
      __syncthreads();
      clear();
      __syncthreads();
      zoom = todo.y;
      ref = row_ref;                                     // (the row's bins)
      for (int j = tid; j < ng; j += kAhead * kSampleThreads) {
        float4 v[kAhead];
        ahead(j, v);
#pragma unroll
        for (int e = 0; e < kAhead; ++e) put4(v[e], std::true_type());
      }
      cluster_barrier<C>();
      for (int i = tid; i < kShareBins; i += kSampleThreads) {
        const int n = rank * kShareBins + i;
        unsigned c = 0;
        u64 w = 0;
#pragma unroll
        for (int from = 0; from < C; ++from) {
          c += ld_peer(&sh.own.cnt[n], from);
          w += ((u64)ld_peer(&sh.own.hi[n], from) << 14) + ld_peer(&sh.own.lo[n], from);
        }
        st_peer(&sh.own.zoom_cnt[n], 0, c);
        st_peer(&sh.own.zoom_mass[n], 0, __double2ull_rn(middle(todo.y - lead, shift - kSampleUnit) * (double)w));
      }
      cluster_barrier<C>();
      if (rank == 0) {
        u64 m2[2], u2[2], b2, all2;
        unsigned c2[2], f2;
#pragma unroll
        for (int e = 0; e < 2; ++e) { m2[e] = sh.own.zoom_mass[2 * tid + e]; c2[e] = sh.own.zoom_cnt[2 * tid + e]; }
        scan2(c2[0] + c2[1], m2[0] + m2[1], sh, f2, b2, all2);
        unsigned k2[2] = {f2 + c2[0], f2 + c2[0] + c2[1]};
        u2[0] = sh.base + b2 + m2[0]; u2[1] = u2[0] + m2[1];
        u64 front, want = todo.x == kShare ? max(reach(lim.p, kept), (u64)1) : exceed(lim.u, kept);
        int s2;
        if (todo.x == kFirst) s2 = bin_of(sh, k2, c2, [&](unsigned c) { return c >= (unsigned)(lim.k - todo.w); }, front);
        else s2 = bin_of(sh, u2, m2, [&](u64 c) { return todo.x == kShare ? c >= want : c > want; }, front);
        if (s2 == kSampleBins) {                         // (rounding: the place is the bin's last element's)
          if (tid == kSampleThreads - 1) sh.found[0] = k2[1];
          __syncthreads();
          const unsigned every = (unsigned)sh.found[0];
          s2 = bin_of(sh, k2, c2, [&](unsigned c) { return c >= every; }, front);
        }
        if (2 * tid <= s2 && s2 < 2 * tid + 2) {
          sh.base = u2[s2 & 1] - m2[s2 & 1];
          sh.rest = kept - m2[s2 & 1];
          sh.found[0] = k2[s2 & 1] - c2[s2 & 1];
        }
        __syncthreads();
        todo.w += (int)sh.found[0];
        __syncthreads();
        if (tid < C) st_peer(&sh.sub, tid, (uint32_t)s2);
      }
      cluster_barrier<C>();
      part = sh.sub;
    }
    // the bins' elements go to the first CTA, the others' by way of a list of their own
    const float from = row_ref - (float)todo.z, to_grid = row_ref - (float)todo.y;
    for (int j = tid; j < ng; j += kAhead * kSampleThreads) {
      float4 v4[kAhead];
      ahead(j, v4);
#pragma unroll
      for (int b = 0; b < kAhead; ++b) {
        if (!(grid(max4(-INFINITY, v4[b])) >= from - 0.5f)) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = (&v4[b].x)[e], p = grid(x);
          if (!(p >= from - 0.5f && p <= to_grid + 0.5f)) continue;
          const float n = whole(p);
          if (!(n >= from && n <= to_grid)) continue;
          if (part >= 0 && part_of(beside(x, p, __fadd_rn(p, kMagic))) != part) continue;
          const unsigned to = atomicAdd(&sh.n_list, 1u);
          if (to < kSampleList) sh.list[to] = element(x, 4 * (g0 + j + b * kSampleThreads) - skew + e);
        }
      }
    }
    if (C > 1) {
      __syncthreads();
      if (rank != 0) {
        const unsigned n = sh.n_list;
        if (tid == 0 && n) sh.at = add_peer(&sh.n_list, 0, n);
        __syncthreads();
        for (unsigned i = tid; i < min(n, (unsigned)kSampleList); i += kSampleThreads)
          if (sh.at + i < kSampleList) st_peer(&sh.list[sh.at + i], 0, sh.list[i]);
        __syncthreads();
        if (tid == 0) sh.n_list = 0;
      }
    }
    cluster_barrier<C>();
    if (rank != 0 && (todo.x == kAll || todo.x == kPick)) return;          // (the last round; what is still too much the first CTA settles alone)
    const bool last = todo.x == kAll || todo.x == kPick;
    if (rank == 0) {
      const int n = (int)sh.n_list;
      if (n > kSampleList || n < 1) {
        todo = make_int4(kAlone, 0, 0, 0);
      } else {
        const u64 base = todo.x == kAll ? 0 : sh.base;
        if (n <= 128) {
          sort_few(sh.list, n);
          if (tid < 32) {
            const u64 left = settle(ListMasses<4, true>(r, sh, n, base), todo);
            if (tid == 0) sh.kept = left;
          }
          __syncthreads();
          kept = sh.kept;
        } else {
          sort_list(sh.list, n);
          kept = n <= kSampleThreads ? settle(ListMasses<1, false>(r, sh, n, base), todo)
                                     : settle(ListMasses<4, false>(r, sh, n, base), todo);
        }
        first = false;
        todo = last ? make_int4(kDone, 0, 0, 0) : next(todo.x);
      }
      __syncthreads();
      if (last) break;
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
  auto k = a.bf16 ? sample_rows_kernel<C, HELD, true> : sample_rows_kernel<C, HELD, false>;
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
  if (a.V < 1 || a.V > (1 << 21) || a.rows > (1 << 27)) return -1;
  // CTAs of a row: as many as find room at a time, two an SM; their serial steps cost a row C times.  us, top-k (top-p), rows of 151936, C = 8 /
  // 4 / 2 / 1: 1 row 15 / 19 / 33 / 51 (31 / 37 / 68 / 107), 64 rows 39 / 31 / 37 / 55 (87 / 73 / 88 / 129), 512 rows 279 / 213 / 179 / 165
  // (491 / 371 / 323 / 313)
  const int fit = a.rows <= 37 ? 8 : a.rows <= 74 ? 4 : a.rows <= 148 ? 2 : 1;
  int c = a.V <= 4096 ? 1 : fit;
  while (c * (1 << 18) < a.V) c *= 2;                    // (a slice's sums of 14-bit parts stay below 2^32)
  // slices of up to 18 Ki elements are held: two CTAs of them share an SM
  const bool held = a.V <= c * 18432;
  if (c == 8) return held ? launch<8, true>(a, st) : launch<8, false>(a, st);
  if (c == 4) return held ? launch<4, true>(a, st) : launch<4, false>(a, st);
  if (c == 2) return held ? launch<2, true>(a, st) : launch<2, false>(a, st);
  return held ? launch<1, true>(a, st) : launch<1, false>(a, st);
}
