// Products of e4m3 rows and e4m3 weights above 64 rows (rows_e4m3.cuh has the form of the rows):
//     Y[t, n] = epilogue( sum_b sx[b, t] sw[n / 128, b] sum_{k in block b} X[t, k] W[n, k] ),
// plain, gated (act(gate) * up, on request as e4m3 rows for the next product) and grouped by expert.
//
// Tokens are the rows of the MMA and features its columns, as in gemm_prefill_tm_kernel (gemm_prefill_sm100.cu), whose pipeline this
// is: one producer warp, one MMA warp, eight warps behind them; with CG = 2 two CTAs share a tile of 256 tokens and each holds half of
// its weight rows.  What differs is that a sum may run over one block of 128 k only: its scales are a number per token and block and a
// number per 128 features and block.  So a block is one accumulator (two in turn), and the eight warps fetch it, scale it and add it to
// registers while the next fills: a thread has one token and 128 columns, whose factor is one product of two scales.  That is 64
// two-wide multiply-adds and 128 words from TMEM per thread and block, against 512 cycles of MMAs in the largest tile; the last
// accumulators of a tile are finished and stored while the next tile's first two fill.
#include "rows_e4m3.cuh"

#include <type_traits>

namespace xft {

int encode_tensor_map(CUtensorMap* out, const void* ptr, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows,
                      uint32_t esize);                                 // gemm_sm100.cu: make_tensor_map without its table

// Three groups of four warps: the issuing ones (producer, MMA; two idle), and eight warps that add up, to which the first group's registers go
// (setmaxnreg: 24 and 240 a thread of the 168 that each was launched with).
constexpr int kRowsThreads = 384;
constexpr int kRowsRing = 192 * 1024;

__device__ __forceinline__ void umma_e4m3(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n"
      :
      : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_e4m3_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n"
      :
      : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// (x, y) += f * (a, b)
__device__ __forceinline__ void fma_pair(float& x, float& y, float f, uint32_t a, uint32_t b) {
  asm("{\n"
      ".reg .b64 c, m, s;\n"
      "mov.b64 c, {%0, %1};\n"
      "mov.b64 m, {%2, %2};\n"
      "mov.b64 s, {%3, %4};\n"
      "fma.rn.f32x2 c, s, m, c;\n"
      "mov.b64 {%0, %1}, c;\n"
      "}\n"
      : "+f"(x), "+f"(y)
      : "f"(f), "r"(a), "r"(b));
}
// waits for the loads from TMEM under way; nothing that uses v moves in front of it
__device__ __forceinline__ void rows_ld_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]),
                 "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]),
                 "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])::"memory");
}
// A bounded wait that also ends when another role of this CTA has given up
__device__ __forceinline__ bool rows_wait(uint64_t* bar, uint32_t parity, int* status, int code, volatile int* lost) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*lost) return false;
    if (clock64() - t0 > kWaitCycles) {
      if (status) atomicCAS(status, 0, code);
      *lost = 1;
      return false;
    }
  }
  return true;
}
// What this arrival orders are the warp's loads from TMEM, which have their own fence and wait; no other memory has to be seen, so it is
// relaxed, and the waits of the issuing threads carry the scope of the CTA also in pairs.  Cluster scope there drops the SM's cached
// lines at every wait: 256 x 256 tiles of 8192 x 8192 x 28672 took 3778 us with it.
__device__ __forceinline__ void rows_arrive(uint32_t addr) {           // in the window of the cluster
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// act of 16 values: one branch for all of them
__device__ __forceinline__ void rows_act(float* x, int act) {
#define XFT_ROWS_ACT(A)                                    \
  case A:                                                  \
    _Pragma("unroll") for (int j = 0; j < 16; ++j) x[j] = apply_act(x[j], A); \
    break;
  switch (act) { XFT_ROWS_ACT(1) XFT_ROWS_ACT(2) XFT_ROWS_ACT(3) XFT_ROWS_ACT(4) XFT_ROWS_ACT(kActGeluErf) XFT_ROWS_ACT(kActTanh) default: break; }
#undef XFT_ROWS_ACT
}

// elements in front of the first 16-byte boundary of a row
template <typename T>
__device__ __forceinline__ int rows_head(const T* p) {
  return (int)((0u - (uint32_t)(reinterpret_cast<uintptr_t>(p) / sizeof(T))) & (16 / sizeof(T) - 1));
}
// N words turned by so many bytes, a multiple of UNIT below 16: left, so that what lay `bytes` behind the start lies at the start, or back
template <int UNIT, bool LEFT, int N>
__device__ __forceinline__ void rows_rotate(uint32_t (&w)[N], int bytes) {
  uint32_t v[N];
#pragma unroll
  for (int s = UNIT; s < 16; s *= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int by = s / 4;                                            // words
      if (LEFT) v[i] = s == 2 ? __funnelshift_r(w[i], w[(i + 1) % N], 16) : w[(i + by) % N];
      else v[i] = s == 2 ? __funnelshift_l(w[(i + N - 1) % N], w[i], 16) : w[(i + N - by) % N];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = bytes & s ? v[i] : w[i];
  }
}

struct RowsTmParams {
  RowsGemm g;
  int n_tiles, t_tiles, num_kb;
  int gn;                                    // feature tiles that walk the token tiles together
};

// NCOL: accumulator columns of a tile; gated: half gate, half up (the other way round as many features).
template <int NCOL, bool DUAL, int CG>
struct RowsTile {
  static constexpr int FEAT = DUAL ? NCOL / 2 : NCOL, TOK = 128 * CG;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = NCOL / CG * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int FIT = kRowsRing / STAGE, STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int LINES = 8 * 4096;     // 32 tokens x 128 bytes of output per summing warp, behind the ring
  static constexpr int SMEM = STAGES * STAGE + LINES + 1024;
  static constexpr int COLS = NCOL / 2;      // of a thread: two warps share 32 tokens
  static_assert((NCOL == 256 || (NCOL == 128 && !DUAL)) && (CG == 1 || CG == 2), "tile");
};

// OUT: how a result leaves.  Each has a kernel of its own: what the others need at the end of a tile takes registers that the sums and their
// scales lack in front of it (8192 x 8192 x 28672 on pairs under the power cap, us: 2285 with kRowsAny for all, 1974 with kRowsPlain).
enum { kRowsCodes = 0, kRowsPlain = 1, kRowsAny = 2 };                // e4m3 rows (gated); bf16 in 16-byte pieces, no bias or activation; anything
template <int NCOL, bool DUAL, int CG, int SPLIT, int OUT>
__global__ void __launch_bounds__(kRowsThreads, 1) gemm_rows_tm_kernel(const __grid_constant__ CUtensorMap tmX,
                                                                       const __grid_constant__ CUtensorMap tmW, const RowsTmParams p) {
  using L = RowsTile<NCOL, DUAL, CG>;
  constexpr int FEAT = L::FEAT, TOK = L::TOK, STAGES = L::STAGES, STAGE = L::STAGE, COLS = L::COLS;
  constexpr uint32_t TMEM_COLS = 2 * NCOL;
  constexpr uint32_t IDESC = umma_idesc(TOK, NCOL, 0, 0, 1);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES], tmem_full[2], tmem_empty[2];
  __shared__ uint32_t tmem_base_s;
  __shared__ int s_lost_mem;
  volatile int* lost = &s_lost_mem;
  int* status = p.g.status;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = CG == 2 ? (int)cluster_ctarank() : 0;              // which 128 tokens of a tile are this CTA's
  const int part = SPLIT > 1 ? (int)cluster_ctarank() : 0;             // which part of k
  const int first = blockIdx.x / (CG * SPLIT), step = gridDim.x / (CG * SPLIT);
  const int k_lo = part * p.num_kb / SPLIT, k_hi = (part + 1) * p.num_kb / SPLIT;
  const int4* groups = reinterpret_cast<const int4*>(p.g.group_tiles);
  const int total = p.n_tiles * (groups ? min(*p.g.num_group_tiles, p.t_tiles) : p.t_tiles);
  struct Item { int nt, row0, rows, w0; };                             // feature tile, first token row, rows, first weight row of its group
  // `gn` feature tiles walk all token tiles together (the tiles of an expert follow one another, so its weights are read once)
  const int per = p.gn * (groups ? min(*p.g.num_group_tiles, p.t_tiles) : p.t_tiles);
  auto entry_of = [&](int item) {
    if (!groups || item >= total) return make_int4(0, 0, 0, 0);
    const int gr = item / per;
    return __ldg(groups + (item - gr * per) / min(p.gn, p.n_tiles - gr * p.gn));
  };
  auto item_of = [&](int item, int4 e) {
    Item r;
    const int gr = item / per, at = item - gr * per, gn = min(p.gn, p.n_tiles - gr * p.gn), tt = at / gn;
    if (groups) r = {gr * p.gn + at - tt * gn, e.y, e.z, e.x * p.g.group_w_rows};
    else r = {gr * p.gn + at - tt * gn, tt * TOK, p.g.T - tt * TOK, 0};
    r.row0 += half * 128;
    r.rows -= half * 128;
    return r;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tmem_full[a], 1); mbar_init(&tmem_empty[a], 8 * CG); }
    s_lost_mem = 0;
    fence_barrier_init();
    fence_proxy_async();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    if constexpr (CG == 2) { tmem_alloc_pair(&tmem_base_s, TMEM_COLS); tmem_relinquish_pair(); }
    else { tmem_alloc(&tmem_base_s, TMEM_COLS); tmem_relinquish(); }
  }
  tcgen05_fence_before();
  __syncthreads();
  if constexpr (CG == 2) {              // both CTAs' barriers and accumulators exist before either touches the other's
    cluster_arrive();
    cluster_wait();
  }
  tcgen05_fence_after();
  const uint32_t tmem_base = tmem_base_s;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
    if (warp == 0) {
      if (elect_one()) {
        const uint32_t lead_bar = CG == 2 ? dsmem_addr(smem_u32(full_bar), 0) : 0;      // the first CTA's full barriers
        // weights that are read about once leave L2 first: 64 experts of 1408 x 2048, 38 rows each, 136 us and 124 so, 8 of 14336 x 4096, 75 rows each,
        // 275 and 266; with three token tiles each the former 366 and 372
        const bool once = groups ? p.n_tiles * (p.g.w_rows / p.g.group_w_rows) * 2 >= total : p.t_tiles == 1;
        const uint64_t hint_w = once ? kEvictFirst : kEvictNormal;
        Ring r = {0, 0};
        bool ok = true;
        for (int item = first; item < total && ok; item += step) {
          const Item im = item_of(item, entry_of(item));
          const int wrow = im.w0 + im.nt * FEAT + half * (DUAL ? p.g.dual_off : NCOL / 2);
          for (int kb = k_lo; kb < k_hi; ++kb, r.next(STAGES)) {
            ok = rows_wait(&empty_bar[r.s], r.ph ^ 1, status, XFT_ERR_WAIT_EMPTY, lost);
            if (!ok) break;
            uint8_t* a = smem + r.s * STAGE;
            if constexpr (CG == 2) {
              if (half == 0) mbar_expect_tx(&full_bar[r.s], 2 * STAGE);
              tma_load_2d_pair(a, &tmX, lead_bar + 8 * r.s, kb * 128, im.row0, kEvictNormal);
              tma_load_2d_pair(a + L::A_BYTES, &tmW, lead_bar + 8 * r.s, kb * 128, wrow, hint_w);
            } else {
              mbar_expect_tx(&full_bar[r.s], STAGE);
              tma_load_2d(a, &tmX, &full_bar[r.s], kb * 128, im.row0, kEvictNormal);
              tma_load_2d(a + L::A_BYTES, &tmW, &full_bar[r.s], kb * 128, wrow, hint_w);
              if (DUAL) tma_load_2d(a + L::A_BYTES + FEAT * 128, &tmW, &full_bar[r.s], kb * 128, wrow + p.g.dual_off, hint_w);
            }
          }
        }
        if (!ok) {                        // copies in flight land before the CTA's shared memory goes
          const long long t0 = clock64();
          while (clock64() - t0 < 2000000LL) {}
        } else if (CG == 2) {
          // the first CTA's commits also arrive here: stay until every stage has been given back
          for (int k = 0; k < STAGES; ++k, r.next(STAGES))
            if (!rows_wait(&empty_bar[r.s], r.ph ^ 1, status, XFT_ERR_WAIT_EMPTY, lost)) break;
        }
      }
    } else if (warp == 1) {
      if (half == 0 && elect_one()) {
        const uint64_t adesc0 = umma_desc_k128(smem_u32(smem)), bdesc0 = umma_desc_k128(smem_u32(smem) + L::A_BYTES);
        Ring r = {0, 0}, b = {0, 0};
        bool ok = true;
        for (int item = first; item < total && ok; item += step) {
          for (int kb = k_lo; kb < k_hi; ++kb, r.next(STAGES), b.next(2)) {
            ok = rows_wait(&tmem_empty[b.s], b.ph ^ 1, status, XFT_ERR_WAIT_TMEM, lost) &&
                 rows_wait(&full_bar[r.s], r.ph, status, XFT_ERR_WAIT_FULL, lost);
            if (!ok) break;
            tcgen05_fence_after();
            const uint64_t off = (uint64_t)(r.s * (STAGE / 16));
            const uint32_t acc = tmem_base + (uint32_t)(b.s * NCOL);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (CG == 2) umma_e4m3_pair(acc, adesc0 + off + 2 * k, bdesc0 + off + 2 * k, IDESC, k > 0);
              else umma_e4m3(acc, adesc0 + off + 2 * k, bdesc0 + off + 2 * k, IDESC, k > 0);
            }
            if constexpr (CG == 2) { tcgen05_commit_pair(&empty_bar[r.s]); tcgen05_commit_pair(&tmem_full[b.s]); }
            else { tcgen05_commit(&empty_bar[r.s]); tcgen05_commit(&tmem_full[b.s]); }
          }
        }
      }
    }
    if constexpr (SPLIT > 1) {          // the parts lie in shared memory
      __syncwarp();
      cluster_arrive();
      cluster_wait();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 240;");
    // ---- a token and COLS columns per thread; gated: COLS / 2 gate columns, then their up columns
    const int q = warp & 3, side = warp >= 8, row = q * 32 + lane;
    constexpr int PART = DUAL ? COLS / 2 : COLS;                       // columns in a row
    const int col0 = side * PART;
    const bool vec = p.g.N % 8 == 0 && p.g.ldo % 8 == 0 && (!p.g.residual || p.g.ldr % 8 == 0) &&
                     ((reinterpret_cast<uintptr_t>(p.g.out) | reinterpret_cast<uintptr_t>(p.g.residual)) & 15) == 0;
    const bool codes32 = p.g.ldo % 32 == 0 && (reinterpret_cast<uintptr_t>(p.g.out) & 31) == 0;
    uint8_t* line = smem + STAGES * STAGE + (warp - 4) * 4096;        // 128 bytes of each of the warp's tokens, their 16-byte pieces interchanged
    auto line_at = [&](int r, int byte) { return line + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15); };
    // bias, activation (the gated form has its own) and residual on C columns from n on of token t, the warp's first `most` tokens being there; all of
    // the residual is on its way before the first value waits for it
    auto apply = [&](auto count, float* x, int t, int n, int most) {
      constexpr int C = decltype(count)::value;
      if constexpr (!DUAL && OUT == kRowsAny) {
        if (p.g.bias) {
          if (n + C <= p.g.N && (reinterpret_cast<uintptr_t>(p.g.bias) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < C; j += 4) {
              const float4 b = __ldg(reinterpret_cast<const float4*>(p.g.bias + n + j));
              x[j] += b.x; x[j + 1] += b.y; x[j + 2] += b.z; x[j + 3] += b.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < C; ++j) x[j] += __ldg(p.g.bias + min(n + j, p.g.N - 1));
          }
        }
        if (p.g.act) {
#pragma unroll
          for (int c = 0; c < C; c += 16) rows_act(x + c, p.g.act);
        }
      }
      if (!p.g.residual) return;
      const __nv_bfloat16* r0 = reinterpret_cast<const __nv_bfloat16*>(p.g.residual) + (size_t)(t - lane) * p.g.ldr + n;
      constexpr int W = C < 64 ? C : 64;
      auto add_line = [&](int c) {                                     // W columns of the residual lie in the warp's lines
#pragma unroll
        for (int j = 0; j < W / 8; ++j) {
          const uint4 u = *reinterpret_cast<const uint4*>(line_at(lane, 16 * j));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&u)[i]);
            x[c + 8 * j + 2 * i] += p.g.res_scale * f.x;
            x[c + 8 * j + 2 * i + 1] += p.g.res_scale * f.y;
          }
        }
      };
      if (OUT == kRowsPlain || vec) {
        // along the rows as well: a lane's own 16 bytes of a row each would touch 32 lines a load (8192 x 28672 x 256 with residual: 320 us,
        // and 228 so)
        constexpr int PIECES = W / 8;
        uint4 v[C / 8];
#pragma unroll
        for (int c = 0; c < C; c += W)
#pragma unroll
          for (int i = 0; i < PIECES; ++i) {
            const int r = 32 / PIECES * i + lane / PIECES, col = c + lane % PIECES * 8;
            v[c / 8 + i] = r < most && n + col < p.g.N
                               ? __ldg(reinterpret_cast<const uint4*>(r0 + (size_t)r * p.g.ldr + col)) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
        for (int c = 0; c < C; c += W) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < PIECES; ++i)
            *reinterpret_cast<uint4*>(line_at(32 / PIECES * i + lane / PIECES, lane % PIECES * 16)) = v[c / 8 + i];
          __syncwarp();
          add_line(c);
        }
        __syncwarp();
      } else if constexpr (OUT == kRowsAny) {
        // rows that do not start on 16 bytes: their 16-byte pieces go into the lines and the elements around those behind them, that is the run
        // rotated, which its lane turns back
        constexpr int PIECES = W / 8, ES = 8 / PIECES;                 // ES: elements of the ends per lane and row
#pragma unroll
        for (int c = 0; c < C; c += W) {
          const int cols = p.g.N - n - c;
          if (cols <= 0) break;
          uint4 v[PIECES];
          __nv_bfloat16 e[PIECES][ES];
          if (cols >= W) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
              const int r = 32 / PIECES * i + lane / PIECES, j = lane % PIECES;
              const __nv_bfloat16* from = r0 + (size_t)r * p.g.ldr + c;
              const int head = rows_head(from);
              v[i] = make_uint4(0, 0, 0, 0);
              if (r < most && (j < PIECES - 1 || !head)) v[i] = __ldg(reinterpret_cast<const uint4*>(from + head) + j);
#pragma unroll
              for (int h = 0; h < ES; ++h)
                e[i][h] = r < most && head ? __ldg(from + ((head + W - 8 + j + h * PIECES) & (W - 1))) : __float2bfloat16(0.f);
            }
          }
          __syncwarp();
          if (cols >= W) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
              const int r = 32 / PIECES * i + lane / PIECES, j = lane % PIECES, head = rows_head(r0 + (size_t)r * p.g.ldr + c);
              if (j < PIECES - 1 || !head) *reinterpret_cast<uint4*>(line_at(r, 16 * j)) = v[i];
#pragma unroll
              for (int h = 0; h < ES; ++h)
                if (head) *reinterpret_cast<__nv_bfloat16*>(line_at(r, 2 * (W - 8 + j + h * PIECES))) = e[i][h];
            }
          } else {                                                     // the last features: one by one, sixteen rows under way
#pragma unroll 1
            for (int r16 = 0; r16 < 32; r16 += 16) {
              constexpr int LC = (W + 31) / 32;                        // columns of a lane
              __nv_bfloat16 u[16][LC];
#pragma unroll
              for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int h = 0; h < LC; ++h) {
                  const int col = 32 * h + lane;
                  u[r][h] = r16 + r < most && col < cols && col < W ? __ldg(r0 + (size_t)(r16 + r) * p.g.ldr + c + col) : __float2bfloat16(0.f);
                }
#pragma unroll
              for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int h = 0; h < LC; ++h) {
                  const int col = 32 * h + lane, head = rows_head(r0 + (size_t)(r16 + r) * p.g.ldr + c);
                  if (col < W) *reinterpret_cast<__nv_bfloat16*>(line_at(r16 + r, 2 * ((col - head) & (W - 1)))) = u[r][h];
                }
            }
          }
          __syncwarp();
          uint32_t w[W / 2];
#pragma unroll
          for (int j = 0; j < W / 8; ++j) reinterpret_cast<uint4*>(w)[j] = *reinterpret_cast<const uint4*>(line_at(lane, 16 * j));
          rows_rotate<2, false>(w, 2 * rows_head(r0 + (size_t)lane * p.g.ldr + c));
#pragma unroll
          for (int j = 0; j < W / 2; ++j) {
            const float2 f = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(w)[j]);
            x[c + 2 * j] += p.g.res_scale * f.x;
            x[c + 2 * j + 1] += p.g.res_scale * f.y;
          }
        }
        __syncwarp();
      }
    };
    // C columns from n on of token t on their way out: 128 bytes of each token at a time through shared memory, so that a store fills lines; rows
    // that do not start on 16 bytes are rotated in their line, so that what leaves in 16 bytes lies so, and the elements around that leave one by one
    // (8192 x 28671 x 256 all one by one 360 us, so 304).  us of 24576 x 2048 x 1408 with a lane's own 32 bytes per store, residual and branches
    // piece by piece / so: 110 / 90 (69 without any store).
    auto leave = [&](auto count, const float* x, int t, int n, int most) {
      constexpr int C = decltype(count)::value;
      auto pieces = [&](auto type, int c0) {                           // the lines hold columns c0 on, W of them
        using OT = decltype(type);
        constexpr int W = C < 128 / (int)sizeof(OT) ? C : 128 / (int)sizeof(OT), PIECES = W * (int)sizeof(OT) / 16;
        OT* out = reinterpret_cast<OT*>(p.g.out) + (size_t)(t - lane) * p.g.ldo + n + c0;
        __syncwarp();
        if (OUT == kRowsPlain || vec) {
#pragma unroll
          for (int i = 0; i < PIECES; ++i) {
            const int r = 32 / PIECES * i + lane / PIECES, j = lane % PIECES;
            const uint4 w = *reinterpret_cast<const uint4*>(line_at(r, 16 * j));
            const int col = j * (16 / (int)sizeof(OT));
            if (r < most && n + c0 + col < p.g.N) *reinterpret_cast<uint4*>(out + (size_t)r * p.g.ldo + col) = w;
          }
        } else if constexpr (OUT == kRowsAny) {
          constexpr int E = 16 / (int)sizeof(OT), ES = E / PIECES < 1 ? 1 : E / PIECES;      // elements of a piece; of the ends per lane and row
          const int cols = p.g.N - n - c0;
          if (cols >= W) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
              const int r = 32 / PIECES * i + lane / PIECES, j = lane % PIECES;
              OT* to = out + (size_t)r * p.g.ldo;
              const int head = rows_head(to);
              if (r >= most) continue;
              if (j < PIECES - 1 || !head) reinterpret_cast<uint4*>(to + head)[j] = *reinterpret_cast<const uint4*>(line_at(r, 16 * j));
#pragma unroll
              for (int h = 0; h < ES; ++h) {
                const int k = W - E + j + h * PIECES;
                if (head && k < W) to[(head + k) & (W - 1)] = *reinterpret_cast<const OT*>(line_at(r, k * (int)sizeof(OT)));
              }
            }
          } else {                                                     // the last features: one by one
#pragma unroll 4
            for (int r = 0; r < 32; ++r) {
              OT* to = out + (size_t)r * p.g.ldo;
              const int head = rows_head(to);
#pragma unroll
              for (int col = lane; col < W; col += 32)
                if (r < most && col < cols) to[col] = *reinterpret_cast<const OT*>(line_at(r, ((col - head) & (W - 1)) * (int)sizeof(OT)));
            }
          }
        }
        __syncwarp();
      };
      if (OUT == kRowsAny && p.g.out_fp32) {
#pragma unroll
        for (int c = 0; c < C; c += 32) {
          constexpr int W = C < 32 ? C : 32;
          uint32_t w[W];
#pragma unroll
          for (int j = 0; j < W; ++j) w[j] = __float_as_uint(x[c + j]);
          if (!vec) rows_rotate<4, true>(w, 4 * rows_head(reinterpret_cast<const float*>(p.g.out) + (size_t)t * p.g.ldo + n + c));
#pragma unroll
          for (int j = 0; j < W / 4; ++j) *reinterpret_cast<uint4*>(line_at(lane, 16 * j)) = reinterpret_cast<const uint4*>(w)[j];
          pieces(float(), c);
        }
      } else {
#pragma unroll
        for (int c = 0; c < C; c += 64) {
          constexpr int W = C < 64 ? C : 64;
          uint32_t w[W / 2];
#pragma unroll
          for (int j = 0; j < W / 2; ++j) reinterpret_cast<__nv_bfloat162*>(w)[j] = __floats2bfloat162_rn(x[c + 2 * j], x[c + 2 * j + 1]);
          if (OUT == kRowsAny && !vec) rows_rotate<2, true>(w, 2 * rows_head(reinterpret_cast<const __nv_bfloat16*>(p.g.out) + (size_t)t * p.g.ldo + n + c));
#pragma unroll
          for (int j = 0; j < W / 8; ++j) *reinterpret_cast<uint4*>(line_at(lane, 16 * j)) = reinterpret_cast<const uint4*>(w)[j];
          pieces(__nv_bfloat16(), c);
        }
      }
    };
    Ring b = {0, 0};
    bool ok = true;
    int turn = 0;
    // Scales of two blocks at a time, asked for two blocks ahead: a load from L2 takes longer than a block, and a value that moves from one
    // register to the next waits for its load.  The first ones of an item are asked for before the item in front of it is finished.
    int t = 0, n0 = 0, nt = 0, rows = 0;
    bool t_ok = false, w_ok = false;
    const float *sx = nullptr, *sw = nullptr, *su = nullptr;
    float xs[2], ws[2], us[2];
    auto fetch_scales = [&](int kb) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = kb + i < k_hi;
        xs[i] = in && t_ok ? __ldg(sx + (size_t)(kb + i) * p.g.x_ld) : 0.f;
        ws[i] = in && w_ok ? __ldg(sw + kb + i) : 0.f;
        if (DUAL) us[i] = in && w_ok ? __ldg(su + kb + i) : 0.f;
      }
    };
    auto begin = [&](int item, int4 e) {
      const Item im = item_of(item, e);
      nt = im.nt;
      t = im.row0 + row;
      n0 = nt * FEAT + col0;
      rows = im.rows;
      t_ok = row < rows;
      w_ok = n0 < p.g.N;                                               // a last tile may have no features on this side
      sx = p.g.x_scale + t;
      sw = p.g.w_scale + (size_t)((im.w0 + n0) >> 7) * p.g.scale_ld;
      su = sw + (size_t)(p.g.dual_off >> 7) * p.g.scale_ld;
      if (!DUAL && SPLIT == 1 && p.g.residual && t_ok && w_ok) {       // on its way to L2 while the item's sums run
        const __nv_bfloat16* r = reinterpret_cast<const __nv_bfloat16*>(p.g.residual) + (size_t)t * p.g.ldr;
#pragma unroll
        for (int c = 0; c < PART; c += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(r + min(n0 + c, p.g.N - 1)));
        if (OUT == kRowsAny) asm volatile("prefetch.global.L2 [%0];" ::"l"(r + min(n0 + PART - 1, p.g.N - 1)));
      }
      fetch_scales(k_lo);
    };
    if (first < total) begin(first, entry_of(first));
    for (int item = first; item < total; item += step, turn ^= 1) {
      const int4 e_next = entry_of(item + step);
      float acc[COLS];
#pragma unroll
      for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
      for (int kb0 = k_lo; kb0 < k_hi && ok; kb0 += 2) {
        float f[2], fu[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) { f[i] = xs[i] * ws[i]; fu[i] = DUAL ? xs[i] * us[i] : 0.f; }
        fetch_scales(kb0 + 2);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (kb0 + i >= k_hi) break;
          ok = __all_sync(0xffffffffu, rows_wait(&tmem_full[b.s], b.ph, status, XFT_ERR_WAIT_TMEM, lost));
          if (!ok) break;
          tcgen05_fence_after();
          const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + (uint32_t)(b.s * NCOL + col0);
          auto at = [&](int c) { return taddr + (DUAL && c >= PART ? FEAT - PART + c : c); };
          auto add = [&](int c, const uint32_t (&v)[32]) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) fma_pair(acc[c + j], acc[c + j + 1], DUAL && c >= PART ? fu[i] : f[i], v[j], v[j + 1]);
          };
#pragma unroll
          for (int c = 0; c < COLS; c += 64) {                         // 64 columns at a time: one wait for two loads
            uint32_t v0[32], v1[32];
            tmem_ld32(at(c), v0);
            tmem_ld32(at(c + 32), v1);
            rows_ld_wait(v0);
            rows_ld_wait(v1);
            if (c + 64 == COLS) {                                      // given back before the last of it is added
              tcgen05_fence_before();
              __syncwarp();
              if (lane == 0) rows_arrive(CG == 2 ? dsmem_addr(smem_u32(&tmem_empty[b.s]), 0) : smem_u32(&tmem_empty[b.s]));
            }
            add(c, v0);
            add(c + 32, v1);
          }
          b.next(2);
        }
      }
      // ---- epilogue of the item (all warps come through here, also after a wait that ran out: the barrier below counts them)
      const int t_now = t, n_now = n0, nt_now = nt, rows_now = rows;
      const bool t_in = t_ok;
      if (item + step < total) begin(item + step, e_next);
      if constexpr (DUAL) {
        if (p.g.bias) {
#pragma unroll
          for (int j = 0; j < PART; ++j) {
            acc[j] += __ldg(p.g.bias + min(n_now + j, p.g.N - 1));
            acc[PART + j] += __ldg(p.g.bias + p.g.dual_off + min(n_now + j, p.g.N - 1));
          }
        }
#pragma unroll
        for (int c = 0; c < PART; c += 16) rows_act(acc + c, p.g.act);
#pragma unroll
        for (int j = 0; j < PART; ++j) acc[j] *= acc[PART + j];
        if constexpr (OUT == kRowsCodes) {
          bool odd;
          float top = e4m3_top<PART>(acc, odd);
          float* tops = reinterpret_cast<float*>(smem + STAGES * STAGE);      // [two items in turn][side][token], where lines would be
          tops[(turn * 2 + side) * 128 + row] = top;
          named_bar_sync(1, 256);
          top = fmaxf(tops[turn * 256 + row], tops[turn * 256 + 128 + row]);
          if (t_in && ok) {
            const E4m3Scale s = e4m3_scale(top);
            uint8_t* to = reinterpret_cast<uint8_t*>(p.g.out) + (size_t)t_now * p.g.ldo + n_now;
#pragma unroll
            for (int j = 0; j < PART; j += 32) {
              uint32_t c[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) c[i] = e4m3_codes(acc + j + 4 * i, s.inv, odd);
              if (codes32) {                                           // whole sectors
                st_global_256(to + j, c);
              } else {
                reinterpret_cast<uint4*>(to + j)[0] = make_uint4(c[0], c[1], c[2], c[3]);
                reinterpret_cast<uint4*>(to + j)[1] = make_uint4(c[4], c[5], c[6], c[7]);
              }
            }
            if (side == 0) p.g.out_scale[(size_t)nt_now * p.g.out_ld + t_now] = s.scale;
          }
          continue;
        }
      }
      if constexpr (SPLIT > 1) {
        // One tile per cluster: every CTA leaves its part of the sums in its shared memory, whose stages the MMAs have all read, [column][token],
        // and finishes NCOL / SPLIT columns from all parts, in the order of k.
        float* mine = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int j = 0; j < COLS; ++j) mine[(col0 + j) * 128 + row] = acc[j];
        cluster_arrive();
        cluster_wait();
        constexpr int OWN = NCOL / SPLIT / 2;                          // columns of a thread
        const int c0 = part * (NCOL / SPLIT) + side * OWN;
        const uint32_t at = smem_u32(mine) + (uint32_t)(c0 * 128 + row) * 4;
#pragma unroll
        for (int j = 0; j < OWN; ++j) acc[j] = 0.f;
#pragma unroll
        for (int r = 0; r < SPLIT; ++r) {
          const uint32_t from = dsmem_addr(at, r);
#pragma unroll
          for (int j = 0; j < OWN; ++j) acc[j] += ld_dsmem(from + j * 512);
        }
        if (nt_now * FEAT + c0 < p.g.N) {
          const int most = ok ? rows_now - q * 32 : 0;
          apply(std::integral_constant<int, OWN>(), acc, t_now, nt_now * FEAT + c0, most);
          leave(std::integral_constant<int, OWN>(), acc, t_now, nt_now * FEAT + c0, most);
        }
        continue;
      }
      if constexpr (OUT != kRowsCodes) {
        if (n_now >= p.g.N) continue;
        const int most = ok ? rows_now - q * 32 : 0;                      // tokens of this warp
        apply(std::integral_constant<int, PART>(), acc, t_now, n_now, most);
        leave(std::integral_constant<int, PART>(), acc, t_now, n_now, most);
      }
    }
  }
  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if constexpr (CG == 2 || SPLIT > 1) { // no CTA's shared memory or accumulator goes while another may still use it
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tcgen05_fence_after();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int NCOL, bool DUAL, int CG, int SPLIT, int OUT>
static int launch_rows_tm(const RowsGemm& g, int sms, cudaStream_t st) {
  using L = RowsTile<NCOL, DUAL, CG>;
  RowsTmParams p{};
  p.g = g;
  p.num_kb = (g.K + 127) / 128;
  p.n_tiles = (g.N + L::FEAT - 1) / L::FEAT;
  p.t_tiles = g.group_tiles ? g.max_tiles : (g.T + L::TOK - 1) / L::TOK;
  p.gn = g.group_tiles && p.n_tiles <= 16 ? p.n_tiles : 8;
  CUtensorMap tmW, tmX;
  int r = make_tensor_map(&tmW, g.w, (uint64_t)g.w_rows, (uint64_t)g.K, (uint64_t)g.ldw, (uint32_t)(DUAL ? L::FEAT : NCOL / CG), 1);
  if (r) return 1000 - r;
  r = encode_tensor_map(&tmX, g.x, (uint64_t)g.x_rows, (uint64_t)g.K, (uint64_t)g.ldx, 128, 1);
  if (r) return 2000 - r;
  const auto kernel = gemm_rows_tm_kernel<NCOL, DUAL, CG, SPLIT, OUT>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  if (e != cudaSuccess) return 3000 + (int)e;
  const long long total = (long long)p.n_tiles * p.t_tiles, slots = SPLIT > 1 ? total : sms / CG > 0 ? sms / CG : 1;      // parts: a tile per cluster
  if (total * CG * SPLIT > 0x7fffffffLL || (SPLIT > 1 && p.num_kb < SPLIT)) return -6;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((total < slots ? total : slots) * CG * SPLIT));
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = L::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG * SPLIT;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG * SPLIT > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kernel, tmX, tmW, (const RowsTmParams)p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// The tile that is expected to take least, or 0 for the weight-stream kernel (gemm_e4m3_sm100.cu), in us: what a launch costs, then rounds of
// tiles, each of its blocks of k and its finish.  Fitted to sweeps on B200; us of tiles 1 / 2 / 3 / 4: 512 x 12288 x 4096 42 / 42 / 39 / 40,
// 4096 x 8192 x 8192 261 / 334 / 254 / 341, 24576 x 2048 x 1408 97 / 119 / 90 / 112; gated 600 x 2 x 11008 x 4096 86 / - / 72, 1500 x 2 x 14336 x
// 4096 205 / - / 224; of 0 / 4 / 5 / 6: 128 x 4096 x 4096 12.1 / 14.2 / 12.1 / 11.3, 389 x 2112 x 7168 25.3 / 20.9 / 15.6 / 31.4, 389 x 1024 x
// 7168 15.8 / 21.3 / 15.1 / 12.3, 600 x 4096 x 1024 20.1 / 12.2 / 21.7 / 36.8.  Under the power cap 1 and 3 are within 4 % of each other.
int rows_form(int T, int N, int K, int gated, int sms) {
  const int kb = (K + 127) / 128, cols = gated ? 2 * N : N;
  auto tiles = [&](int tok, int ncol) { return (long long)((T + tok - 1) / tok) * ((cols + ncol - 1) / ncol); };
  auto cost = [&](int tok, int ncol, int ctas, float block, float finish) {
    const long long slots = sms / ctas > 0 ? sms / ctas : 1;
    return 3.5f + (float)((tiles(tok, ncol) + slots - 1) / slots) * (kb * block + finish);
  };
  const long long small = (long long)((T + 63) / 64) * ((N + 127) / 128);
  int parts = 1;
  while (parts < 8 && small * parts * 2 <= sms && kb / (parts * 2) >= 4) parts *= 2;
  float best = 4.5f + (float)((small * parts + sms - 1) / sms) * ((float)kb / parts * (gated ? 0.7f : 0.35f) + 1.7f);
  int form = 0;
  auto take = [&](int f, float c) { if (c < best) { best = c; form = f; } };
  take(1, cost(256, 256, 2, 0.60f, 1.5f));
  take(3, cost(128, 256, 1, 0.55f, 1.5f));
  if (!gated) {
    take(2, cost(256, 128, 2, 0.35f, 1.2f));
    take(4, cost(128, 128, 1, 0.35f, 1.2f));
    if (tiles(128, 128) * 2 <= sms && kb >= 4) take(5, 6.7f + kb * 0.17f);
    if (tiles(128, 128) * 4 <= sms && kb >= 8) take(6, 7.5f + kb * 0.085f);
  }
  return form;
}

// Tiles: 1 = 256 tokens x 256 columns on two CTAs, 2 = 256 x 128 on two, 3 = 128 x 256, 4 = 128 x 128 (gated: 1 and 3); 5 and 6 = 128 x 128 with k cut into
// two and four parts over a cluster.
int launch_rows_prompt(const RowsGemm& g, int form, cudaStream_t st) {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (sms <= 0) sms = 148;
  if (g.gated && g.out_scale)
    return form == 1 ? launch_rows_tm<256, true, 2, 1, kRowsCodes>(g, sms, st) : launch_rows_tm<256, true, 1, 1, kRowsCodes>(g, sms, st);
  if (g.gated) return launch_rows_tm<256, true, 1, 1, kRowsAny>(g, sms, st);
  if (g.out_scale) return -5;
  // A residual whose rows start between 16 bytes takes its time in front of the stores, and narrow tiles finish in fewer registers: 8192 x 28671 x 256
  // with tiles of 256 and 128 columns 921 and 588 us, 8192 x 28671 x 1024 1078 and 819, 2000 x 5001 x 5000 127 and 111.
  if ((form == 1 || form == 3) && g.residual && g.K <= 5120 && ((g.ldr & 7) || (reinterpret_cast<uintptr_t>(g.residual) & 15))) form = 4;
  const bool plain = !g.bias && !g.act && !g.out_fp32 && g.N % 8 == 0 && g.ldo % 8 == 0 && (!g.residual || g.ldr % 8 == 0) &&
                     ((reinterpret_cast<uintptr_t>(g.out) | reinterpret_cast<uintptr_t>(g.residual)) & 15) == 0;
#define XFT_ROWS_TM(NCOL, CG, SPLIT) \
  (plain ? launch_rows_tm<NCOL, false, CG, SPLIT, kRowsPlain>(g, sms, st) : launch_rows_tm<NCOL, false, CG, SPLIT, kRowsAny>(g, sms, st))
  switch (form) {
    case 1: return XFT_ROWS_TM(256, 2, 1);
    case 2: return XFT_ROWS_TM(128, 2, 1);
    case 3: return XFT_ROWS_TM(256, 1, 1);
    case 5: return XFT_ROWS_TM(128, 1, 2);
    case 6: return XFT_ROWS_TM(128, 1, 4);
    default: return XFT_ROWS_TM(128, 1, 1);
  }
#undef XFT_ROWS_TM
}

}  // namespace xft
