// Attention of the nodes of trees of drafted tokens on the 5th-generation tensor cores: caches in blocks of a multiple of 64, heads of
// 64, 128 or 256 (int8: 128).  The formula, and the kernel for what is left: tree_attention.cu.
//
// The rows (node, query head) of one kv head share its keys: 128 rows a tile, one row per TMEM lane and thread, one tile a CTA, two CTAs
// an SM (heads of 256: one).  CTAs with other rows over the same keys run beside one another and find them in L2; two tiles of rows in a
// CTA over the same keys were no faster (512 rows x 65600 keys, 8 heads: 137 to 147 us, one tile 143 to 147).  For each tile of keys
//
//   S = Q K^T   tcgen05.mma, both operands from shared memory; the keys come by TMA, in pieces of 64 by the block table
//   P = exp2(S - m) as bf16 over S, whole rows in registers; the sum of a row beside it
//   O += P V    tcgen05.mma, P from TMEM, V as it lies in the cache (MN-major)
//
// Bound, for many rows over a key, by the steps between products and softmax (512 rows x 65600 keys, 8 heads, 147 us: tensor pipe and
// exponentials are at work half of the time each; 256 rows x 2100 keys, 16 sequences, 47 us); for few by the keys' bytes and some 4 us of a
// CTA's start and end (8 rows x 1080 keys, 32 sequences of 32 heads, 509 MB, 92 us: 5.5 TB/s).
//
// O stays in TMEM.  m is the largest score only up to a factor of 2^8: O is multiplied again when a row's maximum has grown by more than
// that, behind the product with V that is under way, which after the first tiles hardly ever happens; P and its sum stay below 2^8 per
// key, and their quotient does not depend on m.
//
// The masks matter only in the last tiles, where the nodes' keys are: 128 bits of a row, shifted to the tile's place.  There, and in the tiles
// that a window cuts, two more warps clear the values of keys that no node sees and of slots behind the last key, since 0 x NaN is NaN.
//
// Codes of an int8 cache are expanded on the way, by four warps between the ring that TMA fills and the one that the products read; they are
// exact in bf16, a key's scale multiplies its score and a value's its weight, in 32 bits.  Bound by shared memory: codes, values and the
// scales, which each row's thread reads (104 rows x 3500 keys, 16 sequences of 8 heads, 84 us; without scales 61, without the
// expansion 57).  (There the weights' conversion to bf16 may take the exponentials' unit, which has time.)
//
// Every wait is bounded and reports through the status word.
#include "tree_attention.cuh"

namespace xft {

int encode_tensor_map(CUtensorMap* out, const void* ptr, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows, uint32_t esize);

namespace {

constexpr int kTgRows = 128;

// Heads of 64 * H; I8: int8 cache.  G groups of four softmax warps, two over an int8 cache, which have a tile of rows each, or (TURNS) take
// turns at the key tiles of one.
template <int H, int G, bool I8, bool TURNS>
struct TgShape {
  // tiles of S of a group: with two of 64 keys the next one is made while the softmax is at this one (128 rows x 128 keys 1.62 us, with one
  // of 128 keys 1.74)
  static constexpr int kBufs = I8 ? 1 : 2;
  static constexpr int kKeys = 128 / kBufs;              // of a tile
  static constexpr int R = TURNS ? 1 : G;                // row tiles
  static constexpr int kLead = TURNS ? G : kBufs;        // S of so many tiles is ahead of P V
  static constexpr int kQHalf = kTgRows * 128, kHalf = kKeys * 128;          // 64 features of a tile's rows
  static constexpr int kQTile = H * kQHalf, kTile = H * kHalf;
  static constexpr int kTmem = H == 4 ? 512 : 256 * G;   // columns: of a group 128 of S, half of which becomes P, and O
  static constexpr int kStages = I8 ? (TURNS ? 4 : 2) : H == 4 ? 5 : 8 / H;              // 64 KB: two CTAs an SM, one with heads of 256
  static constexpr int kRaw = I8 ? (TURNS ? 3 : 5) : 0, kRawTile = kKeys * 128;                    // codes as they come
  static constexpr int kScales = I8 ? 4 : 0, kScaleBytes = 2 * kKeys * 4;            // of a tile's keys and values
  static constexpr int kSmem = R * kQTile + kStages * kTile + kRaw * kRawTile + kScales * kScaleBytes + 1024;
  static constexpr int kThreads = 128 + 128 * G + (I8 ? 128 : 0);
  static constexpr int kPerSm = G == 1 ? 2 : 1;
};

__device__ __forceinline__ float tg_max3(float a, float b, float c) {
  float d;
  asm("max.ftz.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float tg_min(float a, float b) {              // NaN where one of them is
  float d;
  asm("min.NaN.ftz.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 tg_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 tg_add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.ftz.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 tg_mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ uint32_t tg_pack(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
// Two weights (not negative) in bf16, rounded to the nearest, halves up.  Whole-number instructions: a conversion takes the unit of the
// exponentials, which bounds the softmax, as long as one of those.  (A NaN may come out as a number: the row's sum has it.)
__device__ __forceinline__ uint32_t tg_round(float lo, float hi) {
  return __byte_perm(__float_as_uint(lo) + 0x8000u, __float_as_uint(hi) + 0x8000u, 0x7632);
}
__device__ __forceinline__ void tg_ld_wait32(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]),
                 "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]),
                 "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])::"memory");
}

// Four codes as bf16, exact: (128 + the low seven bits) - (128 + the sign's 128), each one byte behind the exponent of 128
__device__ __forceinline__ uint32_t tg_sub2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint2 tg_codes(uint32_t c) {
  const uint32_t x = __byte_perm(c, 0x43434343u, 0x5140), y = __byte_perm(c, 0x43434343u, 0x5342);
  return make_uint2(tg_sub2(x & 0xff7fff7fu, x & 0xff80ff80u), tg_sub2(y & 0xff7fff7fu, y & 0xff80ff80u));
}

// Bits of 32 keys from key `first` on that a node with mask `m` (32-bit words) sees: the context's all, then the nodes'
// (of the words, the first two come in registers)
__device__ __forceinline__ uint32_t tg_sees(unsigned long long m01, const uint32_t* m, int first, int ctx, int n) {
  const int o = first - ctx;
  if (o <= -32) return 0xffffffffu;
  auto word = [&](int i) -> uint32_t {
    const int left = n - 32 * i;
    if (left <= 0) return 0;
    const uint32_t w = i == 0 ? (uint32_t)m01 : i == 1 ? (uint32_t)(m01 >> 32) : m[i];
    return left >= 32 ? w : w & ((1u << left) - 1);
  };
  if (o < 0) return (word(0) << -o) | ((1u << -o) - 1);
  return __funnelshift_r(word(o >> 5), word((o >> 5) + 1), o & 31);
}

__device__ __forceinline__ uint32_t tg_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }
// All of 32 keys from key `first` on but those of the context in front of key `from` that are not among the first `keep`
__device__ __forceinline__ uint32_t tg_context(int first, int ctx, int from, int keep) {
  return ~tg_below(ctx - first) | ~tg_below(from - first) | tg_below(keep - first);
}

// Of the same bits those that a window leaves: `pos` is the node's position, `at` the positions of the sequence's nodes
__device__ __forceinline__ uint32_t tg_window(uint32_t sees, int first, int ctx, int pos, const int* at, int window, int keep) {
  const uint32_t context = tg_below(ctx - first);
  sees &= tg_context(first, ctx, pos - window + 1, keep);
  for (uint32_t rest = sees & ~context; rest; rest &= rest - 1) {
    const int i = __ffs(rest) - 1, k = at[first + i - ctx];
    if (!((long long)pos - k < window || k < keep)) sees &= ~(1u << i);
  }
  return sees;
}

// EXT: windows with kept first keys (only tiles with a visible key are visited), and caps on the scores
template <int H, int G, bool I8, bool TURNS, bool EXT>
__global__ void __launch_bounds__(TgShape<H, G, I8, TURNS>::kThreads, TgShape<H, G, I8, TURNS>::kPerSm)
    tree_attention_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const TreeAttnArgs p) {
  using S = TgShape<H, G, I8, TURNS>;
  constexpr int D = 64 * H, ST = S::kStages, R = S::R, L = S::kLead, KT = S::kKeys, NC = KT / 32, NB = S::kBufs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                    // R tiles
  uint8_t* sT = smem + R * S::kQTile;                    // ring: keys and values of the tiles in turn
  uint8_t* sRaw = sT + ST * S::kTile;                    // I8: ring of codes, in the same order
  float* s_scales = reinterpret_cast<float*>(sRaw + S::kRaw * S::kRawTile);           // I8: ring of tiles' scales
  __shared__ uint64_t raw_full[S::kRaw + 1], raw_empty[S::kRaw + 1], c_full[S::kScales + 1], c_empty[S::kScales + 1];
  __shared__ uint64_t q_full, full[ST], empty[ST], v_here, v_clean, s_full[G * S::kBufs], p_half[G], p_full[G * S::kBufs], o_step[G], o_full[G];
  __shared__ float2 s_ml[TURNS ? kTgRows : 1];
  __shared__ uint32_t tmem_base_s, s_union[kTreeWords * 2];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, b = blockIdx.z;
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 4 * R);                           // (TURNS: the first group brings the queries)
    for (int s = 0; s < ST; ++s) { mbar_init(&full[s], I8 ? 4 : 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < S::kRaw; ++s) { mbar_init(&raw_full[s], 1); mbar_init(&raw_empty[s], 4); }
    for (int s = 0; s < S::kScales; ++s) { mbar_init(&c_full[s], 1); mbar_init(&c_empty[s], TURNS ? 4 : 4 * G); }
    mbar_init(&v_here, 1);
    mbar_init(&v_clean, 2);
    for (int g = 0; g < G; ++g) { mbar_init(&p_half[g], 4); mbar_init(&o_step[g], 1); mbar_init(&o_full[g], 1); }
    for (int i = 0; i < G * NB; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); }
    fence_barrier_init();
    fence_proxy_async();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_s, S::kTmem);
    tmem_relinquish();
  }
  grid_dep_launch();
  grid_dep_wait();
  const TreeSeq s(p, b);
  int h0;
  const int heads = tree_heads(p, kvh, h0), rows = s.n * heads;
  const int n_rt = (p.max_q * p.group + R * kTgRows - 1) / (R * kTgRows);
  const int row0 = (blockIdx.x % n_rt) * (R * kTgRows), slice = blockIdx.x / n_rt;
  // tiles: those of the kept first keys, then those from the first key of the widest window
  int lo = 0, n_keep = 0, first_key = 0;
  if (EXT && p.window > 0) {
    int at = 0x7fffffff;
    for (int i = lane; i < s.n; i += 32) at = min(at, p.positions[s.q0 + i]);
    at = __reduce_min_sync(0xffffffffu, at);
    first_key = tree_first(p, s, at);
    lo = first_key / KT;
    n_keep = min((min(p.keep, s.kv) + KT - 1) / KT, lo);
  }
  const int all = n_keep + (s.kv + KT - 1) / KT - lo, per = (all + p.nsplit - 1) / p.nsplit;
  const int t0 = min(all, slice * per), nt = row0 < rows ? min(all, t0 + per) - t0 : 0;
  auto tile_at = [&](int j) -> int { return EXT && t0 + j >= n_keep ? t0 + j - n_keep + lo : t0 + j; };
  const int tail = s.ctx / KT;                           // from this tile on there are keys that are not the context's
  // tile j has keys that no node may see: those that are not the context's, and the ones that the window leaves to none
  auto unseen = [&](int j) -> bool {
    const int t = tile_at(j), k0 = t * KT;
    return t >= tail || (EXT && max(k0, p.keep) < min(k0 + KT, first_key));
  };
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = tmem_base_s;

  // registers at launch: 256 x 128, int8 512 x 128; from here on 128 x 40 + 128 x 216, int8 128 x 40 + 256 x 200 + 128 x 72
  if (I8 && warp >= 4 + 4 * G) {
    // ------------------------------------------------------------------ codes to bf16, a row of a tile per thread
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int r = threadIdx.x & 127;
    Ring raw{0, 0}, ring{0, 1};
    for (int i = 0; i < 2 * nt; ++i) {
      if (!mbar_wait(&raw_full[raw.s], raw.ph, p.status, XFT_ERR_WAIT_FULL)) break;
      if (!mbar_wait(&empty[ring.s], ring.ph, p.status, XFT_ERR_WAIT_EMPTY)) break;
      const uint8_t* from = sRaw + raw.s * S::kRawTile + r * 128;
      uint8_t* to = sT + ring.s * S::kTile + r * 128;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(from + ((c ^ (r & 7)) << 4));
        const uint2 a0 = tg_codes(w.x), a1 = tg_codes(w.y), a2 = tg_codes(w.z), a3 = tg_codes(w.w);
        uint8_t* half = to + (c >> 2) * S::kHalf;
        *reinterpret_cast<uint4*>(half + (((2 * c & 7) ^ (r & 7)) << 4)) = make_uint4(a0.x, a0.y, a1.x, a1.y);
        *reinterpret_cast<uint4*>(half + (((2 * c + 1 & 7) ^ (r & 7)) << 4)) = make_uint4(a2.x, a2.y, a3.x, a3.y);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) { mbar_arrive(&full[ring.s]); mbar_arrive(&raw_empty[raw.s]); }
      raw.next(S::kRaw);
      ring.next(ST);
    }
  } else if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer
      if (elect_one()) {
        const int n_pieces = (s.kv + 63) / 64;
        Ring ring{0, 1};
        // one tile of keys or values, in the order that the products take them
        auto load = [&](int j, bool v) -> bool {
          int at[KT / 64];
          for (int i = 0; i < KT / 64; ++i) {            // past the last keys they are read again
            const int piece = min(KT / 64 * tile_at(j) + i, n_pieces - 1), first = piece * 64;
            at[i] = (tree_block(p, b, first / p.bs) * p.hkv + kvh) * p.bs + first % p.bs;
          }
          if constexpr (I8) {
            if (!v) {
              const int cs = j % S::kScales;
              if (!mbar_wait(&c_empty[cs], (j / S::kScales & 1) ^ 1, p.status, XFT_ERR_WAIT_EMPTY)) return false;
              float* to = s_scales + cs * 2 * KT;
              mbar_expect_tx(&c_full[cs], S::kScaleBytes);
              for (int i = 0; i < KT / 64; ++i) {
                bulk_load(to + i * 64, p.ks + at[i], 256, &c_full[cs]);
                bulk_load(to + KT + i * 64, p.vs + at[i], 256, &c_full[cs]);
              }
            }
            if (!mbar_wait(&raw_empty[ring.s], ring.ph, p.status, XFT_ERR_WAIT_EMPTY)) return false;
            mbar_expect_tx(&raw_full[ring.s], S::kRawTile);
            for (int i = 0; i < KT / 64; ++i)
              tma_load_2d(sRaw + ring.s * S::kRawTile + i * 8192, v ? &tmV : &tmK, &raw_full[ring.s], 0, at[i], kEvictNormal);
            ring.next(S::kRaw);
          } else {
            if (!mbar_wait(&empty[ring.s], ring.ph, p.status, XFT_ERR_WAIT_EMPTY)) return false;
            uint8_t* to = sT + ring.s * S::kTile;
            mbar_expect_tx(&full[ring.s], S::kTile);
            for (int i = 0; i < KT / 64; ++i)
              for (int h = 0; h < H; ++h)
                tma_load_2d(to + h * S::kHalf + i * 8192, v ? &tmV : &tmK, &full[ring.s], h * 64, at[i], kEvictNormal);
            ring.next(ST);
          }
          return true;
        };
        bool ok = true;
        for (int j = 0; j < min(L, nt) && ok; ++j) ok = load(j, false);
        for (int j = 0; j < nt && ok; ++j) ok = load(j, true) && (j + L >= nt || load(j + L, false));
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issuer
      if (nt > 0 && elect_one()) {
        constexpr uint32_t IDESC_S = umma_idesc(128, KT, 1, 1, 1);
        constexpr uint32_t IDESC_O = umma_idesc(128, D, 1, 1, 1) | (1u << 16);       // B = V, MN-major
        Ring ring{0, 0};
        bool ok = mbar_wait(&q_full, 0, p.status, XFT_ERR_WAIT_FULL);
        auto scores = [&](int g, int j, int st) {
          const uint64_t qd = umma_desc_k128(smem_u32(sQ + (TURNS ? 0 : g) * S::kQTile)), kd = umma_desc_k128(smem_u32(sT + st * S::kTile));
          tcgen05_fence_after();
#pragma unroll
          for (int k = 0; k < 4 * H; ++k) {
            const uint32_t q_off = ((k >> 2) * S::kQHalf + (k & 3) * 32) / 16, k_off = ((k >> 2) * S::kHalf + (k & 3) * 32) / 16;
            umma_bf16(tmem_base + g * 256 + j % NB * KT, qd + q_off, kd + k_off, IDESC_S, k > 0);
          }
          tcgen05_commit(&s_full[g * NB + j % NB]);
        };
        for (int j = 0; j < min(L, nt) && ok; ++j) {
          ok = mbar_wait(&full[ring.s], ring.ph, p.status, XFT_ERR_WAIT_FULL);
          if (!ok) break;
          for (int g = TURNS ? j : 0; g < (TURNS ? j + 1 : G); ++g) scores(g, j, ring.s);
          tcgen05_commit(&empty[ring.s]);
          ring.next(ST);
        }
        int cleaned = 0;
        for (int j = 0; j < nt && ok; ++j) {
          const Ring vr = ring;
          ring.next(ST);
          const Ring kr = ring;
          const bool more = j + L < nt;
          if (more) ring.next(ST);
          ok = mbar_wait(&full[vr.s], vr.ph, p.status, XFT_ERR_WAIT_FULL);
          if (!I8 && ok && unseen(j)) {
            mbar_arrive(&v_here);
            ok = mbar_wait(&v_clean, cleaned++ & 1, p.status, XFT_ERR_WAIT_FULL);
          }
          if (!ok) break;
          const uint64_t vd = umma_desc_mn128(smem_u32(sT + vr.s * S::kTile), S::kHalf);
          const int g0 = TURNS ? j % G : 0, g1 = TURNS ? g0 + 1 : G;
          const uint32_t ph = j / L & 1;
          for (int g = g0; g < g1; ++g) {
            const uint32_t pa = tmem_base + g * 256 + j % NB * KT, oa = tmem_base + g * 256 + 128;
            const bool sum = TURNS ? j >= G : j > 0;
            if (NB == 1) {                               // the product may begin with the first half of the keys
              ok = mbar_wait(&p_half[g], ph, p.status, XFT_ERR_WAIT_TMEM);
              if (!ok) break;
              tcgen05_fence_after();
#pragma unroll
              for (int k = 0; k < KT / 32; ++k) umma_bf16_ta(oa, pa + k * 8, vd + k * (2048 / 16), IDESC_O, sum || k > 0);
            }
            ok = mbar_wait(&p_full[g * NB + j % NB], ph, p.status, XFT_ERR_WAIT_TMEM);
            if (!ok) break;
            tcgen05_fence_after();
#pragma unroll
            for (int k = NB == 1 ? KT / 32 : 0; k < KT / 16; ++k) umma_bf16_ta(oa, pa + k * 8, vd + k * (2048 / 16), IDESC_O, sum || k > 0);
            if (g == g1 - 1) tcgen05_commit(&empty[vr.s]);
            if (NB > 1) tcgen05_commit(&o_step[g]);
            if (TURNS ? !more : j == nt - 1) tcgen05_commit(&o_full[g]);
            if (more) {                                  // the next S goes over P, behind the product that reads P
              if (g == g0) ok = mbar_wait(&full[kr.s], kr.ph, p.status, XFT_ERR_WAIT_FULL);
              if (!ok) break;
              scores(g, j + L, kr.s);
              if (g == g1 - 1) tcgen05_commit(&empty[kr.s]);
            }
          }
        }
      }
    } else if (!I8) {
      // ------------------------------------------------------------------ values that no node sees (codes are finite, their scales below)
      if (nt > 0 && tile_at(nt - 1) >= tail) {
        uint32_t seen[kTreeWords * 2] = {};
        const uint32_t* m = reinterpret_cast<const uint32_t*>(p.mask + (long long)s.q0 * p.words);
        for (int i = lane; i < s.n; i += 32) {
          if (EXT && p.window > 0) {
            const int* at = p.positions + s.q0;
            for (int w = 0; w < p.words; ++w) {
              const unsigned long long x = tree_within(p.mask[(long long)(s.q0 + i) * p.words + w], 64 * w, s.n, at[i], at, p.window, p.keep);
#pragma unroll
              for (int e = 0; e < kTreeWords; ++e)
                if (e == w) { seen[2 * e] |= (uint32_t)x; seen[2 * e + 1] |= (uint32_t)(x >> 32); }
            }
            continue;
          }
#pragma unroll
          for (int w = 0; w < kTreeWords * 2; ++w)
            if (w < 2 * p.words) seen[w] |= m[(long long)i * p.words * 2 + w];
        }
#pragma unroll
        for (int w = 0; w < kTreeWords * 2; ++w) {
          const uint32_t x = __reduce_or_sync(0xffffffffu, seen[w]);
          if (lane == 0 && warp == 2) s_union[w] = x;
        }
      }
      named_bar_sync(1, 64);
      for (int j = 0, cleaned = 0; j < nt; ++j) {
        if (!unseen(j)) continue;
        const int i = min(j + L, nt) + j, st = i % ST;   // of the ring's tiles, in order
        const uint32_t ph = i / ST & 1;
        // (these warps do not hold the ring back, so they ask the issuer which round it is in)
        if (!mbar_wait(&v_here, cleaned++ & 1, p.status, XFT_ERR_WAIT_FULL)) break;
        const int key = (warp - 2) * (KT / 2) + lane * (KT / 64);            // one or two keys a lane
        const int k0 = tile_at(j) * KT;
        const int k32 = k0 + (key & ~31);
        uint32_t sees = tg_sees((unsigned long long)s_union[1] << 32 | s_union[0], s_union, k32, s.ctx, s.n);
        if (EXT && p.window > 0) sees &= tg_context(k32, s.ctx, first_key, p.keep);
        sees >>= key & 31;
        if (!mbar_wait(&full[st], ph, p.status, XFT_ERR_WAIT_FULL)) break;
        uint8_t* v = sT + st * S::kTile;
#pragma unroll
        for (int e = 0; e < KT / 64; ++e)
          if (!(sees >> e & 1))
#pragma unroll
            for (int c = 0; c < 8 * H; ++c)
              *reinterpret_cast<uint4*>(v + (c >> 3) * S::kHalf + (key + e) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_clean);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax: one row per thread
    if (I8) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int g = (warp - 4) >> 2, qd = warp & 3;
    const int tile = TURNS ? 0 : g, r = qd * 32 + lane, row = row0 + tile * kTgRows + r;
    const bool mine = row < rows, busy = row0 + tile * kTgRows + qd * 32 < rows;          // the row, some row of the warp
    const int node = mine ? row / heads : 0, h = h0 + (mine ? row - node * heads : 0);
    const long long at = (long long)(s.q0 + node) * p.hq + h;
    if (nt > 0 && (!TURNS || g == 0)) {
      // this row of queries in the order that the product reads: 16-byte pieces exchanged with the row's low bits
      uint8_t* to = sQ + tile * S::kQTile + r * 128;
      uint4 v[8];
#pragma unroll
      for (int half = 0; half < H; ++half) {
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = mine ? *reinterpret_cast<const uint4*>(p.q + at * D + half * 64 + c * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(to + half * S::kQHalf + ((c ^ (r & 7)) << 4)) = v[c];
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    }
    const uint32_t base = tmem_base + g * 256 + (uint32_t(qd * 32) << 16), oa = base + 128;
    const uint32_t* bits = reinterpret_cast<const uint32_t*>(p.mask + (long long)(s.q0 + node) * p.words);
    const unsigned long long first_bits = nt > 0 && tile_at(nt - 1) >= tail ? p.mask[(long long)(s.q0 + node) * p.words] : 0;
    const bool caps = EXT && p.softcap > 0.f;
    const float scale = caps ? 1.f : p.scale * kTreeLog2e;           // (capped scores are in octaves already)
    const float cap = p.softcap * kTreeLog2e, inv_cap = caps ? p.scale / p.softcap : 0.f;
    const int pos = EXT && p.window > 0 && nt > 0 ? p.positions[s.q0 + node] : 0;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    const int first = TURNS ? g : 0;                     // of this group's tiles
    constexpr int kRing = I8 ? S::kScales : 1;
    for (int j = first; j < nt; j += TURNS ? G : 1) {
      const int cs = j % kRing;
      const int buf = j % NB, box = g * NB + buf;
      const uint32_t ph = j / L & 1, sa = base + buf * KT;
      const float* scales = s_scales + cs * 2 * KT;
      if (I8 && !mbar_wait(&c_full[cs], j / kRing & 1, p.status, XFT_ERR_WAIT_FULL)) { ok = false; break; }
      if (!mbar_wait(&s_full[box], ph, p.status, XFT_ERR_WAIT_TMEM)) { ok = false; break; }
      tcgen05_fence_after();
      if (!busy) {
        if (lane == 0) { if (NB == 1) mbar_arrive(&p_half[g]); mbar_arrive(&p_full[box]); if (I8) mbar_arrive(&c_empty[cs]); }
        continue;
      }
      uint32_t x[NC][32];
#pragma unroll
      for (int c = 0; c < NC; ++c) tmem_ld32(sa + 32 * c, x[c]);
#pragma unroll
      for (int c = 0; c < NC; ++c) tg_ld_wait32(x[c]);
      if constexpr (I8) {                                // a key's scale belongs to its scores
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 16) {
            float4 f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = *reinterpret_cast<const float4*>(scales + 32 * c + i + 4 * e);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float2 y = tg_mul2(make_float2(__uint_as_float(x[c][i + e]), __uint_as_float(x[c][i + e + 1])),
                                       make_float2((&f[e >> 2].x)[e & 3], (&f[e >> 2].x)[(e & 3) + 1]));
              x[c][i + e] = __float_as_uint(y.x);
              x[c][i + e + 1] = __float_as_uint(y.y);
            }
          }
      }
      if (caps) {                                        // cap tanh(z), z = score / cap
        float far = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            x[c][i] = __float_as_uint(__uint_as_float(x[c][i]) * inv_cap);
            far = fmaxf(far, fabsf(__uint_as_float(x[c][i])));
          }
        if (__all_sync(0xffffffffu, far <= 1.f)) {
          // tanh(z) / z as a polynomial in z^2, minimax on [0, 1] (off by less than 2e-7), away from the exponentials' unit
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float z = __uint_as_float(x[c][i]), y = z * z;
              float q = 0.0010410224785f;
              q = fmaf(q, y, -0.0062033790164f);
              q = fmaf(q, y, 0.020289981738f);
              q = fmaf(q, y, -0.053457029164f);
              q = fmaf(q, y, 0.13325203957f);
              q = fmaf(q, y, -0.33332839608f);
              q = fmaf(q, y, 0.99999994040f);
              x[c][i] = __float_as_uint(z * cap * q);
            }
        } else {
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              x[c][i] = __float_as_uint(cap - __fdividef(2.f * cap, 1.f + exp2f(tg_min(__uint_as_float(x[c][i]) * 2.8853900817779268f, 120.f))));
        }
      }
      const int k0 = tile_at(j) * KT;
      uint32_t sees[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) sees[c] = 0xffffffffu;
      const bool ends = k0 + KT > s.ctx;
      if (ends || (EXT && p.window > 0)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (ends) sees[c] = tg_sees(first_bits, bits, k0 + 32 * c, s.ctx, s.n);
          if (EXT && p.window > 0) sees[c] = tg_window(sees[c], k0 + 32 * c, s.ctx, pos, p.positions + s.q0, p.window, p.keep);
          if (__any_sync(0xffffffffu, sees[c] != 0xffffffffu))
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(sees[c] >> i & 1)) x[c][i] = 0xff800000u;
        }
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 2) top[(i >> 1) & 3] = tg_max3(top[(i >> 1) & 3], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
      const float mx = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale);
      const bool grown = mx > m + 8.f;
      if (__any_sync(0xffffffffu, grown)) {
        const float f = grown ? exp2f(m - mx) : 1.f;     // 0 where nothing has been seen yet
        if (grown) m = mx;
        l *= f;
        if (j > first) {
          // NB = 2: of the products with V, the last one may be under way (the one before it is not, S came behind that: two phases are
          // possible here, which a parity can tell apart); NB = 1: S came behind the last one
          if (NB > 1 && !mbar_wait(&o_step[g], (j - 1) & 1, p.status, XFT_ERR_WAIT_TMEM)) { ok = false; break; }
          tcgen05_fence_after();
          uint32_t y[32];
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            tmem_ld32(oa + c, y);
            tg_ld_wait32(y);
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
            tmem_st32(oa + c, y);
          }
        }
      }
      const float off = m == -INFINITY ? 0.f : -m;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint32_t w[16];
        float4 f[I8 ? 8 : 1];                            // the values' scales
        if constexpr (I8)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = *reinterpret_cast<const float4*>(scales + KT + 32 * c + 4 * i);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float2 e = tg_fma2(make_float2(__uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1])), make_float2(scale, scale), make_float2(off, off));
          e.x = exp2f(e.x);
          e.y = exp2f(e.y);
          sum[(i >> 1) & 1] = tg_add2(sum[(i >> 1) & 1], e);
          if constexpr (I8) {                            // a value's scale belongs to the product, not to the sum
            e = tg_mul2(e, make_float2((&f[i >> 2].x)[i & 3], (&f[i >> 2].x)[(i & 3) + 1]));
            if (sees[c] != 0xffffffffu) {                // (0 x the scale of a slot behind the last key may be NaN)
              if (!(sees[c] >> i & 1)) e.x = 0.f;
              if (!(sees[c] >> (i + 1) & 1)) e.y = 0.f;
            }
          }
          w[i >> 1] = I8 ? tg_pack(e.x, e.y) : tg_round(e.x, e.y);           // (int8: the other instructions are what is short)
        }
        tmem_st16(sa + 16 * c, w);
        if (NB == 1 && c == NC / 2 - 1) {                // the product may begin with the first half of the keys
          tmem_st_wait();
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_half[g]);
        }
      }
      const float2 t = tg_add2(sum[0], sum[1]);
      l += t.x + t.y;
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) { mbar_arrive(&p_full[box]); if (I8) mbar_arrive(&c_empty[cs]); }
    }
    bool have = ok && busy && nt > first;                // the group has sums
    for (int o = 0; o < G; ++o)                          // (TURNS: the ring is free for the exchange when both are through)
      if (have && (TURNS ? o < nt : o == g)) have = mbar_wait(&o_full[o], 0, p.status, XFT_ERR_WAIT_TMEM);
    tcgen05_fence_after();
    float f = 1.f, f2 = 0.f;
    if constexpr (TURNS) {
      // the second group's sums go through shared memory, column after column
      float* sO = reinterpret_cast<float*>(sT);
      if (g == 1) {
        s_ml[r] = have ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
        if (have)
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t y[32];
            tmem_ld32(oa + c, y);
            tg_ld_wait32(y);
#pragma unroll
            for (int i = 0; i < 32; ++i) sO[(c + i) * kTgRows + r] = __uint_as_float(y[i]);
          }
      }
      named_bar_sync(1, 256);
      const float2 o = s_ml[r];
      if (g == 0 && o.y != 0.f) {
        const float mx = fmaxf(m, o.x);
        f = m == -INFINITY ? 0.f : exp2f(m - mx);
        f2 = o.x == -INFINITY ? 1.f : exp2f(o.x - mx);   // (a NaN among the sums stays one)
        l = l * f + o.y * f2;
        m = mx;
      }
      if (g == 1) have = false;
    }
    if (have) {
      float all = 1.f;
      if (p.nsplit == 1) {
        float sum = l;
        if (p.sinks) {
          const float sink = p.sinks[h] * kTreeLog2e, mx = fmaxf(m, sink);
          all = exp2f(m - mx);
          sum = sum * all + exp2f(sink - mx);
        }
        all = l == 0.f ? 0.f : __fdividef(all, sum);     // a row that sees nothing
      }
      f *= all;
      f2 *= all;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t y[32];
        tmem_ld32(oa + c, y);
        tg_ld_wait32(y);
        if (TURNS && f2 != 0.f) {
          const float* sO = reinterpret_cast<const float*>(sT);
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f + sO[(c + i) * kTgRows + r] * f2);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
        }
        if (mine && p.nsplit == 1) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = tg_pack(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]));
          st_global_256(p.out + at * D + c, w);
          st_global_256(p.out + at * D + c + 16, w + 8);
        } else if (mine) {
          float* o = p.part_o + (at * p.nsplit + slice) * D + c;
#pragma unroll
          for (int i = 0; i < 32; i += 8) st_global_256(o + i, y + i);
        }
      }
    }
    if (mine && p.nsplit > 1 && (!TURNS || g == 0))
      *reinterpret_cast<float2*>(p.part_ml + (at * p.nsplit + slice) * 2) = have ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
  }
  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, S::kTmem);
  }
}

template <int H, int G, bool I8, bool TURNS, bool EXT>
int launch(const TreeAttnArgs& a, cudaStream_t st) {
  using S = TgShape<H, G, I8, TURNS>;
  CUtensorMap tmK, tmV;
  const uint64_t rows = (uint64_t)a.num_blocks * a.hkv * a.bs;
  const uint32_t size = I8 ? 1 : 2;
  if (encode_tensor_map(&tmK, a.kc, rows, a.D, a.D, 64, size) || encode_tensor_map(&tmV, a.vc, rows, a.D, a.D, 64, size)) return -4;
  auto k = tree_attention_tc_kernel<H, G, I8, TURNS, EXT>;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess) return 3000 + (int)cudaGetLastError();
  const int n_rt = (a.max_q * a.group + S::R * kTgRows - 1) / (S::R * kTgRows);
  const cudaError_t e = launch_pdl(k, dim3(n_rt * a.nsplit, a.hkv, a.B), dim3(S::kThreads), (size_t)S::kSmem, st, tmK, tmV, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

template <bool EXT>
int pick(const TreeAttnArgs& a, cudaStream_t st) {
  if (a.ks) return a.form == 2 ? launch<2, 2, true, false, EXT>(a, st) : launch<2, 2, true, true, EXT>(a, st);
  return a.D == 64 ? launch<1, 1, false, false, EXT>(a, st) : a.D == 128 ? launch<2, 1, false, false, EXT>(a, st) : launch<4, 1, false, false, EXT>(a, st);
}

}  // namespace

// 0, -1 where the shape is not one of this kernel's, or an error
int launch_tree_attention_tc(const TreeAttnArgs& a, cudaStream_t st) {
  if (a.bs % 64 || (!(a.scale > 0.f) && !(a.softcap > 0.f)) || (a.D != 64 && a.D != 128 && a.D != 256) || (!a.ks && a.form != 1)) return -1;
  if ((long long)a.num_blocks * a.hkv * a.bs > 0x7fffffffll) return -1;
  if (a.ks && (a.D != 128 || ((reinterpret_cast<uintptr_t>(a.ks) | reinterpret_cast<uintptr_t>(a.vs)) & 15))) return -1;
  return a.window > 0 || a.softcap > 0.f ? pick<true>(a, st) : pick<false>(a, st);
}

}  // namespace xft
