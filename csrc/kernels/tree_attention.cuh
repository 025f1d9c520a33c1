// Arguments of the kernels for trees of drafted tokens over the paged cache, and what they share.
#pragma once
#include "ptx.cuh"

namespace xft {

constexpr int kTreeMaxNodes = 256;           // of one sequence
constexpr int kTreeWords = kTreeMaxNodes / 64;

struct TreeAttnArgs {
  const __nv_bfloat16* q;                    // [T, hq, D]
  __nv_bfloat16* out;                        // [T, hq, D]
  const void* kc; const void* vc;            // [num_blocks, hkv, bs, D] bf16 or int8
  const float* ks; const float* vs;          // int8: [num_blocks, hkv, bs]
  const int* table;                          // [B, table_w], rows table_ld apart
  const int* cu_q; const int* kv_lens;       // [B + 1], [B]
  const unsigned long long* mask;            // [T, words]
  const int* positions;                      // [T], with a window only
  const float* sinks;                        // [hq] or null
  float* part_o;                             // [T, hq, nsplit, D] where nsplit > 1
  float* part_ml;                            // [T, hq, nsplit, 2]
  int* status;
  long long table_ld;
  int B, T, max_q, hq, hkv, group, q_off, D, bs, num_blocks, table_w, words, nsplit, window, keep;
  float scale, softcap;
  int form;                                  // row tiles of a CTA in tree_attention_sm100.cu (2: int8 only), 0: tree_attention.cu
};

// One sequence's rows and keys, cut to what the arrays hold; n = 0 where the lengths cannot be right
struct TreeSeq {
  int q0, n, kv, ctx;
  __device__ __forceinline__ TreeSeq(const TreeAttnArgs& p, int b) {
    q0 = p.cu_q[b];
    n = p.cu_q[b + 1] - q0;
    kv = p.kv_lens[b];
    if (q0 < 0 || n < 0 || n > p.max_q || q0 > p.T - n || kv < n || kv > (long long)p.table_w * p.bs) {
      if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, XFT_ERR_BOUNDS);
      n = 0;
    }
    ctx = kv - n;
  }
};

// Query heads of kv head `kvh`: h0 .. h0 + heads - 1
__device__ __forceinline__ int tree_heads(const TreeAttnArgs& p, int kvh, int& h0) {
  h0 = max(0, kvh * p.group - p.q_off);
  return max(0, min(p.hq, (kvh + 1) * p.group - p.q_off) - h0);
}

// Block `i` of a sequence; one that is outside the pool is reported and read as block 0
__device__ __forceinline__ int tree_block(const TreeAttnArgs& p, int b, int i) {
  int blk = p.table[b * p.table_ld + i];
  if (blk < 0 || blk >= p.num_blocks) {
    if (p.status) atomicCAS(p.status, 0, XFT_ERR_BOUNDS);
    blk = 0;
  }
  return blk;
}

// Of a mask's bits for nodes first .. first + 63, those whose nodes the window leaves to a node at `pos`; `at`: positions of the sequence's n nodes
__device__ __forceinline__ unsigned long long tree_within(unsigned long long m, int first, int n, int pos, const int* at, int window, int keep) {
  if (n - first < 64) m &= n > first ? (1ull << (n - first)) - 1 : 0;
  for (unsigned long long rest = m; rest; rest &= rest - 1) {
    const int i = __ffsll(rest) - 1, k = at[first + i];
    if (!((long long)pos - k < window || k < keep)) m &= ~(1ull << i);
  }
  return m;
}

// The first key of the context that a window leaves to some node, `at` the lowest position of the nodes
__device__ __forceinline__ int tree_first(const TreeAttnArgs& p, const TreeSeq& s, int at) {
  return (int)max(0ll, min((long long)at - p.window + 1, (long long)s.ctx));
}

constexpr float kTreeLog2e = 1.4426950408889634f;

int launch_tree_join(const TreeAttnArgs& a, cudaStream_t st);                 // tree_attention.cu
int launch_tree_attention_tc(const TreeAttnArgs& a, cudaStream_t st);         // tree_attention_sm100.cu

}  // namespace xft
