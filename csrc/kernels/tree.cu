// Trees of drafted tokens: what each node sees, and the path that sampled tokens agree with.
//
// tree_mask_kernel: the nodes on the way from node i to its root, as bits, and their number, which is the node's distance from the
// context.  Latency is all of it (4 bytes in, 12 out per node): one launch, a thread per node that walks its parents in shared memory.  us in a graph: a tree of 26 nodes
// 2.3, 192 trees of up to 64 3.9.
//
// tree_accept_kernel: from node 0 on to the lowest child that carries the token sampled at its parent, until there is none.  Then the
// accepted nodes' cache rows move together: node path[j] of a sequence goes to position context + j of its cache, in every pool.  Every
// CTA walks the path itself, a few steps of one warp, instead of waiting for another launch.  Rows move in ascending order, each
// 16-byte piece by one thread: node path[j] >= j, so what is overwritten by an earlier move has been read before.
// Bound by the walk (a few dozen cycles a step from shared memory) and one trip to memory and back.  us in a graph: a tree of 16 in 32
// layers 3.4; 16 trees of 64 in 80 layers, 20 MB, 7.7.
#include "ptx.cuh"

namespace xft {

constexpr int kTreeNodes = 256;                // of one sequence

struct TreeBatch {
  const int* cu_q;                             // [B + 1]
  const int* kv_lens;                          // [B]
  int B, T;
};

// Rows of sequence b, cut to what the arrays hold; false where they cannot be right
__device__ __forceinline__ bool tree_rows(const TreeBatch& t, int b, int& q0, int& n) {
  q0 = t.cu_q[b];
  n = t.cu_q[b + 1] - q0;
  const bool ok = q0 >= 0 && n >= 0 && n <= kTreeNodes && q0 <= t.T - n;
  if (!ok) n = 0;
  return ok;
}

struct TreeMaskArgs {
  TreeBatch t;
  const int* parents;                          // [T]
  long long* mask;                             // [T, words]
  int* positions;                              // [T]
  int* status;
  int words;
};

__global__ void __launch_bounds__(kTreeNodes) tree_mask_kernel(const TreeMaskArgs a) {
  __shared__ int up[kTreeNodes];
  grid_dep_launch();
  grid_dep_wait();
  const int b = blockIdx.x, i = threadIdx.x;
  int q0, n;
  bool bad = !tree_rows(a.t, b, q0, n);
  if (n > 64 * a.words || n > (int)blockDim.x) { bad = true; n = 0; }
  if (i < n) {
    const int p = a.parents[q0 + i];
    up[i] = p < i ? p : -1;                    // a parent comes before its children: the walk ends
    bad |= p >= i;
  }
  __syncthreads();
  if (bad) atomicCAS(a.status, 0, XFT_ERR_BOUNDS);
  if (i >= n) return;
  unsigned long long w[kTreeNodes / 64] = {};
  int depth = -1;
  for (int at = i; at >= 0; at = up[at], ++depth) {
#pragma unroll
    for (int j = 0; j < kTreeNodes / 64; ++j)
      if (at >> 6 == j) w[j] |= 1ull << (at & 63);
  }
#pragma unroll
  for (int j = 0; j < kTreeNodes / 64; ++j)
    if (j < a.words) a.mask[(long long)(q0 + i) * a.words + j] = (long long)w[j];
  a.positions[q0 + i] = a.t.kv_lens[b] - n + depth;
}

struct TreeAcceptArgs {
  TreeBatch t;
  const long long* tokens;                     // [T]
  const long long* sampled;                    // [T]
  const int* parents;                          // [T]
  const int* table;                            // [B, table_w], rows table_ld apart
  const long long* pools;                      // [n_pools, 3]: address, heads, bytes of a row (a key, a value or a scale of one head)
  long long* emitted;                          // [B, width]
  int* path;                                   // [B, width]
  int* count;                                  // [B]
  int* status;
  long long table_ld;
  int table_w, n_pools, bs, num_blocks, width;
};

constexpr int kAcceptThreads = 256;
constexpr int kAcceptMoves = 2, kAcceptPieces = 4;           // rows that a thread has under way at a time, and pieces of each

template <typename V>
__device__ __forceinline__ void move_rows(char* pool, long long head_rows, int heads, int row_bytes, const int* src, const int* dst, const int* blk_src,
                                          const int* blk_dst, int n) {
  const int pieces = row_bytes / (int)sizeof(V), all = heads * pieces;
  for (int i0 = threadIdx.x & 31; i0 < all; i0 += 32 * kAcceptPieces) {
    for (int j0 = 0; j0 < n; j0 += kAcceptMoves) {
      V v[kAcceptPieces][kAcceptMoves];
      auto each = [&](const int* blk, const int* row, auto use) {
#pragma unroll
        for (int e = 0; e < kAcceptPieces; ++e) {
          const int i = i0 + 32 * e, h = i / pieces, at = (i - h * pieces) * (int)sizeof(V);
#pragma unroll
          for (int j = 0; j < kAcceptMoves; ++j)
            if (i < all && j0 + j < n)
              use(v[e][j], reinterpret_cast<V*>(pool + (((long long)blk[j0 + j] * heads + h) * head_rows + row[j0 + j]) * row_bytes + at));
        }
      };
      each(blk_src, src, [](V& x, const V* from) { x = *from; });
      each(blk_dst, dst, [](const V& x, V* to) { *to = x; });
    }
  }
}

__global__ void __launch_bounds__(kAcceptThreads) tree_accept_kernel(const TreeAcceptArgs a) {
  __shared__ int path[kTreeNodes], src[kTreeNodes], dst[kTreeNodes], blk_src[kTreeNodes], blk_dst[kTreeNodes];
  __shared__ long long says[kTreeNodes];
  __shared__ int s_count, s_moves;
  grid_dep_launch();
  grid_dep_wait();
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pool = blockIdx.x * (kAcceptThreads / 32) + warp;
  long long place[3] = {};
  if (pool < a.n_pools)
    for (int i = 0; i < 3; ++i) place[i] = a.pools[3 * pool + i];
  int q0, n;
  bool bad = !tree_rows(a.t, b, q0, n);
  if (n > a.width) { bad = true; n = 0; }
  const int kv = a.t.kv_lens[b];
  if (kv < n) { bad = true; n = 0; }
  const int ctx = kv - n;
  if (warp == 0) {
    int count = 0;
    // eight nodes a lane
    int up[kTreeNodes / 32];
    long long tok[kTreeNodes / 32];
#pragma unroll
    for (int e = 0; e < kTreeNodes / 32; ++e) {
      const int i = lane + 32 * e;
      up[e] = i < n ? a.parents[q0 + i] : -1;
      tok[e] = i < n ? a.tokens[q0 + i] : 0;
      if (i < n) says[i] = a.sampled[q0 + i];              // (a step that reads it from memory takes ten times as long)
    }
    __syncwarp();
    for (int at = n > 0 ? 0 : -1; at >= 0;) {
      if (lane == 0) path[count] = at;
      ++count;
      const long long said = says[at];
      unsigned next = 0xffffffffu;
#pragma unroll
      for (int e = kTreeNodes / 32 - 1; e >= 0; --e) {
        const int i = lane + 32 * e;
        if (i > at && up[e] == at && tok[e] == said) next = i;
      }
      next = __reduce_min_sync(0xffffffffu, next);
      at = next == 0xffffffffu ? -1 : (int)next;
    }
    __syncwarp();
    int moves = 0;
    for (int j0 = 0; j0 < count; j0 += 32) {               // rows that change their place, in order
      const int j = j0 + lane;
      bool moved = j < count && path[j] != j && a.n_pools > 0;
      int s = 0, d = 0, sb = 0, db = 0;
      if (moved) {
        s = ctx + path[j]; d = ctx + j;
        const bool in = s / a.bs < a.table_w;
        sb = in ? a.table[b * a.table_ld + s / a.bs] : -1;
        db = in ? a.table[b * a.table_ld + d / a.bs] : -1;
        if (sb < 0 || sb >= a.num_blocks || db < 0 || db >= a.num_blocks) { bad = true; moved = false; }
      }
      const unsigned who = __ballot_sync(0xffffffffu, moved);
      if (moved) {
        const int to = moves + __popc(who & ((1u << lane) - 1u));
        src[to] = s % a.bs; dst[to] = d % a.bs; blk_src[to] = sb; blk_dst[to] = db;
      }
      moves += __popc(who);
    }
    if (lane == 0) { s_count = count; s_moves = moves; }
  }
  if (bad && a.status) atomicCAS(a.status, 0, XFT_ERR_BOUNDS);
  __syncthreads();
  const int moves = s_moves, count = s_count;
  if (blockIdx.x == 0) {
    for (int j = threadIdx.x; j < a.width; j += kAcceptThreads) {
      a.path[(long long)b * a.width + j] = j < count ? path[j] : -1;
      a.emitted[(long long)b * a.width + j] = j < count ? says[path[j]] : -1;
    }
    if (threadIdx.x == 0) a.count[b] = count;
  }
  if (!moves || pool >= a.n_pools) return;
  char* base = reinterpret_cast<char*>(place[0]);
  const int heads = (int)place[1], row = (int)place[2];
  if (row % 16 == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0) move_rows<uint4>(base, a.bs, heads, row, src, dst, blk_src, blk_dst, moves);
  else move_rows<uint16_t>(base, a.bs, heads, row, src, dst, blk_src, blk_dst, moves);
}

}  // namespace xft

using namespace xft;

extern "C" int xft_tree_mask(const char* packed, int threads, cudaStream_t st) {
  TreeMaskArgs a;
  memcpy(&a, packed, sizeof(a));
  if (a.t.B <= 0) return 0;
  if (threads < 1 || threads > kTreeNodes || a.words < 1) return -1;
  const cudaError_t e = launch_pdl(tree_mask_kernel, dim3(a.t.B), dim3((threads + 31) / 32 * 32), 0, st, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// tokens, sampled, parents: [T]; pools may be none (then only the path is found).
extern "C" int xft_tree_accept(const char* packed, cudaStream_t st) {
  TreeAcceptArgs a;
  memcpy(&a, packed, sizeof(a));
  if (a.t.B <= 0) return 0;
  if (a.t.B > 65535 || a.width < 1 || a.n_pools < 0 || (a.n_pools > 0 && (a.bs < 1 || !a.table))) return -1;
  const int per = kAcceptThreads / 32;
  const cudaError_t e = launch_pdl(tree_accept_kernel, dim3(a.n_pools ? (a.n_pools + per - 1) / per : 1, a.t.B), dim3(kAcceptThreads), 0, st, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
