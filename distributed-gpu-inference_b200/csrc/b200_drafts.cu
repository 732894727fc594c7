// Trees of drafted tokens: which nodes each node sees, and what becomes of a tree once the model has answered at every node.
//
// A tree has up to 64 nodes, node 0 is its root (the last token that is certain), every other node comes behind its parent.  Sets of nodes
// are 64-bit masks: visible[t] is the node itself and all above it.
//
//   fits[t]   the node's token is what the model chose at its parent, and no earlier sibling has the same token (the root fits)
//   taken[t]  all of visible[t] fits.  At most one child of a node fits, so the taken nodes are one path from the root, in order of
//             their numbers.
//
// accept_drafts_kernel: one CTA per (sequence, layer, keys or values); each finds the path by itself (64 nodes: two ballots), the first of a sequence writes it
// down, and all move their layer's rows.  The k-th taken node's row goes to the k-th place behind the context, never to a later place than
// it has (path[k] >= k), so a thread that walks k upwards with its own piece of the rows reads every row before it is written over.
// Bound by latency where few rows move (three dependent loads: tree, table, rows: with draft_tree_kernel 4.5 us on the device for one sequence and 4 layers),
// by memory where many do (64 sequences, 6 of 24 nodes taken, 32 layers of 8 kv heads of 128: 13 us for 84 MB that move); a call after the other the host's
// two launches and their checks, 29 us, are longer than both.
#include "b200_common.cuh"

namespace b200 {
namespace {

constexpr int kMaxNodes = B200_MAX_DRAFT_NODES;

__global__ void __launch_bounds__(kMaxNodes)
draft_tree_kernel(int64_t* __restrict__ visible, int32_t* __restrict__ depth, const int32_t* __restrict__ parents, int64_t parent_stride,
                  const int32_t* __restrict__ draft_lens, int nodes) {
  __shared__ unsigned long long seen[2][kMaxNodes];
  __shared__ int up[2][kMaxNodes];
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x, n = draft_lens ? min(max(draft_lens[b], 0), nodes) : nodes;
  // a parent that is none, or not before its child: the node sees itself only
  int p = t > 0 && t < n ? parents[b * parent_stride + t] : -1;
  if (p < 0 || p >= t) p = -1;
  unsigned long long m = t < n ? 1ull << t : 0ull;
  for (int step = 1, cur = 0; step < n; step *= 2, cur ^= 1) {    // masks of 1, 2, 4 ... nodes up
    seen[cur][t] = m;
    up[cur][t] = p;
    __syncthreads();
    if (p >= 0) {
      m |= seen[cur][p];
      p = up[cur][p];
    }
  }
  if (t < nodes) {
    visible[b * nodes + t] = static_cast<int64_t>(m);
    depth[b * nodes + t] = max(__popcll(m) - 1, 0);
  }
}

struct Accept {
  int32_t *count, *path;
  int64_t* new_tokens;
  int32_t* new_lens;
  const int64_t *tokens, *chosen, *visible;
  const int32_t* parents;
  int64_t token_stride, chosen_stride, parent_stride, visible_stride;
  void* const* k_pools;
  void* const* v_pools;
  const int32_t* block_tables;
  int table_stride, table_cols;
  const int32_t *context_lens, *draft_lens;
  int nodes, n_layers, Hkv, bs, row_bytes;
  int64_t max_blocks;
};

// rows of `pool` (row_bytes per head) from src[k] to dst[k], k upwards, in pieces of type V
template <typename V>
__device__ __forceinline__ void move_rows(char* pool, const int64_t* src, const int64_t* dst, int count, int Hkv, int64_t head_bytes, int row_bytes) {
  constexpr int kAhead = 4;
  const int per = row_bytes / sizeof(V);
  for (int c = threadIdx.x; c < Hkv * per; c += blockDim.x) {
    const int h = c / per;
    char* mine = pool + h * head_bytes + static_cast<int64_t>(c - h * per) * sizeof(V);
    for (int k = 1; k < count; k += kAhead) {
      V v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (k + u < count && dst[k + u] >= 0) v[u] = *reinterpret_cast<const V*>(mine + src[k + u]);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (k + u < count && dst[k + u] >= 0) *reinterpret_cast<V*>(mine + dst[k + u]) = v[u];
    }
  }
}

__global__ void __launch_bounds__(128)
accept_drafts_kernel(const Accept A) {
  __shared__ int64_t tok[kMaxNodes];
  __shared__ int par[kMaxNodes];
  __shared__ unsigned fits_s[2], taken_s[2];
  __shared__ int64_t src[kMaxNodes], dst[kMaxNodes];
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x, lane = t & 31;
  const int ctx = max(A.context_lens[b], 0);
  const int n = min(A.draft_lens ? max(A.draft_lens[b], 0) : A.nodes, min(A.nodes, ctx));
  const int base = ctx - n;
  if (t < kMaxNodes) {
    tok[t] = t < n ? A.tokens[b * A.token_stride + t] : 0;
    int p = t < n ? A.parents[b * A.parent_stride + t] : -1;
    par[t] = p >= 0 && p < t ? p : -1;
  }
  __syncthreads();
  if (t < kMaxNodes) {
    const int p = par[t];
    bool fits = t == 0;
    if (t > 0 && t < n && p >= 0) {
      fits = tok[t] == A.chosen[b * A.chosen_stride + p];
      for (int s = p + 1; s < t && fits; ++s) fits = par[s] != p || tok[s] != tok[t];
    }
    const unsigned f = __ballot_sync(0xffffffffu, fits && t < n);
    if (lane == 0) fits_s[t >> 5] = f;
  }
  __syncthreads();
  const unsigned long long fits = fits_s[0] | static_cast<unsigned long long>(fits_s[1]) << 32;
  if (t < kMaxNodes) {
    const bool taken = t < n && (fits >> t & 1) && (static_cast<unsigned long long>(A.visible[b * A.visible_stride + t]) & ~fits) == 0;
    const unsigned f = __ballot_sync(0xffffffffu, taken);
    if (lane == 0) taken_s[t >> 5] = f;
  }
  __syncthreads();
  const unsigned long long taken = taken_s[0] | static_cast<unsigned long long>(taken_s[1]) << 32;
  const int count = __popcll(taken);
  const bool writes = blockIdx.y == 0;
  if (writes && t < A.nodes) {      // behind the path
    if (t >= count) {
      A.path[b * A.nodes + t] = -1;
      A.new_tokens[b * A.nodes + t] = -1;
    }
    if (t == 0) {
      A.count[b] = count;
      A.new_lens[b] = base + count;
    }
  }
  if (t < kMaxNodes && (taken >> t & 1)) {
    const int k = __popcll(taken & ((1ull << t) - 1));
    if (writes) {
      A.path[b * A.nodes + k] = t;
      A.new_tokens[b * A.nodes + k] = A.chosen[b * A.chosen_stride + t];
    }
    int64_t from = -1, to = -1;
    if (A.n_layers > 0 && k != t) {
      auto place = [&](int pos) -> int64_t {
        const int col = pos / A.bs, off = pos - col * A.bs;
        const int64_t page = col < A.table_cols ? A.block_tables[b * A.table_stride + col] : -1;
        return page < 0 || page >= A.max_blocks ? -1 : (page * A.Hkv * A.bs + off) * A.row_bytes;
      };
      from = place(base + t);
      to = from < 0 ? -1 : place(base + k);
    }
    src[k] = from;
    dst[k] = to;
  }
  if (A.n_layers == 0) return;
  __syncthreads();
  char* pool = static_cast<char*>((blockIdx.y & 1 ? A.v_pools : A.k_pools)[blockIdx.y >> 1]);
  if ((blockIdx.y & 1) && pool == A.k_pools[blockIdx.y >> 1]) return;       // values that are the keys move once
  const int64_t head_bytes = static_cast<int64_t>(A.bs) * A.row_bytes;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(pool) | static_cast<uintptr_t>(A.row_bytes);
  if ((bits & 15) == 0) move_rows<int4>(pool, src, dst, count, A.Hkv, head_bytes, A.row_bytes);
  else if ((bits & 3) == 0) move_rows<int>(pool, src, dst, count, A.Hkv, head_bytes, A.row_bytes);
  else move_rows<short>(pool, src, dst, count, A.Hkv, head_bytes, A.row_bytes);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200_draft_tree(int64_t* visible, int32_t* depth, const int32_t* parents, int64_t parent_stride, const int32_t* draft_lens, int B,
                    int nodes, void* stream) {
  const char* name = "b200_draft_tree";
  if (B < 0 || nodes <= 0) return fail(B200_EINVAL, "%s: bad sizes", name);
  if (nodes > kMaxNodes) return fail(B200_ESHAPE, "%s: %d nodes, at most %d", name, nodes, kMaxNodes);
  if (B == 0) return 0;
  if (!visible || !depth || !parents) return fail(B200_EINVAL, "%s: null pointer", name);
  draft_tree_kernel<<<B, kMaxNodes, 0, static_cast<cudaStream_t>(stream)>>>(visible, depth, parents, parent_stride, draft_lens, nodes);
  return check_launch(name);
}

int b200_accept_drafts(int32_t* count, int32_t* path, int64_t* new_tokens, int32_t* new_lens, const int64_t* tokens, int64_t token_stride,
                       const int64_t* chosen, int64_t chosen_stride, const int32_t* parents, int64_t parent_stride, const int64_t* visible,
                       int64_t visible_stride, void* const* k_pools, void* const* v_pools, int n_layers, const int32_t* block_tables,
                       int table_stride, int table_cols, const int32_t* context_lens, const int32_t* draft_lens, int B, int nodes, int Hkv, int D,
                       int block_size, int64_t max_blocks, int dtype, void* stream) {
  const char* name = "b200_accept_drafts";
  const int es = dtype_size(dtype);
  if (es == 0) return fail(B200_EINVAL, "%s: unsupported dtype %d", name, dtype);
  if (B < 0 || nodes <= 0 || n_layers < 0) return fail(B200_EINVAL, "%s: bad sizes", name);
  if (n_layers > 0 && (Hkv <= 0 || D <= 0 || block_size <= 0 || max_blocks <= 0 || table_cols <= 0 || table_stride < 0))
    return fail(B200_EINVAL, "%s: bad sizes", name);
  if (nodes > kMaxNodes) return fail(B200_ESHAPE, "%s: %d nodes, at most %d", name, nodes, kMaxNodes);
  if (n_layers > 32767) return fail(B200_ESHAPE, "%s: %d layers", name, n_layers);
  if (n_layers > 0 && static_cast<int64_t>(Hkv) * D * es > INT32_MAX) return fail(B200_ESHAPE, "%s: a token's row", name);
  if (B == 0) return 0;
  if (!count || !path || !new_tokens || !new_lens || !tokens || !chosen || !parents || !visible || !context_lens)
    return fail(B200_EINVAL, "%s: null pointer", name);
  if (n_layers > 0 && (!k_pools || !v_pools || !block_tables)) return fail(B200_EINVAL, "%s: null pointer", name);
  const Accept A{count, path, new_tokens, new_lens, tokens, chosen, visible, parents, token_stride, chosen_stride, parent_stride, visible_stride,
                 k_pools, v_pools, block_tables, table_stride, table_cols, context_lens, draft_lens, nodes, n_layers, Hkv, block_size, D * es, max_blocks};
  accept_drafts_kernel<<<dim3(B, n_layers > 0 ? 2 * n_layers : 1), 128, 0, static_cast<cudaStream_t>(stream)>>>(A);
  return check_launch(name);
}

}  // extern "C"
