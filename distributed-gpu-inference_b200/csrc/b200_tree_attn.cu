// Attention of a tree of drafted tokens over the paged cache: each node sees the context and the nodes of its mask.
//
//   out[t, h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(q[t, h] k_j scale - max),   j in the context, or bit j of visible[t]
#include <algorithm>

#include "b200_common.cuh"

namespace b200 {
namespace {

struct TreeAttn {
  void* out;
  const void *q, *k_pool, *v_pool;
  int64_t q_batch_stride, q_node_stride;
  const int32_t* block_tables;
  int table_stride, table_cols;
  const int32_t *context_lens, *draft_lens;
  const int64_t* visible;
  int64_t visible_stride;
  int B, nodes, Hq, Hkv, D, bs;
  int64_t max_blocks;
  float scale;
};

// a sequence's keys that a call may read, and its nodes
__device__ __forceinline__ void lengths(const TreeAttn& A, int b, int* keys, int* nodes) {
  const int64_t room = static_cast<int64_t>(A.table_cols) * A.bs;
  *keys = static_cast<int>(min(static_cast<int64_t>(max(A.context_lens[b], 0)), room));
  *nodes = min(A.draft_lens ? min(max(A.draft_lens[b], 0), A.nodes) : A.nodes, *keys);
}

// ---- any type, head size and page size ------------------------------------------------------------------------------------------------------
// One CTA per (sequence, node, query head); its warps take 32 keys in turns, a lane a key for the scores and a part of the columns for the
// output, and put their maxima, sums and outputs together at the end.  Bound by the loads' latency; serves what the kernel below does not
// (fp32, head sizes other than 64 and 128, pages that do not divide 64 keys).
constexpr int kAnyWarps = 4, kAnyMostD = 256;

template <typename T>
__global__ void __launch_bounds__(kAnyWarps * 32) tree_attn_any_kernel(const TreeAttn A, bool vec) {
  constexpr int kVec = 16 / sizeof(T), kCols = kAnyMostD / 32;
  __shared__ __align__(16) float q_s[kAnyMostD];
  __shared__ float out_s[kAnyWarps][kAnyMostD], m_s[kAnyWarps], l_s[kAnyWarps];
  const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int keys, n;
  lengths(A, b, &keys, &n);
  T* out = static_cast<T*>(A.out) + ((static_cast<int64_t>(b) * A.nodes + t) * A.Hq + h) * A.D;
  if (t >= n) {
    for (int d = threadIdx.x; d < A.D; d += blockDim.x) out[d] = Cvt<T>::from_f32(0.f);
    return;
  }
  const T* q = static_cast<const T*>(A.q) + b * A.q_batch_stride + t * A.q_node_stride + static_cast<int64_t>(h) * A.D;
  for (int d = threadIdx.x; d < kAnyMostD; d += blockDim.x) q_s[d] = d < A.D ? Cvt<T>::to_f32(q[d]) * A.scale : 0.f;
  __syncthreads();
  const int base = keys - n, g = h / (A.Hq / A.Hkv);
  const uint64_t seen = static_cast<uint64_t>(A.visible[b * A.visible_stride + t]);
  float m = -INFINITY, l = 0.f, acc[kCols] = {};
  for (int j0 = warp * 32; j0 < keys; j0 += kAnyWarps * 32) {
    const int j = j0 + lane;
    const bool live = j < keys && (j < base || (seen >> (j - base) & 1));
    int64_t at = -1;        // element of the pools; outside them: zeros
    float s = 0.f;
    if (live) {
      const int64_t page = A.block_tables[static_cast<int64_t>(b) * A.table_stride + j / A.bs];
      if (page >= 0 && page < A.max_blocks) at = ((page * A.Hkv + g) * A.bs + j % A.bs) * A.D;
    }
    if (at >= 0) {
      const T* k = static_cast<const T*>(A.k_pool) + at;
      if (vec) {
        for (int d = 0; d < A.D; d += kVec) {
          const int4 raw = *reinterpret_cast<const int4*>(k + d);
          const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
          for (int u = 0; u < kVec; ++u) s = fmaf(q_s[d + u], Cvt<T>::to_f32(e[u]), s);
        }
      } else {
        for (int d = 0; d < A.D; ++d) s = fmaf(q_s[d], Cvt<T>::to_f32(k[d]), s);
      }
    }
    const float top = fmaxf(m, warp_max(live ? s : -INFINITY));
    if (top == -INFINITY && !__any_sync(0xffffffffu, live && s != s)) continue;
    const float corr = m == -INFINITY ? 0.f : expf(m - top), w = live ? expf(s - top) : 0.f;
    m = top;
    l = fmaf(l, corr, warp_sum(w));
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[c] *= corr;
    for (int i = 0; i < 32; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const int64_t vi = __shfl_sync(0xffffffffu, at, i);
      if (wi == 0.f || vi < 0) continue;
      const T* v = static_cast<const T*>(A.v_pool) + vi;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        if (c * 32 + lane < A.D) acc[c] = fmaf(wi, Cvt<T>::to_f32(v[c * 32 + lane]), acc[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < kCols; ++c) out_s[warp][c * 32 + lane] = acc[c];
  if (lane == 0) m_s[warp] = m, l_s[warp] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.f, k[kAnyWarps];
#pragma unroll
  for (int w = 0; w < kAnyWarps; ++w) top = fmaxf(top, m_s[w]);
#pragma unroll
  for (int w = 0; w < kAnyWarps; ++w) {
    k[w] = m_s[w] == -INFINITY ? (l_s[w] != l_s[w] ? 1.f : 0.f) : expf(m_s[w] - top);
    sum = fmaf(l_s[w], k[w], sum);
  }
  for (int d = threadIdx.x; d < A.D; d += blockDim.x) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kAnyWarps; ++w) o = fmaf(out_s[w][d], k[w], o);
    out[d] = Cvt<T>::from_f32(sum == 0.f ? 0.f : o / sum);
  }
}

template <typename T>
int launch_any(const TreeAttn& A, cudaStream_t stream) {
  if (A.D > kAnyMostD) return fail(B200_ESHAPE, "b200_paged_tree_attn: head size %d, at most %d", A.D, kAnyMostD);
  if (A.B > 65535) return fail(B200_ESHAPE, "b200_paged_tree_attn: %d sequences", A.B);
  const bool vec = A.D * sizeof(T) % 16 == 0 && aligned16(A.k_pool);
  tree_attn_any_kernel<T><<<dim3(A.Hq, A.nodes, A.B), kAnyWarps * 32, 0, stream>>>(A, vec);
  return check_launch("b200_paged_tree_attn");
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_paged_tree_attn_workspace(int B, int nodes, int Hq, int Hkv, int D, int block_size, int dtype) { return 0; }

int b200_paged_tree_attn(void* out, const void* q, int64_t q_batch_stride, int64_t q_node_stride, const void* k_pool, const void* v_pool,
                         const int32_t* block_tables, int table_stride, int table_cols, const int32_t* context_lens, const int32_t* draft_lens,
                         const int64_t* visible, int64_t visible_stride, int B, int nodes, int Hq, int Hkv, int D, int block_size,
                         int64_t max_blocks, float scale, void* workspace, size_t workspace_bytes, int dtype, unsigned flags, void* stream) {
  const char* name = "b200_paged_tree_attn";
  const int es = dtype_size(dtype);
  if (es == 0) return fail(B200_EINVAL, "%s: unsupported dtype %d", name, dtype);
  if (B < 0 || nodes <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || block_size <= 0 || max_blocks <= 0 || table_cols <= 0 || table_stride < 0)
    return fail(B200_EINVAL, "%s: bad sizes", name);
  if (nodes > B200_MAX_DRAFT_NODES) return fail(B200_ESHAPE, "%s: %d nodes, at most %d", name, nodes, B200_MAX_DRAFT_NODES);
  if (Hq % Hkv != 0) return fail(B200_ESHAPE, "%s: Hq %d is no multiple of Hkv %d", name, Hq, Hkv);
  if (B == 0) return 0;
  if (!out || !q || !k_pool || !v_pool || !block_tables || !context_lens || !visible) return fail(B200_EINVAL, "%s: null pointer", name);
  const TreeAttn A{out, q, k_pool, v_pool, q_batch_stride, q_node_stride, block_tables, table_stride, table_cols, context_lens, draft_lens, visible,
                   visible_stride, B, nodes, Hq, Hkv, D, block_size, max_blocks, scale};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200_DTYPE_F16: return launch_any<__half>(A, s);
    case B200_DTYPE_BF16: return launch_any<__nv_bfloat16>(A, s);
    default: return launch_any<float>(A, s);
  }
}

}  // extern "C"
