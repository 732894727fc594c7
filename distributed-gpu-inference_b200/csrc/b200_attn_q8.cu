// Attention over a key/value cache in 8 bits: one token per sequence, and several.
//
//   out[i, h] = sum_j w_j c_j s_j / sum_j w_j,   w_j = exp(q[i, h] k_j t_j scale - max),   j up to the token's own position
//
// c, s codes and scales of the values, k, t of the keys.
#include <cstdint>
#include <type_traits>

#include "b200_q8.cuh"

namespace b200 {
namespace {

using q8::Cache;
using q8::Rows;

struct Attn {
  Cache c;
  Rows r;
  void* out;
  const void* q;
  int64_t q_stride;
  int Hq;
  float scale;
};

// ---- any type, head size, page size and alignment ------------------------------------------------------------------------------------------
// One CTA per (row, query head); its warps take 32 keys in turns, a lane a key for the scores and a part of the columns for the output, and put their
// maxima, sums and outputs together at the end.  fp32 throughout: what the 32-bit models use, and sizes that the kernels on the tensor cores do not serve.
constexpr int kAnyWarps = 8;

template <typename T, typename C, int COLS>
__global__ void __launch_bounds__(kAnyWarps * 32) attn_any_kernel(const Attn A, bool vec) {
  constexpr int kMostD = 32 * COLS, kAhead = 32 / COLS;
  __shared__ float q_s[kMostD], out_s[kAnyWarps][kMostD], m_s[kAnyWarps], l_s[kAnyWarps];
  __shared__ int b_s;
  const int h = blockIdx.x % A.Hq, row = blockIdx.x / A.Hq, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = A.c.D;
  int b = row, first, count, context;
  if (A.r.starts) {       // the first sequence with the row
    if (threadIdx.x == 0) b_s = A.r.B;
    __syncthreads();
    for (int at = threadIdx.x; at < A.r.B; at += blockDim.x) {
      A.r.of(at, &first, &count, &context);
      if (row >= first && row < first + count) atomicMin(&b_s, at);
    }
    __syncthreads();
    b = b_s;
    if (b >= A.r.B) return;       // nobody's
  }
  A.r.of(b, &first, &count, &context);
  const int keys = row < first + count ? A.c.keys(context - count + (row - first) + 1) : 0;
  T* out = static_cast<T*>(A.out) + (static_cast<int64_t>(row) * A.Hq + h) * D;
  const T* q = static_cast<const T*>(A.q) + row * A.q_stride + static_cast<int64_t>(h) * D;
  for (int d = threadIdx.x; d < kMostD; d += blockDim.x) q_s[d] = d < D ? Cvt<T>::to_f32(q[d]) * A.scale : 0.f;
  __syncthreads();
  const int g = h / (A.Hq / A.c.Hkv);
  float m = -INFINITY, l = 0.f, acc[COLS] = {};
  for (int j0 = warp * 32; j0 < keys; j0 += kAnyWarps * 32) {
    const int j = j0 + lane;
    const bool live = j < keys;
    int64_t at = -1;        // element of the pools; outside them: zeros
    float s = 0.f, v_scale = 0.f;
    if (live) {
      const int page = A.c.page(b, j / A.c.bs);
      if (page >= 0) {
        const int64_t place = static_cast<int64_t>(page) * A.c.Hkv + g;
        at = (place * A.c.bs + j % A.c.bs) * D;
        const uint8_t* k = A.c.k_pool + at;
        if (vec) {
#pragma unroll 4
          for (int d = 0; d < D; d += 16) {
            const int4 raw = *reinterpret_cast<const int4*>(k + d);
            const uint8_t* e = reinterpret_cast<const uint8_t*>(&raw);
#pragma unroll
            for (int u = 0; u < 16; ++u) s = fmaf(q_s[d + u], C::value(e[u]), s);
          }
        } else {
          for (int d = 0; d < D; ++d) s = fmaf(q_s[d], C::value(k[d]), s);
        }
        s *= A.c.k_scale[place];
        v_scale = A.c.v_scale[place];
      }
    }
    const float top = fmaxf(m, warp_max(live ? s : -INFINITY));
    if (top == -INFINITY && !__any_sync(0xffffffffu, live && s != s)) continue;
    const float from = top == -INFINITY ? 0.f : top, corr = m == -INFINITY ? 0.f : expf(m - from), w = live ? expf(s - from) : 0.f, wv = live ? w * v_scale : 0.f;
    m = top;
    l = fmaf(l, corr, warp_sum(w));
#pragma unroll
    for (int c = 0; c < COLS; ++c) acc[c] *= corr;
    for (int i = 0; i < 32; i += kAhead) {
      float wi[kAhead], v[kAhead][COLS];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        wi[u] = __shfl_sync(0xffffffffu, wv, i + u);
        const int64_t vi = __shfl_sync(0xffffffffu, at, i + u);
        const uint8_t* from_v = A.c.v_pool + vi;
#pragma unroll
        for (int c = 0; c < COLS; ++c) v[u][c] = vi >= 0 && c * 32 + lane < D ? C::value(from_v[c * 32 + lane]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[c] = fmaf(wi[u], v[u][c], acc[c]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < COLS; ++c) out_s[warp][c * 32 + lane] = acc[c];
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
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kAnyWarps; ++w) o = fmaf(out_s[w][d], k[w], o);
    out[d] = Cvt<T>::from_f32(sum == 0.f ? 0.f : o / sum);
  }
}

constexpr int kAnyMostD = 256;

template <typename T, typename C>
int launch_any(const char* name, const Attn& A, cudaStream_t stream) {
  if (A.c.D > kAnyMostD) return fail(B200_ESHAPE, "%s: head size %d, at most %d", name, A.c.D, kAnyMostD);
  const int64_t grid = static_cast<int64_t>(A.r.n) * A.Hq;
  if (grid > INT32_MAX) return fail(B200_ESHAPE, "%s: %d rows of %d heads", name, A.r.n, A.Hq);
  auto kern = A.c.D <= 64 ? attn_any_kernel<T, C, 2> : A.c.D <= 128 ? attn_any_kernel<T, C, 4> : attn_any_kernel<T, C, 8>;
  kern<<<static_cast<unsigned>(grid), kAnyWarps * 32, 0, stream>>>(A, A.c.D % 16 == 0 && aligned16(A.c.k_pool));
  return check_launch(name);
}

template <typename T>
int launch_any_of(const char* name, const Attn& A, int codes, cudaStream_t stream) {
  return codes == B200_CODES_INT8 ? launch_any<T, q8::Int8>(name, A, stream) : launch_any<T, q8::E4m3>(name, A, stream);
}
int launch_any_of(const char* name, const Attn& A, int codes, int dtype, cudaStream_t stream) {
  return dtype == B200_DTYPE_F16 ? launch_any_of<__half>(name, A, codes, stream)
         : dtype == B200_DTYPE_BF16 ? launch_any_of<__nv_bfloat16>(name, A, codes, stream) : launch_any_of<float>(name, A, codes, stream);
}

int check_attn(const char* name, const Attn& A, int codes, int dtype) {
  if (dtype_size(dtype) == 0) return fail(B200_EINVAL, "%s: unsupported dtype %d", name, dtype);
  if (int rc = check_cache(name, A.c, codes)) return rc;
  if (A.r.B < 0 || A.r.n < 0 || A.Hq <= 0) return fail(B200_EINVAL, "%s: bad sizes B=%d rows=%d Hq=%d", name, A.r.B, A.r.n, A.Hq);
  if (A.Hq % A.c.Hkv != 0) return fail(B200_ESHAPE, "%s: Hq %d is no multiple of Hkv %d", name, A.Hq, A.c.Hkv);
  if (A.r.B == 0 || A.r.n == 0) return 0;
  if (!A.out || !A.q || !A.c.k_pool || !A.c.v_pool || !A.c.k_scale || !A.c.v_scale || !A.c.tables || !A.r.context_lens) return fail(B200_EINVAL, "%s: null pointer", name);
  return 0;
}

Cache cache_of(const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale, const int32_t* tables, int stride, int cols, int Hkv, int D, int bs,
               int64_t max_blocks) {
  return Cache{static_cast<uint8_t*>(const_cast<void*>(k_pool)), static_cast<uint8_t*>(const_cast<void*>(v_pool)), const_cast<float*>(k_scale), const_cast<float*>(v_scale),
               tables, stride, cols, Hkv, D, bs, max_blocks};
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_paged_decode_attn_q8_workspace(int B, int Hq, int Hkv, int D, int block_size, int max_context_len, int dtype) {
  (void)B, (void)Hq, (void)Hkv, (void)D, (void)block_size, (void)max_context_len, (void)dtype;
  return 0;
}

int b200_paged_decode_attn_q8(void* out, const void* q, int64_t q_stride, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                              const int32_t* block_tables, int table_stride, int table_cols, const int32_t* context_lens, int B, int Hq, int Hkv, int D,
                              int block_size, int64_t max_blocks, float scale, int max_context_len, void* workspace, size_t workspace_bytes, int codes,
                              int dtype, unsigned flags, void* stream) {
  const char* name = "b200_paged_decode_attn_q8";
  const Attn A{cache_of(k_pool, v_pool, k_scale, v_scale, block_tables, table_stride, table_cols, Hkv, D, block_size, max_blocks),
               Rows{nullptr, context_lens, B, B}, out, q, q_stride, Hq, scale};
  if (int rc = check_attn(name, A, codes, dtype)) return rc;
  if (max_context_len < 0) return fail(B200_EINVAL, "%s: negative max_context_len", name);
  if (B == 0) return 0;
  (void)workspace, (void)workspace_bytes, (void)flags;
  return launch_any_of(name, A, codes, dtype, static_cast<cudaStream_t>(stream));
}

size_t b200_paged_prompt_attn_q8_workspace(int B, int max_new, int Hq, int Hkv, int D, int block_size, int max_context_len, int dtype) {
  (void)B, (void)max_new, (void)Hq, (void)Hkv, (void)D, (void)block_size, (void)max_context_len, (void)dtype;
  return 0;
}

int b200_paged_prompt_attn_q8(void* out, const void* q, int64_t q_stride, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                              const int32_t* block_tables, int table_stride, int table_cols, const int32_t* context_lens, const int32_t* row_starts, int B, int rows,
                              int max_new, int Hq, int Hkv, int D, int block_size, int64_t max_blocks, float scale, int max_context_len, void* workspace,
                              size_t workspace_bytes, int codes, int dtype, unsigned flags, void* stream) {
  const char* name = "b200_paged_prompt_attn_q8";
  const Attn A{cache_of(k_pool, v_pool, k_scale, v_scale, block_tables, table_stride, table_cols, Hkv, D, block_size, max_blocks),
               Rows{row_starts, context_lens, B, rows}, out, q, q_stride, Hq, scale};
  if (int rc = check_attn(name, A, codes, dtype)) return rc;
  if (max_context_len < 0 || max_new < 0) return fail(B200_EINVAL, "%s: negative max_context_len or max_new", name);
  if (B == 0 || rows == 0) return 0;
  if (!row_starts) return fail(B200_EINVAL, "%s: null pointer", name);
  (void)workspace, (void)workspace_bytes, (void)flags;
  return launch_any_of(name, A, codes, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
