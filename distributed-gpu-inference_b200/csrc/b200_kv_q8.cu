// Writing a key/value cache in 8 bits, and reading it back.
//
//   s    = max(s_had if the page holds earlier tokens, max |x| / c, 2^-60)        c the largest code, x the page's new keys (or values) of one head
//   code = round(x (1 / s)),   earlier tokens' codes <- round(code (s_had (1 / s)))  where s > s_had
//
// Every product and quotient is rounded to 32 bits by itself: the codes are the same wherever they are computed.
#include <cstdint>
#include <type_traits>

#include "b200_q8.cuh"

namespace b200 {
namespace {

using q8::Cache;
using q8::Rows;

struct Append {
  Cache c;
  Rows r;
  const void *q, *k, *v, *cos_t, *sin_t;      // cos_t NULL: nothing turns
  void* q_out;                                // NULL: keys and values alone
  int64_t q_stride, k_stride, v_stride, out_stride;
  int Hq, pages;                              // pages that a sequence's new tokens touch at most
};

// x[d] and its partner half a head away, turned: x c - y s in the lower half, x c + y s in the upper, each operation rounded
__device__ __forceinline__ float turned(float x, float partner, float c, float s, bool upper) {
  return __fadd_rn(__fmul_rn(x, c), __fmul_rn(upper ? partner : -partner, s));
}

// ---- any type, head size, page size and alignment ------------------------------------------------------------------------------------------
// One CTA per (page that new tokens fall into, kv head, keys or values), behind these one per row of queries.
template <typename T, typename C>
__global__ void __launch_bounds__(128) append_any_kernel(const Append A) {
  __shared__ float most_s[4];
  const int D = A.c.D, bs = A.c.bs, half = D / 2;
  const int64_t units = static_cast<int64_t>(A.r.B) * A.pages * A.c.Hkv * 2;
  auto element = [&](const T* row, int64_t at, int d) -> float {        // of row `at` of the tables
    const float x = Cvt<T>::to_f32(row[d]);
    if (!A.cos_t) return x;
    const bool upper = d >= half;
    return turned(x, Cvt<T>::to_f32(row[upper ? d - half : d + half]), Cvt<T>::to_f32(static_cast<const T*>(A.cos_t)[at * D + d]),
                  Cvt<T>::to_f32(static_cast<const T*>(A.sin_t)[at * D + d]), upper);
  };
  if (blockIdx.x >= units) {
    const int64_t row = blockIdx.x - units;
    const T* q = static_cast<const T*>(A.q) + row * A.q_stride;
    T* out = static_cast<T*>(A.q_out) + row * A.out_stride;
    for (int h = threadIdx.x >> 5; h < A.Hq; h += 4) {        // a warp's head: all of it is read before any of it is written
      for (int d0 = 0; d0 < half; d0 += 32) {
        const int d = d0 + (threadIdx.x & 31);
        float lo = 0.f, hi = 0.f;
        if (d < half) lo = element(q + h * D, row, d), hi = element(q + h * D, row, d + half);
        __syncwarp();
        if (d < half) out[h * D + d] = Cvt<T>::from_f32(lo), out[h * D + d + half] = Cvt<T>::from_f32(hi);
      }
    }
    return;
  }
  const bool values = blockIdx.x & 1;
  const int unit = blockIdx.x >> 1, h = unit % A.c.Hkv, lp = unit / A.c.Hkv % A.pages, b = unit / A.c.Hkv / A.pages;
  int first, count, context;
  A.r.of(b, &first, &count, &context);
  const int held = context - count, at = held / bs + lp;
  const int t0 = max(held, at * bs), t1 = static_cast<int>(min(static_cast<int64_t>(context), static_cast<int64_t>(at + 1) * bs));       // positions
  if (t0 >= t1) return;
  const int page = A.c.page(b, at);
  if (page < 0) return;
  const T* rows = static_cast<const T*>(values ? A.v : A.k) + h * D;
  const int64_t stride = values ? A.v_stride : A.k_stride;
  const int64_t place = static_cast<int64_t>(page) * A.c.Hkv + h;
  uint8_t* codes = (values ? A.c.v_pool : A.c.k_pool) + place * bs * D;
  float* scale = (values ? A.c.v_scale : A.c.k_scale) + place;
  auto number = [&](int i) -> float {        // of the new tokens' elements
    const int t = i / D, d = i - t * D;
    const int64_t row = first + (t0 - held) + t;
    return values ? Cvt<T>::to_f32(rows[row * stride + d]) : element(rows + row * stride, row, d);
  };
  float most = 0.f;
  for (int i = threadIdx.x; i < (t1 - t0) * D; i += blockDim.x) most = q8::max_nan(most, fabsf(number(i)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = q8::max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) most_s[threadIdx.x >> 5] = most;
  const float had = t0 > at * bs ? *scale : 0.f;
  __syncthreads();
  most = q8::max_nan(q8::max_nan(most_s[0], most_s[1]), q8::max_nan(most_s[2], most_s[3]));
  const float now = q8::max_nan(q8::max_nan(had, __fmul_rn(most, 1.f / C::kMost)), q8::kLeastScale), inverse = 1.f / now;
  if (now != had) {
    const float k = __fmul_rn(had, inverse);
    for (int i = threadIdx.x; i < (t0 - at * bs) * D; i += blockDim.x) codes[i] = C::code(__fmul_rn(C::value(codes[i]), k));
    if (threadIdx.x == 0) *scale = now;
  }
  for (int i = threadIdx.x; i < (t1 - t0) * D; i += blockDim.x) codes[(t0 - at * bs) * D + i] = C::code(__fmul_rn(number(i), inverse));
}

// ---- reading back --------------------------------------------------------------------------------------------------------------------------
struct Gather {
  Cache c;
  void *k_out, *v_out;      // [B, Hkv, n, D]
  int B, n;
};

template <typename T, typename C>
__global__ void __launch_bounds__(256) gather_any_kernel(const Gather G) {
  const int D = G.c.D;
  const int64_t all = static_cast<int64_t>(G.B) * G.c.Hkv * G.n * D;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
    const int d = static_cast<int>(i % D), t = static_cast<int>(i / D % G.n), h = static_cast<int>(i / D / G.n % G.c.Hkv), b = static_cast<int>(i / D / G.n / G.c.Hkv);
    const int page = G.c.page(b, t / G.c.bs);
    float k = 0.f, v = 0.f;
    if (page >= 0) {
      const int64_t place = static_cast<int64_t>(page) * G.c.Hkv + h, e = (place * G.c.bs + t % G.c.bs) * D + d;
      k = C::value(G.c.k_pool[e]) * G.c.k_scale[place];
      v = C::value(G.c.v_pool[e]) * G.c.v_scale[place];
    }
    static_cast<T*>(G.k_out)[i] = Cvt<T>::from_f32(k);
    static_cast<T*>(G.v_out)[i] = Cvt<T>::from_f32(v);
  }
}

// calls f(T*, C*) for the types of these ids
template <typename F>
int with_types(int dtype, int codes, F f) {
  auto go = [&](auto* t) {
    return codes == B200_CODES_INT8 ? f(t, static_cast<q8::Int8*>(nullptr)) : f(t, static_cast<q8::E4m3*>(nullptr));
  };
  return dtype == B200_DTYPE_F16 ? go(static_cast<__half*>(nullptr)) : dtype == B200_DTYPE_BF16 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<float*>(nullptr));
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200_rope_kv_append_q8(void* q_out, int64_t q_out_stride, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                           const void* cos_table, const void* sin_table, void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                           const int32_t* block_tables, int table_stride, int table_cols, const int32_t* context_lens, const int32_t* row_starts, int B,
                           int rows, int max_new, int Hq, int Hkv, int D, int block_size, int64_t max_blocks, int codes, int dtype, void* stream) {
  const char* name = "b200_rope_kv_append_q8";
  if (dtype_size(dtype) == 0) return fail(B200_EINVAL, "%s: unsupported dtype %d", name, dtype);
  Append A{};
  A.c = Cache{static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), k_scale, v_scale, block_tables, table_stride, table_cols, Hkv, D, block_size, max_blocks};
  if (int rc = check_cache(name, A.c, codes)) return rc;
  if (B < 0 || rows < 0 || max_new < 0 || (q_out && Hq <= 0)) return fail(B200_EINVAL, "%s: bad sizes B=%d rows=%d max_new=%d Hq=%d", name, B, rows, max_new, Hq);
  if ((cos_table == nullptr) != (sin_table == nullptr) || (q_out && !cos_table)) return fail(B200_EINVAL, "%s: cos and sin come together, and with queries", name);
  if (cos_table && D % 2) return fail(B200_ESHAPE, "%s: head size %d cannot turn", name, D);
  if (B == 0 || rows == 0) return 0;
  if (!k || !v || !k_pool || !v_pool || !k_scale || !v_scale || !block_tables || !context_lens || (q_out && !q)) return fail(B200_EINVAL, "%s: null pointer", name);
  if (!row_starts && rows != B) return fail(B200_EINVAL, "%s: %d rows of %d sequences need row_starts", name, rows, B);
  A.r = Rows{row_starts, context_lens, B, rows};
  A.q = q, A.k = k, A.v = v, A.cos_t = cos_table, A.sin_t = sin_table, A.q_out = q_out;
  A.q_stride = q_stride, A.k_stride = k_stride, A.v_stride = v_stride, A.out_stride = q_out_stride, A.Hq = Hq;
  const int longest = row_starts ? (max_new < rows ? max_new : rows) : 1;
  A.pages = longest == 0 ? 0 : longest == 1 ? 1 : static_cast<int>((longest - 2ll + block_size) / block_size) + 1;
  const int64_t units = static_cast<int64_t>(B) * A.pages * Hkv * 2, grid = units + (q_out ? rows : 0);
  if (grid > INT32_MAX) return fail(B200_ESHAPE, "%s: %d sequences of up to %d pages", name, B, A.pages);
  if (grid == 0) return 0;
  return with_types(dtype, codes, [&](auto* t, auto* c) {
    append_any_kernel<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(c)>><<<static_cast<unsigned>(grid), 128, 0, static_cast<cudaStream_t>(stream)>>>(A);
    return check_launch(name);
  });
}

int b200_kv_gather_dense_q8(void* k_out, void* v_out, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                            const int32_t* block_tables, int table_stride, int table_cols, int B, int n_tokens, int Hkv, int D, int block_size,
                            int64_t max_blocks, int codes, int dtype, void* stream) {
  const char* name = "b200_kv_gather_dense_q8";
  if (dtype_size(dtype) == 0) return fail(B200_EINVAL, "%s: unsupported dtype %d", name, dtype);
  Gather G{};
  G.c = Cache{static_cast<uint8_t*>(const_cast<void*>(k_pool)), static_cast<uint8_t*>(const_cast<void*>(v_pool)), const_cast<float*>(k_scale), const_cast<float*>(v_scale),
              block_tables, table_stride, table_cols, Hkv, D, block_size, max_blocks};
  if (int rc = check_cache(name, G.c, codes)) return rc;
  if (B < 0 || n_tokens < 0) return fail(B200_EINVAL, "%s: bad sizes B=%d n_tokens=%d", name, B, n_tokens);
  if (n_tokens > static_cast<int64_t>(table_cols) * block_size) return fail(B200_EINVAL, "%s: %d tokens do not fit rows of %d blocks", name, n_tokens, table_cols);
  if (B == 0 || n_tokens == 0) return 0;
  if (!k_out || !v_out || !k_pool || !v_pool || !k_scale || !v_scale || !block_tables) return fail(B200_EINVAL, "%s: null pointer", name);
  G.k_out = k_out, G.v_out = v_out, G.B = B, G.n = n_tokens;
  const int64_t blocks = (static_cast<int64_t>(B) * Hkv * n_tokens * D + 255) / 256;
  return with_types(dtype, codes, [&](auto* t, auto* c) {
    gather_any_kernel<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(c)>>
        <<<static_cast<unsigned>(blocks < kNumSMs * 8 ? blocks : kNumSMs * 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(G);
    return check_launch(name);
  });
}

}  // extern "C"
