// Writing a key/value cache in 8 bits, and reading it back.
//
//   s    = max(s_had if the page holds earlier tokens, max |x| / c, 2^-60)        c the largest code, x the page's new keys (or values) of one head
//   code = round(x (1 / s)),   earlier tokens' codes <- round(code (s_had (1 / s)))  where s > s_had
//
// Every product and quotient is rounded to 32 bits by itself: the codes are the same wherever they are computed.
#include <cstdint>
#include <type_traits>

#include "b200_q8.cuh"
#include "b200_tcgen05.cuh"

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
  const int64_t base = static_cast<int64_t>(at) * bs;      // the page's first position
  const int t0 = static_cast<int>(max(held - base, static_cast<int64_t>(0))), t1 = static_cast<int>(min(context - base, static_cast<int64_t>(bs)));     // places of the page
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
    const int64_t row = first + (base + t0 - held) + t;
    return values ? Cvt<T>::to_f32(rows[row * stride + d]) : element(rows + row * stride, row, d);
  };
  float most = 0.f;
  for (int i = threadIdx.x; i < (t1 - t0) * D; i += blockDim.x) most = q8::max_nan(most, fabsf(number(i)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = q8::max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) most_s[threadIdx.x >> 5] = most;
  const float had = t0 > 0 ? *scale : 0.f;
  __syncthreads();
  most = q8::max_nan(q8::max_nan(most_s[0], most_s[1]), q8::max_nan(most_s[2], most_s[3]));
  const float now = q8::max_nan(q8::max_nan(had, __fmul_rn(most, 1.f / C::kMost)), q8::kLeastScale), inverse = 1.f / now;
  if (now != had) {
    const float k = __fmul_rn(had, inverse);
    for (int i = threadIdx.x; i < t0 * D; i += blockDim.x) codes[i] = C::code(__fmul_rn(C::value(codes[i]), k));
    if (threadIdx.x == 0) *scale = now;
  }
  for (int i = threadIdx.x; i < (t1 - t0) * D; i += blockDim.x) codes[t0 * D + i] = C::code(__fmul_rn(number(i), inverse));
}

// ---- 16-bit types, heads of 64 or 128, pages of 16, 32 or 64 -----------------------------------------------------------------------------------
// A warp per P places of a page and kv head's keys or values, 16 of 128 columns, 16 or 32 of 64; the W warps of a page share its maximum.  A lane has 8 columns of the lower and the
// same 8 of the upper half of several rows, which turn into one another: everything is read once and held as it came until the scale is known; turning it a second
// time costs less than the registers of the numbers (136: 12 warps an SM, 8 x 2048 rows of 8 heads of 128 in 98 us with their 32 query heads).  Codes that the page holds
// already are asked for together with its scale, whether or not it grows.  Among or behind these CTAs, those of a warp per row and 16
// query heads.  Bound by memory and its latency: 8 x 2048 rows of 32 query and 8 kv heads of 128 in 62 us, 0.94 of a copy's rate (keys and values alone 22, 0.71: five CTAs an SM,
// a page's rows wait for its largest); 16 x 800 of 16 and 16 of 64 in 33, 0.64 (37 with 16 places a warp); a token for each of 64 sequences 3.7.
constexpr int kHeadsPerWarp = 16, kAppendCTAs = 5;

// Eight numbers as four pairs, two products an instruction.  (Sums stay single: the assembler made one rounding of a pair's product and its sum with a constant,
// whatever their instructions said.)
using Eight = f32x2[4];
template <typename T>
__device__ __forceinline__ void eight(const int4& raw, Eight& x) {
  const uint32_t w[4] = {static_cast<uint32_t>(raw.x), static_cast<uint32_t>(raw.y), static_cast<uint32_t>(raw.z), static_cast<uint32_t>(raw.w)};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      x[u] = pair(__uint_as_float(w[u] << 16), __uint_as_float(w[u] & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[u]));
      x[u] = pair(f.x, f.y);
    }
  }
}
template <typename T>
__device__ __forceinline__ int4 eight_of(const Eight& x) {
  uint32_t w[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    float a, b;
    apart(a, b, x[u]);
    w[u] = pack2<T>(a, b);
  }
  return make_int4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ f32x2 sums(f32x2 x, f32x2 y) {
  float a, b, c, d;
  apart(a, b, x);
  apart(c, d, y);
  return pair(__fadd_rn(a, c), __fadd_rn(b, d));
}
__device__ __forceinline__ f32x2 differences(f32x2 x, f32x2 y) {
  float a, b, c, d;
  apart(a, b, x);
  apart(c, d, y);
  return pair(__fsub_rn(a, c), __fsub_rn(b, d));
}
// lo, hi: the same 8 columns of the two halves
template <typename T>
__device__ __forceinline__ void turn(Eight& lo, Eight& hi, const int4 (&cs)[4]) {
  Eight cl, ch, sl, sh;
  eight<T>(cs[0], cl);
  eight<T>(cs[1], ch);
  eight<T>(cs[2], sl);
  eight<T>(cs[3], sh);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const f32x2 l = differences(mul2(lo[u], cl[u]), mul2(hi[u], sl[u])), h = sums(mul2(hi[u], ch[u]), mul2(lo[u], sh[u]));
    lo[u] = l, hi[u] = h;
  }
}
// the larger of `most` and two pairs' magnitudes, no number if one is none
__device__ __forceinline__ float magnitude(float most, f32x2 x) {
  float a, b;
  apart(a, b, x);
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(most) : "f"(most), "f"(a), "f"(b));
  return most;
}
// of 16 bits, in their type: a comparison rounds nothing
template <typename T>
__device__ __forceinline__ uint32_t magnitudes(uint32_t most, uint32_t two) {
  two &= 0x7fff7fffu;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(most) : "r"(two));
  else asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(most) : "r"(two));
  return most;
}
template <typename C>
__device__ __forceinline__ uint2 codes_of(const Eight& x, float inverse) {
  uint32_t w[2];
  const f32x2 by = both(inverse);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float a, b, c, d;
    if constexpr (std::is_same_v<C, q8::Int8>) {
      // |x / s| <= 127 (1 + 2^-22): the sum's last 8 bits are the nearest whole number's
      apart(a, b, sums(mul2(x[2 * i], by), both(12582912.f)));
      apart(c, d, sums(mul2(x[2 * i + 1], by), both(12582912.f)));
      w[i] = __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
    } else {
      apart(a, b, mul2(x[2 * i], by));
      apart(c, d, mul2(x[2 * i + 1], by));
      w[i] = static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)) |
             static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16;
    }
  }
  return make_uint2(w[0], w[1]);
}
template <typename C>
__device__ __forceinline__ uint2 codes_again(uint2 old, float k) {
  uint8_t* c = reinterpret_cast<uint8_t*>(&old);
#pragma unroll
  for (int u = 0; u < 8; ++u) c[u] = C::code(__fmul_rn(C::value(c[u]), k));
  return old;
}

// q_step: CTAs of queries lie evenly among the others (CTA i is one where i q_step / 2^64 passes a whole number); 0: behind the kv_ctas others
template <typename T, typename C, int D, int P, int W>
__global__ void __launch_bounds__(128, kAppendCTAs) append_kernel(const Append A, unsigned kv_ctas, unsigned long long q_step) {
  constexpr int kCh = D / 16, kRows = 32 / kCh, kPasses = P / kRows;        // pieces of a half; rows of a warp's pass
  __shared__ float most_s[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane % kCh, r = lane / kCh;
  q8::wait_for_ahead();
  const unsigned q_cta = q_step ? static_cast<unsigned>(__umul64hi(blockIdx.x, q_step)) : max(blockIdx.x, kv_ctas) - kv_ctas;        // those before this one
  if (q_step ? __umul64hi(blockIdx.x + 1ull, q_step) != q_cta : blockIdx.x >= kv_ctas) {
    const unsigned groups = (A.Hq + kHeadsPerWarp - 1) / kHeadsPerWarp;
    const unsigned unit = q_cta * 4 + warp, at = unit / groups;        // (a division of 64 bits costs 500 clocks)
    if (at >= static_cast<unsigned>(A.r.n)) return;
    const int64_t row = at;
    const int h0 = static_cast<int>(unit - at * groups) * kHeadsPerWarp + r;
    const T *q = static_cast<const T*>(A.q) + row * A.q_stride + 8 * c, *cs = static_cast<const T*>(A.cos_t) + row * D + 8 * c, *sn = static_cast<const T*>(A.sin_t) + row * D + 8 * c;
    T* out = static_cast<T*>(A.q_out) + row * A.out_stride + 8 * c;
    const int4 angles[4] = {*reinterpret_cast<const int4*>(cs), *reinterpret_cast<const int4*>(cs + D / 2), *reinterpret_cast<const int4*>(sn), *reinterpret_cast<const int4*>(sn + D / 2)};
    constexpr int kSteps = kHeadsPerWarp / kRows;
    int4 raw[kSteps][2];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int h = h0 + i * kRows;
      if (h < A.Hq) {
        raw[i][0] = *reinterpret_cast<const int4*>(q + h * D);
        raw[i][1] = *reinterpret_cast<const int4*>(q + h * D + D / 2);
      }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int h = h0 + i * kRows;
      if (h >= A.Hq) continue;
      Eight lo, hi;
      eight<T>(raw[i][0], lo);
      eight<T>(raw[i][1], hi);
      turn<T>(lo, hi, angles);
      *reinterpret_cast<int4*>(out + h * D) = eight_of<T>(lo);
      *reinterpret_cast<int4*>(out + h * D + D / 2) = eight_of<T>(hi);
    }
    return;
  }
  // ---- keys and values: unit = ((sequence, page), head, keys or values) -----------------------------------------------------------------------
  const unsigned unit = (blockIdx.x - q_cta) * (4 / W) + warp / W, two = unit >> 1, bp = two / A.c.Hkv;
  const bool values = unit & 1;
  const int h = static_cast<int>(two - bp * A.c.Hkv), b = static_cast<int>(bp / A.pages), lp = static_cast<int>(bp - b * A.pages);
  int t0 = 0, t1 = 0, at = 0, first = 0, held = 0;
  if (b < A.r.B) {
    int count, context;
    A.r.of(b, &first, &count, &context);
    held = context - count, at = held / A.c.bs + lp;
    const int64_t base = static_cast<int64_t>(at) * A.c.bs;
    t0 = static_cast<int>(max(held - base, static_cast<int64_t>(0))), t1 = static_cast<int>(min(context - base, static_cast<int64_t>(A.c.bs)));      // places of the page
  }
  if (W == 1 && t0 >= t1) return;
  const int my = warp % W * P + r;       // the place of the lane's row in the first pass
  int4 raw[kPasses][2];       // 8 columns of each half; of earlier tokens their codes, both halves' in the first
  const int64_t stride = values ? A.v_stride : A.k_stride, row = static_cast<int64_t>(first) + static_cast<int64_t>(at) * A.c.bs - held + my;       // of the first pass
  const T* rows = static_cast<const T*>(values ? A.v : A.k) + row * stride + h * D + 8 * c;
  const bool turns = !values && A.cos_t;
  // asked for before the page is known
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int t = my + i * kRows;
    raw[i][0] = raw[i][1] = make_int4(0, 0, 0, 0);
    if (t >= t0 && t < t1) {
      raw[i][0] = q8::ld_once16(rows);
      raw[i][1] = q8::ld_once16(rows + D / 2);
    }
    rows += kRows * stride;
  }
  int4 cs[2][4];       // of a pass, and of the next one
  const T *cos_at = static_cast<const T*>(A.cos_t) + row * D + 8 * c, *sin_at = static_cast<const T*>(A.sin_t) + row * D + 8 * c;
  auto angles = [&](int i) {
    const int t = my + i * kRows;
    if (!(turns && t >= t0 && t < t1)) return;
#pragma unroll
    for (int u = 0; u < 4; ++u) cs[i & 1][u] = *reinterpret_cast<const int4*>((u < 2 ? cos_at : sin_at) + i * kRows * D + u % 2 * (D / 2));
  };
  auto numbers = [&](int i, Eight& lo, Eight& hi) {
    eight<T>(raw[i][0], lo);
    eight<T>(raw[i][1], hi);
    if (turns) turn<T>(lo, hi, cs[i & 1]);
  };
  angles(0);
  const int page = t0 < t1 ? A.c.page(b, at) : -1;
  if (W == 1 && page < 0) return;
  const int64_t place = static_cast<int64_t>(max(page, 0)) * A.c.Hkv + h;
  uint8_t* codes = (values ? A.c.v_pool : A.c.k_pool) + place * A.c.bs * D;
  float* scale = (values ? A.c.v_scale : A.c.k_scale) + place;
  const bool earlier = page >= 0 && t0 > 0;
  float had = earlier ? *scale : 0.f;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int t = my + i * kRows;
    if (earlier && t < t0) {
      const uint2 lo = *reinterpret_cast<const uint2*>(codes + t * D + 8 * c), hi = *reinterpret_cast<const uint2*>(codes + t * D + D / 2 + 8 * c);
      raw[i][0] = make_int4(lo.x, lo.y, hi.x, hi.y);
    }
  }
  float most = 0.f;
  if (turns) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      angles(i + 1 < kPasses ? i + 1 : 0);       // (behind the last the first again: for the codes)
      const int t = my + i * kRows;
      if (!(t >= t0 && t < t1)) continue;
      Eight lo, hi;
      numbers(i, lo, hi);
#pragma unroll
      for (int u = 0; u < 4; ++u) most = magnitude(magnitude(most, lo[u]), hi[u]);
    }
  } else {
    uint32_t two = 0;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int t = my + i * kRows;
      if (!(t >= t0 && t < t1)) continue;
#pragma unroll
      for (int u = 0; u < 2; ++u) two = magnitudes<T>(magnitudes<T>(magnitudes<T>(magnitudes<T>(two, raw[i][u].x), raw[i][u].y), raw[i][u].z), raw[i][u].w);
    }
    const T* e = reinterpret_cast<const T*>(&two);
    most = q8::max_nan(Cvt<T>::to_f32(e[0]), Cvt<T>::to_f32(e[1]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = q8::max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  if constexpr (W > 1) {
    if (lane == 0) most_s[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) most = q8::max_nan(most, most_s[warp / W * W + w]);
    if (page < 0) return;
  }
  const float now = q8::max_nan(q8::max_nan(had, __fmul_rn(most, 1.f / C::kMost)), q8::kLeastScale), inverse = __frcp_rn(now);
  const bool grew = now != had;
  if (grew && warp % W == 0 && lane == 0) *scale = now;       // (the other warps have read what it was: before the barrier)
  const float k = __fmul_rn(had, inverse);
  const bool finite = now < INFINITY;       // else codes are 0
  codes += my * D + 8 * c;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    if (i + 1 < kPasses) angles(i + 1);
    const int t = my + i * kRows;
    uint2* to = reinterpret_cast<uint2*>(codes + i * kRows * D);
    if (t >= t0 && t < t1) {
      Eight lo, hi;
      numbers(i, lo, hi);
      to[0] = finite ? codes_of<C>(lo, inverse) : make_uint2(0u, 0u);
      to[D / 16] = finite ? codes_of<C>(hi, inverse) : make_uint2(0u, 0u);
    } else if (earlier && t < t0 && grew) {
      to[0] = codes_again<C>(make_uint2(raw[i][0].x, raw[i][0].y), k);
      to[D / 16] = codes_again<C>(make_uint2(raw[i][0].z, raw[i][0].w), k);
    }
  }
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

// 16 rows of a page and kv head's keys and values per warp; pages of 16s, rows of D = 64 or 128 codes, 8 of them a lane and step, all asked for before the first is
// turned.  Bound by memory: 8 x 4096 tokens of 8 heads of 128 in 34 us, 0.91 of a copy's rate, 8 x 2048 in 16.3, 0.96.
template <typename C>
__device__ __forceinline__ void values_of(uint2 codes, float s, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w = i ? codes.y : codes.x;
    if constexpr (std::is_same_v<C, q8::Int8>) {
      const uint32_t u = w ^ 0x80808080u;       // code + 128, as the last byte of 2^23 + code + 128
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + e)) - 8388736.f) * s;
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * e)), __NV_E4M3)));
        x[4 * i + 2 * e] = f.x * s, x[4 * i + 2 * e + 1] = f.y * s;
      }
    }
  }
}

template <typename T, typename C, int D>
__global__ void __launch_bounds__(256) gather_kernel(const Gather G, unsigned tiles, unsigned units) {
  constexpr int kSteps = 16 * D / 256;
  const int lane = threadIdx.x & 31;
  const unsigned unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  q8::wait_for_ahead();
  if (unit >= units) return;
  const unsigned bh = unit / tiles;
  const int tile = static_cast<int>(unit - bh * tiles), b = static_cast<int>(bh / G.c.Hkv), h = static_cast<int>(bh - b * G.c.Hkv), at = tile * 16 / G.c.bs;
  const int page = G.c.page(b, at);
  const int64_t place = static_cast<int64_t>(max(page, 0)) * G.c.Hkv + h, from = (place * G.c.bs + (tile * 16 - at * G.c.bs)) * D + lane * 8;
  const float ks = page >= 0 ? G.c.k_scale[place] : 0.f, vs = page >= 0 ? G.c.v_scale[place] : 0.f;
  uint2 k[kSteps], v[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) k[i] = page >= 0 ? q8::ld_once8(G.c.k_pool + from + i * 256) : make_uint2(0u, 0u);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) v[i] = page >= 0 ? q8::ld_once8(G.c.v_pool + from + i * 256) : make_uint2(0u, 0u);
  const int64_t to = (static_cast<int64_t>(bh) * G.n + tile * 16) * D + lane * 8;
  const int live = min(16, G.n - tile * 16) * D;        // elements
#pragma unroll
  for (int i = 0; i < 2 * kSteps; ++i) {
    const int e = i % kSteps * 256 + lane * 8;
    if (e >= live) continue;
    float x[8];
    values_of<C>(i < kSteps ? k[i % kSteps] : v[i % kSteps], i < kSteps ? ks : vs, x);
    T* out = static_cast<T*>(i < kSteps ? G.k_out : G.v_out) + to + i % kSteps * 256;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(out + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<int4*>(out) = make_int4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
  }
}

// Where the CTAs of queries lie.  Evenly among those of keys and values, whose latencies they fill, where there are more than four times as many as are resident and a
// fifth of them at least are theirs; else behind the others, which take longer each.  us evenly / behind: 8 x 2048 rows of 32 heads over 8 62 / 74, 16 x 2048 of 8 74 / 90,
// 8 x 512 17.4 / 18.0, 8 x 256 9.8 / 8.7, 64 x 32 of 64 heads 15.2 / 14.1, 1000 x 1 19.4 / 18.7.
unsigned long long q_step_of(int64_t kv_ctas, int64_t q_ctas) {
  const unsigned long long q = q_ctas, all = kv_ctas + q, whole = ~0ull;
  if (all <= 4ull * kAppendCTAs * kNumSMs || 5 * q < all) return 0;
  return whole / all * q + (whole % all + 1) * q / all + 1;        // 2^64 q / all, rounded up: less than 1 too much in 2^64 / all products
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
  if (k_pool == v_pool || k_scale == v_scale) return fail(B200_EINVAL, "%s: keys and values need pools and scales of their own", name);
  if (!row_starts && rows != B) return fail(B200_EINVAL, "%s: %d rows of %d sequences need row_starts", name, rows, B);
  A.r = Rows{row_starts, context_lens, B, rows};
  A.q = q, A.k = k, A.v = v, A.cos_t = cos_table, A.sin_t = sin_table, A.q_out = q_out;
  A.q_stride = q_stride, A.k_stride = k_stride, A.v_stride = v_stride, A.out_stride = q_out_stride, A.Hq = Hq;
  const int longest = row_starts ? (max_new < rows ? max_new : rows) : 1;
  A.pages = longest == 0 ? 0 : longest == 1 ? 1 : static_cast<int>((longest - 2ll + block_size) / block_size) + 1;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t units = static_cast<int64_t>(B) * A.pages * Hkv * 2, grid = units + (q_out ? rows : 0);
  if (grid * 4 > INT32_MAX) return fail(B200_ESHAPE, "%s: %d sequences of up to %d pages", name, B, A.pages);
  if (grid == 0) return 0;
  const int places = D == 64 && block_size % 32 == 0 ? 32 : 16, warps = block_size / places;        // of a warp; of a page
  const bool pieces = aligned16(k) && aligned16(v) && aligned16(cos_table) && aligned16(sin_table) && aligned16(k_pool) && aligned16(v_pool) && k_stride % 8 == 0 &&
                      v_stride % 8 == 0 && (!q_out || (aligned16(q) && aligned16(q_out) && q_stride % 8 == 0 && q_out_stride % 8 == 0));
  const bool fast = dtype != B200_DTYPE_F32 && (D == 64 || D == 128) && (block_size == 16 || block_size == 32 || block_size == 64) && pieces;
  return with_types(dtype, codes, [&](auto* t, auto* c) {
    using T = std::remove_pointer_t<decltype(t)>;
    using C = std::remove_pointer_t<decltype(c)>;
    if constexpr (sizeof(T) == 2) {
      if (fast) {
        const int64_t ctas = (units * warps + 3) / 4, q_ctas = q_out ? (static_cast<int64_t>(rows) * ((Hq + kHeadsPerWarp - 1) / kHeadsPerWarp) + 3) / 4 : 0;
        auto kern = D == 128 ? (warps == 1 ? append_kernel<T, C, 128, 16, 1> : warps == 2 ? append_kernel<T, C, 128, 16, 2> : append_kernel<T, C, 128, 16, 4>)
                             : (places == 16 ? append_kernel<T, C, 64, 16, 1> : warps == 1 ? append_kernel<T, C, 64, 32, 1> : append_kernel<T, C, 64, 32, 2>);
        return launch_behind(name, kern, static_cast<unsigned>(ctas + q_ctas), 128, 0, s, A, static_cast<unsigned>(ctas), q_step_of(ctas, q_ctas));
      }
    }
    append_any_kernel<T, C><<<static_cast<unsigned>(grid), 128, 0, s>>>(A);
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
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int tiles = static_cast<int>((n_tokens + 15ll) / 16);
  const int64_t blocks = (static_cast<int64_t>(B) * Hkv * n_tokens * D + 255) / 256, units = static_cast<int64_t>(B) * Hkv * tiles;
  const bool fast = (D == 64 || D == 128) && block_size % 16 == 0 && aligned16(k_out) && aligned16(v_out) && aligned16(k_pool) && aligned16(v_pool) && units < INT32_MAX - 8;
  return with_types(dtype, codes, [&](auto* t, auto* c) {
    using T = std::remove_pointer_t<decltype(t)>;
    using C = std::remove_pointer_t<decltype(c)>;
    if (fast) {
      auto kern = D == 128 ? gather_kernel<T, C, 128> : gather_kernel<T, C, 64>;
      return launch_behind(name, kern, static_cast<unsigned>((units + 7) / 8), 256, 0, s, G, static_cast<unsigned>(tiles), static_cast<unsigned>(units));
    }
    gather_any_kernel<T, C><<<static_cast<unsigned>(blocks < kNumSMs * 8 ? blocks : kNumSMs * 8), 256, 0, s>>>(G);
    return check_launch(name);
  });
}

}  // extern "C"
