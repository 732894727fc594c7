// A token for each row of logits, from a given random number, under a temperature, top-k, top-p and min-p of the row's own.
//
//   w_i   = 2^((x_i - max x) * log2(e) / t), 0 for -inf
//   order = descending logits, the lowest index first among equals
//   kept  = the first k of the order; of these the ones before which the weights sum to less than p of theirs all; of these w_i >= min_p:
//           a beginning of the order, down to some (key, index)
//   token = the first index, in the row's own order, up to which the kept weights sum to more than u of them all
//
// Whether a token is the one decides on sums of up to a million weights.  They are summed as multiples of 2^-frac (frac = 62 - log2 of the row's
// length, at most 44) - in doubles while 53 bits hold every sum, a thread's, then as whole numbers -, so no sum depends on its order: neither on how a
// row is spread over CTAs, nor on warps or atomics.  A weight is computed to 2^-31 of itself (the argument in a pair of floats, 256 steps of a power of two from a
// table, a polynomial of degree 3 between them, after Tang's table-driven exponential; set to its exponent and rounded by the double unit, which has
// nothing else to do): errors of independent weights leave one token in 10^7 rows of 128 k another one than 64 bits would.
//
// A row has a cluster of CTAs; each holds its part of the row in shared memory from the only pass over it in memory, if the parts fit; else its three passes
// read it from memory.  Blocks of 256 elements, eight side by side per lane.
//   all rows        load, maximum
//   k, or p         numbers of elements in 1024 ranges of log w (0 .. -46).  k: all elements down to the range that the k-th is in go in a list; p: from
//                   these, to first order in where the elements lie in their ranges, it is known to some 10^-4 where the weights sum to p of all, the elements of these ranges go in
//                   the list, and exact sums are taken of what is above and of all
//   list (4096)     searched by the cluster's first CTA for the last that k keeps, then p; where nothing is above the list, for the token too
//   other rows      kept weights of each block; the block, the lane and the element in which u falls
// Where that does not serve - k over 2048, or ranges of more than 4096 elements, equal logits above all - the last key is found by its digits of 8 bits
// from counts or sums in the whole row.
//
// Bound: a row or a few by the chain of passes and cluster barriers (1500 clocks each; one row of 128256 in 16 bits, k 50 and p 0.9: 13.4 us on the
// device; 64 rows of settings of their own 50, the rows without k the longest); many rows by the instructions of the exact weights, about ninety per element
// in all passes (256 rows of 128256 in 32 bits, p 0.95 with thousands of tokens kept: 137 us; their bytes take 20, read three times 60).
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "b200_common.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBlock = 256;         // elements
constexpr int kRanges = 1024, kRangeColumns = 8;        // columns: lanes that fall in the same range meet at fewer addresses
constexpr float kRange = 11.5f;           // of 1/256 in log2
constexpr int kStepBits = 3, kCountShift = 17, kMostBlocks = 580;       // eight steps a range; elements and steps of a CTA's column share 32 bits
static_assert(32 * kMostBlocks * ((1 << kStepBits) - 1) < 1 << kCountShift && 32 * kMostBlocks < 1 << (32 - kCountShift), "blocks of a CTA");
constexpr int kDigits = 256, kColumns = 8;
constexpr int kList = 4096, kMostK = 2048;
using u64 = unsigned long long;

struct Sample {
  int64_t* out;
  const void* x;
  int64_t row_stride;
  int cols;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float t0, p0, m0;
  int k0;
  int blocks_per_cta, frac, index_bits;
};

// ---- keys: whole numbers in the order of the logits; both zeros are one ------------------------------------------------------------------
template <typename T>
struct Key {
  static constexpr int kBits = 16;
  static __device__ __forceinline__ uint32_t of(uint32_t bits) {
    if (bits == 0x8000u) bits = 0;
    return bits & 0x8000u ? 0xffffu & ~bits : bits | 0x8000u;
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t key) { return key & 0x8000u ? key & 0x7fffu : 0xffffu & ~key; }
};
template <>
struct Key<float> {
  static constexpr int kBits = 32;
  static __device__ __forceinline__ uint32_t of(uint32_t bits) {
    if (bits == 0x80000000u) bits = 0;
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t key) { return key & 0x80000000u ? key & 0x7fffffffu : ~key; }
};
template <typename T>
__device__ __forceinline__ float value(uint32_t bits);
template <>
__device__ __forceinline__ float value<float>(uint32_t bits) { return __uint_as_float(bits); }
template <>
__device__ __forceinline__ float value<__half>(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }
template <>
__device__ __forceinline__ float value<__nv_bfloat16>(uint32_t bits) { return __uint_as_float(bits << 16); }
// largest of two, NaN if one is
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __half>) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
constexpr uint32_t kMinusInf = sizeof(T) == 4 ? 0xff800000u : (std::is_same_v<T, __half> ? 0xfc00u : 0xff80u);

template <typename T>
struct Eight {      // bits of eight elements
  uint32_t w[sizeof(T) * 2];
  __device__ __forceinline__ uint32_t operator[](int e) const {
    if constexpr (sizeof(T) == 4) return w[e];
    else return (w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
  }
};

// 2^(30 + j / 256), as a whole number and as a float's bits
struct Steps {
  uint32_t whole[256];
  float number[256];
};
constexpr Steps make_steps() {
  // 2^(1/256), 2^(1/128) ... 2^(1/2)
  constexpr double roots[8] = {1.0027112750502024854, 1.0054299011128028214, 1.0108892860517004600, 1.0218971486541166782, 1.0442737824274138403,
                               1.0905077326652576592, 1.1892071150027210667, 1.4142135623730950488};
  Steps t{};
  for (int j = 0; j < 256; ++j) {
    double x = 1073741824.0;
    for (int b = 0; b < 8; ++b)
      if (j >> b & 1) x *= roots[b];
    t.whole[j] = static_cast<uint32_t>(x + 0.5) - 0x4b400000u;        // (less the bits of 3 * 2^22, which come with what is added)
    t.number[j] = static_cast<float>(x);
  }
  return t;
}
__device__ constexpr Steps kSteps = make_steps();

constexpr int kMostCtas = 8;      // of a cluster

struct alignas(16) Shared {
  uint2 table[256];             // Steps
  union {
    uint32_t ranges[kRanges * kRangeColumns];
    u64 range_sum[kRanges];             // the cluster's range_count
    struct {
      uint32_t cnt[kDigits * kColumns], lo[kDigits * kColumns], hi[kDigits * kColumns];
    };
    u64 list[kList];
  };
  union {
    u64 range_count[kRanges];           // this CTA's, read by the cluster: elements << 32 | their steps into the range
    struct {
      u64 mass[2][kDigits];             // likewise
      uint32_t count[2][kDigits];
      u64 all_mass[kDigits];            // the cluster's
      uint32_t all_count[kDigits];
    };
  };
  u64 part[kWarps];
  // read by the cluster
  uint32_t best;                        // largest key
  uint32_t first;                       // lowest index of the row's maximum
  uint32_t listed;
  int failed;
  u64 sum_all, sum_above, kept, equal;
  u64 cut;                              // (key, ~index) of the last that is kept
  // this CTA's
  u64 level[4], at[4], ends[2];
  uint32_t few;
  int from, to, n;
};
constexpr int kBins = kThreads, kFew = 256;       // of Shared::range_count, where the list is searched
static_assert(kBins + 2 * kFew <= kRanges, "room for bins and a bin's elements");

// weights: multiples of 2^-frac
struct Weigh {
  // An argument is (x - off) scale - c, scale = 256 log2(e) / t, c = (max - off) scale, each in two parts; one product less than a whole number near it,
  // in one rounding, is what the polynomial takes.  off = 0, and c a multiple of 2^-5 with a rest; where c passes 2^18, off = max, for then what matters is
  // within a twentieth of the maximum, and its difference exact.  (off = max for all rows of 16 bits saves two instructions of thirty, 0.2 - 0.4 us of 13.4
  // for one row of 128256 and 49.9 for 64; but the difference of a logit near zero from a large one has more than 24 bits, and its weight was off by 2^-21.)
  float off, scale, scale_low, c, c_low;
  float floor, end;                     // arguments below `floor` count as it; steps from `end` on give 0
  double one;                           // 2^(52 - frac), whose last bit is 2^-frac
  const uint2* table;
  __device__ __forceinline__ float argument(float x) const { return fmaf(x - off, scale, -c); }
  __device__ __forceinline__ double operator()(float x) const {
    const float d = x - off, shift = 12582912.f, r = fmaxf(argument(x), floor) + shift;        // 3 * 2^22: the nearest whole number n is in the last bits
    const uint32_t n = __float_as_uint(r);
    // (below the floor no number or any: 2^-50 of 32 bits is 0 all the same)
    const float f = fmaf(d, scale, -(c + (r - shift))) + fmaf(d, scale_low, -c_low);
    constexpr float c1 = 0.69314718055994530942 / 256, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;
    const uint2 step = table[n & 255];
    const float q = f * fmaf(fmaf(f, c3, c2), f, c1);
    const uint32_t w = step.x + __float_as_uint(fmaf(q, __uint_as_float(step.y), shift));       // 2^30 times what is left of the exponent
    const double exponent = __hiloint2double((n & ~255u) * 4096u + ((1023u - 30u << 20) - (0x4b400000u << 12)), 0);
    return fma(__hiloint2double(0x43300000, w) - 4503599627370496.0, exponent, one) - one;
  }
  __device__ __forceinline__ u64 whole(double w) const { return __double_as_longlong(w + one) - __double_as_longlong(one); }      // w < one
  __device__ __forceinline__ u64 number(float x) const { return whole((*this)(x)); }
  // place of an argument, in steps; none of no number (-inf without a scale)
  __device__ __forceinline__ float steps(float y) const { return fmaf(y, -(1 << kStepBits) / kRange, 8388608.f); }
};

template <typename V>
__device__ __forceinline__ V warp_sum_of(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// sum of the values of lower lanes
template <typename V>
__device__ __forceinline__ V warp_before(V v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += up;
  }
  const V shifted = __shfl_up_sync(0xffffffffu, v, 1);
  return (threadIdx.x & 31) ? shifted : V(0);
}
// sum of the values of lower threads; *all: of the CTA's
template <typename V>
__device__ __forceinline__ V cta_before(V v, V* part, V* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const V in_warp = warp_before(v);
  __syncthreads();
  if (lane == 31) part[warp] = in_warp + v;
  __syncthreads();
  V upto = part[lane & (kWarps - 1)];
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, upto, o, kWarps);
    if ((lane & (kWarps - 1)) >= o) upto += up;
  }
  const V before = __shfl_sync(0xffffffffu, upto, max(warp - 1, 0), kWarps), total = __shfl_sync(0xffffffffu, upto, kWarps - 1, kWarps);
  *all = total;
  return (warp ? before : V(0)) + in_warp;
}

// f of 2^64, within 0 .. 2^64 - 1; not a number: 0
__device__ __forceinline__ u64 fraction(float f) { return f > 0.f ? (f < 1.f ? static_cast<u64>(static_cast<double>(f) * 18446744073709551616.0) : ~0ull) : 0ull; }
// weights before a kept one sum to less than this: the next whole number from p of `all` on
__device__ __forceinline__ u64 limit_of(float p, u64 all) {
  const u64 f = fraction(p);
  return max(__umul64hi(f, all) + (f * all ? 1 : 0), 1ull);
}

template <typename T, bool HELD>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const Sample A) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  Shared& S = *reinterpret_cast<Shared*>(dynamic);
  cg::cluster_group cluster = cg::this_cluster();
  const int n_cta = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / n_cta;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* x = static_cast<const T*>(A.x) + static_cast<int64_t>(row) * A.row_stride;
  // places count from the 16-byte boundary before the row
  const int head = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T);
  const T* x0 = x - head;
  const int end = head + A.cols;
  const int block0 = rank * A.blocks_per_cta;
  const int n_blocks = max(0, min(A.blocks_per_cta, (end + kBlock - 1) / kBlock - block0));
  u64* block_mass = reinterpret_cast<u64*>(dynamic + sizeof(Shared));
  uint32_t* held = reinterpret_cast<uint32_t*>(block_mass + ((A.blocks_per_cta + 1) & ~1));
  constexpr int kWords = sizeof(T) * 2;     // of eight elements

  auto from_memory = [&](int block) {       // what is not the row's reads as -inf
    Eight<T> v;
    const int at = (block0 + block) * kBlock + lane * 8;
    if (at >= head && at + 8 <= end) {
#pragma unroll
      for (int c = 0; c < kWords; c += 4) {
        const int4 q = __ldg(reinterpret_cast<const int4*>(x0 + at) + c / 4);
        v.w[c] = q.x, v.w[c + 1] = q.y, v.w[c + 2] = q.z, v.w[c + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int c = 0; c < kWords; ++c) v.w[c] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t bits = kMinusInf<T>;
        if (at + e >= head && at + e < end) {
          if constexpr (sizeof(T) == 4) bits = reinterpret_cast<const uint32_t*>(x0)[at + e];
          else bits = reinterpret_cast<const unsigned short*>(x0)[at + e];
        }
        if constexpr (sizeof(T) == 4) v.w[e] = bits;
        else v.w[e >> 1] |= bits << (16 * (e & 1));
      }
    }
    return v;
  };
  auto load = [&](int block) {
    if constexpr (HELD) {
      Eight<T> v;
      const uint4* p = reinterpret_cast<const uint4*>(held + (block * 32 + lane) * kWords);
#pragma unroll
      for (int c = 0; c < kWords; c += 4) {
        const uint4 q = p[c / 4];
        v.w[c] = q.x, v.w[c + 1] = q.y, v.w[c + 2] = q.z, v.w[c + 3] = q.w;
      }
      return v;
    } else {
      return from_memory(block);
    }
  };
  auto bits_at = [&](int block, int e) -> uint32_t {
    using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, unsigned short>;
    if constexpr (HELD) return reinterpret_cast<const Bits*>(held)[(block * 32 + lane) * 8 + e];
    else return __ldg(reinterpret_cast<const Bits*>(x0) + (block0 + block) * kBlock + lane * 8 + e);
  };
  // a warp's blocks, one after another; what comes from memory is asked for a block ahead
  auto each_block = [&](auto&& f) {
    if constexpr (HELD) {
      for (int b = warp; b < n_blocks; b += kWarps) f(b, load(b));
    } else {
      if (warp >= n_blocks) return;
      Eight<T> next = load(warp);
      for (int b = warp; b < n_blocks; b += kWarps) {
        const Eight<T> v = next;
        if (b + kWarps < n_blocks) next = load(b + kWarps);
        f(b, v);
      }
    }
  };
  auto index_of = [&](int block, int e) { return (block0 + block) * kBlock + lane * 8 + e - head; };
  // an element's place in the order: its key over its index, upside down
  const uint32_t index_mask = (1u << A.index_bits) - 1;
  auto composite = [&](uint32_t bits, int index) { return static_cast<u64>(Key<T>::of(bits)) << A.index_bits | (index_mask - static_cast<uint32_t>(index)); };
  auto key_in = [&](u64 c) { return static_cast<uint32_t>(c >> A.index_bits); };
  auto index_in = [&](u64 c) { return index_mask - (static_cast<uint32_t>(c) & index_mask); };
  auto logit_of = [&](u64 c) { return value<T>(Key<T>::bits(key_in(c))); };

  // the CTAs' values of the cluster, all asked for before the first is needed
  auto of_all = [&](auto* mine, auto* values) {
#pragma unroll
    for (int r = 0; r < kMostCtas; ++r) values[r] = r < n_cta ? *cluster.map_shared_rank(mine, r) : 0;
  };
  auto sum_of_all = [&](auto* mine) {
    std::remove_pointer_t<decltype(mine)> v[kMostCtas], sum = 0;
    of_all(mine, v);
#pragma unroll
    for (int r = 0; r < kMostCtas; ++r) sum += v[r];
    return sum;
  };

  // ---- the largest logit ---------------------------------------------------------------------------------------------------------------------
  const float t = A.temperature ? A.temperature[row] : A.t0, p = A.top_p ? A.top_p[row] : A.p0, least = A.min_p ? A.min_p[row] : A.m0, u = A.u[row];
  int k = A.top_k ? A.top_k[row] : A.k0;
  if (tid < 256) S.table[tid] = make_uint2(kSteps.whole[tid], __float_as_uint(kSteps.number[tid]));
  if (tid == 0) S.first = 0xffffffffu, S.listed = 0, S.failed = 0, S.sum_all = S.sum_above = 0, S.best = 0;
  __syncthreads();
  float top = -INFINITY;
  {
    constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;
    [[maybe_unused]] uint32_t top2 = kMinusInf<T> | kMinusInf<T> << 16;
    for (int b = warp; b < n_blocks; b += kAhead * kWarps) {
      Eight<T> v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (b + u * kWarps < n_blocks) v[u] = from_memory(b + u * kWarps);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (b + u * kWarps >= n_blocks) break;
        if constexpr (HELD) {
          uint4* p = reinterpret_cast<uint4*>(held + ((b + u * kWarps) * 32 + lane) * kWords);
#pragma unroll
          for (int c = 0; c < kWords; c += 4) p[c / 4] = make_uint4(v[u].w[c], v[u].w[c + 1], v[u].w[c + 2], v[u].w[c + 3]);
        }
#pragma unroll
        for (int c = 0; c < kWords; ++c) {
          if constexpr (sizeof(T) == 4) top = larger(top, __uint_as_float(v[u].w[c]));
          else top2 = larger2<T>(top2, v[u].w[c]);
        }
      }
    }
    if constexpr (sizeof(T) == 2) top = larger(value<T>(top2 & 0xffffu), value<T>(top2 >> 16));
    const uint32_t mine = __reduce_max_sync(0xffffffffu, top != top ? 0xffffffffu : Key<float>::of(__float_as_uint(top)));
    if (lane == 0) atomicMax(&S.best, mine);
  }
  cluster.sync();
  uint32_t best = 0;
  {
    uint32_t v[kMostCtas];
    of_all(&S.best, v);
#pragma unroll
    for (int r = 0; r < kMostCtas; ++r) best = max(best, v[r]);
  }
  top = __uint_as_float(best == 0xffffffffu ? 0x7fffffffu : Key<float>::bits(best));
  if (!(t > 0.f) || !(fabsf(top) < INFINITY)) {      // no temperature, or a largest logit that is no number: the first of the largest
    uint32_t first = 0xffffffffu;
    each_block([&](int b, const Eight<T>& v) {
#pragma unroll
      for (int e = 7; e >= 0; --e) {
        const float f = value<T>(v[e]);
        const int index = index_of(b, e);
        if ((f == top || (f != f && top != top)) && index >= 0 && index < A.cols) first = min(first, static_cast<uint32_t>(index));
      }
    });
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0 && first != 0xffffffffu) atomicMin(cluster.map_shared_rank(&S.first, 0), first);
    cluster.sync();
    if (rank == 0 && tid == 0) A.out[row] = S.first;
    return;
  }
  if (k <= 0 || k >= A.cols) k = 0;
  const bool by_mass = p < 1.0f;
  // (min_p no number: no limit)
  Weigh weigh;
  {
    const double scale = 369.32993046757463 / static_cast<double>(t);     // 256 log2(e)
    weigh.scale = static_cast<float>(fmin(scale, 3e38));
    weigh.scale_low = scale < 3e38 ? static_cast<float>(scale - weigh.scale) : 0.f;
    const double c = static_cast<double>(top) * (static_cast<double>(weigh.scale) + static_cast<double>(weigh.scale_low));
    const bool apart = fabs(c) <= 262144.0;
    weigh.off = apart ? 0.f : top;
    weigh.c = apart ? static_cast<float>(rint(c * 32.0) / 32.0) : 0.f;
    weigh.c_low = apart ? static_cast<float>(c - static_cast<double>(weigh.c)) : 0.f;
    weigh.floor = -256.0f * (A.frac + 8);
    weigh.end = weigh.steps(-256.0f * (A.frac + 1)) + 1.f;
    weigh.one = __hiloint2double((1023 + 52 - A.frac) << 20, 0);
    weigh.table = S.table;
  }
  const double least_weight = least > 0.f ? ceil(static_cast<double>(fminf(least, 1.0f)) * static_cast<double>(1ull << A.frac)) / static_cast<double>(1ull << A.frac) : 0.0;

  const u64 least_number = weigh.whole(least_weight);
  // a block's sum from the lanes' (of eight weights, 24 bits at a time)
  auto set_block = [&](int b, double mine) {
    const u64 m = weigh.whole(mine);
    const uint32_t low = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(m) & 0xffffffu), high = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(m >> 24));
    if (lane == 0) block_mass[b] = (static_cast<u64>(high) << 24) + low;
  };

  u64 cut = 0;            // kept: (key, ~index) from this on
  bool summed = false;    // the blocks' sums are there already
  bool search = k || by_mass;
  if (search && k <= kMostK) {
    // ---- elements in each range of log w --------------------------------------------------------------------------------------------------------
    for (int i = tid; i < kRanges * kRangeColumns / 4; i += kThreads) reinterpret_cast<uint4*>(S.ranges)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    each_block([&](int, const Eight<T>& v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float step = weigh.steps(weigh.argument(value<T>(v[e])));
        if (step < weigh.end) {
          const uint32_t at = __float_as_uint(step) & 0x7fffffu;
          atomicAdd(&S.ranges[(at >> kStepBits) * kRangeColumns + (lane & (kRangeColumns - 1))], 1u << kCountShift | (at & ((1 << kStepBits) - 1)));
        }
      }
    });
    __syncthreads();
    constexpr int kMine = kRanges / kThreads;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      uint32_t c = 0, steps = 0;
#pragma unroll
      for (int j = 0; j < kRangeColumns; ++j) {
        const uint32_t q = S.ranges[(tid * kMine + i) * kRangeColumns + (j + tid) % kRangeColumns];
        c += q >> kCountShift;
        steps += q & ((1u << kCountShift) - 1);
      }
      S.range_count[tid * kMine + i] = static_cast<u64>(c) << 32 | steps;
    }
    if (tid == 0) S.from = 0, S.to = kRanges - 1;
    cluster.sync();
    // each CTA sums a part of the ranges for all (all of them in every CTA: 10000 clocks instead of 4000)
    for (int i = tid; i < kRanges / n_cta; i += kThreads) {
      const int range = rank * (kRanges / n_cta) + i;
      const u64 sum = sum_of_all(&S.range_count[range]);
#pragma unroll
      for (int r = 0; r < kMostCtas; ++r)
        if (r < n_cta) *cluster.map_shared_rank(&S.range_sum[range], r) = sum;
    }
    cluster.sync();
    // numbers, and weights to second order of the steps (as whole numbers: the same sums in all CTAs)
    uint32_t c[kMine];
    u64 m[kMine], m_mine = 0, m_all, n_mine = 0, n_all;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const u64 both = S.range_sum[tid * kMine + i];
      c[i] = static_cast<uint32_t>(both >> 32);
      const float of = static_cast<float>(c[i]), into = static_cast<float>(static_cast<uint32_t>(both)) / (1 << kStepBits) - 0.5f * of;
      m[i] = static_cast<u64>(exp2f(40.f - (tid * kMine + i + 0.5f) * (kRange / 256.f)) * fmaf(into, -0.69314718f * kRange / 256.f, of));
      n_mine += c[i];
      m_mine += m[i];
    }
    u64 n = cta_before(n_mine, S.part, &n_all);
    int listing;
    if (k) {       // down to the range of the k-th
      if (tid == 0) S.n = static_cast<int>(n_all);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (n < k && k <= n + c[i]) S.to = tid * kMine + i, S.n = static_cast<int>(n + c[i]);
        n += c[i];
      }
      __syncthreads();
      listing = S.n;
    } else {       // the ranges within 0.05 % of the whole around p of it
      u64 before = cta_before(m_mine, S.part, &m_all);
      const u64 low = __umul64hi(fraction(p - 0.0005f), m_all), high = __umul64hi(fraction(p + 0.0005f), m_all) + 1;
      if (tid == 0) S.at[0] = 0, S.at[1] = n_all;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (before < low && low <= before + m[i]) S.from = tid * kMine + i, S.at[0] = n;
        if (before < high && high <= before + m[i]) S.to = tid * kMine + i, S.at[1] = n + c[i];
        n += c[i];
        before += m[i];
      }
      __syncthreads();
      const bool all_of_it = S.at[1] <= kFew;        // nothing above the list: it is compared pairwise (searched, it costs more than the blocks do)
      listing = static_cast<int>(all_of_it ? S.at[1] : S.at[1] - S.at[0]);
      __syncthreads();
      if (all_of_it && tid == 0) S.from = 0;
      __syncthreads();
    }
    const int from = S.from, to = S.to;
    if (listing <= kList) {       // (the same in all CTAs)
      // ---- the list; a row without k: exact sums of all, of what is above the list, and of the blocks' part of that ------------------------------
      double all = 0, above = 0;
      const float from_step = 8388608.f + (from << kStepBits), to_step = fminf(8388608.f + ((to + 1) << kStepBits), weigh.end);
      auto gather = [&](auto sums, auto limited) {
        each_block([&](int b, const Eight<T>& v) {
          double sum = 0;
          unsigned hits = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float f = value<T>(v[e]), step = weigh.steps(weigh.argument(f));
            if (step >= from_step && step < to_step) hits |= 1u << e;
            if constexpr (decltype(sums)::value) {
              const double w = weigh(f);
              all += w;
              if (step < from_step) {
                if (decltype(limited)::value) above += w;
                if (!decltype(limited)::value || w >= least_weight) sum += w;
              }
            }
          }
          if (hits) {       // looked up again, one by one: few
            uint32_t at = atomicAdd(&S.listed, static_cast<uint32_t>(__popc(hits)));
            do {
              const int e = __ffs(hits) - 1;
              hits &= hits - 1;
              if (at < kList) S.list[at++] = composite(bits_at(b, e), index_of(b, e));
            } while (hits);
          }
          if (decltype(sums)::value && from > 0) {
            if (!decltype(limited)::value) above += sum;
            set_block(b, sum);
          }
        });
      };
      if (k) gather(std::false_type{}, std::false_type{});
      else if (least_weight > 0) gather(std::true_type{}, std::true_type{});
      else gather(std::true_type{}, std::false_type{});
      if (!k) {
        const double per_unit = static_cast<double>(1ull << A.frac);
        const u64 all_mine = warp_sum_of(static_cast<u64>(__double2ll_rn(all * per_unit))), above_mine = warp_sum_of(static_cast<u64>(__double2ll_rn(above * per_unit)));
        if (lane == 0) {
          atomicAdd(&S.sum_all, all_mine);
          atomicAdd(&S.sum_above, above_mine);
        }
      }
      cluster.sync();
      if (k && rank > 0) {
        cluster.sync();
        return;
      }
      if (rank == 0) {
        uint32_t lists[kMostCtas];
        of_all(&S.listed, lists);
        int n = lists[0];
        for (int i = tid; i - tid < kList; i += kThreads) {       // a round of all lists at a time
          u64 v[kMostCtas];
          bool more = false;
#pragma unroll
          for (int r = 1; r < kMostCtas; ++r)
            if (r < n_cta && i < lists[r]) v[r] = *cluster.map_shared_rank(&S.list[i], r);
          int to = n;
#pragma unroll
          for (int r = 1; r < kMostCtas; ++r) {
            if (r < n_cta && i < lists[r] && to + i < kList) S.list[to + i] = v[r];
            to += lists[r];
            more = more || i - tid + kThreads < lists[r];
          }
          if (!more) break;
        }
#pragma unroll
        for (int r = 1; r < kMostCtas; ++r) n += lists[r];
        n = min(n, kList);
        if (k) cluster.sync();        // the others are not needed any more
        __syncthreads();
        if (n <= kFew && from == 0) {
          // few elements: every two of them are compared, by 512 threads together
          u64* weights = S.range_count;
          int parts = kThreads;
          while (parts > 32 || (kThreads / parts) < n) parts /= 2;
          const int i = tid / parts, part = tid & (parts - 1);
          const u64 c = i < n ? S.list[i] : 0, w = i < n ? weigh.number(logit_of(c)) : 0;
          if (part == 0 && i < n) weights[i] = w;
          u64 whole = k ? 0 : sum_of_all(&S.sum_all);
          __syncthreads();
          auto before_mine = [&](auto&& earlier, u64* count) {
            u64 sum = 0, n_before = 0;
            for (int j = part; j < n; j += parts)
              if (earlier(S.list[j])) sum += weights[j], ++n_before;
            for (int o = 1; o < parts; o <<= 1) {
              sum += __shfl_xor_sync(0xffffffffu, sum, o);
              n_before += __shfl_xor_sync(0xffffffffu, n_before, o);
            }
            *count = n_before;
            return sum;
          };
          u64 place, unused, sum;
          const u64 heavier = before_mine([&](u64 o) { return o > c; }, &place);
          bool keep = i < n && (!k || place < k);
          if (by_mass) {
            cta_before(keep && part == 0 ? w : 0ull, S.part, &sum);
            const u64 limit = limit_of(p, k ? sum : whole);
            if (!k && sum < limit && tid == 0) S.failed = 1;       // p of all is reached below the list
            keep = keep && heavier < limit;
          }
          keep = keep && w >= least_number;
          __syncthreads();
          if (part == 0 && i < n) weights[i] = keep ? w : 0;
          cta_before(keep && part == 0 ? w : 0ull, S.part, &sum);
          const u64 goal = __umul64hi(fraction(u), sum);
          const u64 lower = before_mine([&](u64 o) { return (o & index_mask) > (c & index_mask); }, &unused);
          if (keep && part == 0 && !S.failed && lower <= goal && goal < lower + w) A.out[row] = index_in(c);
        } else {
          if (tid == 0) S.ends[0] = ~0ull, S.ends[1] = 0;
          __syncthreads();
          {
            u64 lo = ~0ull, hi = 0;
            for (int i = tid; i < n; i += kThreads) lo = min(lo, S.list[i]), hi = max(hi, S.list[i]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
              lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
              hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            if (lane == 0) {
              atomicMin(&S.ends[0], lo);
              atomicMax(&S.ends[1], hi);
            }
          }
          __syncthreads();
          const u64 lowest_listed = S.ends[0], highest_listed = S.ends[1];
          // The element of the list at which the running value (1 or the weight) from `upto` on reaches `target`, of those from `lowest` on, in the
          // list's order or by index: by the sums of 512 equal parts of what is left, until a part has few elements.
          u64* bins = S.range_count;
          u64 *few = bins + kBins, *few_value = few + kFew;
          auto find = [&](auto by_index, u64 lo, u64 hi, u64 lowest, auto&& value_of, u64 upto, u64 target) -> u64 {
            auto order = [&](u64 c) { return decltype(by_index)::value ? c & index_mask : c; };
            while (true) {
              int shift = 63;       // one part
              u64 bin = 0;
              bins[tid] = 0;
              if (tid == 0) S.few = 0, S.at[0] = ~0ull, S.at[2] = 0;
              __syncthreads();
              if (n > kFew) {
                shift = max(0, 64 - __clzll(hi - lo) - 9);
                for (int i = tid; i < n; i += kThreads) {
                  const u64 c = S.list[i], o = order(c);
                  if (c >= lowest && o >= lo && o <= hi) atomicAdd(&bins[(hi - o) >> shift], value_of(c));
                }
                __syncthreads();
                u64 unused;
                const u64 in = bins[tid], before = upto + cta_before(in, S.part, &unused);
                if (before < target && target <= before + in) S.at[0] = tid, S.at[1] = before;
                __syncthreads();
                if (S.at[0] == ~0ull) return 0;       // not in the list
                bin = S.at[0];
                upto = S.at[1];
              }
              for (int i = tid; i < n; i += kThreads) {
                const u64 c = S.list[i], o = order(c);
                if (c >= lowest && o >= lo && o <= hi && (hi - o) >> shift == bin) {
                  const uint32_t at = atomicAdd(&S.few, 1u);
                  if (at < kFew) few[at] = c, few_value[at] = value_of(c);
                }
              }
              __syncthreads();
              const int m = S.few;
              if (m <= kFew) {
                if (tid < m) {
                  u64 before_mine = upto;
                  for (int j = 0; j < m; ++j)
                    if (order(few[j]) > order(few[tid])) before_mine += few_value[j];
                  if (before_mine < target && target <= before_mine + few_value[tid]) S.at[2] = few[tid];
                }
                __syncthreads();
                const u64 c = S.at[2];
                __syncthreads();
                return c;
              }
              hi -= bin << shift;
              lo = max(lo, hi - ((1ull << shift) - 1));
              __syncthreads();
            }
          };
          auto weight_of = [&](u64 c) { return weigh.number(logit_of(c)); };
          auto kept_of = [&](u64 c) -> u64 {
            const u64 w = weigh.number(logit_of(c));
            return w >= least_number ? w : 0;
          };
          auto sum_from = [&](u64 lowest, auto&& value_of) {
            u64 mine = 0, sum;
            for (int i = tid; i < n; i += kThreads) mine += S.list[i] >= lowest ? value_of(S.list[i]) : 0;
            cta_before(mine, S.part, &sum);
            return sum;
          };
          u64 whole = 0, over = 0, mine = 0;
          if (k) {
            if (n > k) mine = find(std::false_type{}, lowest_listed, highest_listed, 0ull, [](u64) { return 1ull; }, 0ull, static_cast<u64>(k));
            if (by_mass) whole = sum_from(mine, weight_of);
          } else {
            whole = sum_of_all(&S.sum_all);
            over = sum_of_all(&S.sum_above);
          }
          bool failed = false;
          if (by_mass) {
            const u64 limit = limit_of(p, whole);
            const u64 last = over < limit ? find(std::false_type{}, lowest_listed, highest_listed, mine, weight_of, over, limit) : 0;
            failed = last == 0;     // p of all is reached above the list, or below it
            mine = last;
          }
          if (failed) {
            if (tid == 0) S.failed = 1;
          } else if (from > 0) {      // kept ones to their blocks
            for (int i = tid; i < n; i += kThreads) {
              const u64 c = S.list[i], w = c >= mine ? kept_of(c) : 0;
              if (w) {
                const int place = static_cast<int>(index_in(c)) + head, b = place / kBlock, r = b / A.blocks_per_cta;
                u64* sums = reinterpret_cast<u64*>(cluster.map_shared_rank(dynamic, r) + sizeof(Shared));
                atomicAdd(&sums[b - r * A.blocks_per_cta], w);
              }
            }
            if (tid == 0) S.cut = mine;
          } else {        // all that is kept is in the list
            const u64 goal = __umul64hi(fraction(u), sum_from(mine, kept_of));
            const u64 c = find(std::true_type{}, static_cast<u64>(index_mask + 1 - A.cols), static_cast<u64>(index_mask), mine, kept_of, 0ull, goal + 1);
            if (tid == 0) A.out[row] = index_in(c);
          }
        }
      }
      if (k) return;
      cluster.sync();
      if (*cluster.map_shared_rank(&S.failed, 0) == 0) {
        cut = *cluster.map_shared_rank(&S.cut, 0);
        search = false;
        summed = true;
      }
      cluster.sync();       // the others read the first CTA's; and the list is where digits are counted
      if (summed && from == 0) return;
    }
  }

  if (search) {
    // ---- by digits: the key that a number of elements, or a sum of weights, ends in -----------------------------------------------------------
    // Of the elements of key >= lowest: the key at which the running count (by weight: sum) from the largest on reaches `target`.  What is still
    // to be reached in it is left in *rest, its elements in *equal.  target 0: `p` of the sum of all, less `minus`.
    int parity = 0;
    auto select = [&](auto weighted, uint32_t lowest, u64 target, u64 minus, u64* rest, u64* equal) -> uint32_t {
      constexpr bool WEIGHTED = decltype(weighted)::value;
      uint32_t prefix = 0;
      for (int shift = Key<T>::kBits - 8; shift >= 0; shift -= 8) {
        for (int i = tid; i < kDigits * kColumns; i += kThreads) {
          S.cnt[i] = 0;
          if (WEIGHTED) S.lo[i] = S.hi[i] = 0;
        }
        __syncthreads();
        each_block([&](int, const Eight<T>& v) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t key = Key<T>::of(v[e]);
            if (key < lowest || (shift + 8 < 32 && key >> (shift + 8) != prefix)) continue;
            const int slot = ((key >> shift) & 255) * kColumns + (lane & (kColumns - 1));
            atomicAdd(&S.cnt[slot], 1u);
            if constexpr (WEIGHTED) {
              const u64 w = weigh.number(value<T>(v[e]));
              if (w) {
                const uint32_t old = atomicAdd(&S.lo[slot], static_cast<uint32_t>(w));
                const uint32_t up = static_cast<uint32_t>(w >> 32) + (old + static_cast<uint32_t>(w) < old ? 1u : 0u);
                if (up) atomicAdd(&S.hi[slot], up);
              }
            }
          }
        });
        __syncthreads();
        if (tid < kDigits) {
          uint32_t n = 0;
          u64 m = 0;
#pragma unroll
          for (int c = 0; c < kColumns; ++c) {
            n += S.cnt[tid * kColumns + c];
            if (WEIGHTED) m += S.lo[tid * kColumns + c] + (static_cast<u64>(S.hi[tid * kColumns + c]) << 32);
          }
          S.count[parity][tid] = n;
          if (WEIGHTED) S.mass[parity][tid] = m;
        }
        cluster.sync();
        if (tid < kDigits) {
          S.all_count[tid] = sum_of_all(&S.count[parity][tid]);
          if (WEIGHTED) S.all_mass[tid] = sum_of_all(&S.mass[parity][tid]);
        }
        parity ^= 1;      // the others read this level's until they come to the next level's barrier
        __syncthreads();
        if (warp == 0) {        // eight digits a lane, the largest first
          u64 mine = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int d = kDigits - 1 - (lane * 8 + j);
            mine += WEIGHTED ? S.all_mass[d] : S.all_count[d];
          }
          u64 above = warp_before(mine);
          if (WEIGHTED && target == 0) target = limit_of(p, warp_sum_of(mine) - minus);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int d = kDigits - 1 - (lane * 8 + j);
            const u64 in = WEIGHTED ? S.all_mass[d] : S.all_count[d];
            if (above < target && target <= above + in) {
              S.level[0] = d;
              S.level[1] = target - above;
              S.level[2] = S.all_count[d];
            }
            above += in;
          }
        }
        __syncthreads();
        prefix = prefix << 8 | static_cast<uint32_t>(S.level[0]);
        target = S.level[1];
        *equal = S.level[2];
      }
      *rest = target;
      return prefix;
    };
    uint32_t last = 0;
    u64 equals = 0, there = 0, rest = 0, in = 0;      // kept: keys above `last` and the first `equals` of it
    if (k) last = select(std::false_type{}, 0u, static_cast<u64>(k), 0ull, &equals, &there);
    if (by_mass) {
      const u64 each = k ? weigh.number(value<T>(Key<T>::bits(last))) : 0ull;
      last = select(std::true_type{}, last, 0ull, (there - equals) * each, &rest, &in);
      const u64 w = weigh.number(value<T>(Key<T>::bits(last)));
      equals = (rest + w - 1) / w;
    }
    // where the last of them is
    uint32_t same_mine = 0;
    const int per = (n_blocks + kWarps - 1) / kWarps, b0 = min(warp * per, n_blocks), b1 = min(b0 + per, n_blocks);        // a warp's blocks are side by side here
    for (int b = b0; b < b1; ++b) {
      const Eight<T> v = load(b);
#pragma unroll
      for (int e = 0; e < 8; ++e) same_mine += Key<T>::of(v[e]) == last;
    }
    same_mine = __reduce_add_sync(0xffffffffu, same_mine);
    u64 same = 0;
    u64 seen = cta_before(lane == 0 ? static_cast<u64>(same_mine) : 0ull, S.part, &same);
    seen = __shfl_sync(0xffffffffu, seen, 0);
    if (tid == 0) S.equal = same;
    cluster.sync();
    for (int r = 0; r < rank; ++r) seen += *cluster.map_shared_rank(&S.equal, r);
    if (seen < equals && equals <= seen + same_mine) {        // this warp's
      for (int b = b0; b < b1; ++b) {
        const Eight<T> v = load(b);
        uint32_t here = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) here += Key<T>::of(v[e]) == last;
        u64 upto = seen + warp_before(here);
        seen += __reduce_add_sync(0xffffffffu, here);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (Key<T>::of(v[e]) == last && ++upto == equals) {
            const u64 c = composite(v[e], index_of(b, e));
            for (int r = 0; r < n_cta; ++r) *cluster.map_shared_rank(&S.cut, r) = c;
          }
        }
        if (seen >= equals) break;
      }
    }
    cluster.sync();
    cut = S.cut;
  }

  const uint32_t cut_key = key_in(cut), cut_index = index_in(cut);
  auto kept_weight = [&](uint32_t bits, int index) -> double {
    const uint32_t key = Key<T>::of(bits);
    if (key < cut_key || (key == cut_key && static_cast<uint32_t>(index) > cut_index)) return 0.0;
    const double w = weigh(value<T>(bits));
    return w >= least_weight ? w : 0.0;
  };
  // ---- kept weights of each block ----------------------------------------------------------------------------------------------------------------
  if (!summed) {
    auto sum_blocks = [&](auto&& weight_of) {
      each_block([&](int b, const Eight<T>& v) {
        double sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += weight_of(v[e], index_of(b, e));
        set_block(b, sum);
      });
    };
    if (cut || least_weight > 0) sum_blocks(kept_weight);
    else sum_blocks([&](uint32_t bits, int) { return weigh(value<T>(bits)); });
    __syncthreads();
  }
  const int per = (n_blocks + kThreads - 1) / kThreads, b0 = min(tid * per, n_blocks), b1 = min(b0 + per, n_blocks);
  u64 mine = 0, all = 0;
  for (int b = b0; b < b1; ++b) mine += block_mass[b];
  u64 before = cta_before(mine, S.part, &all);
  if (tid == 0) S.kept = all, S.at[0] = ~0ull;
  cluster.sync();
  u64 total = 0, lower = 0;
  {
    u64 v[kMostCtas];
    of_all(&S.kept, v);
#pragma unroll
    for (int r = 0; r < kMostCtas; ++r) {
      total += v[r];
      if (r < rank) lower += v[r];
    }
  }
  const u64 goal = __umul64hi(fraction(u), total);
  before += lower;
  if (before <= goal && goal < before + mine) {
    for (int b = b0; b < b1; ++b) {
      if (goal < before + block_mass[b]) {
        S.at[0] = b;
        S.at[1] = goal - before;
        break;
      }
      before += block_mass[b];
    }
  }
  __syncthreads();
  if (warp == 0 && S.at[0] != ~0ull) {
    const int b = static_cast<int>(S.at[0]);
    const u64 to = S.at[1];
    const Eight<T> v = load(b);
    u64 w[8], sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = weigh.whole(kept_weight(v[e], index_of(b, e)));
      sum += w[e];
    }
    u64 run = warp_before(sum);
    if (run <= to && to < run + sum) {
      int found = 7;
      run += sum;
#pragma unroll
      for (int e = 7; e >= 0; --e) {       // the first whose running sum passes
        if (run > to) found = e;
        run -= w[e];
      }
      A.out[row] = index_of(b, found);
    }
  }
  cluster.sync();       // the others may still read this CTA's
}

template <typename T>
int launch_sample(Sample A, int rows, cudaStream_t stream) {
  const char* name = "b200_sample_rows";
  const int blocks = (A.cols + 7 + kBlock - 1) / kBlock;      // with the places before the row
  auto bytes = [&](int ctas, bool held) {
    const size_t per = (blocks + ctas - 1) / ctas;
    return sizeof(Shared) + ((per + 1) & ~size_t{1}) * 8 + (held ? per * kBlock * sizeof(T) : 0);
  };
  // Two CTAs per SM.  As many for a row as the rows leave room for in one round, each with a part worth a cluster's barriers (1500 clocks each); the parts
  // stay in shared memory if they fit, else they are read again.  (256 rows of 128 k in 32 bits, a call after the other: 148 - 154 us; with more instructions a
  // weight 160; then cut until they fit, in seven rounds of CTAs, 288; every other pass backwards, for what the cache still holds, 162.  37 rows of 32003 in 16 bits: 12.3 us by four CTAs each,
  // 16.8 by eight.)
  constexpr size_t kHalf = 113 * 1024;
  int ctas = 1;
  while (ctas < kMostCtas && (blocks > kMostBlocks * ctas || (2 * ctas * static_cast<int64_t>(rows) <= (blocks >= 128 * ctas ? 2 : 1) * kNumSMs && blocks >= 16 * ctas))) ctas *= 2;
  const bool held = bytes(ctas, true) <= kHalf;
  const size_t smem = bytes(ctas, held);
  if (smem > kMaxSmem) return fail(B200_ESHAPE, "%s: rows of %d", name, A.cols);
  A.blocks_per_cta = (blocks + ctas - 1) / ctas;
  int bits = 0;
  while ((1ll << bits) < A.cols) ++bits;
  A.frac = std::min(62 - bits, 44);
  A.index_bits = std::max(bits, 1);
  auto kern = held ? sample_rows_kernel<T, true> : sample_rows_kernel<T, false>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, A);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(static_cast<int>(e), "%s: %s", name, cudaGetErrorString(e));
  }
  return 0;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_sample_rows(int64_t* out, const void* x, int64_t rows, int64_t cols, int64_t row_stride, const float* u,
                                const float* temperature, float temperature_all, const int32_t* top_k, int top_k_all, const float* top_p,
                                float top_p_all, const float* min_p, float min_p_all, int dtype, void* stream) {
  const char* name = "b200_sample_rows";
  const int es = dtype_size(dtype);
  if (es == 0) return fail(B200_EINVAL, "%s: unsupported dtype %d", name, dtype);
  if (rows < 0 || cols <= 0 || row_stride < 0) return fail(B200_EINVAL, "%s: bad sizes", name);
  if (cols > B200_MAX_SAMPLE_COLS || rows > (1 << 24)) return fail(B200_ESHAPE, "%s: %lld rows of %lld", name, static_cast<long long>(rows), static_cast<long long>(cols));
  if (rows == 0) return 0;
  if (!out || !x || !u) return fail(B200_EINVAL, "%s: null pointer", name);
  if (reinterpret_cast<uintptr_t>(x) % es) return fail(B200_EINVAL, "%s: logits not aligned to their type", name);
  const Sample A{out, x, row_stride, static_cast<int>(cols), u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, 0, 0};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200_DTYPE_F16: return launch_sample<__half>(A, static_cast<int>(rows), s);
    case B200_DTYPE_BF16: return launch_sample<__nv_bfloat16>(A, static_cast<int>(rows), s);
    default: return launch_sample<float>(A, static_cast<int>(rows), s);
  }
}
