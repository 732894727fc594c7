// A token for each row of logits, from a given random number, under a temperature, top-k, top-p and min-p of the row's own.
//
//   w_i   = 2^((x_i - max x) * log2(e) / t), 0 for -inf
//   order = descending logits, the lowest index first among equals
//   kept  = the first k of the order; of these the ones before which the weights sum to less than p of theirs all; of these w_i >= min_p
//           (each a beginning of the order: what is kept is the keys above some key, and the first m of that key itself)
//   token = the first index, in the row's own order, up to which the kept weights sum to more than u of them all
//
// Whether a token is the one decides on sums of up to a quarter of a million weights, next to a border more often than 32 bits tell apart: the
// weights are computed in 64 bits (argument reduced to 1/256 of a power of two, table and a polynomial of degree 4 after Tang's table-driven exponential,
// 2^-52) and summed as whole numbers of 2^-frac (frac = 62 - log2 of the row's length, 45 for 128 k): sums do not depend on their order, so
// neither does the token on how rows are spread over CTAs, on warps or on atomics.
//
// A row has a cluster of CTAs; each holds its part of the row in shared memory from the only pass over it, if the parts fit.  Blocks of 256 elements, eight
// side by side per lane.  Passes: (1) load, maximum; (2) where k limits: the k-th key by its digits of 8 bits, from counts; (3) where p does: the same from
// sums of weights; (4) kept weights per block; then the block, the lane and the element in which u falls.  Digits are counted in 16 columns per
// digit, one for every other lane, so that logits of few exponents do not meet at few addresses.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "b200_common.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kBlock = 256;         // elements
constexpr int kDigits = 256, kColumns = 16;
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
  int blocks_per_cta, frac;
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

struct alignas(16) Shared {
  double table[256];                            // 2^(j / 256)
  uint32_t cnt[kDigits * kColumns], lo[kDigits * kColumns], hi[kDigits * kColumns];
  u64 mass[2][kDigits];                         // this CTA's sums, read by the cluster
  uint32_t count[2][kDigits];
  u64 all_mass[kDigits];                        // the cluster's
  uint32_t all_count[kDigits];
  u64 warp_part[kWarps];
  u64 best;                                     // read by the cluster
  u64 kept;
  u64 equal;
  u64 level[4];                                 // digit, sum above it, count and mass in it
  u64 at[4];
};

// weights
struct Weigh {
  double top, scale;        // maximum; 256 log2(e) / t
  double one, least;        // 2^(52 - frac), whose last bit is 2^-frac; arguments below this are weights of 0
  const double* table;
  __device__ __forceinline__ double operator()(float x) const {
    const double y = (static_cast<double>(x) - top) * scale;
    if (!(y > least)) return 0.0;
    const double shift = 6755399441055744.0;     // 3 * 2^51: the nearest whole number is in the last bits
    const double r = y + shift;
    const int n = __double2loint(r);
    const double f = y - (r - shift);
    constexpr double c1 = 0.69314718055994530942 / 256, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4;
    const double p = fma(fma(fma(fma(f, c4, c3), f, c2), f, c1), f, 1.0);
    const double w = table[n & 255] * p;
    return __hiloint2double(__double2hiint(w) + ((n >> 8) << 20), __double2loint(w));
  }
  __device__ __forceinline__ u64 whole(double w) const { return __double_as_longlong(w + one) - __double_as_longlong(one); }
};

template <typename V>
__device__ __forceinline__ V warp_sum_of(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// sum of the values of lower lanes
__device__ __forceinline__ u64 warp_before(u64 v) {
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) >= o) s += up;
  }
  return s - v;
}
// sum of the values of lower threads; *all: of the CTA's
__device__ __forceinline__ u64 cta_before(u64 v, u64* part, u64* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const u64 in_warp = warp_before(v);
  __syncthreads();
  if (lane == 31) part[warp] = in_warp + v;
  __syncthreads();
  u64 before = 0, total = 0;
  const u64 mine = part[lane];
  before = warp_sum_of(lane < warp ? mine : 0ull);
  total = warp_sum_of(mine);
  *all = total;
  return before + in_warp;
}

template <typename T, bool HELD>
__global__ void __launch_bounds__(kThreads, 1) sample_rows_kernel(const Sample A) {
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
  uint32_t* block_equal = reinterpret_cast<uint32_t*>(block_mass + ((A.blocks_per_cta + 1) & ~1));
  uint32_t* held = block_equal + ((A.blocks_per_cta + 3) & ~3);
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

  // ---- the largest logit and where it is first ---------------------------------------------------------------------------------------------
  if (tid < 256) S.table[tid] = exp2(tid / 256.0);
  u64 best = 0;
  for (int b = warp; b < n_blocks; b += kWarps) {
    const Eight<T> v = from_memory(b);
    if constexpr (HELD) {
      uint4* p = reinterpret_cast<uint4*>(held + (b * 32 + lane) * kWords);
#pragma unroll
      for (int c = 0; c < kWords; c += 4) p[c / 4] = make_uint4(v.w[c], v.w[c + 1], v.w[c + 2], v.w[c + 3]);
    }
    const int at = (block0 + b) * kBlock + lane * 8 - head;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = value<T>(v[e]);
      const uint32_t order = f != f ? 0xffffffffu : Key<float>::of(__float_as_uint(f));
      const u64 key = static_cast<u64>(order) << 32 | (0xffffffffu - static_cast<uint32_t>(at + e));
      if (at + e >= 0 && at + e < A.cols && key > best) best = key;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) S.warp_part[warp] = best;
  __syncthreads();
  if (warp == 0) {
    best = S.warp_part[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) S.best = best;
  }
  cluster.sync();
  best = 0;
  for (int r = 0; r < n_cta; ++r) best = max(best, *cluster.map_shared_rank(&S.best, r));
  const float top = __uint_as_float(Key<float>::bits(static_cast<uint32_t>(best >> 32)));
  const float t = A.temperature ? A.temperature[row] : A.t0;
  // no temperature, or a largest logit that is no number: the greedy token
  if (!(t > 0.f) || !(fabsf(top) < INFINITY)) {
    if (rank == 0 && tid == 0) A.out[row] = 0xffffffffu - static_cast<uint32_t>(best);
    cluster.sync();       // the others may still read this CTA's
    return;
  }
  int k = A.top_k ? A.top_k[row] : A.k0;
  float p = A.top_p ? A.top_p[row] : A.p0, least = A.min_p ? A.min_p[row] : A.m0, u = A.u[row];
  if (k <= 0 || k >= A.cols) k = 0;
  const bool by_mass = p < 1.0f;
  least = least > 0.f ? fminf(least, 1.0f) : 0.f;       // not a number: no limit
  Weigh weigh;
  weigh.top = top;
  weigh.scale = 369.32993046757463 / static_cast<double>(t);     // 256 log2(e)
  weigh.one = __hiloint2double((1023 + 52 - A.frac) << 20, 0);
  weigh.least = -256.0 * (A.frac + 2);
  weigh.table = S.table;

  // ---- the key that a number of elements, or a sum of weights, ends in ----------------------------------------------------------------------
  // Of the elements of key >= lowest: the key at which the running count (by weight: sum) from the largest on reaches `target`.  What is still
  // to be reached in it is left in *rest, its elements in *equal.  target 0: `share` of the sum of all, less `minus`.
  int parity = 0;
  auto select = [&](auto weighted, uint32_t lowest, u64 target, float share, u64 minus, u64* rest, u64* equal) -> uint32_t {
    constexpr bool WEIGHTED = decltype(weighted)::value;
    uint32_t prefix = 0;
    for (int shift = Key<T>::kBits - 8; shift >= 0; shift -= 8) {
      for (int i = tid; i < kDigits * kColumns; i += kThreads) {
        S.cnt[i] = 0;
        if (WEIGHTED) S.lo[i] = S.hi[i] = 0;
      }
      __syncthreads();
      for (int b = warp; b < n_blocks; b += kWarps) {
        const Eight<T> v = load(b);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = Key<T>::of(v[e]);
          if (key < lowest || (shift + 8 < 32 && key >> (shift + 8) != prefix)) continue;
          const int slot = ((key >> shift) & 255) * kColumns + (lane & (kColumns - 1));
          atomicAdd(&S.cnt[slot], 1u);
          if constexpr (WEIGHTED) {
            const u64 w = weigh.whole(weigh(value<T>(v[e])));
            if (w) {
              const uint32_t old = atomicAdd(&S.lo[slot], static_cast<uint32_t>(w));
              const uint32_t up = static_cast<uint32_t>(w >> 32) + (old + static_cast<uint32_t>(w) < old ? 1u : 0u);
              if (up) atomicAdd(&S.hi[slot], up);
            }
          }
        }
      }
      __syncthreads();
      for (int i = tid; i < kDigits * 4; i += kThreads) {       // four threads a digit
        const int first = (i >> 2) * kColumns + (i & 3) * (kColumns / 4);
        uint32_t n = 0;
        u64 m = 0;
#pragma unroll
        for (int c = 0; c < kColumns / 4; ++c) {
          n += S.cnt[first + c];
          if (WEIGHTED) m += S.lo[first + c] + (static_cast<u64>(S.hi[first + c]) << 32);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          n += __shfl_xor_sync(0xffffffffu, n, o);
          if (WEIGHTED) m += __shfl_xor_sync(0xffffffffu, m, o);
        }
        if ((i & 3) == 0) {
          S.count[parity][i >> 2] = n;
          if (WEIGHTED) S.mass[parity][i >> 2] = m;
        }
      }
      cluster.sync();
      if (tid < kDigits) {
        uint32_t n = 0;
        u64 m = 0;
        for (int r = 0; r < n_cta; ++r) {
          n += *cluster.map_shared_rank(&S.count[parity][tid], r);
          if (WEIGHTED) m += *cluster.map_shared_rank(&S.mass[parity][tid], r);
        }
        S.all_count[tid] = n;
        if (WEIGHTED) S.all_mass[tid] = m;
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
        if (WEIGHTED && target == 0) {
          const u64 all = warp_sum_of(mine) - minus;
          // the weights before a kept one sum to less than share * all: to less than the next whole number
          const u64 f = share > 0.f ? static_cast<u64>(static_cast<double>(share) * 18446744073709551616.0) : 0ull;
          target = max(__umul64hi(f, all) + (f * all ? 1 : 0), 1ull);
        }
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

  // kept: keys above `cut`, and the first `equals` of key `cut`
  uint32_t cut = 0;
  u64 equals = 0;
  if (k) {
    u64 there = 0;
    cut = select(std::false_type{}, 0u, static_cast<u64>(k), 0.f, 0ull, &equals, &there);
    if (by_mass) {
      const u64 each = weigh.whole(weigh(value<T>(Key<T>::bits(cut))));
      u64 rest = 0, in = 0;
      const uint32_t at = select(std::true_type{}, cut, 0ull, p, (there - equals) * each, &rest, &in);
      const u64 w = weigh.whole(weigh(value<T>(Key<T>::bits(at))));
      equals = (rest + w - 1) / w;
      cut = at;
    }
  } else if (by_mass) {
    u64 rest = 0, in = 0;
    cut = select(std::true_type{}, 0u, 0ull, p, 0ull, &rest, &in);
    const u64 w = weigh.whole(weigh(value<T>(Key<T>::bits(cut))));
    equals = (rest + w - 1) / w;
  }
  const double cut_weight = weigh(value<T>(Key<T>::bits(cut)));
  const u64 each = weigh.whole(cut_weight);
  if (equals && cut_weight < least) equals = 0;

  // ---- kept weights of each block, without those of key `cut`, which are counted ------------------------------------------------------------
  for (int b = warp; b < n_blocks; b += kWarps) {
    const Eight<T> v = load(b);
    u64 sum = 0;
    uint32_t same = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t key = Key<T>::of(v[e]);
      if (key > cut) {
        const double w = weigh(value<T>(v[e]));
        if (w >= least) sum += weigh.whole(w);
      }
      same += key == cut;
    }
    sum = warp_sum_of(sum);
    same = warp_sum_of(same);
    if (lane == 0) {
      block_mass[b] = sum;
      block_equal[b] = same;
    }
  }
  __syncthreads();
  const int per = (n_blocks + kThreads - 1) / kThreads, b0 = min(tid * per, n_blocks), b1 = min(b0 + per, n_blocks);
  u64 same = 0, all = 0;
  for (int b = b0; b < b1; ++b) same += block_equal[b];
  u64 same_before = cta_before(same, S.warp_part, &all);
  if (tid == 0) S.equal = all;
  cluster.sync();
  for (int r = 0; r < rank; ++r) same_before += *cluster.map_shared_rank(&S.equal, r);
  u64 mine = 0, seen = same_before;
  for (int b = b0; b < b1; ++b) {
    const u64 left = equals > seen ? equals - seen : 0;
    mine += block_mass[b] + min(left, static_cast<u64>(block_equal[b])) * each;
    seen += block_equal[b];
  }
  u64 before = cta_before(mine, S.warp_part, &all);
  if (tid == 0) S.kept = all;
  cluster.sync();
  u64 total = 0, lower = 0;
  for (int r = 0; r < n_cta; ++r) {
    const u64 m = *cluster.map_shared_rank(&S.kept, r);
    total += m;
    if (r < rank) lower += m;
  }
  // u of the sum, rounded down; u below 0 or no number counts as 0, 1 and above as the largest below 1
  const u64 f = u > 0.f ? (u < 1.f ? static_cast<u64>(static_cast<double>(u) * 18446744073709551616.0) : ~0ull) : 0ull;
  const u64 goal = __umul64hi(f, total);
  before += lower;
  if (tid == 0) S.at[0] = ~0ull;
  __syncthreads();
  if (before <= goal && goal < before + mine) {
    seen = same_before;
    for (int b = b0; b < b1; ++b) {
      const u64 left = equals > seen ? equals - seen : 0;
      const u64 in = block_mass[b] + min(left, static_cast<u64>(block_equal[b])) * each;
      if (goal < before + in) {
        S.at[0] = b;
        S.at[1] = goal - before;
        S.at[2] = left;
        break;
      }
      before += in;
      seen += block_equal[b];
    }
  }
  __syncthreads();
  if (warp == 0 && S.at[0] != ~0ull) {
    const int b = static_cast<int>(S.at[0]);
    const u64 to = S.at[1], left = S.at[2];
    const Eight<T> v = load(b);
    uint32_t mine_same = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) mine_same += Key<T>::of(v[e]) == cut;
    u64 rank_of = warp_before(mine_same), w[8], sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t key = Key<T>::of(v[e]);
      w[e] = 0;
      if (key > cut) {
        const double d = weigh(value<T>(v[e]));
        if (d >= least) w[e] = weigh.whole(d);
      } else if (key == cut && rank_of++ < left) {
        w[e] = each;
      }
      sum += w[e];
    }
    u64 run = warp_before(sum);
    if (run <= to && to < run + sum) {
      int found = 0;
#pragma unroll
      for (int e = 7; e >= 0; --e) {       // the first whose running sum passes
        u64 upto = run;
#pragma unroll
        for (int i = 0; i < 8; ++i) upto += i <= e ? w[i] : 0;
        if (upto > to) found = e;
      }
      A.out[row] = static_cast<int64_t>(block0 + b) * kBlock + lane * 8 + found - head;
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
    return sizeof(Shared) + ((per + 1) & ~size_t{1}) * 8 + ((per + 3) & ~size_t{3}) * 4 + (held ? per * kBlock * sizeof(T) : 0);
  };
  int ctas = 1;
  while (ctas < 8 && bytes(ctas, true) > kMaxSmem) ctas *= 2;
  const bool held = bytes(ctas, true) <= kMaxSmem;
  while (ctas < 8 && 2 * ctas * static_cast<int64_t>(rows) <= kNumSMs && blocks >= 16 * ctas) ctas *= 2;
  const size_t smem = bytes(ctas, held);
  if (smem > kMaxSmem) return fail(B200_ESHAPE, "%s: rows of %d", name, A.cols);
  A.blocks_per_cta = (blocks + ctas - 1) / ctas;
  int bits = 0;
  while ((1ll << bits) < A.cols) ++bits;
  A.frac = std::min(62 - bits, 50);
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
  if (rows < 0 || cols <= 0 || row_stride < cols) return fail(B200_EINVAL, "%s: bad sizes", name);
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
