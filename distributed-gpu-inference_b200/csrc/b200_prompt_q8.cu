// Causal attention of several tokens per sequence over a key/value cache in 8 bits, on the fifth-generation tensor cores: 16-bit types, heads of 64 or
// 128, pages of 16s.  Formula: b200_attn_q8.cu.
//
// The rows of a sequence and kv head - its new tokens times the G query heads of the group, token by token - go in blocks of 128; a CTA has RB of them and
// walks the keys up to its last row's in tiles of 64.
//
//   codes -> fp16   four warps, 16 codes of a key a thread and step: asked for a tile ahead, turned (exact) and stored in 128-byte swizzled lines, once for all
//                   RB x 128 rows
//   S = Q K^T       tcgen05.mma, 128 x 64, both operands in shared memory, S in tensor memory, two of them; queries in fp16 by a power of two of their own, the
//                   largest of a row between 2^14 and 2^15
//   w               a warp per 32 rows, thread = row: w = 2^(S t + log2 s - m) with the page's scales t and s, so that weights meet bare codes; the sum counts w / s; rounded to
//                   fp16 into the tensor memory S was in: by 2^-11 of a weight at most (half a step), down to 2^-20 of the largest.  One pass: m is the maximum so far less 6, the weights
//                   of a tile are made with it while the tile's own maximum is found, and made again where that lies more than 15 above m (the first tile's is looked for
//                   first); the largest weight lies between 2^6 and 2^15
//   O += w V        tcgen05.mma, w from tensor memory, O in tensor memory in fp32
//
// Few rows: the keys are divided among `splits` CTAs, whose parts prompt_merge_kernel puts together in their order.
//
// Bound, for many rows, by the latencies of a tile's steps: of a tile's 2000 clocks the warps that make weights are busy 1900 (the exponential unit 1000), those that turn codes 1800, the tensor
// cores and the shared memory that feeds them some 1300 (a tile of 64 keys reads Q once more for each, 6 KB in the 32 clocks in which 4 KB can be read).  32 heads over 8 of 128, on the
// device: one sequence of 8192 tokens 537 us, 1.02 PFLOP/s; 8 x 2048 361 us, 0.76 PFLOP/s: 6 us of a CTA's 26 go to its beginning and its output (queries are there after 3, the first
// weights after 6); 512 tokens behind 8k 93 us.  What did not pay: tiles of 128 keys with one S (1 x 8192 659 us when this took 583), one row block and two CTAs an SM (674), CTAs that stay
// and take one unit after another (8 x 2048 385, then the same), twice the warps for codes (362), two threads a row (384 - 401), S in smaller pieces (392, then 374).
// Up to 128 rows (one block, two CTAs an SM): by the latency of a tile's steps, one tile behind the other, and of its codes: 64 x 8 tokens of 4 heads behind 2k 100 us, where
// memory would allow 43; without reading codes a quarter less, without turning them or without weights the same.  Codes asked for two tiles ahead, or brought to the second level of
// the cache three tiles ahead, changed nothing; that warps without rows make no weights, 115 -> 104.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "b200_prompt_q8.cuh"
#include "b200_tcgen05.cuh"

namespace b200 {
namespace {

using q8::Cache;
using q8::Divisor;
using q8::PromptAttn;

constexpr int kRows = 128, kGroup = 16;
constexpr float kLog2e = 1.4426950408889634f;

template <int D, int RB>
struct Plan {
  static constexpr int kKeys = 64, kS = 2, kBufs = RB == 1 ? 2 : 3;       // keys of a tile; S in tensor memory for a row block; buffers of keys, and of values
  static constexpr int kGroups = kKeys / kGroup, kBlk = kKeys * 128;
  static constexpr int kSoft = 128 * RB, kConvert = 128, kThreads = kSoft + kConvert + 32;
  static constexpr int kQBlock = (D / 64) * kRows * 128, kTile = (D / 64) * kBlk;       // bytes
  static constexpr int kQ = 0, kK = kQ + RB * kQBlock, kV = kK + kBufs * kTile, kScales = kV + kBufs * kTile;       // scales: [warp][3][32] numbers
  static constexpr int kFactor = kScales + 4 * RB * 3 * 32 * 4, kBar = kFactor + RB * kRows * 4, kFlags = kBar + 8 * (4 * kBufs + RB * 7), kEnd = kFlags + 16;
  static constexpr int kSmem = kEnd + 1024;
  static constexpr int kO = kS * kKeys, kTm = 256;      // columns of a row block's tensor memory: S, two | O
  static_assert(RB == 2 ? kSmem <= kMaxSmem : 2 * (kSmem + 1024) <= 228 * 1024, "shared memory");
  static_assert(kO + D <= kTm, "tensor memory");
};

__device__ __forceinline__ uint32_t line(uint32_t base, int r, int ch, int rows) {     // 16-byte piece ch of row r: blocks of 64 columns, swizzled lines
  return base + (ch >> 3) * (rows * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void st16(uint32_t to, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {      // of two pairs of whole numbers
  asm("max.u16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}

// What a CTA works on
struct Work {
  int b, kvh, row0, split;       // sequence, kv head, first row, part of the keys
  int first, n, base, room;      // packed row of the sequence's first new token, new tokens, tokens before them, keys that the table holds
  int rows, t0, t1;              // of the sequence and head that are worked on; tiles
  // where a row's part of the result goes
  __device__ __forceinline__ int64_t part(const PromptAttn& A, int row) const {
    return ((static_cast<int64_t>(b) * A.c.Hkv + kvh) * A.max_rows + row) * A.splits + split;
  }
  // tiles up to those of the `count` rows from `from` on
  template <int KEYS>
  __device__ __forceinline__ int tiles(const PromptAttn& A, int from, int count) const {
    return from < rows ? (min(base + min(n, A.by_G.of(from + count - 1) + 1), room) + KEYS - 1) / KEYS : 0;
  }
};
template <int RB, int KEYS>
__device__ __forceinline__ Work work_of(const PromptAttn& A, int unit) {
  Work w;
  const int head = A.by_splits.of(unit), b = A.by_heads.of(head), block = A.by_B.of(b);
  w.split = unit - head * A.splits, w.kvh = head - b * A.c.Hkv, w.b = b - block * A.r.B;
  w.row0 = (A.blocks - 1 - block) * kRows * RB;       // the longest walks first
  int context;
  A.r.of(w.b, &w.first, &w.n, &context);
  w.base = context - w.n;
  w.room = A.c.keys(context);
  w.rows = min(w.n * A.G, A.max_rows);
  const int tiles = w.tiles<KEYS>(A, w.row0, kRows * RB), per = A.by_splits.of(tiles + A.splits - 1);
  w.t0 = min(w.split * per, tiles);
  w.t1 = min(w.t0 + per, tiles);
  return w;
}

template <typename T, typename C, int D, int RB>
__global__ void __launch_bounds__(Plan<D, RB>::kThreads, 3 - RB)
prompt_kernel(const PromptAttn A) {
  using P = Plan<D, RB>;
  constexpr int NB = P::kBufs, kKeys = P::kKeys, kGroups = P::kGroups, kBlk = P::kBlk;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* sm = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
  const uint32_t sm0 = smem_u32(sm);
  // keys of a buffer in, and read; values of a buffer in, and read; of a row block: queries in, S of a buffer done, w written, w V done
  const uint32_t bar_k = sm0 + P::kBar, bar_ke = bar_k + 8 * NB, bar_v = bar_ke + 8 * NB, bar_ve = bar_v + 8 * NB, bar_rb = bar_ve + 8 * NB;
  auto bar_q = [&](int rb) { return bar_rb + 56 * rb; };
  auto bar_s = [&](int rb, int i) { return bar_rb + 56 * rb + 8 + 8 * (i & 1); };
  auto bar_p = [&](int rb, int i) { return bar_rb + 56 * rb + 24 + 8 * (i & 1); };
  auto bar_o = [&](int rb, int i) { return bar_rb + 56 * rb + 40 + 8 * (i & 1); };
  volatile uint32_t* tm_slot = reinterpret_cast<volatile uint32_t*>(sm + P::kFlags);
  volatile int* dead = reinterpret_cast<volatile int*>(sm + P::kFlags + 4);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const Cache& c = A.c;
  const int G = A.G;

  asm volatile("griddepcontrol.launch_dependents;");
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm0 + P::kFlags), "n"(P::kTm * RB) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const Work w = work_of<RB, kKeys>(A, blockIdx.x);
  const int run = w.t1 - w.t0, rows = w.rows;
  const bool weighs = warp < P::kSoft / 32 && w.row0 + 32 * warp < rows;        // warps that have rows
  // Queries are read and outputs written by kCh lanes a row, kPer rows at a time: in step u a lane has row `y` + u kPer of the CTA.  Its token, from the CTA's first one: a
  // division costs 30 instructions; at most 4096 + 256 rows, the product is exact enough.
  constexpr int kCh = D / 8, kPer = 32 / kCh, kSteps = 32 / kPer;
  const int ch = lane % kCh, r = lane / kCh, y = 32 * warp + r, token0 = A.by_G.of(w.row0), head0 = w.row0 - token0 * G;
  const float per_head = 1.0f / static_cast<float>(G), y_f = static_cast<float>(head0 + y) + 0.5f;
  // rows of a token lie D apart, tokens `stride`
  auto place_of = [&](int u, int64_t stride) {
    const int token = __float_as_int(__fadd_rd((y_f + static_cast<float>(u * kPer)) * per_head, 0x1p23f)) - 0x4b000000;        // (rounded down: the sum's last digits)
    return token * (stride - static_cast<int64_t>(G) * D) + (y + u * kPer) * D;
  };
  auto first_place = [&](int64_t stride) { return (static_cast<int64_t>(w.first) + token0) * stride + static_cast<int64_t>(w.kvh * G + head0) * D + ch * 8; };
  int4 raw[kSteps];       // (asked for before the barriers stand)
  if (weighs && run > 0) {
    const T* q = static_cast<const T*>(A.q) + first_place(A.q_stride);
#pragma unroll
    for (int u = 0; u < kSteps; ++u) raw[u] = w.row0 + y + u * kPer < rows ? ld_stream16(q + place_of(u, A.q_stride)) : make_int4(0, 0, 0, 0);
  }
  if (tid == 32) {
    auto init = [](uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); };
    for (int b = 0; b < NB; ++b) {
      init(bar_k + 8 * b, P::kConvert);
      init(bar_ke + 8 * b, 1);
      init(bar_v + 8 * b, P::kConvert);
      init(bar_ve + 8 * b, 1);
    }
    for (int rb = 0; rb < RB; ++rb) {
      const int with_rows = max(1, min(128, (rows - w.row0 - rb * kRows + 31) & ~31));        // threads of warps that have rows
      init(bar_q(rb), with_rows);
      for (int i = 0; i < 2; ++i) {
        init(bar_s(rb, i), 1);
        init(bar_p(rb, i), with_rows);
        init(bar_o(rb, i), 1);
      }
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *dead = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = __shfl_sync(0xffffffffu, *tm_slot, 0);
  const int per_page = c.bs / kGroup;
  if (run == 0) {       // no keys, or no rows (the whole CTA): nothing but the statistics that say so
    for (int x = tid; x < kRows * RB; x += P::kThreads) {
      const int row = w.row0 + x;
      if (row < rows) A.ml[w.part(A, row)] = make_float2(-INFINITY, 0.f);
    }
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(P::kTm * RB));
    return;
  }

  if (warp >= P::kSoft / 32 && warp < (P::kSoft + P::kConvert) / 32) {
    // ---- codes to fp16 -----------------------------------------------------------------------------------------------------------------------
    constexpr int kCh = D / 16, kStep = P::kConvert / kCh, kPasses = kKeys / kStep;       // pieces of a key; keys of a pass
    const int me = tid - P::kSoft, ch = me % kCh, r = me / kCh;
    const int keys = min(w.room, w.base + w.n);
    // the pool's rows of 32 groups of 16 keys, a lane each, the next ones under way; -1: zeros
    auto look_up = [&](int group) -> int {
      if (group >= w.t1 * kGroups) return -1;
      const int place = A.by_page.of(group), page = c.page(w.b, place);
      return page < 0 ? -1 : (page * c.Hkv + w.kvh) * c.bs + (group - place * per_page) * kGroup;
    };
    const int g0 = w.t0 * kGroups;
    int at = look_up(g0 + lane), later = look_up(g0 + 32 + lane);
    int4 k[2][kPasses], v[2][kPasses];       // of a tile, and of the next one
    auto load = [&](int i, auto odd) {
      constexpr int kOdd = decltype(odd)::value;
      if (i > 0 && i % (32 / kGroups) == 0) {
        at = later;
        later = look_up(g0 + i * kGroups + 32 + lane);
      }
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int key = p * kStep + r, row = __shfl_sync(0xffffffffu, at, (i * kGroups + key / kGroup) & 31);
        const bool in = row >= 0 && (w.t0 + i) * kKeys + key < keys;
        const int64_t e = (static_cast<int64_t>(row) + key % kGroup) * D + ch * 16;
        k[kOdd][p] = in ? ld_stream16(c.k_pool + e) : make_int4(0, 0, 0, 0);
        v[kOdd][p] = in ? ld_stream16(c.v_pool + e) : make_int4(0, 0, 0, 0);
      }
    };
    auto store = [&](uint32_t to, const int4 (&x)[kPasses]) {
      const int odd = ch >> 2 & 1;       // pieces 2 ch and 2 ch + 1, the lanes of the second block in the other order: eight lanes, eight banks
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        uint32_t h[8];
        const uint32_t* e = reinterpret_cast<const uint32_t*>(&x[p]);
#pragma unroll
        for (int u = 0; u < 4; ++u) q8::halves<C, false>(e[u], h[2 * u], h[2 * u + 1]);
        const int key = p * kStep + r;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bool second = u != odd;
          st16(line(to, key, 2 * ch + second, kKeys), second ? h[4] : h[0], second ? h[5] : h[1], second ? h[6] : h[2], second ? h[7] : h[3]);
        }
      }
      fence_smem_to_mma();
    };
    load(0, std::integral_constant<int, 0>{});
    auto tile = [&](int i, auto odd) {       // (registers have no indexes: the parity is known to the compiler)
      constexpr int kOdd = decltype(odd)::value;
      const int buf = i % NB;
      if (i >= NB) bar_wait(bar_ke + 8 * buf, (i / NB - 1) & 1, dead);
      store(sm0 + P::kK + buf * P::kTile, k[kOdd]);
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_k + 8 * buf) : "memory");
      if (i >= NB) bar_wait(bar_ve + 8 * buf, (i / NB - 1) & 1, dead);
      store(sm0 + P::kV + buf * P::kTile, v[kOdd]);
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_v + 8 * buf) : "memory");
    };
    for (int i = 0; i < run; i += 2) {
      if (i + 1 < run) load(i + 1, std::integral_constant<int, 1>{});
      tile(i, std::integral_constant<int, 0>{});
      if (i + 2 < run) load(i + 2, std::integral_constant<int, 0>{});
      if (i + 1 < run) tile(i + 1, std::integral_constant<int, 1>{});
    }
  } else if (warp == P::kThreads / 32 - 1) {
    // ---- products ----------------------------------------------------------------------------------------------------------------------------
    int runs[RB];        // tiles of a row block: a part of the CTA's first ones
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) runs[rb] = max(min(w.tiles<kKeys>(A, w.row0 + rb * kRows, kRows), w.t1) - w.t0, 0);
    auto scores = [&](int i, int rb) {
      const uint32_t kk = sm0 + P::kK + (i % NB) * P::kTile, q = sm0 + P::kQ + rb * P::kQBlock, to = tm + rb * P::kTm + (i % P::kS) * kKeys;
      if (i >= P::kS) bar_wait(bar_o(rb, i - P::kS), ((i - P::kS) >> 1) & 1, dead);        // S goes where the weights of an earlier tile were read
      tc_fence_after();
#pragma unroll
      for (int u = 0; u < D / 16; ++u)
        mma_ss(to, operand(q + (u >> 2) * (kRows * 128) + (u & 3) * 32, 16, 1024), operand(kk + (u >> 2) * kBlk + (u & 3) * 32, 16, 1024), instr<__half>(kKeys, false), u > 0);
      mma_commit(bar_s(rb, i));
    };
    auto outputs = [&](int i, int rb) {
      const uint32_t v = sm0 + P::kV + (i % NB) * P::kTile, from = tm + rb * P::kTm;
      bar_wait(bar_p(rb, i), (i >> 1) & 1, dead);
      tc_fence_after();
#pragma unroll
      for (int u = 0; u < kKeys / 16; ++u)
        mma_ts(from + P::kO, from + (i % P::kS) * kKeys + 8 * u, operand(v + u * 2048, kBlk, 1024), instr<__half>(D, true), i > 0 || u > 0);
      mma_commit(bar_o(rb, i));
    };
    bar_wait(bar_k, 0, dead);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      if (runs[rb] == 0) continue;
      bar_wait(bar_q(rb), 0, dead);
      scores(0, rb);
    }
    mma_commit(bar_ke);
    for (int i = 0; i < run; ++i) {
      const bool more = i + 1 < run;
      if (more) bar_wait(bar_k + 8 * ((i + 1) % NB), ((i + 1) / NB) & 1, dead);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        if (i + 1 < runs[rb]) scores(i + 1, rb);
      if (more) mma_commit(bar_ke + 8 * ((i + 1) % NB));
      bar_wait(bar_v + 8 * (i % NB), (i / NB) & 1, dead);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        if (i < runs[rb]) outputs(i, rb);
      mma_commit(bar_ve + 8 * (i % NB));
    }
    __syncwarp();
  } else if (weighs) {
    // ---- weights: thread = row (of a warp without rows queries and weights are what memory held: rows of a product are apart) ----------------------
    const int rb = warp >> 2, in_block = tid & 127, row = w.row0 + tid;
    const int my_run = max(min(w.tiles<kKeys>(A, w.row0 + rb * kRows, kRows), w.t1) - w.t0, 0);
    const uint32_t q_at = sm0 + P::kQ + rb * P::kQBlock, tm_row = tm + rb * P::kTm + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    float* factor = reinterpret_cast<float*>(sm + P::kFactor);
    const float sign = A.scale < 0.f ? -1.f : 1.f;
    // scales of 32 groups of keys: the keys', log2 of the values', 1 / the values'; the next ones under way
    float* scales = reinterpret_cast<float*>(sm + P::kScales) + warp * 96;
    const int g0 = w.t0 * kGroups;
    auto page_of = [&](int group) { return group < w.t1 * kGroups ? c.page(w.b, A.by_page.of(group)) : -1; };
    auto scales_of = [&](int page, float& ks, float& vs) {
      ks = vs = q8::kAbsentScale;
      if (page >= 0) {
        ks = c.k_scale[static_cast<int64_t>(page) * c.Hkv + w.kvh];
        vs = q8::max_nan(c.v_scale[static_cast<int64_t>(page) * c.Hkv + w.kvh], q8::kLeastScale);
      }
    };
    int page = page_of(g0 + lane);
    float ks, vs;
    {
      scales_of(page, ks, vs);        // (under way beside the queries)
      page = page_of(g0 + 32 + lane);
      // the rows' largest, two rows a register: magnitudes order like whole numbers
      uint32_t most[kSteps / 2];
#pragma unroll
      for (int u = 0; u < kSteps; u += 2) {
        uint32_t two[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t* e = reinterpret_cast<const uint32_t*>(&raw[u + x]);
          two[x] = larger(larger(e[0] & 0x7fff7fffu, e[1] & 0x7fff7fffu), larger(e[2] & 0x7fff7fffu, e[3] & 0x7fff7fffu));
        }
        most[u / 2] = larger(__byte_perm(two[0], two[1], 0x5410), __byte_perm(two[0], two[1], 0x7632));
      }
#pragma unroll
      for (int o = kCh / 2; o > 0; o >>= 1) {
#pragma unroll
        for (int u = 0; u < kSteps / 2; ++u) most[u] = larger(most[u], __shfl_xor_sync(0xffffffffu, most[u], o));
      }
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const T* e = reinterpret_cast<const T*>(&raw[u]);
        const T row_most = reinterpret_cast<const T*>(&most[u / 2])[u & 1];
        const int p = max(static_cast<int>(__float_as_uint(Cvt<T>::to_f32(row_most)) >> 23) - 127, -100) - 14;       // the largest = 2^(p + 14) .. 2^(p + 15)
        const float down = __uint_as_float(static_cast<uint32_t>(127 - p) << 23) * sign;
        const int my = u * kPer + r;
        st16(line(q_at, 32 * (warp & 3) + my, ch, kRows), pack2<__half>(Cvt<T>::to_f32(e[0]) * down, Cvt<T>::to_f32(e[1]) * down),
             pack2<__half>(Cvt<T>::to_f32(e[2]) * down, Cvt<T>::to_f32(e[3]) * down), pack2<__half>(Cvt<T>::to_f32(e[4]) * down, Cvt<T>::to_f32(e[5]) * down),
             pack2<__half>(Cvt<T>::to_f32(e[6]) * down, Cvt<T>::to_f32(e[7]) * down));
        if (ch == 0) factor[32 * warp + my] = fabsf(A.scale) * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + p) << 23);
      }
      fence_smem_to_mma();
      tc_fence_before();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_q(rb)) : "memory");
      __syncwarp();
    }
    const float f = factor[tid];
    const int token = A.by_G.of(row), see = min(w.base + min(token, w.n - 1) + 1, w.room);       // keys that the row sees
    const int see_all = __shfl_sync(0xffffffffu, see, 0);                                 // the warp's rows see these
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < my_run; ++i) {
      const int in = i % (32 / kGroups);
      if (in == 0) {
        __syncwarp();
        const float lv = log2f(vs);
        scales[lane] = ks, scales[32 + lane] = lv, scales[64 + lane] = exp2_fast(-lv);
        __syncwarp();
        scales_of(page, ks, vs);
        page = page_of(g0 + i * kGroups + 64 + lane);
      }
      ok = bar_wait(bar_s(rb, i), (i >> 1) & 1, dead) && ok;
      tc_fence_after();
      const uint32_t s_at = tm_row + (i % P::kS) * kKeys;
      const int left = see - (w.t0 + i) * kKeys;       // keys of the tile that the row sees
      uint32_t p[kKeys / 2];
      float top, sum;
      // 32 keys at a time: their maximum, and (kWeigh) their weights.  kMasked: some rows of the warp do not see all of the tile, whatever the scales of a page that
      // they do not see
      auto pass = [&](auto masked, auto weigh) {
        constexpr bool kMasked = decltype(masked)::value, kWeigh = decltype(weigh)::value;
        const float from = m == -INFINITY ? 0.f : m;       // a row that sees no key yet: weights 0
        top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int y = 0; y < kKeys / 32; ++y) {
          float s[32];
          tm_ld32(s, s_at + 32 * y);
          const float2 kt = *reinterpret_cast<const float2*>(scales + in * kGroups + 2 * y), lv = *reinterpret_cast<const float2*>(scales + 32 + in * kGroups + 2 * y),
                       iv = *reinterpret_cast<const float2*>(scales + 64 + in * kGroups + 2 * y);
          const float kg[2] = {q8::max_nan(f * kt.x, 1e-30f), q8::max_nan(f * kt.y, 1e-30f)}, ls[2] = {lv.x, lv.y}, per[2] = {iv.x, iv.y};
          tc_wait_ld();
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            float* e = s + g * kGroup;
            const int here = left - 32 * y - g * kGroup;       // keys of the group that the row sees
            if constexpr (kMasked) {
#pragma unroll
              for (int x = 0; x < kGroup; ++x)
                if (x >= here) e[x] = -INFINITY;
            }
            float a = max3(e[0], e[1], e[2]), b = max3(e[3], e[4], e[5]);
            a = max3(a, e[6], e[7]), b = max3(b, e[8], e[9]);
            a = max3(a, e[10], e[11]), b = max3(b, e[12], e[13]);
            a = max3(a, e[14], e[15]);
            top = fmaxf(top, fmaf(fmaxf(a, b), kg[g], ls[g]));
            if constexpr (kWeigh) {
              const f32x2 kk = both(kg[g]), mm = both(ls[g] - from);
              f32x2 two = 0ull;
#pragma unroll
              for (int x = 0; x < kGroup; x += 2) {
                float u = e[x], v = e[x + 1];
                scale_shift(u, v, kk, mm);
                u = exp2_fast(u), v = exp2_fast(v);
                if constexpr (kMasked) {
                  if (x >= here) u = 0.f;
                  if (x + 1 >= here) v = 0.f;
                }
                two = add2(two, pair(u, v));
                p[16 * y + 8 * g + (x >> 1)] = pack2<__half>(u, v);
              }
              apart(a, b, two);
              if (!kMasked || here > 0) sum = fmaf(a + b, per[g], sum);
            }
          }
        }
      };
      auto walk = [&](auto masked) {
        if (i == 0) pass(masked, std::false_type{});
        else pass(masked, std::true_type{});
        const bool grow = top > m + 15.f;
        if (i == 0 || __any_sync(0xffffffffu, grow)) {
          float corr = 1.f;
          if (grow) {
            const float now = top - 6.f;
            corr = m == -INFINITY ? 0.f : exp2_fast(m - now);
            m = now;
          }
          if (i > 0) {
            ok = bar_wait(bar_o(rb, i - 1), ((i - 1) >> 1) & 1, dead) && ok;
            tc_fence_after();
            scale_rows<D, 16>(tm_row + P::kO, corr);
          }
          l *= corr;
          pass(masked, std::true_type{});
        }
      };
      if (see_all < (w.t0 + i + 1) * kKeys) walk(std::true_type{});
      else walk(std::false_type{});
      l += sum;
#pragma unroll
      for (int y = 0; y < kKeys / 32; ++y) tm_st16(s_at + 16 * y, *reinterpret_cast<uint32_t(*)[16]>(p + 16 * y));
      tc_wait_st();
      tc_fence_before();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_p(rb, i)) : "memory");
    }
    if (my_run > 0) ok = bar_wait(bar_o(rb, my_run - 1), ((my_run - 1) >> 1) & 1, dead) && ok;
    tc_fence_after();
    ok = ok && !*dead;
    if (!ok) l = NAN;
    if (A.splits > 1) {
      const int64_t part = w.part(A, row);
      if (row < rows) A.ml[part] = make_float2(m, l);
#pragma unroll 1
      for (int x = 0; x < D && my_run > 0; x += 32) {
        float o[32];
        tm_ld32(o, tm_row + P::kO + x);
        tc_wait_ld();
        if (row < rows) {
#pragma unroll
          for (int u = 0; u < 32; u += 4) *reinterpret_cast<float4*>(A.acc + part * D + x + u) = make_float4(o[u], o[u + 1], o[u + 2], o[u + 3]);
        }
      }
    } else {
      // by way of where the warp's queries were (every product that reads them is done), rows side by side
      const float k = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int x = 0; x < D; x += 32) {
        float o[32];
        tm_ld32(o, tm_row + P::kO + x);
        tc_wait_ld();
#pragma unroll
        for (int u = 0; u < 32; u += 8)
          st16(line(q_at, in_block, (x + u) / 8, kRows), pack2<T>(o[u] * k, o[u + 1] * k), pack2<T>(o[u + 2] * k, o[u + 3] * k), pack2<T>(o[u + 4] * k, o[u + 5] * k),
               pack2<T>(o[u + 6] * k, o[u + 7] * k));
      }
      __syncwarp();
      T* out = static_cast<T*>(A.out) + first_place(static_cast<int64_t>(A.Hq) * D);
#pragma unroll 8
      for (int u = 0; u < kSteps; ++u) {
        if (w.row0 + y + u * kPer < rows) {
          uint4 x;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(line(q_at, 32 * (warp & 3) + r + u * kPer, ch, kRows)) : "memory");
          *reinterpret_cast<uint4*>(out + place_of(u, static_cast<int64_t>(A.Hq) * D)) = x;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*dead) {      // a wait gave up: what is still under way gets 10 ms to end before its memory is another's
    for (const long long begun = clock64(); clock64() - begun < 20000000ll;) {}
  }
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(P::kTm * RB));
}

// A warp per row: the parts of its keys, in their order
template <typename T, int D>
__global__ void __launch_bounds__(256) prompt_merge_kernel(const PromptAttn A) {
  const int lane = threadIdx.x & 31, per_unit = (A.max_rows + 7) / 8, unit = blockIdx.x / per_unit, kvh = unit % A.c.Hkv, b = unit / A.c.Hkv;
  const int row = (blockIdx.x - unit * per_unit) * 8 + (threadIdx.x >> 5);
  int first, n, context;
  A.r.of(b, &first, &n, &context);
  const bool live = row < n * A.G && row < A.max_rows;
  const int64_t out_row = (static_cast<int64_t>(first) + row / A.G) * A.Hq + kvh * A.G + row % A.G, parts = (static_cast<int64_t>(unit) * A.max_rows + row) * A.splits;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!live) return;
  const float2* ml = A.ml + parts;
  float top = -INFINITY, sum = 0.f, o[D / 32] = {};
  for (int s = lane; s < A.splits; s += 32) top = fmaxf(top, ml[s].x);
  top = warp_max(top);
#pragma unroll 4
  for (int s = 0; s < A.splits; ++s) {
    const float2 one = ml[s];
    if (one.x == -INFINITY && one.y == one.y) continue;
    const float k = one.x == -INFINITY ? 1.f : exp2_fast(one.x - top);
    sum = fmaf(one.y, k, sum);
    const float* acc = A.acc + (parts + s) * D;
#pragma unroll
    for (int u = 0; u < D / 32; ++u) o[u] = fmaf(acc[u * 32 + lane], k, o[u]);
  }
  const float k = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int u = 0; u < D / 32; ++u) static_cast<T*>(A.out)[out_row * D + u * 32 + lane] = Cvt<T>::from_f32(o[u] * k);
}

// How a call is cut
struct Cut {
  int row_blocks, blocks, splits;      // of a CTA; CTAs of a sequence and kv head; parts of the keys
  // The workspace: statistics of [sequence][kv head][row][part], then outputs of the same.  The statistics' number is brought to an even one: outputs are stored 16 bytes at once
  size_t statistics(int B, int Hkv, int64_t max_rows) const { return (static_cast<size_t>(B) * Hkv * max_rows * splits + 1) / 2 * 2; }
  size_t bytes(int B, int Hkv, int64_t max_rows, int D) const {
    return splits == 1 ? 0 : statistics(B, Hkv, max_rows) * sizeof(float2) + static_cast<size_t>(B) * Hkv * max_rows * splits * D * sizeof(float);
  }
};
Cut cut_of(int B, int max_new, int Hq, int Hkv, int longest) {
  const int64_t rows = static_cast<int64_t>(max_new) * (Hq / Hkv);
  Cut x;
  x.row_blocks = rows > kRows ? 2 : 1;
  x.blocks = static_cast<int>((rows + kRows * x.row_blocks - 1) / (kRows * x.row_blocks));
  const int64_t units = static_cast<int64_t>(B) * Hkv * std::max(x.blocks, 1), slots = kNumSMs * (x.row_blocks == 1 ? 2 : 1), tiles = (longest + 63ll) / 64;
  int64_t splits = units >= slots ? 1 : slots / units;
  splits = std::min(splits, std::max<int64_t>(tiles / 4, 1));
  x.splits = static_cast<int>(std::max<int64_t>(splits, 1));
  return x;
}

bool serves(int Hq, int Hkv, int D, int bs, int dtype) { return dtype != B200_DTYPE_F32 && (D == 64 || D == 128) && bs % kGroup == 0 && Hq / Hkv <= 1 << 12; }

template <typename T, typename C, int D, int RB>
int launch_as(const char* name, const PromptAttn& A, unsigned grid, cudaStream_t stream) {
  auto kern = prompt_kernel<T, C, D, RB>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Plan<D, RB>::kSmem);
  kern<<<grid, Plan<D, RB>::kThreads, Plan<D, RB>::kSmem, stream>>>(A);
  if (int rc = check_launch(name)) return rc;
  return A.splits == 1 ? 0 : launch_behind(name, prompt_merge_kernel<T, D>, static_cast<unsigned>((A.max_rows + 7) / 8 * A.r.B * A.c.Hkv), 256, 0, stream, A);
}

}  // namespace

size_t prompt_q8_workspace(int B, int max_new, int Hq, int Hkv, int D, int bs, int longest, int dtype) {
  if (B <= 0 || max_new <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || bs <= 0 || longest < 0 || !serves(Hq, Hkv, D, bs, dtype)) return 0;
  return cut_of(B, max_new, Hq, Hkv, longest).bytes(B, Hkv, static_cast<int64_t>(max_new) * (Hq / Hkv), D);
}

bool prompt_q8_serves(const PromptAttn& A, int max_new, int longest, int dtype) {
  if (!serves(A.Hq, A.c.Hkv, A.c.D, A.c.bs, dtype) || max_new <= 0) return false;
  if (!aligned16(A.c.k_pool) || !aligned16(A.c.v_pool) || !aligned16(A.q) || !aligned16(A.out) || A.q_stride % 8) return false;
  const Cut x = cut_of(A.r.B, max_new, A.Hq, A.c.Hkv, longest);
  return (A.c.max_blocks + 1) * A.c.Hkv * A.c.bs < INT32_MAX && static_cast<int64_t>(max_new) * A.Hq < INT32_MAX / 2 && static_cast<int64_t>(A.r.n) * A.Hq < INT32_MAX &&
         static_cast<int64_t>(A.r.B) * A.c.Hkv * x.blocks * x.splits < INT32_MAX && static_cast<int64_t>(A.r.B) * A.c.Hkv * (static_cast<int64_t>(max_new) * (A.Hq / A.c.Hkv) / 8 + 1) < INT32_MAX;
}

int prompt_q8(const char* name, PromptAttn A, int max_new, int longest, void* workspace, int codes, int dtype, cudaStream_t stream) {
  const Cut x = cut_of(A.r.B, max_new, A.Hq, A.c.Hkv, longest);
  A.G = A.Hq / A.c.Hkv, A.blocks = x.blocks, A.splits = x.splits, A.max_rows = max_new * A.G;
  A.by_G = Divisor::by(A.G), A.by_splits = Divisor::by(A.splits), A.by_heads = Divisor::by(A.c.Hkv), A.by_B = Divisor::by(A.r.B), A.by_page = Divisor::by(A.c.bs / kGroup);
  A.ml = static_cast<float2*>(workspace);
  A.acc = reinterpret_cast<float*>(A.ml + x.statistics(A.r.B, A.c.Hkv, A.max_rows));
  const unsigned grid = static_cast<unsigned>(A.r.B * A.c.Hkv * x.blocks * x.splits);
  auto go = [&](auto* t, auto* c, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    using C = std::remove_pointer_t<decltype(c)>;
    return x.row_blocks == 2 ? launch_as<T, C, d.value, 2>(name, A, grid, stream) : launch_as<T, C, d.value, 1>(name, A, grid, stream);
  };
  auto with_d = [&](auto* t, auto* c) { return A.c.D == 128 ? go(t, c, std::integral_constant<int, 128>{}) : go(t, c, std::integral_constant<int, 64>{}); };
  auto with_c = [&](auto* t) { return codes == B200_CODES_INT8 ? with_d(t, static_cast<q8::Int8*>(nullptr)) : with_d(t, static_cast<q8::E4m3*>(nullptr)); };
  return dtype == B200_DTYPE_BF16 ? with_c(static_cast<__nv_bfloat16*>(nullptr)) : with_c(static_cast<__half*>(nullptr));
}

}  // namespace b200
