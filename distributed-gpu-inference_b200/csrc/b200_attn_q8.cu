// Attention over a key/value cache in 8 bits: one token per sequence, and several.
//
//   out[i, h] = sum_j w_j c_j s_j / sum_j w_j,   w_j = exp(q[i, h] k_j t_j scale - max),   j up to the token's own position
//
// c, s codes and scales of the values, k, t of the keys.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "b200_prompt_q8.cuh"
#include "b200_q8.cuh"
#include "b200_tcgen05.cuh"

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

// ---- one token per sequence: 16-bit types, heads of 64 or 128, pages of 16s ---------------------------------------------------------------------
// A CTA of four warps per (part of the keys, kv head and up to 8 of its query heads, sequence); a warp takes every fourth tile of 16 tokens and keeps kStages of them
// under way, a TMA copy of 16 x D codes for the keys and one for the values each, in 128-byte lines whose 16-byte pieces are swizzled.  (Many short items: a warp
// per item, which then waits for nobody.)
//
//   S^T[token, head] = K Q^T   mma.m16n8k16, the codes as fp16: exact, for both kinds.  Queries in fp16 too, by a power of two of their own brought to 2^14 .. 2^15
//                              at the largest, so that what fp16 loses lies 2^-38 below it; the 8-wide side holds the heads, nothing is padded.  (int8 products of the
//                              codes as they are with queries in two digits of 8 bits, 80 instructions a tile fewer, took the same time.)
//   w = 2^(S t + log2 s - m)   t the page's key scale with all else, s its value scale: the weights carry it, so that they meet bare codes; the sum counts w / s.
//                              m moves when a score is 2^8 above it; the largest weight lies between 2^6 and 2^14, and rounding to fp16 is by 2^-11 of
//                              a weight at most (half a step), for weights down to 2^-20 of the largest; the sum is of the weights before they are rounded
//   O^T[d, head] += V^T w^T    the values by ldmatrix.trans, whose pairs of bytes are two tokens' codes of neighbouring columns
//
// The order of columns inside a product is free as long as both sides agree: a lane's 4 bytes of a key's 16 are its 4 columns there, and its rows of the
// output are two neighbouring columns.  A byte becomes fp16 as the low byte of 1024 + code + 128 (int8) or by the conversion that the hardware has (e4m3).
//
// Bound by memory and its latency: four CTAs an SM (shared memory and registers) keep up to 192 KB under way.  32 heads over 8 of 128, int8, on the device: 64 x 2048 51 us (0.82 of
// a copy's rate, 512 CTAs on 592 places, SMs are not served alike), 64 x 8192 174 (0.95), 8 x 32768 of 64 heads, e4m3, ragged 74 (0.83); one sequence of 160 tokens 4.9.
// What did not pay: tiles of 32 tokens and three CTAs an SM (64 x 2048 70), a CTA for each place with equal shares of all tokens (59, and more in most other calls).
constexpr int kWarps = 4, kTok = 16;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A warp's unit of work is kTiles tiles, one barrier for their copies.
template <int D>
struct DecodePlan {
  static constexpr int kTiles = 128 / D, kStages = 3, kTile = kTok * D, kStage = 2 * kTiles * kTile;       // bytes: keys of the tiles, then their values
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kBars = kRing, kDead = kBars + kWarps * kStages * 8, kEnd = kDead + 16;
  static constexpr int kSmem = kEnd + 1024;
  static_assert(kWarps * 16 * (D + 2) * 4 <= kRing, "outputs go where the tiles were");
  static_assert(4 * (kSmem + 1024) <= 228 * 1024, "shared memory");
};
// byte of (token, 16-byte piece) in a tile: lines of 128 bytes, a token each or two
template <int D>
__device__ __forceinline__ uint32_t tile_at(int token, int piece) {
  const int line = D == 128 ? token : token >> 1, p = D == 128 ? piece : (token & 1) * 4 + piece;
  return line * 128 + ((p ^ (line & 7)) << 4);
}

// A sequence, kv head and block of up to 8 of its query heads is an item.  The tokens of an item are divided among `splits` CTAs in equal parts (of kLeastPart
// at least, the last ones may have none), which leave maximum, sum and output in the workspace for decode_merge_kernel.
struct Decode {
  Attn a;
  int G, max_rows, blocks;        // query heads of a kv head; rows of a sequence and kv head at most, blocks of up to 8 NB of them
  int items, splits;
  float2* ml;                     // [item][part][row of the block]: maximum (of scores in powers of two), sum
  float* o;                       // [item][part][row of the block][D]
};
// The rows of an item: a single token's query heads, or several tokens' one after another
struct Item {
  int block, kvh, b;
  int first, base, rows, keys;    // packed row of the first token, tokens before it, rows of the sequence and kv head, keys that the block's rows see
  template <int MOST>
  __device__ __forceinline__ static Item of(const Decode& P, int item) {
    Item x;
    x.block = item % P.blocks, x.kvh = item / P.blocks % P.a.c.Hkv, x.b = item / P.blocks / P.a.c.Hkv;
    int n, context;
    P.a.r.of(x.b, &x.first, &n, &context);
    x.keys = P.a.c.keys(context);
    if (!P.a.r.starts) {       // (a sequence without keys has a row all the same: 0)
      x.base = context - 1, x.rows = P.G;
      return x;
    }
    x.base = context - n, x.rows = min(n * P.G, P.max_rows);
    x.keys = x.block * MOST < x.rows ? min(x.keys, x.base + min(n, (x.block * MOST + MOST - 1) / P.G + 1)) : 0;
    return x;
  }
  // element of queries or outputs, rows `stride` apart
  __device__ __forceinline__ int64_t at(const Decode& P, int row, int64_t stride) const {
    const int token = P.a.r.starts ? row / P.G : 0;
    return (static_cast<int64_t>(first) + token) * stride + static_cast<int64_t>(kvh * P.G + row - token * P.G) * P.a.c.D;
  }
};
constexpr int kLeastPart = 256;      // tokens

// tokens of a part of a sequence's: 32s for each of the four warps
__device__ __forceinline__ int part_of(int keys, int splits) {
  constexpr int kOf = 32 * kWarps;
  return splits == 1 ? keys : max((keys + splits - 1) / splits + kOf - 1 - ((keys + splits - 1) / splits + kOf - 1) % kOf, kLeastPart);
}

// NB blocks of 8 rows meet a tile, which is turned to fp16 once for them.  CAUSAL: several tokens, each sees the keys up to its own.
template <typename T, typename C, int D, int NB, bool CAUSAL, bool WARPITEM>
__global__ void __launch_bounds__(kWarps * 32, NB == 1 ? 4 : 3)
decode_kernel(const Decode P, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using S = DecodePlan<D>;
  constexpr int kStages = S::kStages, kTiles = S::kTiles, kUnit = kTiles * kTok, kPieces = D / 16, kStep = WARPITEM ? 1 : kWarps;
  const Cache& c = P.a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, tq = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;");
  const int unit = WARPITEM ? blockIdx.x * kWarps + warp : blockIdx.x, ofs = WARPITEM ? 0 : warp;
  if (WARPITEM && unit >= P.items) return;
  constexpr int kMost = 8 * NB;
  const int split = WARPITEM ? 0 : unit % P.splits, item = WARPITEM ? unit : unit / P.splits;
  const Item it = Item::of<kMost>(P, item);
  const int b = it.b, kvh = it.kvh, keys = it.keys, row0 = it.block * kMost, rows = min(kMost, it.rows - row0);
  if (CAUSAL && rows <= 0) return;
  const int part = WARPITEM ? keys : part_of(keys, P.splits), first = split * part, run = first < keys ? (min(part, keys - first) + kUnit - 1) / kUnit : 0, u0 = first / kUnit;
  const int mine = run > ofs ? (run - ofs + kStep - 1) / kStep : 0;       // units u0 + ofs, and every kStep-th

  extern __shared__ unsigned char raw_smem[];
  unsigned char* sm = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
  const uint32_t ring = smem_u32(sm) + warp * kStages * S::kStage, bars = smem_u32(sm + S::kBars) + warp * kStages * 8;
  volatile int* dead = reinterpret_cast<volatile int*>(sm + S::kDead) + (WARPITEM ? warp : 0);
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + s * 8));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (WARPITEM || warp == 0) *dead = 0;
  }
  if constexpr (WARPITEM) __syncwarp();
  else __syncthreads();
  const int per_page = c.bs / kTok, my_token = (lane >> 3 & 1) * 8 + (lane & 7), my_piece = lane >> 4;       // of four 8 x 8 matrices: tokens 0 - 7, 8 - 15, the next piece's
  uint32_t at[kPieces / 2];
#pragma unroll
  for (int p = 0; p < kPieces; p += 2) at[p / 2] = tile_at<D>(my_token, p + my_piece);
  // Pages of 32 units at a time, a lane each, and their scales: the next ones under way while these are used
  auto place_of = [&](int j, int h) -> int {        // page and head of the unit's tile h; -1: none, or outside the pool
    const int tile = kTiles * (u0 + ofs + j * kStep) + h;
    if (j >= mine || tile * kTok >= keys) return -1;
    const int p = c.page(b, tile / per_page);
    return p < 0 ? -1 : p * c.Hkv + kvh;
  };
  auto line_of = [&](int place, int j, int h) -> int {        // where copies begin: behind the pool they bring zeros
    const int tile = kTiles * (u0 + ofs + j * kStep) + h;
    return (place < 0 ? static_cast<int>(c.max_blocks) * c.Hkv * c.bs : place * c.bs + tile % per_page * kTok) / (128 / D);
  };
  auto scale_of = [&](const float* scales, int place) { return place < 0 ? q8::kAbsentScale : scales[place]; };
  int place[kTiles], lines[kTiles];
  float ks[kTiles], vs[kTiles], ks_next[kTiles], vs_next[kTiles];
#pragma unroll
  for (int h = 0; h < kTiles; ++h) place[h] = place_of(lane, h);
#pragma unroll
  for (int h = 0; h < kTiles; ++h) lines[h] = line_of(place[h], lane, h);
  auto issue = [&](int j, int buf) {
    int from[kTiles];
#pragma unroll
    for (int h = 0; h < kTiles; ++h) from[h] = __shfl_sync(0xffffffffu, lines[h], j & 31);
    if (lane == 0) {
      const uint32_t to = ring + buf * S::kStage, bar = bars + buf * 8;
      auto copy = [&](uint32_t at, const CUtensorMap* map, int line) {
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(at), "l"(map), "r"(0), "r"(line), "r"(bar) : "memory");
      };
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(S::kStage) : "memory");
#pragma unroll
      for (int h = 0; h < kTiles; ++h) {
        copy(to + h * S::kTile, &k_map, from[h]);
        copy(to + (kTiles + h) * S::kTile, &v_map, from[h]);
      }
    }
  };
  const int ahead = min(kStages, mine);
  for (int j = 0; j < ahead; ++j) issue(j, j);
#pragma unroll
  for (int h = 0; h < kTiles; ++h) {
    ks[h] = scale_of(c.k_scale, place[h]), vs[h] = scale_of(c.v_scale, place[h]);
    place[h] = place_of(32 + lane, h);
  }

  // queries: head quad's columns 16 i + 4 tq .. + 3
  uint32_t qf[NB][kPieces][2];
  float factor[NB][2];        // of rows 2 tq and 2 tq + 1 of a block of 8
  int see[NB][2];             // keys that they see
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const bool in = 8 * nb + quad < rows;
    const T* q = static_cast<const T*>(P.a.q) + (in ? it.at(P, row0 + 8 * nb + quad, P.a.q_stride) : 0) + 4 * tq;
    uint2 raw[kPieces];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) raw[i] = in ? *reinterpret_cast<const uint2*>(q + 16 * i) : make_uint2(0u, 0u);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
      for (int u = 0; u < 4; ++u) most = q8::max_nan(most, fabsf(Cvt<T>::to_f32(e[u])));
    }
    most = q8::max_nan(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = q8::max_nan(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100) - 14;       // most = 2^(e + 14) .. 2^(e + 15)
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23), f = P.a.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const T* x = reinterpret_cast<const T*>(&raw[i]);
      qf[nb][i][0] = pack2<__half>(Cvt<T>::to_f32(x[0]) * down, Cvt<T>::to_f32(x[1]) * down);
      qf[nb][i][1] = pack2<__half>(Cvt<T>::to_f32(x[2]) * down, Cvt<T>::to_f32(x[3]) * down);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      factor[nb][h] = __shfl_sync(0xffffffffu, f, 8 * tq + 4 * h);
      see[nb][h] = CAUSAL ? min(it.base + min(row0 + 8 * nb + 2 * tq + h, it.rows - 1) / P.G + 1, keys) : keys;
    }
  }
#pragma unroll
  for (int h = 0; h < kTiles; ++h) vs[h] = log2f(q8::max_nan(vs[h], q8::kLeastScale));

  float m[NB][2], l[NB][2], o[NB][kPieces][4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb][0] = m[nb][1] = -INFINITY, l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) o[nb][i][0] = o[nb][i][1] = o[nb][i][2] = o[nb][i][3] = 0.f;
  }
  bool ok = true;
  int buf = 0, left = keys - kUnit * (u0 + ofs);        // tokens from the unit's first on
  uint32_t parity = 0;
#pragma unroll 1
  for (int i = 0; i < mine; ++i, left -= kUnit * kStep) {
    if ((i & 31) == 0 && i > 0) {
#pragma unroll
      for (int h = 0; h < kTiles; ++h) ks[h] = ks_next[h], vs[h] = log2f(q8::max_nan(vs_next[h], q8::kLeastScale));
    }
    const uint32_t tiles = ring + buf * S::kStage;
    ok = __all_sync(0xffffffffu, bar_wait1(bars + buf * 8, parity, dead));
    if (!ok) break;
    float x[kTiles][NB][4], ls[kTiles];
#pragma unroll
    for (int h = 0; h < kTiles; ++h) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) x[h][nb][0] = x[h][nb][1] = x[h][nb][2] = x[h][nb][3] = 0.f;
#pragma unroll
      for (int p = 0; p < kPieces; p += 2) {
        uint32_t r[4];
        ldsm4(r, tiles + h * S::kTile + at[p / 2]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t a0, a1, a2, a3;
          q8::halves<C, false>(r[2 * u], a0, a2);
          q8::halves<C, false>(r[2 * u + 1], a1, a3);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma16(x[h][nb], a0, a1, a2, a3, qf[nb][p + u][0], qf[nb][p + u][1]);
        }
      }
      // [0], [1]: token quad, rows 2 tq and 2 tq + 1; [2], [3]: token quad + 8
      const float kt = __shfl_sync(0xffffffffu, ks[h], i & 31);
      ls[h] = __shfl_sync(0xffffffffu, vs[h], i & 31);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float f0 = factor[nb][0] * kt, f1 = factor[nb][1] * kt;
        float* s = x[h][nb];
        s[0] = fmaf(s[0], f0, ls[h]), s[1] = fmaf(s[1], f1, ls[h]), s[2] = fmaf(s[2], f0, ls[h]), s[3] = fmaf(s[3], f1, ls[h]);
      }
    }
    // of several tokens, the first one's last key (which may lie behind what the table holds)
    const bool masked = left < kUnit || (CAUSAL && keys - left + kUnit > it.base + 1);
    if (masked) {
#pragma unroll
      for (int h = 0; h < kTiles; ++h) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (h * kTok + quad + 8 * (e >> 1) >= left - keys + see[nb][e & 1]) x[h][nb][e] = -INFINITY;
        }
      }
      if constexpr (std::is_same_v<C, q8::E4m3>) {       // what is behind the last token may be no number
        for (int e = max(left, 0) * kPieces + lane; e < kUnit * kPieces; e += 32) {
          const int token = e / kPieces;
          asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(tiles + (kTiles + token / kTok) * S::kTile + tile_at<D>(token % kTok, e % kPieces)), "r"(0) : "memory");
        }
        __syncwarp();
      }
    }
    bool grow = false;
    float top[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float a = fmaxf(x[0][nb][y], x[0][nb][y + 2]);
#pragma unroll
        for (int h = 1; h < kTiles; ++h) a = fmaxf(a, fmaxf(x[h][nb][y], x[h][nb][y + 2]));
        top[nb][y] = a;
        grow = grow || a > m[nb][y] + 14.f;
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float a = top[nb][h];
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 4));
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 8));
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 16));
          const float now = fmaxf(m[nb][h], a - 6.f), corr = m[nb][h] == -INFINITY ? 0.f : exp2_fast(m[nb][h] - now);
          m[nb][h] = now;
          l[nb][h] *= corr;
#pragma unroll
          for (int p = 0; p < kPieces; ++p) o[nb][p][h] *= corr, o[nb][p][h + 2] *= corr;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < kTiles; ++h) {
      const float per = exp2_fast(-ls[h]);
      uint32_t w01[NB], w23[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = exp2_fast(x[h][nb][e] - (m[nb][e & 1] == -INFINITY ? 0.f : m[nb][e & 1]));      // (a row that sees no key yet, or scores below all numbers: 0)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float sum = w[y] + w[y + 2];
          l[nb][y] = fmaf(sum, CAUSAL && sum == 0.f ? 0.f : per, l[nb][y]);        // (whatever the scale of a page that a row does not see)
        }
        w01[nb] = transposed(pack2<__half>(w[0], w[1])), w23[nb] = transposed(pack2<__half>(w[2], w[3]));
      }
#pragma unroll
      for (int p = 0; p < kPieces; p += 2) {
        uint32_t r[4];
        ldsm4_trans(r, tiles + (kTiles + h) * S::kTile + at[p / 2]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t a0, a1, a2, a3;
          q8::halves<C, true>(r[2 * u], a0, a1);
          q8::halves<C, true>(r[2 * u + 1], a2, a3);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma16(o[nb][p + u], a0, a1, a2, a3, w01[nb], w23[nb]);
        }
      }
    }
    __syncwarp();       // every lane has read the buffer
    const int next = i + kStages;
    if (next < mine) {
      if ((next & 31) == 0) {
#pragma unroll
        for (int h = 0; h < kTiles; ++h) {
          lines[h] = line_of(place[h], next + lane, h);
          ks_next[h] = scale_of(c.k_scale, place[h]), vs_next[h] = scale_of(c.v_scale, place[h]);
          place[h] = place_of(next + 32 + lane, h);
        }
      }
      issue(next, buf);
    }
    if (++buf == kStages) buf = 0, parity ^= 1;
  }
  if (!ok || *dead) {      // a wait gave up: what is under way gets 10 ms to end; no number comes out
    for (const long long begun = clock64(); clock64() - begun < 20000000ll;) {}
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) l[nb][0] = l[nb][1] = NAN;
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[nb][h] += __shfl_xor_sync(0xffffffffu, l[nb][h], 4);
      l[nb][h] += __shfl_xor_sync(0xffffffffu, l[nb][h], 8);
      l[nb][h] += __shfl_xor_sync(0xffffffffu, l[nb][h], 16);
    }
  }
  // ---- outputs: columns 16 p + 2 quad and + 1, rows 2 tq and 2 tq + 1, of the warps' parts, where the tiles were -------------------------------
  constexpr int kSets = WARPITEM ? 1 : kWarps;
  if constexpr (WARPITEM) __syncwarp();
  else __syncthreads();
  float* o_s = reinterpret_cast<float*>(sm + (WARPITEM ? warp * kStages * S::kStage : 0));      // [set][row][D]
  float *m_s = o_s + kSets * kMost * D, *l_s = m_s + kSets * kMost;
  const int set = WARPITEM ? 0 : warp;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = set * kMost + 8 * nb + 2 * tq + h;
#pragma unroll
      for (int p = 0; p < kPieces; ++p) *reinterpret_cast<float2*>(o_s + row * D + 16 * p + 2 * quad) = make_float2(o[nb][p][h], o[nb][p][h + 2]);
      if (quad == 0) m_s[row] = m[nb][h], l_s[row] = l[nb][h];
    }
  }
  if constexpr (WARPITEM) __syncwarp();
  else __syncthreads();
  for (int e = WARPITEM ? lane : threadIdx.x; e < rows * (D / 2); e += WARPITEM ? 32 : kWarps * 32) {
    const int g = e / (D / 2), d = e % (D / 2) * 2;
    float top = -INFINITY, sum = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int w = 0; w < kSets; ++w) top = fmaxf(top, m_s[w * kMost + g]);
#pragma unroll
    for (int w = 0; w < kSets; ++w) {
      const float mw = m_s[w * kMost + g], lw = l_s[w * kMost + g], k = mw == -INFINITY ? (lw != lw ? 1.f : 0.f) : exp2_fast(mw - top);
      const float2 v = *reinterpret_cast<const float2*>(o_s + (w * kMost + g) * D + d);
      sum = fmaf(lw, k, sum);
      a0 = fmaf(v.x, k, a0);
      a1 = fmaf(v.y, k, a1);
    }
    if (WARPITEM || P.splits == 1) {
      const float f = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint32_t*>(static_cast<T*>(P.a.out) + it.at(P, row0 + g, static_cast<int64_t>(P.a.Hq) * D) + d) = pack2<T>(a0 * f, a1 * f);
    } else {
      const int64_t piece = static_cast<int64_t>(unit) * kMost + g;
      *reinterpret_cast<float2*>(P.o + piece * D + d) = make_float2(a0, a1);
      if (d == 0) P.ml[piece] = make_float2(top, sum);
    }
  }
}

// A CTA per item and row: the parts in the order of the keys, by four groups of threads.  (All that needs no part is done before the kernel ahead ends.)
template <typename T, int D, int NB>
__global__ void __launch_bounds__(2 * D) decode_merge_kernel(const Decode P) {
  constexpr int kCols = D / 2, kAhead = 4;      // two columns a thread
  __shared__ float2 part_s[3][kCols];
  __shared__ float sum_s[4], top_s[4];
  constexpr int kMost = 8 * NB;
  const int most = min(P.max_rows, kMost), g = blockIdx.x % most, item = blockIdx.x / most;
  const Item it = Item::of<kMost>(P, item);
  const int row = it.block * kMost + g, col = threadIdx.x % kCols, group = threadIdx.x / kCols, keys = it.keys, part = part_of(keys, P.splits), parts = keys > 0 ? (keys + part - 1) / part : 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row >= it.rows) return;
  float top = -INFINITY, sum = 0.f;
  float2 o = make_float2(0.f, 0.f);
  for (int p0 = group; p0 < parts; p0 += 4 * kAhead) {
    float2 ml[kAhead], v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int p = p0 + 4 * u;
      const int64_t piece = (static_cast<int64_t>(item) * P.splits + p) * kMost + g;
      ml[u] = make_float2(-INFINITY, 0.f), v[u] = make_float2(0.f, 0.f);
      if (p < parts) ml[u] = P.ml[piece], v[u] = *reinterpret_cast<const float2*>(P.o + piece * D + 2 * col);
    }
    float now = top;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) now = fmaxf(now, ml[u].x);
    const float was = top == -INFINITY ? (sum != sum ? 1.f : 0.f) : exp2_fast(top - now);
    top = now;
    sum *= was, o.x *= was, o.y *= was;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float k = ml[u].x == -INFINITY ? (ml[u].y != ml[u].y ? 1.f : 0.f) : exp2_fast(ml[u].x - now);
      sum = fmaf(ml[u].y, k, sum), o.x = fmaf(v[u].x, k, o.x), o.y = fmaf(v[u].y, k, o.y);
    }
  }
  if (col == 0) top_s[group] = top, sum_s[group] = sum;
  if (group > 0) part_s[group - 1][col] = o;
  __syncthreads();
  if (group > 0) return;
  float all_top = -INFINITY, k[4];
#pragma unroll
  for (int y = 0; y < 4; ++y) all_top = fmaxf(all_top, top_s[y]);
  sum = 0.f;
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    k[y] = top_s[y] == -INFINITY ? (sum_s[y] != sum_s[y] ? 1.f : 0.f) : exp2_fast(top_s[y] - all_top);
    sum = fmaf(sum_s[y], k[y], sum);
  }
  o.x *= k[0], o.y *= k[0];
#pragma unroll
  for (int y = 1; y < 4; ++y) o.x = fmaf(part_s[y - 1][col].x, k[y], o.x), o.y = fmaf(part_s[y - 1][col].y, k[y], o.y);
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint32_t*>(static_cast<T*>(P.a.out) + it.at(P, row, static_cast<int64_t>(P.a.Hq) * D) + 2 * col) = pack2<T>(o.x * f, o.y * f);
}

// The pool as lines of 128 bytes, fetched 16 tokens at a time; lines behind the pool read as zeros
bool code_map(CUtensorMap* map, const void* pool, const Cache& c) {
  const Encode encode = tensor_map_encode();
  if (!encode) return false;
  const cuuint64_t dims[2] = {128, static_cast<cuuint64_t>(c.max_blocks) * c.Hkv * c.bs / (128 / c.D)}, strides[1] = {128};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(kTok / (128 / c.D))}, step[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool decode_serves(int D, int bs, int dtype) { return dtype != B200_DTYPE_F32 && (D == 64 || D == 128) && bs % kTok == 0; }

// Parts of an item.  Items of up to 512 tokens are not divided (a second launch costs the host 5 us and the device 3).  592 CTAs are resident (444 of the kernel of two blocks of 8 rows, for
// which the same rule stands): what fits is
// divided until there are some 400 of them; long contexts go on to 1024, parts of 2048 tokens, which evens out that SMs are not served alike.  32 heads over 8
// of 128, us with 1 / 2 / 3 / 4 / 6 / 8 / 16 parts: 1 x 4096 39 / 22 / 17 / 14 / 12 / 9 / 7; 8 x 8192 80 / 44 / 39 / 31 / 29 / 30 / 32; 16 x 4096 43 / 31 / 29 / 31 / 35 / 32 / 37;
// 32 x 2048 30 / 32 / 35 / 34 / 36 / 39 / 46; 64 x 2048 51 / 56 / 58 / 58 / 61 / 67 / 83; 64 x 8192 185 / 173 / 179 / 176 / 177 / 176; 128 x 2048 90 / 103 / 102 / 104; 8 x 32768 of
// e4m3, ragged, 274 / 152 / 111 / 86 / 75 / 75 / 72.
constexpr int kShort = 512;
int splits_of(int64_t items, int longest) {
  if (longest <= kShort) return 1;
  int64_t splits = 400 / items;
  if (longest >= 8192) splits = std::max(splits, std::min<int64_t>(longest / 2048, 1024 / items));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(splits, (longest + kLeastPart - 1ll) / kLeastPart)));
}
// Rows of a sequence and kv head, in blocks of 8 or 16
int most_of(int rows) { return rows <= 8 ? 8 : 16; }
int64_t items_of(int B, int Hkv, int rows) { return static_cast<int64_t>(B) * Hkv * ((rows + most_of(rows) - 1) / most_of(rows)); }
size_t decode_bytes(int B, int Hkv, int D, int rows, int longest) {
  const int most = most_of(rows);
  const int64_t items = items_of(B, Hkv, rows), splits = splits_of(items, longest);
  return splits > 1 ? static_cast<size_t>(items * splits) * most * (D + 2) * sizeof(float) : 0;
}

template <typename T, typename C, int D, int NB, bool CAUSAL, bool WARPITEM>
int launch_decode_as(const char* name, const Decode& P, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t stream) {
  auto kern = decode_kernel<T, C, D, NB, CAUSAL, WARPITEM>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodePlan<D>::kSmem);
  kern<<<WARPITEM ? (P.items + kWarps - 1) / kWarps : P.items * P.splits, kWarps * 32, DecodePlan<D>::kSmem, stream>>>(P, k_map, v_map);
  if (int rc = check_launch(name)) return rc;
  if (P.splits == 1) return 0;
  return launch_behind(name, decode_merge_kernel<T, D, NB>, static_cast<unsigned>(P.items) * static_cast<unsigned>(std::min(P.max_rows, 8 * NB)), 2 * D, 0, stream, P);
}

// rows: of a sequence and kv head at most
template <typename T>
int launch_decode(const char* name, const Attn& A, int rows, int longest, void* workspace, int codes, cudaStream_t stream) {
  Decode P{};
  const int most = most_of(rows);
  P.a = A, P.G = A.Hq / A.c.Hkv, P.max_rows = rows, P.blocks = (rows + most - 1) / most, P.items = static_cast<int>(items_of(A.r.B, A.c.Hkv, rows));
  P.splits = splits_of(P.items, longest);
  P.ml = static_cast<float2*>(workspace), P.o = static_cast<float*>(workspace) + static_cast<int64_t>(P.items) * P.splits * 2 * most;
  CUtensorMap k_map, v_map;
  if (!code_map(&k_map, A.c.k_pool, A.c) || !code_map(&v_map, A.c.v_pool, A.c)) return fail(B200_EINVAL, "%s: no tensor map of the pools", name);
  const bool warps = longest <= kShort && most == 8 && P.items > 4 * kNumSMs;       // more than are resident at once
  auto go = [&](auto* c, auto d) {
    using C = std::remove_pointer_t<decltype(c)>;
    if (A.r.starts)
      return most == 16 ? launch_decode_as<T, C, d.value, 2, true, false>(name, P, k_map, v_map, stream)
             : warps    ? launch_decode_as<T, C, d.value, 1, true, true>(name, P, k_map, v_map, stream)
                        : launch_decode_as<T, C, d.value, 1, true, false>(name, P, k_map, v_map, stream);
    return most == 16 ? launch_decode_as<T, C, d.value, 2, false, false>(name, P, k_map, v_map, stream)
           : warps    ? launch_decode_as<T, C, d.value, 1, false, true>(name, P, k_map, v_map, stream)
                      : launch_decode_as<T, C, d.value, 1, false, false>(name, P, k_map, v_map, stream);
  };
  auto of = [&](auto* c) { return A.c.D == 128 ? go(c, std::integral_constant<int, 128>{}) : go(c, std::integral_constant<int, 64>{}); };
  return codes == B200_CODES_INT8 ? of(static_cast<q8::Int8*>(nullptr)) : of(static_cast<q8::E4m3*>(nullptr));
}

// Whether these kernels take a call: sizes, alignment, numbers that fit
bool decode_takes(const Attn& A, int rows, int longest, int dtype) {
  const int most = most_of(rows);
  const int64_t items = items_of(A.r.B, A.c.Hkv, rows);
  return decode_serves(A.c.D, A.c.bs, dtype) && aligned16(A.c.k_pool) && aligned16(A.c.v_pool) && !(reinterpret_cast<uintptr_t>(A.q) & 7) && A.q_stride % 4 == 0 &&
         !(reinterpret_cast<uintptr_t>(A.out) & 3) && (A.c.max_blocks + 1) * A.c.Hkv * A.c.bs < INT32_MAX && items * most * splits_of(items, longest) < INT32_MAX;
}
int run_decode(const char* name, const Attn& A, int rows, int longest, void* workspace, size_t workspace_bytes, int codes, int dtype, cudaStream_t stream) {
  const size_t need = decode_bytes(A.r.B, A.c.Hkv, A.c.D, rows, longest);
  if (need && (!workspace || workspace_bytes < need)) return fail(B200_ENOSPC, "%s: workspace of %zu bytes", name, workspace ? workspace_bytes : 0);
  if (need && !aligned16(workspace)) return fail(B200_EINVAL, "%s: workspace not aligned to 16 bytes", name);
  return dtype == B200_DTYPE_BF16 ? launch_decode<__nv_bfloat16>(name, A, rows, longest, workspace, codes, stream)
                                  : launch_decode<__half>(name, A, rows, longest, workspace, codes, stream);
}
// Several tokens per sequence: whether they are few enough for these kernels rather than those of b200_prompt_q8.cu, which take 128 rows at once.  Always where one block of
// up to 16 rows holds them; else while all the blocks' walks are few and short: each reads and turns its sequence's codes again, and beyond 32 of them they fill the SMs sooner.
// us here / there, 8 kv heads and 4 query heads to each, D = 128, but where it says otherwise.  One block: 64 x 2 tokens at 2k 53 / 103, 64 x 4 81 / 103, 16 x 9 of one head of 64 at 3k
// 20 / 32.  32 walks and fewer: 1 x 16 at 100 tokens 8.3 / 8.9, at 2k 13 / 15, at 8k 24 / 28, at 16k 36 / 38, at 24k 50 / 45; 1 x 8 at 32k 38 / 44, at 64k 81 / 63.  48: 1 x 24 at 1.5k 14 / 16,
// at 4k 22 / 20, at 8k 31 / 30, at 12k 41 / 39.  64: 2 x 16 at 100 8.4 / 8.9, at 1k 17 / 14, at 2k 19.5 / 17, at 4k 26 / 24, at 8k 38 / 33; 4 x 8 at 2k 19.5 / 20, at 4k 27 / 26, at 8k 39 / 35; 1 x 64
// over 4 heads at 1.5k 19 / 23, at 4k 26 / 23, at 8k 37 / 30.  Heads of 64: 3 x 32 of one head, 48 walks, at 8k 20 / 23; 16 x 17 of one over 2, 64 walks, at 8k 23 / 24.  More: 4 x 12 at 1k 20 / 15.
bool few_rows(int B, int Hkv, int D, int64_t rows, int longest) {
  const int64_t walks = static_cast<int64_t>(B) * Hkv * ((rows + 15) / 16);
  return rows <= 16 || (walks <= 64 && walks * longest <= (walks <= 32 || D == 64 ? 600000 : 200000));
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
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || block_size <= 0 || max_context_len < 0 || !decode_serves(D, block_size, dtype)) return 0;
  return decode_bytes(B, Hkv, D, Hq / Hkv, max_context_len);
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
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!(flags & B200_ATTN_FORCE_GENERIC) && decode_takes(A, Hq / Hkv, max_context_len, dtype))
    return run_decode(name, A, Hq / Hkv, max_context_len, workspace, workspace_bytes, codes, dtype, s);
  return launch_any_of(name, A, codes, dtype, s);
}

size_t b200_paged_prompt_attn_q8_workspace(int B, int max_new, int Hq, int Hkv, int D, int block_size, int max_context_len, int dtype) {
  if (B <= 0 || max_new <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || block_size <= 0 || max_context_len < 0) return 0;
  const int64_t rows = static_cast<int64_t>(max_new) * (Hq / Hkv);
  const size_t few = few_rows(B, Hkv, D, rows, max_context_len) && decode_serves(D, block_size, dtype) ? decode_bytes(B, Hkv, D, static_cast<int>(rows), max_context_len) : 0;
  return std::max(few, prompt_q8_workspace(B, max_new, Hq, Hkv, D, block_size, max_context_len, dtype));
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
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  q8::PromptAttn P{};
  P.c = A.c, P.r = A.r, P.out = out, P.q = q, P.q_stride = q_stride, P.Hq = Hq, P.scale = scale;
  if (max_new == 0) return 0;
  const int64_t of_head = static_cast<int64_t>(max_new) * (Hq / Hkv);
  if (!(flags & B200_ATTN_FORCE_GENERIC) && few_rows(B, Hkv, D, of_head, max_context_len) && decode_takes(A, static_cast<int>(of_head), max_context_len, dtype))
    return run_decode(name, A, static_cast<int>(of_head), max_context_len, workspace, workspace_bytes, codes, dtype, s);
  if (!(flags & B200_ATTN_FORCE_GENERIC) && prompt_q8_serves(P, max_new, max_context_len, dtype)) {
    const size_t need = prompt_q8_workspace(B, max_new, Hq, Hkv, D, block_size, max_context_len, dtype);
    if (need && (!workspace || workspace_bytes < need)) return fail(B200_ENOSPC, "%s: workspace of %zu bytes", name, workspace ? workspace_bytes : 0);
    if (need && !aligned16(workspace)) return fail(B200_EINVAL, "%s: workspace not aligned to 16 bytes", name);
    return prompt_q8(name, P, max_new, max_context_len, workspace, codes, dtype, s);
  }
  return launch_any_of(name, A, codes, dtype, s);
}

}  // extern "C"
