// Attention of a tree of drafted tokens over the paged cache: each node sees the context and the nodes of its mask.
//
//   out[t, h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(q[t, h] k_j scale - max),   j in the context, or bit j of visible[t]
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "b200_common.cuh"
#include "b200_tcgen05.cuh"

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
// output, and put their maxima, sums and outputs together at the end.  Bound by the loads' latency: 4 sequences x 13 nodes x 8 heads of 64 at 160 keys
// in fp32 11 - 14 us on the device (four warps, eight rows of values under way: 20).  Serves what neither kernel below does: few rows behind short tables, rows
// that are not of 16-byte pieces.
constexpr int kAnyWarps = 8, kAnyMostD = 256;

template <typename T, int COLS>
__global__ void __launch_bounds__(kAnyWarps * 32) tree_attn_any_kernel(const TreeAttn A, bool vec) {
  constexpr int kVec = 16 / sizeof(T), kAhead = 32 / COLS, kMostD = 32 * COLS;        // rows of values under way
  __shared__ __align__(16) float q_s[kMostD];
  __shared__ float out_s[kAnyWarps][kMostD], m_s[kAnyWarps], l_s[kAnyWarps];
  const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int keys, n;
  lengths(A, b, &keys, &n);
  T* out = static_cast<T*>(A.out) + ((static_cast<int64_t>(b) * A.nodes + t) * A.Hq + h) * A.D;
  if (t >= n) {
    for (int d = threadIdx.x; d < A.D; d += blockDim.x) out[d] = Cvt<T>::from_f32(0.f);
    return;
  }
  const T* q = static_cast<const T*>(A.q) + b * A.q_batch_stride + t * A.q_node_stride + static_cast<int64_t>(h) * A.D;
  for (int d = threadIdx.x; d < kMostD; d += blockDim.x) q_s[d] = d < A.D ? Cvt<T>::to_f32(q[d]) * A.scale : 0.f;
  __syncthreads();
  const int base = keys - n, g = h / (A.Hq / A.Hkv);
  const uint64_t seen = static_cast<uint64_t>(A.visible[b * A.visible_stride + t]);
  float m = -INFINITY, l = 0.f, acc[COLS] = {};
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
#pragma unroll 16
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
    for (int c = 0; c < COLS; ++c) acc[c] *= corr;
    for (int i = 0; i < 32; i += kAhead) {
      float wi[kAhead], v[kAhead][COLS];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        wi[u] = __shfl_sync(0xffffffffu, w, i + u);
        const int64_t vi = __shfl_sync(0xffffffffu, at, i + u);
        const T* row = static_cast<const T*>(A.v_pool) + vi;
#pragma unroll
        for (int c = 0; c < COLS; ++c) v[u][c] = wi[u] != 0.f && vi >= 0 && c * 32 + lane < A.D ? Cvt<T>::to_f32(row[c * 32 + lane]) : 0.f;
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
  for (int d = threadIdx.x; d < A.D; d += blockDim.x) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kAnyWarps; ++w) o = fmaf(out_s[w][d], k[w], o);
    out[d] = Cvt<T>::from_f32(sum == 0.f ? 0.f : o / sum);
  }
}

// The same for many keys: a CTA per (sequence, kv head, block of R = 8 RW rows) - or a cluster of them with a part of the keys each, where there are few -
// walks tiles of KT keys that its copies bring to shared memory as they are.  A warp has RW rows, a lane KT / 32 keys of each for the scores; for the output
// a thread has two columns of some rows.  The next tile's keys are under way while this one's weights meet its values, and the values while the next scores are
// formed.  fp32 arithmetic without tensor cores; bound by shared memory, 12 wavefronts for 32 products a lane at RW = 4: 4 sequences x 64 nodes x 32 heads over 8
// of 128 at 4k in fp32 746 us, three times what the products alone take at 70 TFLOP/s (each row by itself: 5470).  Values of drafted tokens count only where their weight is not 0.
template <typename T, int DM, int RW>
struct RowsPlan {
  static constexpr int kTile = DM == 256 ? 32 : 64, kRowsOf = 8 * RW;
  static constexpr int kKeyRow = DM * sizeof(T) + 16, kWeightRow = kRowsOf + 4;      // bytes; numbers
  static constexpr int kK = 0, kV = kK + kTile * kKeyRow, kQ = kV + kTile * DM * static_cast<int>(sizeof(T)), kP = kQ + kRowsOf * DM * 4,
                       kStats = kP + kTile * kWeightRow * 4, kPlaces = kStats + 3 * kRowsOf * 4 + (kRowsOf * 4 % 8), kEnd = kPlaces + 2 * kTile * 8;
  static_assert(kQ >= kRowsOf * DM * 4, "outputs go where keys and values were");
  static_assert(kPlaces % 8 == 0 && kP % 16 == 0 && kV % 16 == 0 && kQ % 16 == 0, "alignment");
};

// 16 bytes as numbers
template <typename T>
__device__ __forceinline__ void numbers_of(const int4& raw, float* to) {
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int u = 0; u < static_cast<int>(16 / sizeof(T)); ++u) to[u] = Cvt<T>::to_f32(e[u]);
}

template <typename T, int DM, int RW>
__global__ void __launch_bounds__(256, 2) tree_attn_rows_kernel(const TreeAttn A, int blocks) {
  using P = RowsPlan<T, DM, RW>;
  constexpr int KT = P::kTile, R = P::kRowsOf, KPL = KT / 32, kVec = 16 / sizeof(T), kGroups = 512 / DM, RG = R / kGroups > 0 ? R / kGroups : 1;
  extern __shared__ __align__(16) unsigned char sm[];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int unit = blockIdx.x / ctas, block = unit % blocks, b = unit / blocks / A.Hkv, g = unit / blocks - b * A.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rep = A.Hq / A.Hkv, row0 = block * R, rows = A.nodes * rep;
  int keys, n;
  lengths(A, b, &keys, &n);
  auto place_out = [&](int row) { return (static_cast<int64_t>(b) * A.nodes + row / rep) * A.Hq + g * rep + row % rep; };
  T* out = static_cast<T*>(A.out);
  if (row0 >= n * rep) {        // (the same in the cluster)
    for (int r = rank; r < min(R, rows - row0); r += ctas)
      for (int d = tid; d < A.D; d += blockDim.x) out[place_out(row0 + r) * A.D + d] = Cvt<T>::from_f32(0.f);
    return;
  }
  float* q_s = reinterpret_cast<float*>(sm + P::kQ);
  float* p_s = reinterpret_cast<float*>(sm + P::kP);
  float *corr_s = reinterpret_cast<float*>(sm + P::kStats), *m_s = corr_s + R, *l_s = m_s + R;
  int64_t* places = reinterpret_cast<int64_t*>(sm + P::kPlaces);
  const int tiles = (keys + KT - 1) / KT, per = (tiles + ctas - 1) / ctas, t0 = min(rank * per, tiles), t1 = min(t0 + per, tiles), base = keys - n;

  auto look_up = [&](int tile) {        // element of the pools; outside them, and behind the last key: zeros
    if (tid < KT) {
      const int j = tile * KT + tid;
      int64_t at = -1;
      if (j < keys) {
        const int64_t page = A.block_tables[static_cast<int64_t>(b) * A.table_stride + j / A.bs];
        if (page >= 0 && page < A.max_blocks) at = ((page * A.Hkv + g) * A.bs + j % A.bs) * A.D;
      }
      places[(tile & 1) * KT + tid] = at;
    }
  };
  auto copy = [&](int tile, const void* pool, uint32_t to, int row_bytes) {
    constexpr int kCh = DM / kVec;
    const int ch_of = A.D / kVec;
    for (int c = tid; c < KT * kCh; c += 256) {
      const int key = c / kCh, ch = c % kCh;
      const int64_t at = places[(tile & 1) * KT + key];
      if (ch < ch_of) cp16(to + key * row_bytes + ch * 16, static_cast<const T*>(pool) + (at >= 0 ? at + ch * kVec : 0), at >= 0);
    }
  };
  const uint32_t k_at = smem_u32(sm + P::kK), v_at = smem_u32(sm + P::kV);
  look_up(t0);
  look_up(t0 + 1);
  __syncthreads();
  if (t0 < t1) copy(t0, A.k_pool, k_at, P::kKeyRow);
  cp_commit();
  if (t0 < t1) copy(t0, A.v_pool, v_at, DM * sizeof(T));
  cp_commit();
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int r = warp * RW + i, row = row0 + r, t = row / rep;
    const T* q = static_cast<const T*>(A.q) + b * A.q_batch_stride + t * A.q_node_stride + static_cast<int64_t>(g * rep + row - t * rep) * A.D;
#pragma unroll
    for (int d = lane; d < DM; d += 32) q_s[r * DM + d] = d < A.D && t < n ? Cvt<T>::to_f32(q[d]) * A.scale : 0.f;
  }
  uint64_t seen[RW];
  bool live[RW];
  float m[RW], l[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const int t = (row0 + warp * RW + r) / rep;
    live[r] = t < n;
    seen[r] = live[r] ? static_cast<uint64_t>(A.visible[b * A.visible_stride + t]) : 0ull;
    m[r] = -INFINITY;
    l[r] = 0.f;
  }
  const int pair = tid % (DM / 2), first = tid / (DM / 2) * RG;        // columns 2 pair, 2 pair + 1 of rows first ..
  const bool mine = first < R;
  float acc[RG][2] = {};
  for (int tile = t0; tile < t1; ++tile) {
    cp_wait<1>();
    __syncthreads();
    float s[RW][KPL] = {};
    const int4* k_row[KPL];
#pragma unroll
    for (int i = 0; i < KPL; ++i) k_row[i] = reinterpret_cast<const int4*>(sm + P::kK + (i * 32 + lane) * P::kKeyRow);
#pragma unroll 4
    for (int d = 0; d < A.D; d += kVec) {
      float k[KPL][kVec];
#pragma unroll
      for (int i = 0; i < KPL; ++i) numbers_of<T>(k_row[i][d / kVec], k[i]);
#pragma unroll
      for (int r = 0; r < RW; ++r) {
#pragma unroll
        for (int u = 0; u < kVec; u += 4) {
          const float4 q = *reinterpret_cast<const float4*>(q_s + (warp * RW + r) * DM + d + u);
#pragma unroll
          for (int i = 0; i < KPL; ++i) s[r][i] = fmaf(q.x, k[i][u], fmaf(q.y, k[i][u + 1], fmaf(q.z, k[i][u + 2], fmaf(q.w, k[i][u + 3], s[r][i]))));
        }
      }
    }
    float p[KPL][RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      bool sees[KPL];
      float top = m[r];
#pragma unroll
      for (int i = 0; i < KPL; ++i) {
        const int j = tile * KT + i * 32 + lane;
        sees[i] = live[r] && j < keys && (j < base || (seen[r] >> (j - base) & 1));
        top = fmaxf(top, sees[i] ? s[r][i] : -INFINITY);
      }
      top = warp_max(top);
      const float from = top == -INFINITY ? 0.f : top, corr = m[r] == -INFINITY ? 0.f : expf(m[r] - from);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < KPL; ++i) {
        p[i][r] = sees[i] ? expf(s[r][i] - from) : 0.f;
        sum += p[i][r];
      }
      l[r] = fmaf(l[r], corr, warp_sum(sum));
      m[r] = top;
      if (lane == 0) corr_s[warp * RW + r] = corr;
    }
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
      float* to = p_s + (i * 32 + lane) * P::kWeightRow + warp * RW;
      if constexpr (RW == 4) *reinterpret_cast<float4*>(to) = make_float4(p[i][0], p[i][1], p[i][2], p[i][3]);
      else
#pragma unroll
        for (int r = 0; r < RW; ++r) to[r] = p[i][r];
    }
    if (tile + 1 < t1) look_up(tile + 2);
    __syncthreads();
    if (tile + 1 < t1) copy(tile + 1, A.k_pool, k_at, P::kKeyRow);
    cp_commit();
    cp_wait<1>();
    __syncthreads();
    if (mine) {
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        const float corr = corr_s[first + r];
        acc[r][0] *= corr;
        acc[r][1] *= corr;
      }
      auto weigh = [&](auto drafted) {
#pragma unroll 4
        for (int key = 0; key < KT; ++key) {
          float v[2], w[RG];
          const T* e = reinterpret_cast<const T*>(sm + P::kV) + key * DM + 2 * pair;
          if constexpr (sizeof(T) == 4) {
            const float2 two = *reinterpret_cast<const float2*>(e);
            v[0] = two.x, v[1] = two.y;
          } else {
            const uint32_t two = *reinterpret_cast<const uint32_t*>(e);
            const T* h = reinterpret_cast<const T*>(&two);
            v[0] = Cvt<T>::to_f32(h[0]), v[1] = Cvt<T>::to_f32(h[1]);
          }
          const float* from = p_s + key * P::kWeightRow + first;
#pragma unroll
          for (int r = 0; r < RG; ++r) w[r] = from[r];
#pragma unroll
          for (int r = 0; r < RG; ++r) {
            const bool counts = !decltype(drafted)::value || w[r] != 0.f;
            acc[r][0] = fmaf(w[r], counts ? v[0] : 0.f, acc[r][0]);
            acc[r][1] = fmaf(w[r], counts ? v[1] : 0.f, acc[r][1]);
          }
        }
      };
      if (tile * KT + KT > base) weigh(std::true_type{});
      else weigh(std::false_type{});
    }
    __syncthreads();
    if (tile + 1 < t1) copy(tile + 1, A.v_pool, v_at, DM * sizeof(T));
    cp_commit();
  }
  // ---- outputs, of the cluster's parts of the keys -------------------------------------------------------------------------------------------
  cp_wait<0>();
  __syncthreads();
  if (lane == 0) {
#pragma unroll
    for (int r = 0; r < RW; ++r) m_s[warp * RW + r] = m[r], l_s[warp * RW + r] = l[r];
  }
  float* o_s = reinterpret_cast<float*>(sm);
  if (mine) {
#pragma unroll
    for (int r = 0; r < RG; ++r) *reinterpret_cast<float2*>(o_s + (first + r) * DM + 2 * pair) = make_float2(acc[r][0], acc[r][1]);
  }
  cluster.sync();
  for (int r = rank + ctas * warp; r < min(R, rows - row0); r += ctas * 8) {        // a warp a row, a lane a CTA's part of it
    const float mc = lane < ctas ? *cluster.map_shared_rank(m_s + r, lane) : -INFINITY, lc = lane < ctas ? *cluster.map_shared_rank(l_s + r, lane) : 0.f;
    const float top = warp_max(mc), k = mc == -INFINITY ? (lc != lc ? 1.f : 0.f) : expf(mc - top), sum = warp_sum(lc * k);
    T* to = out + place_out(row0 + r) * A.D;
#pragma unroll
    for (int d0 = 0; d0 < DM; d0 += 32) {
      float o = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float kc = __shfl_sync(0xffffffffu, k, c);
        if (c < ctas) o = fmaf(*cluster.map_shared_rank(o_s + r * DM + d0 + lane, c), kc, o);
      }
      if (d0 + lane < A.D) to[d0 + lane] = Cvt<T>::from_f32(sum == 0.f ? 0.f : o / sum);
    }
  }
  cluster.sync();       // the others may still read this CTA's
}

// ---- 16-bit types, heads of 64 or 128, pages that divide 64 keys (or are multiples of 64) ------------------------------------------------------
// The rows of a sequence and kv head - its nodes times the rep = Hq / Hkv query heads, node by node - go in blocks of 128; a CTA keeps to one
// block's number.  Keys go in tiles of 64, and the tiles of all sequences and kv heads, one after another, in equal shares to the workers: a CTA
// per row block that walk the same keys side by side.  Whole walks (a sequence's and head's every tile) are written out; what a share's
// ends cut leaves (maximum, sum, output) in the workspace, at most two pieces a worker, for tree_merge_kernel, which puts a row's pieces together in the order of
// their keys and writes the zeros of rows without a node.
//
//   S = Q K^T   tcgen05.mma, 128 x 64, both operands in shared memory (128-byte swizzled lines), S in tensor memory, two of them
//   P           four warps, one thread per row: mask, running maximum, exp2 in fp32; rounded to the storage type into the tensor memory S
//               was in: by half a step of each weight, wherever it lies (the largest lies between 1 and 2^8, the reference moves late); the sum is taken
//               before.  Error against 64 bits 0.0023 (bf16), 0.00029 (fp16) of the outputs' size, 0.0017 and 0.00021 with weights in fp32, which is
//               the outputs' own rounding
//   O += P V    tcgen05.mma, P from tensor memory, O in tensor memory in fp32
//
// Three warps copy (one keys, two values), boxes of a page by 64 columns; the tiles that reach into the drafted tokens have their values copied by the
// threads themselves, zeros for slots behind the last token and for values that are no numbers: 0 x NaN would reach rows that do not see
// them.  Rows that do get them in the end.
//
// Bound.  Few rows: memory, 64 sequences x 8 nodes at 2k (32 heads over 8 of 128) 84 us on the device, 4.9 TB/s of the 6.55 that a copy reaches: SMs are
// not served evenly, and each walk begins with three dependent loads (lengths, table, keys).  Two to four times the workers, so that late ones do less:
// 98 to 114 us for 90.  Many rows: the softmax's chain of a tile, 8 x 64 nodes at 32k (64 heads over 8) 514 us on the device and 607 a call after the
// other, 1.05 PFLOP/s; at 8k exponential unit 55 %, tensor cores 53 %, issue slots 56 %.  A part of the exponentials as polynomials took 656 for 590.
constexpr int kRows = 128, kKeys = 64, kBlk = kKeys * 128;
// threads: rows, copies of keys and of values, products.  Eight warps: two CTAs' leave each thread 128 registers (nine: 96)
constexpr int kSoft = 128, kLoadK = 32, kLoadV = 64, kNT = kSoft + kLoadK + kLoadV + 32;
constexpr int kCtasPerSm = 2;
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct Plan {
  static constexpr int kBufs = D == 128 ? 2 : 4;        // of keys, and of values
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + (D / 64) * kRows * 128;
  static constexpr int kV = kK + kBufs * (D / 64) * kBlk;
  static constexpr int kBar = kV + kBufs * (D / 64) * kBlk;
  static constexpr int kFlags = kBar + 8 * (1 + 4 * kBufs + 4);     // tensor memory's address, failure, values that are no numbers
  static constexpr int kEnd = kFlags + 16;
  static constexpr int kO = 2 * kKeys, kTm = 256;     // columns of tensor memory: S0 | S1 | O
  static_assert((kEnd + 1024 + 1024) * kCtasPerSm <= 228 * 1024, "shared memory");
};

struct Shares {
  float2* ml;               // [worker][row block][2][rows]: maximum (of scores in powers of two), sum
  float4* o;                // [worker][row block][2][D / 4][rows]
  int rows, blocks, workers;        // of a block that are kept (multiple of 32)
  bool whole;               // a worker for each sequence and kv head: no pieces, and nothing behind this kernel
};

// Tiles of a sequence
__device__ __forceinline__ int tiles_of(const TreeAttn& A, int b) {
  int keys, n;
  lengths(A, b, &keys, &n);
  return n > 0 ? (keys + kKeys - 1) / kKeys : 0;
}

// A worker's way through the tiles
struct Walk {
  int b, g, t, nt;          // sequence, kv head, tile of nt
  int left;                 // tiles
  __device__ __forceinline__ int run() const { return min(nt - t, left); }       // tiles of this sequence and head
  __device__ __forceinline__ void skip(const TreeAttn& A, int tiles) {        // no more than these
    left -= tiles;
    t += tiles;
    if (t < nt || left <= 0) return;
    t = 0;
    if (++g < A.Hkv) return;
    g = 0;
    do
      if (++b >= A.B) {
        left = 0;
        return;
      }
    while ((nt = tiles_of(A, b)) == 0);
  }
};

// (tiles have numbers of 31 bits: the launch sees to it; a division of 64 costs 500 clocks)
__device__ __forceinline__ int share_of(int total, int workers) { return max(static_cast<int>((static_cast<unsigned>(total) + workers - 1) / workers), 1); }

// Tiles of 32 sequences at a time, a lane each; the first 128 are looked up once
struct Lookup {
  int n[4];
  __device__ __forceinline__ explicit Lookup(const TreeAttn& A) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = i * 32 + (threadIdx.x & 31);
      n[i] = b < A.B ? tiles_of(A, b) : 0;
    }
  }
  __device__ __forceinline__ int at(const TreeAttn& A, int round) const {
    if (round < 4) return round == 0 ? n[0] : round == 1 ? n[1] : round == 2 ? n[2] : n[3];
    const int b = round * 32 + (threadIdx.x & 31);
    return b < A.B ? tiles_of(A, b) : 0;
  }
};

// Tiles of a head of the sequences before b, and of all
__device__ __forceinline__ void tiles_before(const TreeAttn& A, const Lookup& look, int b, int* before, int* all) {
  *before = *all = 0;
  for (int round = 0; round * 32 < A.B; ++round) {
    const int n = look.at(A, round);
    *all += __reduce_add_sync(0xffffffffu, n);
    *before += __reduce_add_sync(0xffffffffu, round * 32 + static_cast<int>(threadIdx.x & 31) < b ? n : 0);
  }
}

// Where a worker begins; by a whole warp
__device__ __forceinline__ Walk walk_of(const TreeAttn& A, int worker, int workers) {
  const Lookup look(A);
  int none, total;
  tiles_before(A, look, 0, &none, &total);
  total *= A.Hkv;
  const int share = share_of(total, workers);
  if (worker > total / share) return Walk{0, 0, 0, 0, 0};
  const int from = worker * share;
  Walk w{0, 0, 0, 0, min(share, total - from)};
  if (w.left <= 0) return w;
  int before = 0;       // tiles of a head of the sequences before
  for (int round = 0; round * 32 < A.B; ++round) {
    const int lane = threadIdx.x & 31, n = look.at(A, round);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    const unsigned here = __ballot_sync(0xffffffffu, from < (before + upto) * A.Hkv);
    if (here) {
      const int first = __ffs(here) - 1, nt = __shfl_sync(0xffffffffu, n, first);
      const int in = from - (before + __shfl_sync(0xffffffffu, upto - n, first)) * A.Hkv;
      w.b = round * 32 + first;
      w.nt = nt;
      w.g = in / nt;
      w.t = in - w.g * nt;
      return w;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return w;
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// by a whole warp
__device__ __forceinline__ void copy_box(uint32_t to, const CUtensorMap* map, int col, int row, uint32_t bar) {
  asm volatile(
      "{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\n"
      "@p cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}\n" ::"r"(to),
      "l"(map), "r"(col), "r"(row), "r"(bar)
      : "memory");
}

__device__ __forceinline__ uint32_t line(uint32_t base, int r, int ch, int rows) {     // 16-byte piece ch of row r: blocks of 64 columns, swizzled lines
  return base + (ch >> 3) * (rows * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
}

// the larger magnitudes of two pairs, no number if one is none
template <typename T>
__device__ __forceinline__ uint32_t magnitudes(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7fff7fffu), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7fff7fffu), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ bool no_number(uint32_t two) {        // either half
  constexpr uint32_t e = std::is_same_v<T, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
  return (two & e) == e || ((two >> 16) & e) == e;
}
template <typename T>
__device__ __forceinline__ int numbers_only(int two) {
  constexpr int e = std::is_same_v<T, __nv_bfloat16> ? 0x7f80 : 0x7c00;
  if ((two & e) == e) two &= 0xffff0000;
  if (((two >> 16) & e) == e) two &= 0xffff;
  return two;
}

// What was left out of the products: values of drafted tokens that are no numbers, `cols` columns from c on of head g, for a row that sees the tokens
// `seen` of the keys k0 .. k1 - 1.  Hardly ever called.
template <typename T, int D>
__device__ __noinline__ void add_no_numbers(float* o, const TreeAttn& A, int b, int g, int base, int k0, int k1, uint64_t seen, int c, int cols) {
  for (int j = max(k0, base); j < k1; ++j) {
    if (!(seen >> (j - base) & 1)) continue;
    const int64_t page = A.block_tables[static_cast<int64_t>(b) * A.table_stride + j / A.bs];
    if (page < 0 || page >= A.max_blocks) continue;
    const T* v = static_cast<const T*>(A.v_pool) + ((page * A.Hkv + g) * A.bs + j % A.bs) * D + c;
    for (int x = 0; x < cols; ++x) {
      const float f = Cvt<T>::to_f32(v[x]);
      if (!(fabsf(f) < INFINITY)) o[x] += f;
    }
  }
}

// SPLIT > 1: 128 / SPLIT rows, each in the lanes of SPLIT warps, which take a part of a tile's keys each: with 32 rows in one warp, its
// exponentials alone were 512 clocks a tile.  Their outputs, each of its own keys, are put together at the end of a walk.
template <typename T, int D, int SPLIT>
__global__ void __launch_bounds__(kNT, kCtasPerSm)
tree_attn_kernel(const TreeAttn A, const Shares W, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using P = Plan<D>;
  constexpr int NB = P::kBufs, kRowWarps = 4 / SPLIT, kMine = kKeys / SPLIT;      // warps with rows of their own; keys of a tile for a warp
  extern __shared__ unsigned char raw_smem[];
  unsigned char* sm = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
  const uint32_t sm0 = smem_u32(sm);
  // queries in; keys of a buffer in, and read; values of a buffer in; P V of a value buffer done; S of a buffer done, P of a buffer written
  const uint32_t bar_q = sm0 + P::kBar, bar_k = bar_q + 8, bar_ke = bar_k + 8 * NB, bar_v = bar_ke + 8 * NB, bar_o = bar_v + 8 * NB, bar_s = bar_o + 8 * NB, bar_p = bar_s + 16;
  volatile uint32_t* tm_slot = reinterpret_cast<volatile uint32_t*>(sm + P::kFlags);
  volatile int* dead = reinterpret_cast<volatile int*>(sm + P::kFlags + 4);
  volatile int* strange = reinterpret_cast<volatile int*>(sm + P::kFlags + 8);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int worker = blockIdx.x / W.blocks, block = blockIdx.x - worker * W.blocks;
  const int rep = A.Hq / A.Hkv, row0 = block * kRows;
  const int row_warps = (min(kRows, A.nodes * rep - row0) + 31) / 32, soft_warps = SPLIT > 1 ? 4 : row_warps;       // SPLIT > 1: no more rows than fit

  asm volatile("griddepcontrol.launch_dependents;");
  if (tid == 0) {
    auto init = [](uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); };
    init(bar_q, soft_warps * 32);
    for (int b = 0; b < NB; ++b) {
      init(bar_k + 8 * b, kLoadK);
      init(bar_ke + 8 * b, 1);
      init(bar_v + 8 * b, kLoadV);
      init(bar_o + 8 * b, 1);
    }
    for (int b = 0; b < 2; ++b) {
      init(bar_s + 8 * b, 1);
      init(bar_p + 8 * b, soft_warps * 32);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *dead = 0;
    *strange = 0;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm0 + P::kFlags), "n"(P::kTm) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  Walk w;
  if (W.whole) {
    const int b = worker / A.Hkv, nt = tiles_of(A, b);
    w = Walk{b, worker - b * A.Hkv, 0, nt, nt};
  } else {
    w = walk_of(A, worker, W.workers);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = __shfl_sync(0xffffffffu, *tm_slot, 0);

  if (warp >= kSoft / 32 && warp < (kSoft + kLoadK + kLoadV) / 32) {
    // ---- copies ------------------------------------------------------------------------------------------------------------------------------
    const bool values = warp >= (kSoft + kLoadK) / 32;
    const int me = tid - kSoft - kLoadK;        // of those that copy values
    // rows of a copy, copies of a tile, tiles of a look-up (below): powers of two
    const int box = min(A.bs, kKeys), box_bits = __ffs(box) - 1, page_bits = 6 - box_bits, n_pages = 1 << page_bits, ahead = 32 >> page_bits;
    const uint32_t bar_in = values ? bar_v : bar_k, bar_free = values ? bar_o : bar_ke, bufs = sm0 + (values ? P::kV : P::kK);
    const CUtensorMap* map = values ? &v_map : &k_map;
    for (int i = 0; w.left > 0;) {
      const int b = w.b, g = w.g, run = w.run(), t0 = w.t;
      int keys, n;
      lengths(A, b, &keys, &n);
      const int32_t* table = A.block_tables + static_cast<int64_t>(b) * A.table_stride;
      // 32 pages at a time, the next ones under way: of tile at + lane / n_pages; -1: none, behind the pool (copies bring zeros): outside it
      auto look_up = [&](int at) -> int {
        const int t = at + (lane >> page_bits), j = t * kKeys + ((lane & (n_pages - 1)) << box_bits), col = A.bs > kKeys ? j / A.bs : j >> box_bits;
        const int page = col < A.table_cols ? table[col] : 0;       // (asked for before it is known how many keys there are)
        if (t >= t0 + run || j >= keys) return -1;
        return page < 0 || page >= A.max_blocks ? static_cast<int>(A.max_blocks) : page;
      };
      int pages = look_up(t0), later = look_up(t0 + ahead);
      for (int x = 0; x < run; ++x, ++i) {
        const int in = x & (ahead - 1);
        if (x > 0 && in == 0) {
          pages = later;
          later = look_up(t0 + x + ahead);
        }
        auto free_again = [&] {
          if (i >= NB) bar_wait(bar_free + 8 * (i % NB), (i / NB - 1) & 1, dead);
        };
        const uint32_t base = bufs + (i % NB) * (D / 64) * kBlk, bar = bar_in + 8 * (i % NB);
        const int j0 = (t0 + x) * kKeys, in_page = A.bs > kKeys ? j0 % A.bs : 0;
        if (!values || j0 + kKeys <= keys - n) {
          free_again();
          // One thread asks for all of them: a copy for each of several lanes took 150 clocks each, 1200 for a tile's keys.  The two warps of the values
          // take turns with the pages.
          const int turns = values ? 2 : 1, mine = values ? me / 32 : 0;
          const int there = __popc(__ballot_sync(0xffffffffu, lane >> page_bits == in && (lane & (n_pages - 1) & (turns - 1)) == mine && pages >= 0));
          if (there > 0 && elect_one())
            asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(there * (D / 64) * box * 128) : "memory");
          __syncwarp();
          for (int y = mine; y < n_pages; y += turns) {
            const int page = __shfl_sync(0xffffffffu, pages, (in << page_bits) + y);
            if (page < 0) break;
            const int row = (page * A.Hkv + g) * A.bs + in_page;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) copy_box(base + c * kBlk + y * box * 128, map, 64 * c, row, bar);
          }
        } else {
          // all loads before the buffer is free and the first store
          constexpr int kCh = D / 8, kPer = kKeys * kCh / kLoadV;
          int4 v[kPer];
          uint32_t most = 0;
#pragma unroll
          for (int u = 0; u < kPer; ++u) {
            const int c = me + u * kLoadV, key = c / kCh, ch = c - key * kCh;
            const int page = __shfl_sync(0xffffffffu, pages, (in << page_bits) + (key >> box_bits));
            v[u] = make_int4(0, 0, 0, 0);
            if (j0 + key < keys && page < A.max_blocks)
              v[u] = *reinterpret_cast<const int4*>(static_cast<const T*>(A.v_pool) + ((static_cast<int64_t>(page) * A.Hkv + g) * A.bs + in_page + (key & (box - 1))) * D + ch * 8);
          }
#pragma unroll
          for (int u = 0; u < kPer; ++u) most = magnitudes<T>(v[u].x, magnitudes<T>(v[u].y, magnitudes<T>(v[u].z, magnitudes<T>(v[u].w, most))));
          if (no_number<T>(most)) {       // hardly ever; the context's stay (every row sees them)
            *strange = 1;
#pragma unroll
            for (int u = 0; u < kPer; ++u)
              if (j0 + (me + u * kLoadV) / kCh >= keys - n)
                v[u] = make_int4(numbers_only<T>(v[u].x), numbers_only<T>(v[u].y), numbers_only<T>(v[u].z), numbers_only<T>(v[u].w));
          }
          free_again();
#pragma unroll
          for (int u = 0; u < kPer; ++u) {
            const int c = me + u * kLoadV, key = c / kCh, ch = c - key * kCh;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(line(base, key, ch, kKeys)), "r"(v[u].x), "r"(v[u].y), "r"(v[u].z), "r"(v[u].w) : "memory");
          }
          fence_smem_to_mma();
        }
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
      }
      w.skip(A, run);
    }
  } else if (warp == kNT / 32 - 1) {
    // ---- products ----------------------------------------------------------------------------------------------------------------------------
    auto scores = [&](int i) {
      const uint32_t k = sm0 + P::kK + (i % NB) * (D / 64) * kBlk;
      bar_wait(bar_k + 8 * (i % NB), (i / NB) & 1, dead);
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        mma_ss(tm + (i & 1) * kKeys, operand(sm0 + P::kQ + (kk >> 2) * (kRows * 128) + (kk & 3) * 32, 16, 1024),
               operand(k + (kk >> 2) * kBlk + (kk & 3) * 32, 16, 1024), instr<T>(kKeys, false), kk > 0);
      mma_commit(bar_s + 8 * (i & 1));
      mma_commit(bar_ke + 8 * (i % NB));
    };
    int i = 0;
    for (int seg = 0; w.left > 0; ++seg) {
      const int run = w.run();
      bar_wait(bar_q, seg & 1, dead);       // queries are in, the rows before them out
      tc_fence_after();
      scores(i);
      for (int x = 0; x < run; ++x, ++i) {
        if (x + 1 < run) {
          // S of the next tile goes where P of the one before is being read
          if (x > 0) bar_wait(bar_o + 8 * ((i - 1) % NB), ((i - 1) / NB) & 1, dead);
          scores(i + 1);
        }
        bar_wait(bar_v + 8 * (i % NB), (i / NB) & 1, dead);
        bar_wait(bar_p + 8 * (i & 1), (i >> 1) & 1, dead);
        tc_fence_after();
        const uint32_t v = sm0 + P::kV + (i % NB) * (D / 64) * kBlk;
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          mma_ts(tm + P::kO, tm + (i & 1) * kKeys + 8 * kk, operand(v + kk * 2048, kBlk, 1024), instr<T>(D, true), x > 0 || kk > 0);
        mma_commit(bar_o + 8 * (i % NB));
      }
      w.skip(A, run);
    }
    __syncwarp();
  } else if (warp < soft_warps) {
    // ---- softmax: thread = row ---------------------------------------------------------------------------------------------------------------
    const int my_row = warp % kRowWarps * 32 + lane, part = warp / kRowWarps, node = (row0 + my_row) / rep;       // part: of the keys
    const uint32_t tm_row = tm + (static_cast<uint32_t>(32 * warp) << 16);
    const float k2 = A.scale > 0.f ? A.scale * kLog2e : 1.f;       // weight = 2^(s k2 - m)
    const int per = W.rows;
    const float per_rep = 1.0f / rep;
    auto node_of = [&](int row) { return static_cast<int>((row + 0.5f) * per_rep); };        // (exact: rows have 18 bits; a division takes a hundred clocks)
    const int whole_b = w.b, whole_g = w.g;
    int i = 0;
    while (w.left > 0) {
      const int b = w.b, g = w.g, t0 = w.t, run = w.run();
      int keys, n;
      uint64_t seen = node < A.nodes ? static_cast<uint64_t>(A.visible[b * A.visible_stride + node]) : 0ull;
      lengths(A, b, &keys, &n);
      const int base = keys - n;
      const bool live = node < n;
      if (!live) seen = 0;
      if (n < 64) seen &= (1ull << n) - 1;
      {
        constexpr int kCh = D / 8;
        const T* q = static_cast<const T*>(A.q) + b * A.q_batch_stride;
#pragma unroll 8
        for (int u = 0; u < kCh; ++u) {
          const int c = lane + u * 32, r = c / kCh, ch = c % kCh, at = row0 + warp % kRowWarps * 32 + r;       // a warp's rows by itself
          const int t = node_of(at), h = g * rep + at - t * rep;
          const bool in = t < n;
          cp16(line(sm0 + P::kQ, 32 * warp + r, ch, kRows), in ? q + t * A.q_node_stride + static_cast<int64_t>(h) * D + ch * 8 : q, in);
        }
        cp_commit();
        cp_wait<0>();
        fence_smem_to_mma();
        tc_fence_before();
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_q) : "memory");
      }
      float m_ref = -INFINITY, l = 0.f;     // a power of two that the weights are relative to; -inf until the row sees a key
      bool ok = true;
      for (int x = 0; x < run; ++x, ++i) {
        const int j0 = (t0 + x) * kKeys;
        ok = bar_wait(bar_s + 8 * (i & 1), (i >> 1) & 1, dead) && ok;
        tc_fence_after();
        float s[kMine];
        if constexpr (SPLIT == 1) {
          tm_ld32(*reinterpret_cast<float(*)[32]>(s), tm_row + (i & 1) * kKeys);
          tm_ld32(*reinterpret_cast<float(*)[32]>(s + 32), tm_row + (i & 1) * kKeys + 32);
        } else if constexpr (SPLIT == 2) {
          tm_ld32(*reinterpret_cast<float(*)[32]>(s), tm_row + (i & 1) * kKeys + 32 * part);
        } else {
          tm_ld16(*reinterpret_cast<float(*)[16]>(s), tm_row + (i & 1) * kKeys + 16 * part);
        }
        tc_wait_ld();
        if (!(A.scale > 0.f)) {
#pragma unroll
          for (int c = 0; c < kMine; ++c) s[c] *= A.scale * kLog2e;
        }
        if (j0 + kKeys > base) {        // bit c: key j0 + c is seen
          const int past = base - j0;
          uint64_t keep = past > 0 ? (seen << past) | ((1ull << past) - 1) : (past > -64 ? seen >> -past : 0ull);
          if (SPLIT > 1) keep >>= part * kMine;
          const uint32_t half[2] = {static_cast<uint32_t>(keep), static_cast<uint32_t>(keep >> 32)};
#pragma unroll
          for (int c = 0; c < kMine; ++c)
            if (!(half[c >> 5] >> (c & 31) & 1)) s[c] = -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < kMine - 4; c += 8) {
#pragma unroll
          for (int u = 0; u < 4; ++u) mx[u] = max3(mx[u], s[c + u], s[c + 4 + u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = fmaxf(mx[u], s[kMine - 4 + u]);
        const float m_new = max3(mx[0], mx[1], fmaxf(mx[2], mx[3])) * k2;
        // the reference moves once the maximum is 2^8 above it: weights keep their digits wherever they lie, sums and outputs are fp32
        const bool grow = m_new > m_ref + 8.f;
        const float corr = grow ? exp2_fast(m_ref - m_new) : 1.0f;      // 0 where nothing was seen before
        if (grow) m_ref = m_new;
        if (x > 0 && __any_sync(0xffffffffu, grow)) {
          ok = bar_wait(bar_o + 8 * ((i - 1) % NB), ((i - 1) / NB) & 1, dead) && ok;
          tc_fence_after();
          scale_rows<D, 16>(tm_row + P::kO, corr);
        }
        const f32x2 kk = both(k2), mm = both(m_ref == -INFINITY ? 0.f : -m_ref);      // a row that sees no key yet keeps weights 0
        f32x2 sum[2] = {0ull, 0ull};
        uint32_t p[32];
#pragma unroll
        for (int c = 0; c < kMine; c += 2) {
          float u = s[c], v = s[c + 1];
          scale_shift(u, v, kk, mm);
          u = exp2_fast(u);
          v = exp2_fast(v);
          sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], pair(u, v));
          p[c >> 1] = pack2<T>(u, v);
          if constexpr (SPLIT == 1) {
            if (c % 32 == 30) tm_st16(tm_row + (i & 1) * kKeys + c / 32 * 16, *reinterpret_cast<uint32_t(*)[16]>(p + c / 32 * 16));
          }
        }
        if constexpr (SPLIT > 1) {      // the other warps' keys: 0
          uint32_t z[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) z[c] = SPLIT == 4 ? ((c < 8) == (part % 2 == 0) ? p[c & 7] : 0u) : p[c];
          uint32_t none[16] = {};
          const bool second = SPLIT == 4 ? part >= 2 : part == 1;
          tm_st16(tm_row + (i & 1) * kKeys + (second ? 16 : 0), z);
          tm_st16(tm_row + (i & 1) * kKeys + (second ? 0 : 16), none);
        }
        float some[4];
        apart(some[0], some[1], sum[0]);
        apart(some[2], some[3], sum[1]);
        l = fmaf(l, corr, (some[0] + some[1]) + (some[2] + some[3]));
        tc_wait_st();
        tc_fence_before();
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_p + 8 * (i & 1)) : "memory");
      }
      ok = bar_wait(bar_o + 8 * ((i - 1) % NB), ((i - 1) / NB) & 1, dead) && ok;
      tc_fence_after();
      ok = ok && !*dead;
      const bool whole = t0 == 0 && run == w.nt, odd = *strange != 0;
      const int64_t piece = (static_cast<int64_t>(worker) * W.blocks + block) * 2 + (t0 == 0);
      auto others_too = [&] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
      float scaled = 1.f;      // this warp's output to the row's common reference
      if constexpr (SPLIT > 1) {
        float2* ml = reinterpret_cast<float2*>(sm + P::kK - 1024);        // (of the room below)
        ml[tid] = make_float2(m_ref, ok ? l : NAN);
        others_too();
        float top = -INFINITY;
#pragma unroll
        for (int y = 0; y < SPLIT; ++y) top = fmaxf(top, ml[my_row + y * (kRows / SPLIT)].x);
        l = 0.f;
#pragma unroll
        for (int y = 0; y < SPLIT; ++y) {
          const float2 one = ml[my_row + y * (kRows / SPLIT)];
          l = fmaf(one.y, one.x == -INFINITY ? 0.f : exp2_fast(one.x - top), l);
        }
        scaled = m_ref == -INFINITY ? 0.f : exp2_fast(m_ref - top);
        m_ref = top;
        ok = l == l;
      }
      const float f = !whole ? 1.f : ok ? (l == 0.f ? 0.f : 1.0f / l) : NAN;
      if (!whole && part == 0) W.ml[piece * per + my_row] = make_float2(m_ref, ok ? l : NAN);
      T* out = static_cast<T*>(A.out) + static_cast<int64_t>(b) * A.nodes * A.Hq * D;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        constexpr int kCols = 32 / SPLIT;       // of the 32 that this warp finishes, from c + part * kCols on
        float o[32];
        __syncwarp();
        tm_ld32(o, tm_row + P::kO + c);
        tc_wait_ld();
        if constexpr (SPLIT > 1) {
          // [part][column / 4][row] of four columns
          constexpr int kSet = kRows / SPLIT;
          float4* all = reinterpret_cast<float4*>(sm + P::kQ) + (D == 128 && c % 64 ? 32 * kSet * SPLIT / 4 : 0);        // in turns, where there is room for two
          if (D == 64 || c == 0) others_too();
#pragma unroll
          for (int u = 0; u < 32; u += 4) all[(part * 8 + u / 4) * kSet + my_row] = make_float4(o[u] * scaled, o[u + 1] * scaled, o[u + 2] * scaled, o[u + 3] * scaled);
          others_too();
#pragma unroll
          for (int u = 0; u < kCols; u += 4) {
            float4 sum = all[(part * kCols + u) / 4 * kSet + my_row];
#pragma unroll
            for (int y = 1; y < SPLIT; ++y) {
              const float4 more = all[(y * 8 + (part * kCols + u) / 4) * kSet + my_row];
              sum.x += more.x, sum.y += more.y, sum.z += more.z, sum.w += more.w;
            }
            o[u] = sum.x, o[u + 1] = sum.y, o[u + 2] = sum.z, o[u + 3] = sum.w;
          }
        }
        const int c0 = c + part * kCols;
        if (odd && live) {
          float other[kCols];      // (an array that a function sees is kept in memory)
#pragma unroll
          for (int u = 0; u < kCols; ++u) other[u] = o[u];
          add_no_numbers<T, D>(other, A, b, g, base, t0 * kKeys, min((t0 + run) * kKeys, keys), seen, c0, kCols);
#pragma unroll
          for (int u = 0; u < kCols; ++u) o[u] = other[u];
        }
        if (!whole) {
#pragma unroll
          for (int u = 0; u < kCols; u += 4) W.o[(piece * (D / 4) + (c0 + u) / 4) * per + my_row] = make_float4(o[u], o[u + 1], o[u + 2], o[u + 3]);
        } else {
#pragma unroll
          for (int u = 0; u < kCols; u += 8) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = pack2<T>(o[u + 2 * e] * f, o[u + 2 * e + 1] * f);
            if constexpr (SPLIT == 1) {
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(line(sm0 + P::kQ, tid, (c + u) / 8, kRows)), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
            } else if (live) {
              const int t = node, h = g * rep + row0 + my_row - t * rep;
              *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(t) * A.Hq + h) * D + c0 + u) = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
        }
      }
      if (SPLIT == 1 && whole) {      // from where the warp's queries were (they have been read), rows side by side
        __syncwarp();
        constexpr int kCh = D / 8;
#pragma unroll 4
        for (int u = 0; u < kCh; ++u) {
          const int c = lane + u * 32, r = c / kCh, ch = c % kCh, at = row0 + 32 * warp + r, t = node_of(at), h = g * rep + at - t * rep;
          if (t < n) {
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(line(sm0 + P::kQ, 32 * warp + r, ch, kRows)) : "memory");
            *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(t) * A.Hq + h) * D + ch * 8) = v;
          }
        }
      }
      if constexpr (SPLIT > 1) others_too();       // the next queries go where the outputs were
      __syncwarp();
      w.skip(A, run);
    }
    if (W.whole) {        // rows without a node
      int keys, n;
      lengths(A, whole_b, &keys, &n);
      constexpr int kCh = D / 8;
      for (int c = n < A.nodes ? tid : kRows * kCh; c < kRows * kCh; c += soft_warps * 32) {
        const int at = row0 + c / kCh, t = node_of(at);
        if (t >= n && t < A.nodes)
          *reinterpret_cast<uint4*>(static_cast<T*>(A.out) + ((static_cast<int64_t>(whole_b) * A.nodes + t) * A.Hq + whole_g * rep + at - t * rep) * D + c % kCh * 8) = make_uint4(0, 0, 0, 0);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*dead) {      // a wait gave up: what is still under way gets 10 ms to end before its memory is another's
    for (const long long t0 = clock64(); clock64() - t0 < 20000000ll;) {}
  }
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(P::kTm));
}

// One CTA per (sequence and kv head, 32 rows, a part of the columns): what the workers' ends cut in pieces is put together, rows without a node become 0.
// Bound by the latency of its loads: all that it needs before the pieces is done before the kernel ahead ends, and pieces are asked for several at a
// time (one after another: 7 us behind a walk of three tiles, and 11 behind the 64 sequences of 2k).
template <typename T, int D, int PER>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeAttn A, const Shares W) {
  const int b = blockIdx.x / A.Hkv, g = blockIdx.x - b * A.Hkv, rep = A.Hq / A.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y * 32 + lane, t = row / rep, h = g * rep + row - t * rep;
  int keys, n, before, all;
  lengths(A, b, &keys, &n);
  const int nt = n > 0 ? (keys + kKeys - 1) / kKeys : 0;
  tiles_before(A, Lookup(A), b, &before, &all);
  const int share = share_of(all * A.Hkv, W.workers), from = before * A.Hkv + g * nt;
  const int first = from / share, last = nt > 0 ? (from + nt - 1) / share : first;
  const bool live = t < n;
  const bool nothing = row >= A.nodes * rep || (live && first == last);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (__all_sync(0xffffffffu, nothing)) return;
  const int in_block = row % kRows, block = row / kRows, c0 = (blockIdx.z * 8 + warp) * PER;
  auto piece_of = [&](int p) { return (static_cast<int64_t>(p) * W.blocks + block) * 2 + (p == first); };
  float top = -INFINITY, sum = 0.f;
  bool odd = false;
  float4 o[PER];
#pragma unroll
  for (int c = 0; c < PER; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live && !nothing) {
    constexpr int kAhead = PER == 1 ? 16 : 8 / PER;
    for (int p0 = first; p0 <= last; p0 += kAhead) {
      float2 ml[kAhead];
      float4 v[kAhead][PER];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (p0 + u > last) continue;
        const int64_t piece = piece_of(p0 + u);
        ml[u] = W.ml[piece * W.rows + in_block];
#pragma unroll
        for (int c = 0; c < PER; ++c) v[u][c] = W.o[(piece * (D / 4) + c0 + c) * W.rows + in_block];
      }
      float now = top;
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (p0 + u <= last) {
          odd = odd || ml[u].y != ml[u].y;
          now = fmaxf(now, ml[u].x);
        }
      if (now == -INFINITY) continue;
      const float was = top == -INFINITY ? 0.f : exp2_fast(top - now);
      top = now;
      sum *= was;
#pragma unroll
      for (int c = 0; c < PER; ++c) o[c].x *= was, o[c].y *= was, o[c].z *= was, o[c].w *= was;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (p0 + u > last || ml[u].x == -INFINITY) continue;
        const float k = exp2_fast(ml[u].x - now);
        sum = fmaf(ml[u].y, k, sum);
#pragma unroll
        for (int c = 0; c < PER; ++c)
          o[c].x = fmaf(v[u][c].x, k, o[c].x), o[c].y = fmaf(v[u][c].y, k, o[c].y), o[c].z = fmaf(v[u][c].z, k, o[c].z), o[c].w = fmaf(v[u][c].w, k, o[c].w);
      }
    }
  }
  if (nothing) return;
  const float f = odd ? NAN : (sum == 0.f ? 0.f : 1.0f / sum);
  T* out = static_cast<T*>(A.out) + ((static_cast<int64_t>(b) * A.nodes + t) * A.Hq + h) * D + c0 * 4;
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const uint2 y = live ? make_uint2(pack2<T>(o[c].x * f, o[c].y * f), pack2<T>(o[c].z * f, o[c].w * f)) : make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>(out + c * 4) = y;
  }
}

// The pool as rows, fetched in boxes of 64 columns x a page (or 64 rows of one); rows behind the pool read as zeros.  Made for the launch and not kept.
template <typename T>
bool pool_map(CUtensorMap* map, const void* pool, const TreeAttn& A) {
  const Encode encode = tensor_map_encode();
  if (!encode) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(A.D), static_cast<cuuint64_t>(A.max_blocks * A.Hkv * A.bs)}, strides[1] = {2ull * A.D};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(std::min(A.bs, kKeys))}, step[2] = {1, 1};
  return encode(map, std::is_same_v<T, __nv_bfloat16> ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(pool),
                dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

Shares shares_of(int nodes, int Hq, int Hkv) {
  Shares W{};
  const int rows = nodes * (Hq / Hkv);
  W.blocks = (rows + kRows - 1) / kRows;
  W.rows = std::min(kRows, (rows + 31) / 32 * 32);
  W.workers = std::max(1, kCtasPerSm * kNumSMs / W.blocks);
  return W;
}
// Walks of up to eight tiles are not divided: a second launch costs the host 5 us and the device 2, each tile here one.  (One sequence at 160 behind
// 8 kv heads of 128, a call after the other: undivided 16.9 us, divided 20.4.)
bool whole_walks(int B, int nodes, int Hq, int Hkv, int bs, int table_cols) {
  return static_cast<int64_t>(table_cols) * bs <= B200_TREE_SHORT_KEYS && static_cast<int64_t>(B) * Hkv * shares_of(nodes, Hq, Hkv).blocks <= INT32_MAX;
}
size_t sums_bytes(const Shares& W) { return static_cast<size_t>(W.workers) * W.blocks * 2 * W.rows * sizeof(float2); }

bool tiles_serve(int Hq, int Hkv, int D, int bs, int dtype) {
  return (dtype == B200_DTYPE_BF16 || dtype == B200_DTYPE_F16) && (D == 64 || D == 128) && ((bs >= 8 && kKeys % bs == 0) || bs % kKeys == 0) && Hq / Hkv <= 1 << 12;
}

template <typename T, int D>
int launch_tiles(const TreeAttn& A, const CUtensorMap& k_map, const CUtensorMap& v_map, void* workspace, cudaStream_t stream) {
  const char* name = "b200_paged_tree_attn";
  Shares W = shares_of(A.nodes, A.Hq, A.Hkv);
  W.ml = static_cast<float2*>(workspace);
  W.o = reinterpret_cast<float4*>(static_cast<char*>(workspace) + sums_bytes(W));
  const int rows = A.nodes * (A.Hq / A.Hkv);
  W.whole = whole_walks(A.B, A.nodes, A.Hq, A.Hkv, A.bs, A.table_cols);
  if (W.whole) W.workers = A.B * A.Hkv;
  auto kern = rows <= 32 ? tree_attn_kernel<T, D, 4> : rows <= 64 ? tree_attn_kernel<T, D, 2> : tree_attn_kernel<T, D, 1>;
  constexpr int smem = Plan<D>::kEnd + 1024;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  kern<<<W.workers * W.blocks, kNT, smem, stream>>>(A, W, k_map, v_map);
  if (int rc = check_launch(name)) return rc;
  if (W.whole) return 0;
  cudaLaunchConfig_t cfg{};
  // columns are divided while there are fewer CTAs than SMs
  constexpr int kMost = D / 32;
  const unsigned groups = static_cast<unsigned>(rows + 31) / 32;
  const bool divided = static_cast<int64_t>(A.B) * A.Hkv * groups < kNumSMs;
  cfg.gridDim = dim3(static_cast<unsigned>(A.B) * A.Hkv, groups, divided ? kMost : 1);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = divided ? cudaLaunchKernelEx(&cfg, tree_merge_kernel<T, D, 1>, A, static_cast<const Shares>(W))
                                : cudaLaunchKernelEx(&cfg, tree_merge_kernel<T, D, kMost>, A, static_cast<const Shares>(W));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(static_cast<int>(e), "%s: %s", name, cudaGetErrorString(e));
  }
  return 0;
}

// Rows share their keys where block tables hold more tokens than this, or where there are more rows in all.  (fp32, heads of 64, 1 x 8 rows behind 200 / 400 /
// 800 / 1600 tokens: each by itself 9 / 14 / 26 / 43 us, sharing 10 / 16 / 16 / 16; 416 rows 14 / 23 / 42 / 75 and 16 / 25 / 24 / 33; 2048 rows behind 30: 32
// and 13, behind 1600: 340 and 54.)
constexpr int kRowsFromTokens = 512, kRowsFromRows = 1024;

template <typename T, int DM, int RW>
int launch_rows(const TreeAttn& A, cudaStream_t stream) {
  using P = RowsPlan<T, DM, RW>;
  const char* name = "b200_paged_tree_attn";
  const int blocks = (A.nodes * (A.Hq / A.Hkv) + P::kRowsOf - 1) / P::kRowsOf;
  const int64_t units = static_cast<int64_t>(A.B) * A.Hkv * blocks, tiles = (static_cast<int64_t>(A.table_cols) * A.bs + P::kTile - 1) / P::kTile;
  int ctas = 1;
  while (ctas < 8 && units * ctas * 2 <= 2 * kNumSMs && tiles >= ctas * 4) ctas *= 2;
  if (units * ctas > INT32_MAX) return fail(B200_ESHAPE, "%s: %d sequences", name, A.B);
  auto kern = tree_attn_rows_kernel<T, DM, RW>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kEnd);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(units * ctas));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = P::kEnd;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, A, blocks);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(static_cast<int>(e), "%s: %s", name, cudaGetErrorString(e));
  }
  return 0;
}
template <typename T, int DM>
int launch_rows_of(const TreeAttn& A, cudaStream_t stream) {
  const int rows = A.nodes * (A.Hq / A.Hkv);
  return rows <= 8 ? launch_rows<T, DM, 1>(A, stream) : rows <= 16 ? launch_rows<T, DM, 2>(A, stream) : launch_rows<T, DM, 4>(A, stream);
}

template <typename T>
int launch_any(const TreeAttn& A, cudaStream_t stream) {
  if (A.D > kAnyMostD) return fail(B200_ESHAPE, "b200_paged_tree_attn: head size %d, at most %d", A.D, kAnyMostD);
  const bool vec = A.D * sizeof(T) % 16 == 0 && aligned16(A.k_pool);
  if (vec && aligned16(A.v_pool) && (static_cast<int64_t>(A.table_cols) * A.bs > kRowsFromTokens || static_cast<int64_t>(A.B) * A.nodes * A.Hq > kRowsFromRows))
    return A.D <= 64 ? launch_rows_of<T, 64>(A, stream) : A.D <= 128 ? launch_rows_of<T, 128>(A, stream) : launch_rows_of<T, 256>(A, stream);
  if (A.B > 65535) return fail(B200_ESHAPE, "b200_paged_tree_attn: %d sequences", A.B);
  auto kern = A.D <= 64 ? tree_attn_any_kernel<T, 2> : A.D <= 128 ? tree_attn_any_kernel<T, 4> : tree_attn_any_kernel<T, 8>;
  kern<<<dim3(A.Hq, A.nodes, A.B), kAnyWarps * 32, 0, stream>>>(A, vec);
  return check_launch("b200_paged_tree_attn");
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_paged_tree_attn_workspace(int B, int nodes, int Hq, int Hkv, int D, int block_size, int dtype) {
  if (nodes <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || block_size <= 0 || !tiles_serve(Hq, Hkv, D, block_size, dtype)) return 0;
  const Shares W = shares_of(nodes, Hq, Hkv);
  return sums_bytes(W) + static_cast<size_t>(W.workers) * W.blocks * 2 * W.rows * D * sizeof(float);
}

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
  // rows of 16-byte pieces, pages and rows whose numbers fit
  const bool pieces = aligned16(q) && aligned16(out) && aligned16(k_pool) && aligned16(v_pool) && q_batch_stride % 8 == 0 && q_node_stride % 8 == 0;
  if (tiles_serve(Hq, Hkv, D, block_size, dtype) && !(flags & B200_ATTN_FORCE_GENERIC) && pieces && max_blocks < INT32_MAX / (static_cast<int64_t>(Hkv) * block_size) - 1 &&
      (static_cast<int64_t>(table_cols) * block_size / kKeys + 1) * B < INT32_MAX / Hkv - 1024 && nodes * static_cast<int64_t>(Hq / Hkv) <= 32 * 65535) {
    if (workspace ? workspace_bytes < b200_paged_tree_attn_workspace(B, nodes, Hq, Hkv, D, block_size, dtype) : !whole_walks(B, nodes, Hq, Hkv, block_size, table_cols))
      return fail(B200_ENOSPC, "%s: workspace of %zu bytes", name, workspace_bytes);
    if (!aligned16(workspace)) return fail(B200_EINVAL, "%s: workspace not aligned to 16 bytes", name);
    CUtensorMap k_map, v_map;
    auto go = [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      if (!pool_map<T>(&k_map, k_pool, A) || !pool_map<T>(&v_map, v_pool, A)) return fail(B200_EINVAL, "%s: no tensor map of the pools", name);
      return D == 128 ? launch_tiles<T, 128>(A, k_map, v_map, workspace, s) : launch_tiles<T, 64>(A, k_map, v_map, workspace, s);
    };
    return dtype == B200_DTYPE_BF16 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<__half*>(nullptr));
  }
  switch (dtype) {
    case B200_DTYPE_F16: return launch_any<__half>(A, s);
    case B200_DTYPE_BF16: return launch_any<__nv_bfloat16>(A, s);
    default: return launch_any<float>(A, s);
  }
}

}  // extern "C"
