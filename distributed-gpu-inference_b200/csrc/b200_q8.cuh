// What the kernels of the cache in 8 bits share (b200_kv_q8.cu, b200_attn_q8.cu, b200_prompt_q8.cu): the codes, the cache, a sequence's rows.
//
// A page of a kv head holds block_size x D codes and has one scale for its keys and one for its values; a code stands for code * scale.
#pragma once
#include <cuda_fp8.h>

#include <type_traits>

#include "b200_common.cuh"

namespace b200 {
namespace q8 {

// Whole numbers -127 .. 127
struct Int8 {
  static constexpr float kMost = 127.f;
  static __device__ __forceinline__ float value(uint8_t c) { return static_cast<float>(static_cast<int8_t>(c)); }
  // ties to even; what is no number becomes 0
  static __device__ __forceinline__ uint8_t code(float y) {
    return static_cast<uint8_t>(static_cast<int8_t>(max(-127, min(127, __float2int_rn(y)))));
  }
};
// 8-bit floating point, 4 bits of exponent, 3 of mantissa, largest 448
struct E4m3 {
  static constexpr float kMost = 448.f;
  static __device__ __forceinline__ float value(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }
  // (what is no number becomes 0 here too: a row that does not see it must not meet it)
  static __device__ __forceinline__ uint8_t code(float y) { return __nv_cvt_float_to_fp8(y == y ? y : 0.f, __NV_SATFINITE, __NV_E4M3); }
};

constexpr float kLeastScale = 0x1p-60f;     // of a page that holds nothing but zeros, or numbers below 127 * 2^-60

// The values' scale of a page that is outside the pool.  Its codes are zeros whatever it is, but weights carry it, and those of a row are rounded to fp16 relative to the largest: far
// below ordinary scales, so that small values keep their digits beside it, and not so far that its weights leave fp32 beside large ones
constexpr float kAbsentScale = 0x1p-30f;

// the larger of two, no number if one is none
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// four codes as two pairs of fp16: (0, 1) and (2, 3), or across (0, 2) and (1, 3)
template <typename C, bool ACROSS>
__device__ __forceinline__ void halves(uint32_t codes, uint32_t& a, uint32_t& b) {
  if constexpr (std::is_same_v<C, Int8>) {
    const uint32_t u = codes ^ 0x80808080u, bias = 0x64806480u;       // 1024 + 128
    a = __byte_perm(u, 0x64646464u, ACROSS ? 0x4240 : 0x4140);
    b = __byte_perm(u, 0x64646464u, ACROSS ? 0x4341 : 0x4342);
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(a) : "r"(bias));
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(b) : "r"(bias));
  } else {
    uint32_t lo, hi;
    asm("{\n.reg .b16 x, y;\nmov.b32 {x, y}, %2;\ncvt.rn.f16x2.e4m3x2 %0, x;\ncvt.rn.f16x2.e4m3x2 %1, y;\n}\n" : "=r"(lo), "=r"(hi) : "r"(codes));
    a = ACROSS ? __byte_perm(lo, hi, 0x5410) : lo;
    b = ACROSS ? __byte_perm(lo, hi, 0x7632) : hi;
  }
}

struct Cache {
  uint8_t *k_pool, *v_pool;       // [max_blocks, Hkv, bs, D]
  float *k_scale, *v_scale;       // [max_blocks, Hkv]
  const int32_t* tables;
  int table_stride, table_cols;
  int Hkv, D, bs;
  int64_t max_blocks;
  // the pool's page behind a place of a sequence's table; -1 outside the table or the pool
  __device__ __forceinline__ int page(int b, int at) const {
    if (at < 0 || at >= table_cols) return -1;
    const int p = tables[static_cast<int64_t>(b) * table_stride + at];
    return p < 0 || p >= max_blocks ? -1 : p;
  }
  // keys of a sequence that a call may read
  __device__ __forceinline__ int keys(int context) const {
    return static_cast<int>(min(static_cast<int64_t>(max(context, 0)), static_cast<int64_t>(table_cols) * bs));
  }
};

// What is ahead on the stream has ended, and the kernel behind may take its places.  First thing in a kernel of launch_behind that runs behind any other.  Such a kernel is
// there while the one ahead writes what it will read: its loads are coherent ones (ld.global.nc is for what nobody writes as long as the kernel lives)
__device__ __forceinline__ void wait_for_ahead() {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// 16 and 8 bytes read once
__device__ __forceinline__ int4 ld_once16(const void* p) {
  int4 r;
  asm volatile("ld.global.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 ld_once8(const void* p) {
  uint2 r;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}

// The packed rows of a call: sequence b's new tokens are rows starts[b] .. starts[b + 1] - 1 (row b where starts is NULL), the last tokens of its
// context_lens[b]
struct Rows {
  const int32_t *starts, *context_lens;
  int B, n;
  // first row, number of rows, tokens of the sequence with them; numbers that do not fit one another give no rows
  __device__ __forceinline__ void of(int b, int* first, int* count, int* context) const {
    const int a = starts ? starts[b] : b, e = starts ? starts[b + 1] : b + 1, c = context_lens[b];
    const bool fits = a >= 0 && e >= a && e <= n && c >= e - a;
    *first = a;
    *count = fits ? e - a : 0;
    *context = c;
  }
};

}  // namespace q8

// host side

// A launch whose CTAs may take their places while the kernel ahead on the stream ends; each waits for it before it touches what that kernel writes.
// For appends, gathers and the merges of parts.  Not for the attention kernels: their CTAs are to lie evenly over the SMs, and do not where some still hold CTAs of
// the kernel ahead, and their merges could look nothing up before they end (4 x 2048 8.7 -> 11.8 us, 32 x 2048 30 -> 38, ragged portions of 1 to 9 tokens 23 -> 28).
template <typename... P, typename... A>
int launch_behind(const char* name, void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(static_cast<int>(e), "%s: %s", name, cudaGetErrorString(e));
  }
  return 0;
}

inline int check_cache(const char* name, const q8::Cache& c, int codes) {
  if (codes != B200_CODES_INT8 && codes != B200_CODES_E4M3) return fail(B200_EINVAL, "%s: unsupported codes %d", name, codes);
  if (c.Hkv <= 0 || c.D <= 0 || c.bs <= 0 || c.max_blocks <= 0 || c.max_blocks > INT32_MAX || c.table_cols <= 0 || c.table_stride < 0)
    return fail(B200_EINVAL, "%s: bad sizes Hkv=%d D=%d block_size=%d max_blocks=%lld table of %d", name, c.Hkv, c.D, c.bs,
                static_cast<long long>(c.max_blocks), c.table_cols);
  return 0;
}

}  // namespace b200
