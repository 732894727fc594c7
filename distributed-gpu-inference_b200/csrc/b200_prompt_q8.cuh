// Between the entry points of attention over a cache in 8 bits (b200_attn_q8.cu) and its kernels for several tokens per sequence (b200_prompt_q8.cu).
#pragma once
#include "b200_q8.cuh"

namespace b200 {
namespace q8 {

// Quotients of whole numbers below 2^31 by a number that the host knows: with l = ceil(log2 d) and m = ceil(2^(31 + l) / d), n m / 2^(31 + l) is less than 1 / d above n / d.  (A division
// costs a kernel's beginning some 150 clocks, one behind the other.)
struct Divisor {
  unsigned m = 0;      // 0: by 1
  int s = 0;
  static Divisor by(int d) {
    Divisor x;
    if (d <= 1) return x;
    int l = 0;
    while ((1ll << l) < d) ++l;
    x.m = static_cast<unsigned>(((1ull << (31 + l)) + d - 1) / d), x.s = l - 1;
    return x;
  }
  __device__ __forceinline__ int of(int n) const { return m ? static_cast<int>(__umulhi(static_cast<unsigned>(n), m) >> s) : n; }
};

struct PromptAttn {
  Cache c;
  Rows r;
  void* out;
  const void* q;
  int64_t q_stride;
  int Hq;
  float scale;
  // set by the launch: query heads of a kv head, CTAs and rows of a sequence and kv head at most, parts of the keys and where their results go
  int G, blocks, max_rows, splits;
  float2* ml;
  float* acc;
  Divisor by_G, by_splits, by_heads, by_B, by_page;      // (of kv heads, of sequences, of groups of 16 keys to a page)
};

}  // namespace q8

size_t prompt_q8_workspace(int B, int max_new, int Hq, int Hkv, int D, int bs, int longest, int dtype);
bool prompt_q8_serves(const q8::PromptAttn& A, int max_new, int longest, int dtype);
int prompt_q8(const char* name, q8::PromptAttn A, int max_new, int longest, void* workspace, int codes, int dtype, cudaStream_t stream);

}  // namespace b200
