// Between the entry points of attention over a cache in 8 bits (b200_attn_q8.cu) and its kernels for several tokens per sequence (b200_prompt_q8.cu).
#pragma once
#include "b200_q8.cuh"

namespace b200 {
namespace q8 {

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
};

}  // namespace q8

size_t prompt_q8_workspace(int B, int max_new, int Hq, int Hkv, int D, int bs, int longest, int dtype);
bool prompt_q8_serves(const q8::PromptAttn& A, int max_new, int longest, int dtype);
int prompt_q8(const char* name, q8::PromptAttn A, int max_new, int longest, void* workspace, int codes, int dtype, cudaStream_t stream);

}  // namespace b200
