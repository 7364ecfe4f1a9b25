// What the cross-attention kernels share: the addressed tensors of one call.
#pragma once
#include "host_common.cuh"
#include "sm100_primitives.cuh"

namespace b200 {

struct CrossArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int32_t* kv_lens;
  long long q_st[3], k_st[3], v_st[3], o_st[3];  // batch, head, position, in elements
  int B, Hq, Hkv, Sq, Skv, group, dtype;
  float scale_log2;  // softmax scale times log2(e)
};

// Encoder states that batch row b may look at, 0..Skv.
__device__ __forceinline__ int cross_kv_len(const CrossArgs& a, int b) {
  if (!a.kv_lens) return a.Skv;
  const int n = a.kv_lens[b];
  return n < 0 ? 0 : (n < a.Skv ? n : a.Skv);
}

constexpr float kLn2 = 0.6931471805599453f;

cudaError_t launch_cross_simt(const CrossArgs& a, int D, cudaStream_t st);   // fp32 arithmetic
cudaError_t launch_cross_token(const CrossArgs& a, int D, cudaStream_t st);  // 16-bit types, up to 64 query rows per KV head
cudaError_t launch_cross_prompt(const CrossArgs& a, int D, cudaStream_t st); // 16-bit types, many query rows
cudaError_t cross_wait_timeouts(unsigned int* count);    // bounded waits that ran out, per kernel
cudaError_t cross_prompt_timeouts(unsigned int* count);

}  // namespace b200
