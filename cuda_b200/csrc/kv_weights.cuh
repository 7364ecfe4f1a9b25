// What the kernels of the accumulated weights share: the addressed tensors and the division of a call among CTAs.
#pragma once
#include "host_common.cuh"
#include "sm100_primitives.cuh"

namespace b200 {

struct WeightsArgs {
  const void* q;
  const uint8_t* kc;
  const uint8_t* ks;
  const int32_t *bt, *ctx, *cuq;
  const float* lse;
  float* scores;
  uint32_t* status;
  long long st_seq, st_head;
  int S, total_q, Hq, Hkv, group, D, page, max_blocks, num_blocks, max_tokens, q_dtype, k_format, scale_mode, causal, keep_old;
  int group_shift;  // log2(group), or -1
  int q_first;  // query row of the first sequence when there are no offsets
  float scale_log2, decay;
};

constexpr int kWgtSeqs = 1024;  // sequences per launch (their prefix sums live in shared memory)

// The plan of a CTA: its range of stages (of `tok_stage` tokens, `n_hg` head groups per sequence) and the prefix sums to find
// sequences by.
struct WeightsPlan {
  const int *pre, *lens;
  int w0, w1, s0;
};
template <int THREADS>
__device__ __forceinline__ WeightsPlan make_plan(const WeightsArgs& a, int tok_stage, int n_hg, int* pre, int* lens) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int cap = (int)min((long long)a.max_blocks * a.page, (long long)a.max_tokens);
  for (int s = tid; s < a.S; s += THREADS) {
    int n = a.ctx[s];
    if (n > cap) {
      if (a.status && blockIdx.x == 0) atomicOr(a.status, CUDA_LLM_ST_BAD_CTX);
      n = cap;
    }
    lens[s] = max(n, 0);
  }
  __syncthreads();
  if (tid < 32) {
    int sum = 0;
    if (lane == 0) pre[0] = 0;
    for (int s0 = 0; s0 < a.S; s0 += 32) {
      const int s = s0 + lane;
      int x = s < a.S ? (lens[s] + tok_stage - 1) / tok_stage * n_hg : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (s < a.S) pre[s + 1] = sum + x;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  __syncthreads();
  WeightsPlan p;
  p.pre = pre;
  p.lens = lens;
  const long long total = pre[a.S];
  p.w0 = (int)(total * blockIdx.x / gridDim.x);
  p.w1 = (int)(total * (blockIdx.x + 1) / gridDim.x);
  int lo = 0, hi = a.S - 1;  // the last sequence with pre[s] <= w0
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= p.w0) lo = mid;
    else hi = mid - 1;
  }
  p.s0 = lo;
  return p;
}

// One launch of the kernel for windows of a prompt (16-bit queries; `a`: up to kWgtSeqs sequences of up to `cap` tokens).
cudaError_t launch_kv_weights_window(const WeightsArgs& a, long long cap, int sms, cudaStream_t st);

}  // namespace b200
