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

// Batch rows in the order of falling length: blocks of the longest start first and the short ones fill the last wave.
// (Block-uniform; every thread counts for one row how many go before it.  `pick`: a word of shared memory.)
template <int THREADS>
__device__ __forceinline__ int longest_first(const CrossArgs& c, int z, volatile int* pick) {
  if (!c.kv_lens || c.B == 1 || c.B > THREADS) return z;
  const int b = threadIdx.x;
  if (b < c.B) {
    const int n = cross_kv_len(c, b);
    int before = 0;
    for (int x = 0; x < c.B; ++x) {
      const int y = cross_kv_len(c, x);
      before += (y > n || (y == n && x < b)) ? 1 : 0;
    }
    if (before == z) *pick = b;
  }
  __syncthreads();
  return *pick;
}

// ---- clusters: the CTAs that share the states of one (sequence, KV head) and join their parts
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 dsmem_ld128(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [ra];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
  return v;
}
__device__ __forceinline__ float2 dsmem_ld64(uint32_t addr, uint32_t rank) {
  float2 v;
  asm volatile(
      "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %2, %3;\n\tld.shared::cluster.v2.f32 {%0, %1}, [ra];\n\t}"
      : "=f"(v.x), "=f"(v.y) : "r"(addr), "r"(rank) : "memory");
  return v;
}

constexpr int kMaxParts = 8;
struct JoinedWord {
  float4 x;    // sum of the parts' O, weighted
  float M, L;  // their common maximum and sum
};
// Four elements of one row from the parts of all CTAs: {m, l} of the row at `ml_at`, the elements at `o_at` (the same places in
// every CTA).  All loads first: one after another they would cost a remote latency each.
__device__ __forceinline__ JoinedWord join_parts(uint32_t ml_at, uint32_t o_at, int parts) {
  float2 ml[kMaxParts];
  float4 y[kMaxParts];
#pragma unroll
  for (int q = 0; q < kMaxParts; ++q) {
    ml[q] = make_float2(-__builtin_huge_valf(), 0.f);
    y[q] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (q < parts) {
      ml[q] = dsmem_ld64(ml_at, q);
      y[q] = dsmem_ld128(o_at, q);
    }
  }
  JoinedWord j;
  j.M = ml[0].x;
#pragma unroll
  for (int q = 1; q < kMaxParts; ++q) j.M = fmaxf(j.M, ml[q].x);
  const float ref = j.M == -__builtin_huge_valf() ? 0.f : j.M;
  j.L = 0.f;
  j.x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int q = 0; q < kMaxParts; ++q) {
    const float w = exp2f(ml[q].x - ref);
    j.L = fmaf(ml[q].y, w, j.L);
    j.x.x = fmaf(y[q].x, w, j.x.x);
    j.x.y = fmaf(y[q].y, w, j.x.y);
    j.x.z = fmaf(y[q].z, w, j.x.z);
    j.x.w = fmaf(y[q].w, w, j.x.w);
  }
  return j;
}

// CTAs per (sequence, KV head, row block): enough for two CTAs on every SM, at most 8 and at most one per `tiles`.  More parts even
// out lengths, fewer join less (bf16 token form, us for 1 / 2 / 4 parts where the rule says 1, 2, 2, 4): 512 pairs of
// 1000-4096 states 102 / 119 / 141, 160 pairs of 2000-8192 104 / 76 / 80, 256 pairs of 1000-4096 68 / 60 / 73, 128 pairs of
// 4096 - / 49 / 54.
inline int cross_parts(long long blocks, int tiles) {
  const int sms = current_sm_count();
  int parts = 1;
  while (parts < kMaxParts && parts * 2 <= tiles && blocks * parts < 2ll * sms) parts *= 2;
  return parts;
}

constexpr float kLn2 = 0.6931471805599453f;

cudaError_t launch_cross_simt(const CrossArgs& a, int D, cudaStream_t st);   // fp32 tensors
cudaError_t launch_cross_stream(const CrossArgs& a, int D, cudaStream_t st); // fp32 tensors, up to 16 query rows per KV head
cudaError_t launch_cross_token(const CrossArgs& a, int D, cudaStream_t st);  // 16-bit types, up to 64 query rows per KV head
cudaError_t launch_cross_prompt(const CrossArgs& a, int D, cudaStream_t st); // 16-bit types, many query rows
cudaError_t cross_wait_timeouts(unsigned int* count);    // bounded waits that ran out, per kernel
cudaError_t cross_prompt_timeouts(unsigned int* count);

}  // namespace b200
