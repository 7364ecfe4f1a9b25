// Accumulated attention weight of cached tokens: scores[s, h, t] = decay * old + sum_rows 2^(scale_log2 q . k_t - lse2).
#include <cmath>

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
  int S, total_q, Hq, Hkv, group, D, page, max_blocks, num_blocks, max_tokens, q_dtype, k_format, scale_mode, causal;
  float scale_log2, decay;
};

__device__ __forceinline__ float load_q(const void* q, size_t i, int dtype) {
  if (dtype == CUDA_LLM_F32) return static_cast<const float*>(q)[i];
  if (dtype == CUDA_LLM_F16) return __half2float(static_cast<const __half*>(q)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(q)[i]);
}

// One thread per cached token of one KV head; the queries of the sequence pass through shared memory eight rows at a time.
__global__ void __launch_bounds__(128) kv_weights_kernel(const WeightsArgs a) {
  constexpr int R = 8;
  __shared__ float sq[R][128];
  __shared__ float slse[R];
  const int s = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  const int cap = min(a.max_blocks * (long long)a.page, (long long)a.max_tokens);
  int ctx = a.ctx[s];
  if (ctx > cap) {
    if (a.status && blockIdx.x == 0 && h == 0 && tid == 0) atomicOr(a.status, CUDA_LLM_ST_BAD_CTX);
    ctx = cap;
  }
  int q0 = a.cuq ? a.cuq[s] : s, q1 = a.cuq ? a.cuq[s + 1] : s + 1;
  if (q0 < 0 || q1 < q0 || q1 > a.total_q) {
    if (a.status && blockIdx.x == 0 && h == 0 && tid == 0) atomicOr(a.status, CUDA_LLM_ST_BAD_QLEN);
    q0 = q1 = 0;
  }
  const int t0 = blockIdx.x * 128;
  if (t0 >= ctx) return;
  const int n_q = q1 - q0, rows = n_q * a.group, t = t0 + tid;
  const int blk = t < ctx ? a.bt[(size_t)s * a.max_blocks + t / a.page] : 0, off = t % a.page;
  bool live = t < ctx;
  if (live && (blk < 0 || blk >= a.num_blocks)) {
    if (a.status) atomicOr(a.status, CUDA_LLM_ST_BAD_BLOCK);
    live = false;
  }
  const size_t base = ((size_t)(live ? blk : 0) * a.Hkv + h) * a.D * a.page + off;
  float sum = 0.f;
  for (int r0 = 0; r0 < rows; r0 += R) {
    __syncthreads();
    for (int i = tid; i < R * a.D; i += 128) {
      const int r = r0 + i / a.D, d = i % a.D;
      sq[i / a.D][d] = r < rows ? load_q(a.q, ((size_t)(q0 + r / a.group) * a.Hq + h * a.group + r % a.group) * a.D + d, a.q_dtype) : 0.f;
    }
    if (tid < R && r0 + tid < rows) slse[tid] = a.lse[(size_t)(q0 + (r0 + tid) / a.group) * a.Hq + h * a.group + (r0 + tid) % a.group] * 1.4426950408889634f;
    __syncthreads();
    if (!live) continue;
    float acc[R] = {}, part[R];
    for (int b = 0; b < a.D / 32; ++b) {
#pragma unroll
      for (int r = 0; r < R; ++r) part[r] = 0.f;
      for (int d = b * 32; d < b * 32 + 32; ++d) {
        const size_t e = base + (size_t)d * a.page;
        float k;
        if (a.k_format == CUDA_LLM_KV_FP8_E4M3) k = f16x2_lo(e4m3x2_to_f16x2_lo(a.kc[e]));
        else if (a.k_format == CUDA_LLM_KV_F16) k = __half2float(reinterpret_cast<const __half*>(a.kc)[e]);
        else k = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.kc)[e]);
#pragma unroll
        for (int r = 0; r < R; ++r) part[r] = fmaf(k, sq[r][d], part[r]);
      }
      const float f = a.scale_mode == CUDA_LLM_SCALE_MX_E8M0 && a.ks
                          ? e8m0_to_f32(a.ks[(((size_t)blk * a.Hkv + h) * (a.D / 32) + b) * a.page + off]) : 1.f;
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r] = fmaf(part[r], f, acc[r]);
    }
    float f = a.scale_log2;
    const float* ks = reinterpret_cast<const float*>(a.ks);
    if (a.ks && a.scale_mode == CUDA_LLM_SCALE_PER_HEAD) f *= ks[h];
    if (a.ks && a.scale_mode == CUDA_LLM_SCALE_PER_BLOCK) f *= ks[(size_t)blk * a.Hkv + h];
    if (a.ks && a.scale_mode == CUDA_LLM_SCALE_PER_TOKEN) f *= ks[((size_t)blk * a.Hkv + h) * a.page + off];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = (r0 + r) / a.group;
      if (r0 + r < rows && (!a.causal || t < ctx - n_q + 1 + j) && slse[r] != -__builtin_huge_valf())
        sum += exp2f(fmaf(acc[r], f, -slse[r]));
    }
  }
  if (!live) return;
  float* sp = a.scores + s * a.st_seq + h * a.st_head + t;
  if (a.decay != 0.f && t < ctx - n_q) sum = fmaf(*sp, a.decay, sum);
  *sp = sum;
}

}  // namespace b200

using namespace b200;

extern "C" int cuda_llm_kv_accumulate_weights(const CudaLlmKvWeightsParams* p, void* stream) {
  if (!p) return refuse(CUDA_LLM_EINVAL, "params is null");
  if (p->num_seqs < 0 || p->total_q < 0 || p->max_tokens < 0) return refuse(CUDA_LLM_EINVAL, "sizes must not be negative");
  if (p->num_q_heads <= 0 || p->num_kv_heads <= 0 || p->num_q_heads % p->num_kv_heads)
    return refuse(CUDA_LLM_EINVAL, "num_q_heads must be a positive multiple of num_kv_heads");
  if (p->head_dim != 64 && p->head_dim != 128) return refuse(CUDA_LLM_EINVAL, "Only head_dim 64 and 128 supported");
  if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64) return refuse(CUDA_LLM_EINVAL, "Only page_size 16, 32 and 64 supported");
  if (p->q_dtype < CUDA_LLM_F32 || p->q_dtype > CUDA_LLM_BF16) return refuse(CUDA_LLM_EINVAL, "q_dtype must be fp32, fp16 or bf16");
  const bool kv16 = p->k_format == CUDA_LLM_KV_F16 || p->k_format == CUDA_LLM_KV_BF16;
  if (!kv16 && p->k_format != CUDA_LLM_KV_FP8_E4M3) return refuse(CUDA_LLM_EINVAL, "K must be E4M3, fp16 or bf16");
  if (kv16 && p->q_dtype != (p->k_format == CUDA_LLM_KV_F16 ? CUDA_LLM_F16 : CUDA_LLM_BF16))
    return refuse(CUDA_LLM_EINVAL, "a 16-bit cache needs queries of its own type");
  if (!kv16 && (p->scale_mode < CUDA_LLM_SCALE_PER_HEAD || p->scale_mode > CUDA_LLM_SCALE_MX_E8M0))
    return refuse(CUDA_LLM_EINVAL, "unknown scale mode");
  if (!(p->softmax_scale > 0.f) || !std::isfinite(p->softmax_scale))
    return refuse(CUDA_LLM_EINVAL, "softmax_scale must be positive and finite");
  if (!(p->decay >= 0.f && p->decay <= 1.f)) return refuse(CUDA_LLM_EINVAL, "decay must be between 0 and 1");
  if (p->num_seqs == 0 || p->max_tokens == 0 || p->max_blocks_per_seq == 0) return CUDA_LLM_OK;
  if (p->max_blocks_per_seq < 0 || p->num_blocks <= 0) return refuse(CUDA_LLM_EINVAL, "block table and pool must not be empty");
  if (p->num_seqs > 65535 || p->num_kv_heads > 65535) return refuse(CUDA_LLM_EINVAL, "more than 65535 sequences or KV heads");
  if (!p->key_cache || !p->block_tables || !p->context_lens || !p->scores || (!kv16 && !p->k_scale) ||
      (p->total_q > 0 && (!p->query || !p->lse)))
    return refuse(CUDA_LLM_EINVAL, "null tensor");
  if (!p->cu_q_lens && p->total_q != p->num_seqs) return refuse(CUDA_LLM_EINVAL, "query has more or fewer rows than sequences: pass cu_q_lens");
  if (((uintptr_t)p->query | (uintptr_t)p->key_cache | (uintptr_t)(kv16 ? nullptr : p->k_scale)) & 15)
    return refuse(CUDA_LLM_EALIGN, "query, cache and scales must be 16-byte aligned");
  if (((uintptr_t)p->block_tables | (uintptr_t)p->context_lens | (uintptr_t)p->cu_q_lens | (uintptr_t)p->lse | (uintptr_t)p->scores | (uintptr_t)p->status) & 3)
    return refuse(CUDA_LLM_EALIGN, "tables, lengths, lse, scores and status must be 4-byte aligned");
  int rc = check_current_device();
  if (rc != CUDA_LLM_OK) return rc;
  WeightsArgs a;
  a.q = p->query; a.kc = (const uint8_t*)p->key_cache; a.ks = kv16 ? nullptr : (const uint8_t*)p->k_scale;
  a.bt = p->block_tables; a.ctx = p->context_lens; a.cuq = p->cu_q_lens; a.lse = p->lse; a.scores = p->scores; a.status = p->status;
  a.st_seq = p->score_strides[0]; a.st_head = p->score_strides[1];
  a.S = p->num_seqs; a.total_q = p->total_q; a.Hq = p->num_q_heads; a.Hkv = p->num_kv_heads; a.group = a.Hq / a.Hkv;
  a.D = p->head_dim; a.page = p->page_size; a.max_blocks = p->max_blocks_per_seq; a.num_blocks = p->num_blocks;
  a.max_tokens = p->max_tokens; a.q_dtype = p->q_dtype; a.k_format = p->k_format; a.scale_mode = p->scale_mode;
  a.causal = p->is_causal ? 1 : 0; a.scale_log2 = p->softmax_scale * 1.4426950408889634f; a.decay = p->decay;
  const long long cap = (long long)a.max_blocks * a.page < a.max_tokens ? (long long)a.max_blocks * a.page : a.max_tokens;
  kv_weights_kernel<<<dim3((unsigned)((cap + 127) / 128), a.Hkv, a.S), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return cuda_result(cudaGetLastError(), "kv_weights_kernel launch");
}
