// C entry of the cross attention: checks, strides, choice of the kernel.
#include "cross_attention.cuh"

#include <climits>
#include <cmath>

using namespace b200;

// The 16-bit kernels read their inputs through tensor maps, whose boxes step over positions: a map can hold one batch row or head for
// all (a dimension of one element), but not one position for all.
static bool take_strides(const int64_t* st, int B, int H, int S, int D, int eb, bool output, long long* out) {
  const int extent[3] = {B, H, S};
  if (eb == 2 && !output && S > 1 && st[2] == 0) return false;
  for (int i = 0; i < 3; ++i) {
    out[i] = extent[i] == 1 ? D : st[i];  // never multiplied by anything but 0
    if (out[i] < 0 || (out[i] * eb) % 16 || out[i] > (1ll << 36)) return false;
    if (output && extent[i] > 1 && out[i] < D) return false;
  }
  return true;
}

extern "C" int cuda_llm_cross_attention(const CudaLlmCrossAttentionParams* p, void* stream) {
  if (!p) return refuse(CUDA_LLM_EINVAL, "params is null");
  if (p->batch_size < 0 || p->q_len < 0 || p->kv_len < 0) return refuse(CUDA_LLM_EINVAL, "sizes must not be negative");
  if (p->num_q_heads <= 0 || p->num_kv_heads <= 0 || p->num_q_heads % p->num_kv_heads)
    return refuse(CUDA_LLM_EINVAL, "num_q_heads must be a positive multiple of num_kv_heads");
  if (p->head_dim != 64 && p->head_dim != 128) return refuse(CUDA_LLM_EINVAL, "Only head_dim 64 and 128 supported");
  if (p->dtype < CUDA_LLM_F32 || p->dtype > CUDA_LLM_BF16) return refuse(CUDA_LLM_EINVAL, "dtype must be fp32, fp16 or bf16");
  if (!(p->softmax_scale > 0.f) || !std::isfinite(p->softmax_scale))
    return refuse(CUDA_LLM_EINVAL, "softmax_scale must be positive and finite");
  if (p->batch_size == 0 || p->q_len == 0) return CUDA_LLM_OK;
  if (p->batch_size > 65535 || p->num_kv_heads > 65535) return refuse(CUDA_LLM_EINVAL, "more than 65535 batch rows or KV heads");
  const int group = p->num_q_heads / p->num_kv_heads;
  if ((long long)group * p->q_len > INT_MAX / 2 || p->kv_len > INT_MAX / 2)
    return refuse(CUDA_LLM_EINVAL, "more than 2^30 query rows of a KV head, or states");
  if (!p->q || !p->out || (p->kv_len > 0 && (!p->k || !p->v))) return refuse(CUDA_LLM_EINVAL, "null tensor");
  const int eb = p->dtype == CUDA_LLM_F32 ? 4 : 2;
  if (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->out) & 15)
    return refuse(CUDA_LLM_EALIGN, "q, k, v and out must be 16-byte aligned");
  if (((uintptr_t)p->lse | (uintptr_t)p->kv_lens) & 3) return refuse(CUDA_LLM_EALIGN, "lse and kv_lens must be 4-byte aligned");
  CrossArgs a;
  a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out; a.lse = p->lse; a.kv_lens = p->kv_lens;
  a.B = p->batch_size; a.Hq = p->num_q_heads; a.Hkv = p->num_kv_heads; a.Sq = p->q_len; a.Skv = p->kv_len;
  a.group = group; a.dtype = p->dtype;
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  const int D = p->head_dim;
  if (!take_strides(p->q_strides, a.B, a.Hq, a.Sq, D, eb, false, a.q_st) || !take_strides(p->k_strides, a.B, a.Hkv, a.Skv, D, eb, false, a.k_st) ||
      !take_strides(p->v_strides, a.B, a.Hkv, a.Skv, D, eb, false, a.v_st) || !take_strides(p->out_strides, a.B, a.Hq, a.Sq, D, eb, true, a.o_st))
    return refuse(CUDA_LLM_EALIGN, "strides must be multiples of 16 bytes, not negative, no less than head_dim for out, and not 0 for the positions of a 16-bit input");
  int rc = check_current_device();
  if (rc != CUDA_LLM_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // Which kernel: with few rows per KV head the states' bytes bound the call, with many the products.
  const long long rows = (long long)group * a.Sq, pairs = (long long)a.B * a.Hkv;
  if (a.dtype == CUDA_LLM_F32)
    return rows <= 16 ? cuda_result(launch_cross_stream(a, D, st), "cross_stream_kernel launch") : cuda_result(launch_cross_simt(a, D, st), "cross_simt_kernel launch");
  // 16 bit, 16 x 8 pairs of 4 heads (groups that are no power of two were not timed), 4096 states: 32 rows take 57 us streamed and 74 us on the tensor cores' 256-row blocks, 64 rows 96 and
  // 74 us.  Those blocks walk all states in turn: where they leave SMs idle, 64 rows are streamed as well.
  if (rows <= 32 || (rows <= 64 && pairs < current_sm_count() / 2)) return cuda_result(launch_cross_token(a, D, st), "cross_token_kernel launch");
  return cuda_result(launch_cross_prompt(a, D, st), "cross_prompt_kernel launch");
}

extern "C" int cuda_llm_cross_attention_wait_timeouts(uint32_t* count) {
  if (!count) return refuse(CUDA_LLM_EINVAL, "count is null");
  *count = 0;
  const int rc = check_current_device();
  if (rc != CUDA_LLM_OK) return rc;
  unsigned int token = 0, prompt = 0;
  // the copies below wait for the default stream alone, not for streams that run beside it
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cross_wait_timeouts(&token);
  if (e == cudaSuccess) e = cross_prompt_timeouts(&prompt);
  *count = token + prompt;
  return cuda_result(e, "reading the counters");
}
