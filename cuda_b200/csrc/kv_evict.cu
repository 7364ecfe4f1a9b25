// Eviction from a paged KV cache: which tokens stay (a selection by rank per sequence and KV head), and their move to the
// front of the same or of other pages.
#include "host_common.cuh"
#include "sm100_primitives.cuh"

namespace b200 {

struct EvictArgs {
  const float* scores;
  float* new_scores;
  const int32_t *bt, *new_bt, *ctx;
  int32_t *new_ctx, *kept;
  uint32_t* status;
  long long st_seq, st_head, nst_seq, nst_head;
  int S, Hkv, page, max_blocks, new_max_blocks, num_blocks, max_tokens, budget, sink, recent, in_place;
};

// tokens of sequence s that the table and the score row hold
__device__ __forceinline__ int evict_ctx(const EvictArgs& a, int s, bool report) {
  const int cap = (int)min((long long)a.max_blocks * a.page, (long long)a.max_tokens);
  int ctx = a.ctx[s];
  if (ctx > cap) {
    if (report && a.status) atomicOr(a.status, CUDA_LLM_ST_BAD_CTX);
    ctx = cap;
  }
  return max(ctx, 0);
}

// Scores as unsigned integers of the same order: NaN lowest, then -inf .. +inf (-0 and +0 alike), protected tokens on top.
__device__ __forceinline__ uint32_t rank_key(float x, bool is_protected) {
  if (is_protected) return 0xffffffffu;
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;

// One CTA per (KV head, sequence): the budget-th largest key by four passes over its bytes (histograms in shared memory),
// then the kept positions in order by a running prefix sum.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_prefix, s_left;
  __shared__ uint32_t warp_gt[32], warp_eq[32];
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ctx = evict_ctx(a, s, h == 0 && tid == 0);
  const int n_keep = min(ctx, a.budget);
  const float* sc = a.scores + s * a.st_seq + h * a.st_head;
  float* ns = a.new_scores ? a.new_scores + s * a.nst_seq + h * a.nst_head : nullptr;
  int32_t* kept = a.kept + ((size_t)s * a.Hkv + h) * a.budget;
  if (h == 0 && tid == 0) a.new_ctx[s] = n_keep;
  for (int i = n_keep + tid; i < a.budget; i += kSelThreads) kept[i] = -1;
  auto key_at = [&](int t) { return rank_key(sc[t], t < a.sink || t >= ctx - a.recent); };
  if (ctx <= a.budget) {
    for (int t = tid; t < ctx; t += kSelThreads) {
      kept[t] = t;
      if (ns) ns[t] = sc[t];
    }
    return;
  }
  if (tid == 0) {
    s_prefix = 0;
    s_left = (uint32_t)n_keep;
  }
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int t = tid; t < ctx; t += kSelThreads) {
      const uint32_t k = key_at(t);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t left = s_left;
      int b = 255;
      while (b > 0 && hist[b] < left) left -= hist[b--];
      s_left = left;
      s_prefix = prefix | ((uint32_t)b << shift);
    }
    __syncthreads();
  }
  const uint32_t edge = s_prefix, n_edge = s_left;  // keep all above the edge and the first n_edge on it
  uint32_t base_gt = 0, base_eq = 0;
  for (int t0 = 0; t0 < ctx; t0 += kSelThreads) {
    const int t = t0 + tid;
    const uint32_t k = t < ctx ? key_at(t) : 0u;
    const float x = t < ctx ? sc[t] : 0.f;
    const bool gt = t < ctx && k > edge, eq = t < ctx && k == edge;
    const uint32_t bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) {
      warp_gt[warp] = __popc(bg);
      warp_eq[warp] = __popc(be);
    }
    __syncthreads();  // and every score of this tile is read: new_scores may be scores
    uint32_t g = base_gt, e = base_eq;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) {
        g += warp_gt[w];
        e += warp_eq[w];
      }
      base_gt += warp_gt[w];
      base_eq += warp_eq[w];
    }
    g += __popc(bg & ((1u << lane) - 1));
    e += __popc(be & ((1u << lane) - 1));
    if (gt || (eq && e < n_edge)) {
      const uint32_t i = g + min(e, n_edge);
      kept[i] = t;
      if (ns) ns[i] = x;
    }
    __syncthreads();
  }
}

struct MoveTensor {
  void* p;
  int rows;     // rows of a (page, head): head_dim, head_dim / 2, head_dim / 32 or 1
  int task0;    // first 32-row slice of this tensor among all slices of a head
};
struct MoveArgs {
  EvictArgs e;
  MoveTensor t[4];
  int n_tensors, slices;
};

// One warp per (sequence, KV head, 32 rows of one tensor): it walks the new positions in groups of 16 tokens, a lane
// takes the group's 16 elements of one row.  Within a row old positions never lie before new ones, so walking
// upwards is safe in place, and no two warps touch the same row.
template <typename E>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const MoveTensor& mt, int s, int h, int row, int g0, int g_step) {
  const int ctx = evict_ctx(a, s, false), n = min(ctx, a.budget);
  if (a.in_place && ctx <= a.budget) return;
  const int32_t* kept = a.kept + ((size_t)s * a.Hkv + h) * a.budget;
  const int32_t* bt = a.bt + (size_t)s * a.max_blocks;
  const int32_t* nbt = a.new_bt + (size_t)s * a.new_max_blocks;
  E* p = static_cast<E*>(mt.p);
  for (int g = g0; g * 16 < n; g += g_step) {
    E x[16];
    uint32_t have = 0;
    for (int k = 0; k < 16; ++k) {
      const int i = g * 16 + k;
      if (i >= n) break;
      const int t = kept[i];
      if (t < 0 || t >= ctx) continue;
      const int blk = bt[t / a.page];
      if (blk < 0 || blk >= a.num_blocks) {
        if (a.status) atomicOr(a.status, CUDA_LLM_ST_BAD_BLOCK);
        continue;
      }
      x[k] = p[(((size_t)blk * a.Hkv + h) * mt.rows + row) * a.page + t % a.page];
      have |= 1u << k;
    }
    const int to = nbt[g * 16 / a.page];
    if (to < 0 || to >= a.num_blocks) {
      if (a.status) atomicOr(a.status, CUDA_LLM_ST_BAD_BLOCK);
      continue;
    }
    E* dst = p + (((size_t)to * a.Hkv + h) * mt.rows + row) * a.page + g * 16 % a.page;
    for (int k = 0; k < 16; ++k)
      if (have >> k & 1) dst[k] = x[k];
  }
}

template <typename EK, typename EV>
__global__ void __launch_bounds__(128) evict_move_kernel(const MoveArgs m) {
  const int task = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, h = blockIdx.y % m.e.Hkv, s = blockIdx.y / m.e.Hkv;
  if (task >= m.slices) return;
  int i = 0;
  while (i + 1 < m.n_tensors && task >= m.t[i + 1].task0) ++i;
  const int row = (task - m.t[i].task0) * 32 + lane;
  if (row >= m.t[i].rows) return;
  if (i == 0) move_rows<EK>(m.e, m.t[i], s, h, row, blockIdx.z, gridDim.z);
  else if (i == 1) move_rows<EK>(m.e, m.t[i], s, h, row, blockIdx.z, gridDim.z);
  else move_rows<EV>(m.e, m.t[i], s, h, row, blockIdx.z, gridDim.z);
}

}  // namespace b200

using namespace b200;

static int format_bytes(int f) { return f == CUDA_LLM_KV_F32 ? 4 : (f == CUDA_LLM_KV_F16 || f == CUDA_LLM_KV_BF16) ? 2 : 1; }

extern "C" int cuda_llm_kv_evict(const CudaLlmKvEvictParams* p, void* stream) {
  if (!p) return refuse(CUDA_LLM_EINVAL, "params is null");
  if (p->num_seqs < 0 || p->max_tokens < 0) return refuse(CUDA_LLM_EINVAL, "sizes must not be negative");
  if (p->num_kv_heads <= 0) return refuse(CUDA_LLM_EINVAL, "num_kv_heads must be positive");
  if (p->head_dim != 64 && p->head_dim != 128) return refuse(CUDA_LLM_EINVAL, "Only head_dim 64 and 128 supported");
  if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64) return refuse(CUDA_LLM_EINVAL, "Only page_size 16, 32 and 64 supported");
  const bool wide = p->k_format >= CUDA_LLM_KV_F16 && p->k_format <= CUDA_LLM_KV_F32;
  if (wide ? p->v_format != p->k_format
           : p->k_format != CUDA_LLM_KV_FP8_E4M3 || (p->v_format != CUDA_LLM_KV_FP8_E4M3 && p->v_format != CUDA_LLM_KV_FP4_E2M1))
    return refuse(CUDA_LLM_EINVAL, "K must be E4M3 with V in E4M3 or E2M1, or both fp16, bf16 or fp32");
  if (!wide) {
    if (p->scale_mode == CUDA_LLM_SCALE_PER_BLOCK)
      return refuse(CUDA_LLM_EINVAL, "per-block scales: tokens of pages with different scales cannot share a page without being quantised again");
    if (p->scale_mode != CUDA_LLM_SCALE_PER_HEAD && p->scale_mode != CUDA_LLM_SCALE_PER_TOKEN && p->scale_mode != CUDA_LLM_SCALE_MX_E8M0)
      return refuse(CUDA_LLM_EINVAL, "unknown scale mode");
    if (p->v_format == CUDA_LLM_KV_FP4_E2M1 && p->scale_mode != CUDA_LLM_SCALE_MX_E8M0)
      return refuse(CUDA_LLM_EINVAL, "an E2M1 V cache needs E8M0 block scales");
  }
  if (p->budget < 1 || p->sink < 0 || p->recent < 0 || (long long)p->sink + p->recent > p->budget)
    return refuse(CUDA_LLM_EINVAL, "budget must be at least 1 and at least sink + recent");
  if (p->max_tokens > CUDA_LLM_EVICT_MAX_TOKENS) return refuse(CUDA_LLM_EINVAL, "score rows of more than CUDA_LLM_EVICT_MAX_TOKENS entries");
  if (p->num_seqs == 0) return CUDA_LLM_OK;
  if (p->max_blocks_per_seq < 0 || p->new_max_blocks_per_seq < 0 || p->num_blocks <= 0)
    return refuse(CUDA_LLM_EINVAL, "block tables and pool must not be empty");
  if ((long long)p->num_seqs * p->num_kv_heads > 65535) return refuse(CUDA_LLM_EINVAL, "more than 65535 (sequence, KV head) pairs");
  const bool scaled = !wide && p->scale_mode != CUDA_LLM_SCALE_PER_HEAD;
  if (!p->scores || !p->key_cache || !p->value_cache || !p->block_tables || !p->new_block_tables || !p->context_lens ||
      !p->new_context_lens || !p->kept || (scaled && (!p->k_scale || !p->v_scale)))
    return refuse(CUDA_LLM_EINVAL, "null tensor");
  if (p->new_context_lens == p->context_lens) return refuse(CUDA_LLM_EINVAL, "new_context_lens must not be context_lens");
  const bool in_place = p->new_block_tables == p->block_tables;
  if (in_place && p->new_max_blocks_per_seq != p->max_blocks_per_seq)
    return refuse(CUDA_LLM_EINVAL, "the same block table with another width");
  long long most = (long long)p->max_blocks_per_seq * p->page_size;
  if (most > p->max_tokens) most = p->max_tokens;
  if (most > p->budget) most = p->budget;
  if ((long long)p->new_max_blocks_per_seq * p->page_size < most) return refuse(CUDA_LLM_EINVAL, "new_block_tables is too narrow for the kept tokens");
  if (((uintptr_t)p->key_cache | (uintptr_t)p->value_cache | (scaled ? (uintptr_t)p->k_scale | (uintptr_t)p->v_scale : 0)) & 15)
    return refuse(CUDA_LLM_EALIGN, "caches and scales must be 16-byte aligned");
  if (((uintptr_t)p->scores | (uintptr_t)p->new_scores | (uintptr_t)p->block_tables | (uintptr_t)p->new_block_tables | (uintptr_t)p->context_lens |
       (uintptr_t)p->new_context_lens | (uintptr_t)p->kept | (uintptr_t)p->status) & 3)
    return refuse(CUDA_LLM_EALIGN, "tables, lengths, scores, kept and status must be 4-byte aligned");
  int rc = check_current_device();
  if (rc != CUDA_LLM_OK) return rc;
  MoveArgs m;
  EvictArgs& a = m.e;
  a.scores = p->scores; a.new_scores = p->new_scores; a.bt = p->block_tables; a.new_bt = p->new_block_tables; a.ctx = p->context_lens;
  a.new_ctx = p->new_context_lens; a.kept = p->kept; a.status = p->status;
  a.st_seq = p->score_strides[0]; a.st_head = p->score_strides[1];
  a.nst_seq = p->new_score_strides[0]; a.nst_head = p->new_score_strides[1];
  a.S = p->num_seqs; a.Hkv = p->num_kv_heads; a.page = p->page_size; a.max_blocks = p->max_blocks_per_seq;
  a.new_max_blocks = p->new_max_blocks_per_seq; a.num_blocks = p->num_blocks; a.max_tokens = p->max_tokens; a.budget = p->budget;
  a.sink = p->sink; a.recent = p->recent; a.in_place = in_place;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  evict_select_kernel<<<dim3(a.Hkv, a.S), kSelThreads, 0, st>>>(a);
  rc = cuda_result(cudaGetLastError(), "evict_select_kernel launch");
  if (rc != CUDA_LLM_OK) return rc;
  const int D = p->head_dim;
  m.n_tensors = 0;
  m.slices = 0;
  auto add = [&](void* t, int rows) {
    m.t[m.n_tensors++] = MoveTensor{t, rows, m.slices};
    m.slices += (rows + 31) / 32;
  };
  add(p->key_cache, D);
  add(p->value_cache, p->v_format == CUDA_LLM_KV_FP4_E2M1 ? D / 2 : D);
  if (scaled) {
    const int rows = p->scale_mode == CUDA_LLM_SCALE_PER_TOKEN ? 1 : D / 32;
    add(p->k_scale, rows);
    add(p->v_scale, rows);
  }
  const dim3 grid((m.slices + 3) / 4, a.Hkv * a.S, in_place ? 1 : 16);
  const int eb = format_bytes(p->k_format);
  if (eb == 4) evict_move_kernel<uint32_t, uint32_t><<<grid, 128, 0, st>>>(m);
  else if (eb == 2) evict_move_kernel<uint16_t, uint16_t><<<grid, 128, 0, st>>>(m);
  else if (p->scale_mode == CUDA_LLM_SCALE_PER_TOKEN) evict_move_kernel<uint8_t, uint32_t><<<grid, 128, 0, st>>>(m);
  else evict_move_kernel<uint8_t, uint8_t><<<grid, 128, 0, st>>>(m);
  return cuda_result(cudaGetLastError(), "evict_move_kernel launch");
}
