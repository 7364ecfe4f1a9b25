// Cross attention of few query rows (16-bit types): the states are streamed once, HBM-bound.
//
//   per warp and 16 states:  S = Q K^T (16 rows x 16 states), m' = max(m, rowmax S), P = 2^(S - m'),
//                            l = l 2^(m - m') + rowsum P, O = O 2^(m - m') + P V
//   joined over warps and CTAs:  M = max m_i, L = sum l_i 2^(m_i - M), out = sum O_i 2^(m_i - M) / L
//
// The query rows of a KV head (its heads x positions, up to 64) ride on the M side of mma.m16n8k16.  A thread-block cluster
// shares the states of one (sequence, KV head): CTA r takes the r-th part of its 64-state tiles and the parts are joined
// through distributed shared memory, so that one launch without a workspace serves one stream and large batches alike and
// nothing depends on the order in which CTAs finish.  One producer warp keeps a ring of K / V tiles in flight by TMA
// (128-byte swizzle, so the row addresses of ldmatrix carry the XOR of their row); four warps share a tile: each its
// own 16 states of one row block, or (more than 16 rows) each its own row block of more states.
//
// P is rounded to the operand type (half a step of it, against the row's own maximum); sums, maxima and O stay in fp32.
//
// Measured (bf16, 32 query and 8 KV heads of 128, one token): 64 sequences of 1000-4096 states 102 us = 6.5 TB/s, the measured
// copy peak; 16 sequences of 4096 states 54 us; one sequence of 1500 states 8.2 us, of which the launch, the first
// copies' latency and the join are nearly all.
#include "cross_attention.cuh"
#include "tcgen05_primitives.cuh"

namespace b200 {

__device__ unsigned int g_cross_wait_timeouts = 0;

constexpr int kTokTile = 64;       // states per ring slot
constexpr int kTokThreads = 160;   // four computing warps, one producer warp

struct alignas(64) CrossTokenArgs {
  CUtensorMap k, v;
  CrossArgs c;
  int k_hmul, k_bmul, v_hmul, v_bmul;  // 0: one tile serves all heads / batch rows (stride 0)
};

__device__ __forceinline__ void tma_tile_4d(uint32_t dst, const void* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
template <int D>
constexpr int tok_stages() { return D == 128 ? 3 : 6; }
template <int D>
constexpr size_t tok_smem() { return 1024 + (size_t)tok_stages<D>() * 2 * kTokTile * D * 2; }

template <int D, bool BF16, int MT>
__global__ void __launch_bounds__(kTokThreads) cross_token_kernel(const __grid_constant__ CrossTokenArgs a) {
  constexpr int NST = tok_stages<D>(), NCH = D / 64;
  constexpr uint32_t CH = kTokTile * 128, TILE = NCH * CH, STAGE = 2 * TILE;
  constexpr float NEG_INF = -__builtin_huge_valf();
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t full = base, empty = base + 8 * NST, ring = base + 1024;
  volatile uint32_t* fail_ptr = reinterpret_cast<volatile uint32_t*>(smem + 16 * NST);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.y, b = longest_first<kTokThreads>(a.c, blockIdx.z, reinterpret_cast<volatile int*>(smem + 512));
  const int rank = (int)cluster_rank(), parts = (int)cluster_size();

  if (tid == 0) {
    for (int i = 0; i < NST; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 4);
    }
    *fail_ptr = 0;
    mbar_fence_init();
  }
  const int len = cross_kv_len(a.c, b);
  const int tiles = (len + kTokTile - 1) / kTokTile;
  const int j0 = (int)((long long)tiles * rank / parts), j1 = (int)((long long)tiles * (rank + 1) / parts);
  __syncthreads();

  const int g = lane >> 2, t = lane & 3;
  const int mtile = warp % MT, tslot = warp / MT;
  float o[D / 8][4], m[2] = {NEG_INF, NEG_INF}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const int rows = a.c.group * a.c.Sq;

  if (warp == 4) {
    if (lane == 0) {
      int j = j0;
      for (; j < j1; ++j) {
        const int i = j - j0, st = i % NST;
        if (i >= NST && !tc_wait(empty + 8 * st, ((i / NST) - 1) & 1)) {
          *fail_ptr = 1;
          break;
        }
        mbar_arrive_expect_tx(full + 8 * st, STAGE);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          tma_tile_4d(ring + st * STAGE + c * CH, &a.k, c * 64, j * kTokTile, kvh * a.k_hmul, b * a.k_bmul, full + 8 * st);
          tma_tile_4d(ring + st * STAGE + TILE + c * CH, &a.v, c * 64, j * kTokTile, kvh * a.v_hmul, b * a.v_bmul, full + 8 * st);
        }
      }
      // copies in flight land before the ring is used for anything else, also after a wait that ran out
      for (int x = max(0, j - j0 - NST); x < j - j0; ++x) tc_wait(full + 8 * (x % NST), (x / NST) & 1);
    }
  } else {
    // query fragments: rows g and g + 8 of this warp's block, two 16-bit elements per register
    uint32_t qf[D / 16][4];
    const uint16_t* qp = static_cast<const uint16_t*>(a.c.q) + b * a.c.q_st[0];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = mtile * 16 + g + half * 8;
      const uint16_t* p = qp + (kvh * a.c.group + r % a.c.group) * a.c.q_st[1] + (r / a.c.group) * a.c.q_st[2];
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[kk][half] = r < rows ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + 2 * t) : 0u;
        qf[kk][half + 2] = r < rows ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + 2 * t + 8) : 0u;
      }
    }
    const uint32_t x7 = lane & 7;
    const int k_tok = ((lane >> 4) << 3) + (lane & 7), k_chunk = (lane >> 3) & 1;       // ldmatrix rows of K
    const int v_tok = (((lane >> 3) & 1) << 3) + (lane & 7), v_chunk = lane >> 4;       // and of V
    for (int j = j0; j < j1; ++j) {
      const int i = j - j0, st = i % NST;
      if (!tc_wait(full + 8 * st, (i / NST) & 1)) {
        *fail_ptr = 1;
        break;
      }
      const bool edge = (j + 1) * kTokTile > len;
#pragma unroll 1
      for (int u = 0; u < MT; ++u) {
        const int tok0 = (tslot * MT + u) * 16, tok_abs = j * kTokTile + tok0;
        if (edge && tok_abs >= len) break;
        const uint32_t kb = ring + st * STAGE + (tok0 + k_tok) * 128, vb = ring + st * STAGE + TILE + (tok0 + v_tok) * 128;
        float s[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t r[4];
          ldmatrix_x4(r, kb + (kk >> 2) * CH + ((((kk & 3) * 2 + k_chunk) ^ x7) << 4));
          if (BF16) {
            mma_bf16(s[0], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], r[0], r[1]);
            mma_bf16(s[1], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], r[2], r[3]);
          } else {
            mma_f16(s[0], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], r[0], r[1]);
            mma_f16(s[1], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], r[2], r[3]);
          }
        }
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;  // states 2t, 2t + 1 and 2t + 8, 2t + 9 of V
        if (edge) {
          const int n = len - tok_abs - 2 * t;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (n <= h * 8) s[h][0] = s[h][2] = NEG_INF;
            if (n <= h * 8 + 1) s[h][1] = s[h][3] = NEG_INF;
          }
          keep0 = n <= 0 ? 0u : n == 1 ? 0xffffu : 0xffffffffu;
          keep1 = n <= 8 ? 0u : n == 9 ? 0xffffu : 0xffffffffu;
        }
        uint32_t p[4];
        float alpha[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1])) * a.c.scale_log2;
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m[h], mx), ref = m_new == NEG_INF ? 0.f : m_new;
          alpha[h] = fast_exp2(m[h] - ref);
          m[h] = m_new;
          const float p0 = fast_exp2(fmaf(s[0][2 * h], a.c.scale_log2, -ref)), p1 = fast_exp2(fmaf(s[0][2 * h + 1], a.c.scale_log2, -ref));
          const float p2 = fast_exp2(fmaf(s[1][2 * h], a.c.scale_log2, -ref)), p3 = fast_exp2(fmaf(s[1][2 * h + 1], a.c.scale_log2, -ref));
          l[h] = l[h] * alpha[h] + ((p0 + p1) + (p2 + p3));
          p[h] = BF16 ? pack_bf16x2(p0, p1) : pack_f16x2(p0, p1);
          p[h + 2] = BF16 ? pack_bf16x2(p2, p3) : pack_f16x2(p2, p3);
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][0] *= alpha[0];
            o[n][1] *= alpha[0];
            o[n][2] *= alpha[1];
            o[n][3] *= alpha[1];
          }
        }
#pragma unroll
        for (int n = 0; n < D / 8; n += 2) {
          uint32_t r[4];
          ldmatrix_x4_trans(r, vb + (n >> 3) * CH + ((((n & 7) + v_chunk) ^ x7) << 4));
          if (edge) {
            r[0] &= keep0;
            r[1] &= keep1;
            r[2] &= keep0;
            r[3] &= keep1;
          }
          if (BF16) {
            mma_bf16(o[n], p[0], p[1], p[2], p[3], r[0], r[1]);
            mma_bf16(o[n + 1], p[0], p[1], p[2], p[3], r[2], r[3]);
          } else {
            mma_f16(o[n], p[0], p[1], p[2], p[3], r[0], r[1]);
            mma_f16(o[n + 1], p[0], p[1], p[2], p[3], r[2], r[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * st);
    }
  }

  // ---- join: warps through shared memory (the ring is idle), CTAs through distributed shared memory
  __syncthreads();
  if (*fail_ptr && tid == 0) atomicAdd(&g_cross_wait_timeouts, 1u);
  constexpr int LD = D + 4;
  float* part_o = reinterpret_cast<float*>(smem + 1024);              // [4 warps][16][LD]
  float2* part_ml = reinterpret_cast<float2*>(part_o + 4 * 16 * LD);  // [4 warps][16]
  float* cta_o = reinterpret_cast<float*>(part_ml + 64);              // [16 MT][D]
  float2* cta_ml = reinterpret_cast<float2*>(cta_o + 16 * MT * D);    // [16 MT]
  if (warp < 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (t == 0) part_ml[warp * 16 + g + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2*>(part_o + (warp * 16 + g + 8 * h) * LD + n * 8 + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
    }
  }
  __syncthreads();
  const int live_rows = min(rows, 16 * MT);
  auto emit = [&](int r, int c, float4 x, float M, float L) {
    const float inv = L == 0.f ? 0.f : 1.f / L;  // nothing seen: zeros
    const int head = kvh * a.c.group + r % a.c.group, pos = r / a.c.group;
    uint16_t* op = static_cast<uint16_t*>(a.c.out) + b * a.c.o_st[0] + head * a.c.o_st[1] + pos * a.c.o_st[2] + 4 * c;
    *reinterpret_cast<uint2*>(op) = BF16 ? make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv))
                                         : make_uint2(pack_f16x2(x.x * inv, x.y * inv), pack_f16x2(x.z * inv, x.w * inv));
    if (c == 0 && a.c.lse) a.c.lse[((size_t)b * a.c.Hq + head) * a.c.Sq + pos] = L == 0.f ? NEG_INF : kLn2 * (M + log2f(L));
  };
  for (int e = tid; e < live_rows * (D / 4); e += kTokThreads) {
    const int r = e / (D / 4), c = e % (D / 4);
    float M = NEG_INF;
#pragma unroll
    for (int x = 0; x < 4 / MT; ++x) M = fmaxf(M, part_ml[(x * MT + r / 16) * 16 + (r & 15)].x);
    const float ref = M == NEG_INF ? 0.f : M;
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < 4 / MT; ++x) {
      const int at = (x * MT + r / 16) * 16 + (r & 15);
      const float2 ml = part_ml[at];
      const float w = fast_exp2(ml.x - ref);
      const float4 y = *reinterpret_cast<const float4*>(part_o + at * LD + 4 * c);
      L = fmaf(ml.y, w, L);
      acc.x = fmaf(y.x, w, acc.x);
      acc.y = fmaf(y.y, w, acc.y);
      acc.z = fmaf(y.z, w, acc.z);
      acc.w = fmaf(y.w, w, acc.w);
    }
    if (parts == 1) {
      emit(r, c, acc, M, L);
    } else {
      *reinterpret_cast<float4*>(cta_o + r * D + 4 * c) = acc;
      if (c == 0) cta_ml[r] = make_float2(M, L);
    }
  }
  if (parts > 1) {
    cluster_sync_all();
    const uint32_t o_at = smem_u32(cta_o), ml_at = smem_u32(cta_ml);
    for (int e = rank * kTokThreads + tid; e < live_rows * (D / 4); e += parts * kTokThreads) {
      const int r = e / (D / 4), c = e % (D / 4);
      const JoinedWord w = join_parts(ml_at + r * 8, o_at + (r * D + 4 * c) * 4, parts);
      emit(r, c, w.x, w.M, w.L);
    }
    cluster_sync_all();  // no CTA leaves while another still reads its parts
  }
}

// Tensor map of states [B, H, S, D] by their strides: boxes of 64 head_dim elements x `box_rows` positions, 128-byte
// swizzle.  A stride of 0 is a dimension of one element (`hmul`, `bmul` 0); positions have none (refused by the entry).
bool encode_cross_map(CUtensorMap* map, const void* p, const long long* st, int B, int H, int S, int D, int box_rows, int* hmul, int* bmul) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (!enc) return false;
  *hmul = H > 1 && st[1] == 0 ? 0 : 1;
  *bmul = B > 1 && st[0] == 0 ? 0 : 1;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)(*hmul ? H : 1), (cuuint64_t)(*bmul ? B : 1)};
  const cuuint64_t strides[3] = {(cuuint64_t)st[2] * 2, (cuuint64_t)(st[1] ? st[1] : D) * 2, (cuuint64_t)(st[0] ? st[0] : D) * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, estr[4] = {1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16, int MT>
static cudaError_t go(const CrossTokenArgs& a, int parts, cudaStream_t st) {
  auto kern = cross_token_kernel<D, BF16, MT>;
  static int configured[64] = {0};
  cudaError_t e = allow_shared_memory((const void*)kern, (int)tok_smem<D>(), configured);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts, a.c.Hkv, a.c.B);
  cfg.blockDim = dim3(kTokThreads);
  cfg.dynamicSmemBytes = tok_smem<D>();
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}
template <int D, bool BF16>
static cudaError_t go_rows(const CrossTokenArgs& a, int parts, cudaStream_t st) {
  const int rows = a.c.group * a.c.Sq;
  return rows <= 16 ? go<D, BF16, 1>(a, parts, st) : rows <= 32 ? go<D, BF16, 2>(a, parts, st) : go<D, BF16, 4>(a, parts, st);
}

cudaError_t launch_cross_token(const CrossArgs& c, int D, cudaStream_t st) {
  CrossTokenArgs a;
  a.c = c;
  if (c.Skv > 0) {
    if (!encode_cross_map(&a.k, c.k, c.k_st, c.B, c.Hkv, c.Skv, D, kTokTile, &a.k_hmul, &a.k_bmul) ||
        !encode_cross_map(&a.v, c.v, c.v_st, c.B, c.Hkv, c.Skv, D, kTokTile, &a.v_hmul, &a.v_bmul))
      return cudaErrorInvalidValue;
  }
  const int tiles = (c.Skv + kTokTile - 1) / kTokTile;
  const int parts = cross_parts((long long)c.B * c.Hkv, tiles);
  const bool bf16 = c.dtype == CUDA_LLM_BF16;
  if (D == 64) return bf16 ? go_rows<64, true>(a, parts, st) : go_rows<64, false>(a, parts, st);
  return bf16 ? go_rows<128, true>(a, parts, st) : go_rows<128, false>(a, parts, st);
}

cudaError_t cross_wait_timeouts(unsigned int* count) { return cudaMemcpyFromSymbol(count, g_cross_wait_timeouts, sizeof(unsigned int)); }

}  // namespace b200
