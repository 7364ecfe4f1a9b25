// Cross attention of many query rows (16-bit types) on the 5th-generation tensor cores: tensor-bound.
//
//   S = Q K^T (128 rows x 128 states), P = 2^(scale S - m), l += rowsum P, O += P V;  out = O / l, lse = ln2 (m + log2 l)
//
// One CTA per (batch row, KV head, 256 query rows): the rows are the heads that share the KV head x consecutive positions,
// as two accumulator tiles of 128 rows, so that the tensor cores work on one tile while the softmax of the other runs:
//   warps 0..3, 4..7  softmax of tile 0 and tile 1, one thread per row (= per TMEM lane): S with tcgen05.ld, maximum,
//                     exponentials, P (16-bit) back over the columns of S
//   warp 8            TMA: Q once, then K and V tiles of 128 states into a ring of 32 KB slots
//   warp 9            (10, 11 idle) allocates TMEM, issues the MMAs of both tiles in turn: PV_0(j), S_0(j+1), PV_1(j), S_1(j+1)
// Tensor memory, head_dim 128: S0/P0 | S1/P1 | O0 | O1, 128 columns each, all there is.  P overwrites S: every MMA that reads P
// of step j is issued before the S of step j + 1, and the tensor pipe works in order.  The same order makes "S(j) is complete"
// mean "P V (j - 1) is complete", so a softmax thread may rescale O without another barrier.
// head_dim 64 leaves columns for P of its own (S0 | S1 | O0 | O1 | P0 | P1): S(j + 1) then follows as soon as the softmax has
// read S(j), and is ready when it comes back; P and O wait for the P V before instead.  O is rescaled only when a row maximum grew
// by more than 2^8 (P stays below 256), which after the first tiles is rare.
// What lies behind a sequence's length inside the last tile may be NaN: S is replaced by -inf there and the V rows are
// zeroed in shared memory before the last P V.
//
// Measured: bf16, 4 x 32 / 8 heads of 128, 2048 positions, 4096-8192 states: 717 us = 1150 TFLOP/s cold, 790 us back to back under
// the power cap (0.74 of the sustained cuBLAS rate).  fp16, 8 x 16 heads of 64, 447 positions, 201-1500 states: 37 us.
// A pair of tiles took about 3440 cycles per 128 states (by the clock register, before the last steps), 2048 of them MMA at the
// nominal rate; the tensor pipe counts 1.46 times its nominal cycles, since an MMA of 128 x 128 with both operands in shared memory
// reads them at exactly the rate of the memory, beside the TMA's writes.  Tried and slower, each against this form in the same
// run: a polynomial exponential on the FMA pipe for 25 / 33 / 50 % of the weights (765 -> 797 / 835 / 844 us), P handed over in
// four parts (725 -> 879-887) or two (754 -> 787-804); two threads per row (717 -> 750, separate runs).  Two CTAs per MMA (half
// of B from each) would relieve the operand reads.
// All waits are bounded; one that runs out raises a counter and the CTA falls through to the exit that frees TMEM.
#include "cross_attention.cuh"
#include "softmax_math.cuh"
#include "tcgen05_primitives.cuh"

namespace b200 {

bool encode_cross_map(CUtensorMap* map, const void* p, const long long* st, int B, int H, int S, int D, int box_rows, int* hmul, int* bmul);

__device__ unsigned int g_cross_prompt_timeouts = 0;

struct alignas(64) CrossPromptArgs {
  CUtensorMap q, k, v;
  CrossArgs c;
  int q_hmul, q_bmul, k_hmul, k_bmul, v_hmul, v_bmul;
  int gsz;  // query heads per CTA: 1, 2, 4, 8 or 16, divides the group
};

constexpr int kPromptThreads = 384;  // three warpgroups: registers are dealt out per warpgroup
constexpr int kPromptKeys = 128;
constexpr int kPromptRows = 256;

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

template <int D>
constexpr int prompt_slots() { return D == 128 ? 5 : 8; }
template <int D>
constexpr size_t prompt_smem() { return 1024 + (size_t)kPromptRows * D * 2 + (size_t)prompt_slots<D>() * kPromptKeys * D * 2; }

template <int D, bool BF16>
__global__ void __launch_bounds__(kPromptThreads, 1) cross_prompt_kernel(const __grid_constant__ CrossPromptArgs a) {
  constexpr int NCH = D / 64, NS = prompt_slots<D>();
  constexpr bool OWN_P = D == 64;                        // P has tensor memory of its own
  constexpr uint32_t T_O = 256, T_P = OWN_P ? 256 + 2 * D : 0, P_STEP = OWN_P ? 64 : 128, O_STEP = OWN_P ? D : 128;
  constexpr uint32_t QCH = kPromptRows * 128, KCH = kPromptKeys * 128, SLOT = NCH * KCH;
  constexpr float NEG_INF = -__builtin_huge_valf();
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t q_full = base, full = base + 8, empty = full + 8 * NS, s_full = empty + 8 * NS, p_full = s_full + 16, o_full = p_full + 16,
                 v_fixed = o_full + 16, s_read = v_fixed + 8, pv_done = s_read + 16, tmem_slot = pv_done + 16;
  const uint32_t sQ = base + 1024, ring = sQ + NCH * QCH;
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem + (tmem_slot - base));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = longest_first<kPromptThreads>(a.c, blockIdx.z, reinterpret_cast<volatile int*>(smem + 1020));
  const int BQ = kPromptRows / a.gsz;  // positions per CTA
  const int q_blocks = gridDim.x / (a.c.group / a.gsz), chunk = blockIdx.x / q_blocks;
  const int kvh = blockIdx.y, head0 = kvh * a.c.group + chunk * a.gsz;
  const int q0 = (blockIdx.x - chunk * q_blocks) * BQ;
  const int len = cross_kv_len(a.c, b);
  const int n_tiles = (len + kPromptKeys - 1) / kPromptKeys;
  // the second tile may hold no row at all (its heads' or positions' part starts behind the last)
  const int n_q = (a.gsz == 1 && q0 + 128 >= a.c.Sq) ? 1 : 2;
  const bool fix_v = len < a.c.Skv && len % kPromptKeys != 0;

  if (tid == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);  // one arrival per softmax warp of the tile
      mbar_init(o_full + 8 * i, 1);
      mbar_init(s_read + 8 * i, 4);
      mbar_init(pv_done + 8 * i, 1);
    }
    mbar_init(v_fixed, 1);
    mbar_fence_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot_ptr;
  auto give_up = [&]() { atomicAdd(&g_cross_prompt_timeouts, 1u); };

  // 384 threads x 168 registers at launch = 128 x (88 + 208 + 208): the softmax threads hold a row of 128 scores
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 8) {
    if (n_tiles > 0) {
      bool ok = true;
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, NCH * QCH);
        for (int i = 0; i < a.gsz; ++i)
          for (int c = 0; c < NCH; ++c)
            tma_load_4d(sQ + c * QCH + i * BQ * 128, &a.q, c * 64, q0, (head0 + i) * a.q_hmul, b * a.q_bmul, q_full);
        int st = 0;
        uint32_t par = 1;  // parity of the wait for a free slot: the first round passes at once
        int x = 0;
        for (; ok && x < 2 * n_tiles; ++x) {  // K0 V0 K1 V1 ...
          if (!tc_wait(empty + 8 * st, par)) { ok = false; break; }
          mbar_arrive_expect_tx(full + 8 * st, SLOT);
          for (int c = 0; c < NCH; ++c) {
            if (x & 1) tma_load_4d(ring + st * SLOT + c * KCH, &a.v, c * 64, (x >> 1) * kPromptKeys, kvh * a.v_hmul, b * a.v_bmul, full + 8 * st);
            else tma_load_4d(ring + st * SLOT + c * KCH, &a.k, c * 64, (x >> 1) * kPromptKeys, kvh * a.k_hmul, b * a.k_bmul, full + 8 * st);
          }
          if (++st == NS) {
            st = 0;
            par ^= 1;
          }
        }
        // copies in flight land before anybody leaves (after a wait that ran out; otherwise the consumers have waited)
        for (int y = x > NS ? x - NS : 0; y < x; ++y) tc_wait(full + 8 * (y % NS), (y / NS) & 1);
        if (!ok) give_up();
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (ok && fix_v) {  // rows of V behind the length become zeros before the last P V reads them
        const int x = 2 * n_tiles - 1, st = x % NS;
        ok = tc_wait(full + 8 * st, (x / NS) & 1);
        const int r0 = len - (n_tiles - 1) * kPromptKeys;
        for (int i = lane; ok && i < (kPromptKeys - r0) * 8 * NCH; i += 32) {
          const int c = i / ((kPromptKeys - r0) * 8), e = i % ((kPromptKeys - r0) * 8);
          sts128(ring + st * SLOT + c * KCH + r0 * 128 + e * 16, 0, 0, 0, 0);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (ok) mbar_arrive(v_fixed);
          else give_up();
        }
      }
    }
  } else if (warp == 9) {
    if (lane == 0 && n_tiles > 0) {
      const uint32_t idesc_s = instr_desc_f16(BF16 ? 1 : 0, 0, 128, kPromptKeys);
      const uint32_t idesc_o = instr_desc_f16(BF16 ? 1 : 0, 1, 128, D);
      const uint32_t hi = smem_desc_hi_sw128(1024);
      const uint32_t q_lo = smem_desc_lo(sQ, 16), k_lo = smem_desc_lo(ring, 16), v_lo = smem_desc_lo(ring, KCH);
      int st = 0;  // ring position of the next tile to wait for
      uint32_t par = 0;
      auto next_slot = [&](int& slot) -> bool {
        slot = st;
        const bool ok = tc_wait(full + 8 * st, par);
        if (++st == NS) {
          st = 0;
          par ^= 1;
        }
        return ok;
      };
      auto issue_s = [&](int i, int slot) {
        const uint32_t kl = k_lo + ((slot * SLOT) >> 4), ql = q_lo + ((i * 128 * 128) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16_parts(tmem + i * 128, ql + (((kk >> 2) * QCH + (kk & 3) * 32) >> 4), hi, kl + (((kk >> 2) * KCH + (kk & 3) * 32) >> 4), hi,
                         idesc_s, kk > 0 ? 1u : 0u);
        umma_commit(s_full + 8 * i);
      };
      int ks = 0, vs = 0;
      bool ok = tc_wait(q_full, 0) && next_slot(ks);
      if (ok) {
        tc_fence_after();
        for (int i = 0; i < n_q; ++i) issue_s(i, ks);
        umma_commit(empty + 8 * ks);
      }
      for (int j = 0; ok && j < n_tiles; ++j) {
        ok = next_slot(vs);
        if (ok && j + 1 < n_tiles) ok = next_slot(ks);
        if (ok && fix_v && j + 1 == n_tiles) ok = tc_wait(v_fixed, 0);
        for (int i = 0; ok && i < n_q; ++i) {
          if (OWN_P && j + 1 < n_tiles) {
            ok = tc_wait(s_read + 8 * i, j & 1);
            if (!ok) break;
            tc_fence_after();
            issue_s(i, ks);
            if (i == n_q - 1) umma_commit(empty + 8 * ks);
          }
          ok = tc_wait(p_full + 8 * i, j & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t vl = v_lo + ((vs * SLOT) >> 4);
#pragma unroll
          for (int kk = 0; kk < kPromptKeys / 16; ++kk)
            umma_f16_ts_parts(tmem + T_O + i * O_STEP, tmem + T_P + i * P_STEP + kk * 8, vl + ((kk * 2048) >> 4), hi, idesc_o,
                              (j > 0 || kk > 0) ? 1u : 0u);
          if (OWN_P) umma_commit(pv_done + 8 * i);
          if (i == n_q - 1) umma_commit(empty + 8 * vs);
          if (j + 1 == n_tiles) {
            umma_commit(o_full + 8 * i);
          } else if (!OWN_P) {
            issue_s(i, ks);
            if (i == n_q - 1) umma_commit(empty + 8 * ks);
          }
        }
      }
      if (!ok) give_up();
    }
  }
  } else {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
  if ((warp >> 2) < n_q) {
    const int i = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + i * 128, tO = tmem + lanes + T_O + i * O_STEP, tP = tmem + lanes + T_P + i * P_STEP;
    const int r = i * 128 + row, head = head0 + r / BQ, pos = q0 + r % BQ;
    float m_run = -3.0e38f, l_run = 0.f;  // below every score but -inf, whose weight is then zero
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      if (!tc_wait(s_full + 8 * i, j & 1)) { ok = false; break; }
      tc_fence_after();
      uint32_t sr[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, sr[c]);
      tc_wait_ld();
      if (OWN_P) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_read + 8 * i);
      }
      const int left = len - j * kPromptKeys;
      if (left < kPromptKeys) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c * 32 + e >= left) sr[c][e] = __float_as_uint(NEG_INF);
      }
      float mx8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) mx8[e] = NEG_INF;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          mx8[(e >> 1) & 7] = fmax3(mx8[(e >> 1) & 7], __uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1]));
      const float mx = fmaxf(fmax3(mx8[0], mx8[1], mx8[2]), fmaxf(fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
      const float m_tile = mx * a.c.scale_log2;
      if (OWN_P && j > 0) {  // O and P are free
        if (!tc_wait(pv_done + 8 * i, (j - 1) & 1)) { ok = false; break; }
        tc_fence_after();
      }
      if (__any_sync(0xffffffffu, m_tile > m_run + 8.f)) {  // some row of the warp needs a new reference
        const float m_new = (m_tile > m_run + 8.f) ? m_tile : m_run;
        const float alpha = fast_exp2(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t x[32];
            tmem_ld32(tO + c * 32, x);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * alpha);
            tmem_st32(tO + c * 32, x);
          }
        }
      }
      float ps[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const float neg_m = -m_run;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float x0, x1, p0, p1;
          ffma2(x0, x1, __uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1]), a.c.scale_log2, a.c.scale_log2, neg_m, neg_m);
          p0 = fast_exp2(x0);
          p1 = fast_exp2(x1);
          const int k = (e >> 1) & 3;
          fadd2(ps[2 * k], ps[2 * k + 1], ps[2 * k], ps[2 * k + 1], p0, p1);
          pk[e >> 1] = BF16 ? pack_bf16x2(p0, p1) : pack_f16x2(p0, p1);
        }
        tmem_st16(tP + c * 16, pk);
      }
      tc_wait_st();
      l_run += (((ps[0] + ps[1]) + (ps[2] + ps[3])) + ((ps[4] + ps[5]) + (ps[6] + ps[7])));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + 8 * i);
    }
    if (ok && n_tiles > 0 && !tc_wait(o_full + 8 * i, 0)) ok = false;
    if (!ok) {
      if (lane == 0) give_up();
    } else {
      tc_fence_after();
      const bool seen = l_run != 0.f;  // the largest score weighs 1 at least, unless all are -inf
      const float inv = seen ? 1.f / l_run : 0.f;
      const bool store = pos < a.c.Sq;
      uint16_t* op = static_cast<uint16_t*>(a.c.out) + b * a.c.o_st[0] + head * a.c.o_st[1] + (store ? pos : 0) * a.c.o_st[2];
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t x[32];
        if (n_tiles > 0) {
          tmem_ld32(tO + c * 32, x);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = 0u;
        }
        if (store) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x0 = __uint_as_float(x[8 * u + 2 * e]) * inv, x1 = __uint_as_float(x[8 * u + 2 * e + 1]) * inv;
              w[e] = BF16 ? pack_bf16x2(x0, x1) : pack_f16x2(x0, x1);
            }
            *reinterpret_cast<uint4*>(op + c * 32 + u * 8) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (store && a.c.lse)
        a.c.lse[((size_t)b * a.c.Hq + head) * a.c.Sq + pos] = seen ? kLn2 * (m_run + log2f(l_run)) : NEG_INF;
    }
  }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

template <int D, bool BF16>
static cudaError_t go(const CrossPromptArgs& a, cudaStream_t st) {
  auto kern = cross_prompt_kernel<D, BF16>;
  static int configured[64] = {0};
  cudaError_t e = allow_shared_memory((const void*)kern, (int)prompt_smem<D>(), configured);
  if (e != cudaSuccess) return e;
  const int bq = kPromptRows / a.gsz;
  // position blocks of a group's head chunks in x: the grid's y would end at 65535 query heads
  const dim3 grid((a.c.Sq + bq - 1) / bq * (a.c.group / a.gsz), a.c.Hkv, a.c.B);
  kern<<<grid, kPromptThreads, prompt_smem<D>(), st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_cross_prompt(const CrossArgs& c, int D, cudaStream_t st) {
  CrossPromptArgs a = {};
  a.c = c;
  a.gsz = 1;  // the largest power of two up to 16 that divides the group: a K / V tile is fetched once for those heads
  while (a.gsz < 16 && c.group % (2 * a.gsz) == 0) a.gsz *= 2;
  if (c.Skv > 0) {
    if (!encode_cross_map(&a.q, c.q, c.q_st, c.B, c.Hq, c.Sq, D, kPromptRows / a.gsz, &a.q_hmul, &a.q_bmul) ||
        !encode_cross_map(&a.k, c.k, c.k_st, c.B, c.Hkv, c.Skv, D, kPromptKeys, &a.k_hmul, &a.k_bmul) ||
        !encode_cross_map(&a.v, c.v, c.v_st, c.B, c.Hkv, c.Skv, D, kPromptKeys, &a.v_hmul, &a.v_bmul))
      return cudaErrorInvalidValue;
  }
  const bool bf16 = c.dtype == CUDA_LLM_BF16;
  if (D == 64) return bf16 ? go<64, true>(a, st) : go<64, false>(a, st);
  return bf16 ? go<128, true>(a, st) : go<128, false>(a, st);
}

cudaError_t cross_prompt_timeouts(unsigned int* count) { return cudaMemcpyFromSymbol(count, g_cross_prompt_timeouts, sizeof(unsigned int)); }

}  // namespace b200
