// Accumulated attention weight of cached tokens:
//
//   scores[s, h, t] = decay * old + sum over the rows r that see t of 2^(scale_log2 q_r . k_t - lse2_r)
//
// The log-sum-exp is known, so tokens are independent: one pass over K, no join, no atomics.  A decode step (up to 16 rows per
// KV head) is bound by the bytes of K: 64 sequences of 1000-8192 tokens, 8 heads of 128, E4M3 with per-token scales, 64 us =
// 5.1 TB/s (0.79 of the measured copy peak; what is missing is issue slots: 165 warp instructions per 16 tokens and head, counted
// when it took 77 us).
// Windows of a prompt with more rows go to kv_weights_window_kernel; those of up to 64 (or 128) rows stay here, bound by the latency
// of warp-level products and exponentials (tensor pipe 35 % busy at 128 rows), and so do all with fp32 queries (three bf16 terms) or
// with fp16 queries on block-scaled keys (f16 has no room for the block scale in the key): they pay 2.6 to 10 times.
//
// Arithmetic: K as E4M3 codes (widened exactly to f16) or as 16-bit elements, products on mma.m16n8k16 with fp32 sums, tokens on
// the 16-wide side and query rows on the 8-wide side.  bf16 and fp32 queries against 8-bit codes are brought into f16's range by a
// power of two per row, fp32 ones as two f16 terms (22 bits); scales multiply the fp32 sums, block scales the sums
// of their 32 elements.
#include <cmath>

#include "kv_weights.cuh"
#include "tcgen05_primitives.cuh"

namespace b200 {

// ---------------------------------------------------------------------------------------------------------------------
// Geometry.  A stage of the ring holds K of `hg` KV heads of one sequence for tok_stage consecutive tokens (whole pages, one
// bulk copy per page: the heads of a page are contiguous) and their scales.  Its 16-token units, one head each, go to the
// computing warps.  All stages of the call, in (sequence, head group, token) order, are cut into equal contiguous
// ranges, one per CTA; every CTA finds its range from a prefix sum over the context lengths.
constexpr int kWgtWarps = 8;          // computing warps; a stage is 2 or 4 16-token units for each (streamed rows: 16 warps, one each)
constexpr int kWgtMaxStages = 8;
constexpr uint32_t kWgtHeader = 9 * 1024;  // barriers, page masks, flag, prefix sums, lengths
static_assert(192 + 4 * (2 * kWgtSeqs + 4) <= kWgtHeader, "header");
constexpr int kWgtRows = 128;         // query rows of a KV head kept in shared memory
constexpr uint32_t kWgtBudget = 224 * 1024;

struct WeightsGeom {
  int hg, n_hg, pages, tok_stage, units;   // pages, tokens and units (head x 16 tokens) of a stage
  int n_stages;
  int box_rows;                            // pages as swizzled TMA boxes of this many head_dim rows; 0: as bulk copies
  uint32_t q_off, smem;                    // where streamed rows are kept in shared memory; bytes of it in all
  uint32_t k_head, s_head;                 // bytes of one head of one page, K / scales
  uint32_t k_bytes, s_bytes, stage_bytes;  // of the head group of one page; of a stage
};

// Pages with rows of 64 or 128 bytes arrive as TMA boxes with the swizzle of that width, which spreads the eight rows of an
// ldmatrix over all banks; shorter rows do that by themselves (16 bytes) or conflict in pairs (32).
struct alignas(64) WeightsMap {
  CUtensorMap k;  // [num_blocks][Hkv * D][page]
};
__device__ __forceinline__ void tma_box_3d(uint32_t dst, const void* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}

// B fragments of mma.m16n8k16 for 8 query rows: lane (g, t) holds 8 consecutive elements of every 32 of row g, d = 32 p + 8 t ..
// 8 t + 7.  Word w of them meets matrix (w - t) & 3 of the ldmatrix below, which for lane t brings K at d = 32 p + 8 t +
// 2 ((m + t) & 3): every product finds its partner, and the eight rows of a matrix lie in different banks.
__device__ __forceinline__ void rotate_words(uint32_t (&w)[4], int t) {
  if (t & 1) {
    const uint32_t x = w[0];
    w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = x;
  }
  if (t & 2) {
    uint32_t x = w[0];
    w[0] = w[2]; w[2] = x;
    x = w[1];
    w[1] = w[3]; w[3] = x;
  }
}

enum { KF_E4M3 = 0, KF_F16 = 1, KF_BF16 = 2 };

// m16n8k16, fp32 accumulation.  (Not volatile: the products of several tokens and rows may be interleaved.)
template <bool BF>
__device__ __forceinline__ void mma_any(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What the rows of one 8-column block need after the product, for the two columns 2t, 2t + 1 of a lane.
struct RowPair {
  float lse2[2], inv[2];  // log-sum-exp in units of log2; 1 / (power of two the query row was multiplied by)
  int limit[2];           // tokens below it are seen
};

// row r of a sequence: query token r / group, head r % group of the KV head's group
__device__ __forceinline__ void row_pair(const WeightsArgs& a, int r0, int rows, int q0, int n_q, int ctx, int h, int t, RowPair& rp) {
  float v[2];  // both on their way before the first is looked at
  int j[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = r0 + 2 * t + x;  // the lane's two columns
    j[x] = a.group_shift >= 0 ? r >> a.group_shift : r / a.group;
    v[x] = __builtin_huge_valf();
    if (r < rows) v[x] = a.lse[(size_t)(q0 + j[x]) * a.Hq + h * a.group + (r - j[x] * a.group)];
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    // a row that saw nothing (-inf), or is not there, sees no token: its products may be NaN
    const bool none = v[x] == -__builtin_huge_valf();
    rp.lse2[x] = none ? __builtin_huge_valf() : v[x] * 1.4426950408889634f;
    rp.limit[x] = none || r0 + 2 * t + x >= rows ? 0 : a.causal ? ctx - n_q + 1 + j[x] : ctx;
    rp.inv[x] = 1.f;
  }
}

// 8 query rows as B fragments in their own 16-bit type, or an fp32 row as three bf16 terms (24 bits).
template <int D, int QT>
__device__ __forceinline__ void load_rows(const void* q, size_t at, bool live, int t, uint32_t (&w)[QT == CUDA_LLM_F32 ? 3 : 1][D / 32][4]) {
#pragma unroll
  for (int p = 0; p < D / 32; ++p) {
    if (QT != CUDA_LLM_F32) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (live) u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(q) + at + p * 32 + 8 * t);
      w[0][p][0] = u.x; w[0][p][1] = u.y; w[0][p][2] = u.z; w[0][p][3] = u.w;
      rotate_words(w[0][p], t);
    } else {
      // fp32 as three bf16 terms: 24 bits
      float f[8] = {};
      if (live) {
        const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(q) + at + p * 32 + 8 * t);
        const float4 x = src[0], y = src[1];
        f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w; f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
      }
#pragma unroll
      for (int term = 0; term < (QT == CUDA_LLM_F32 ? 3 : 1); ++term) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[term][p][e] = pack_bf16x2(f[2 * e], f[2 * e + 1]);
          f[2 * e] -= __uint_as_float(w[term][p][e] << 16);
          f[2 * e + 1] -= __uint_as_float(w[term][p][e] & 0xffff0000u);
        }
        rotate_words(w[term][p], t);
      }
    }
  }
}

// K fragments of 16 tokens and 32 elements of head_dim (two k-steps): E4M3 codes widened to f16 (exact), or 16-bit elements as
// they are.  `at` comes from key_row().  Rows of the result: tokens 2g and 2g + 1 (8 bit) or g and g + 8 (16 bit).
// `chunk`: which 16 bytes of a row hold the unit's tokens (its first 8 tokens, 16 bit).
template <int KF>
__device__ __forceinline__ uint32_t key_row(int lane, uint32_t row_bytes, int chunk, int x) {
  const int m = lane >> 3, i = lane & 7;
  uint32_t row;
  if (KF == KF_E4M3) {
    row = 8 * (i >> 1) + 2 * ((m + (i >> 1)) & 3) + (i & 1);
  } else {  // matrices of k-step x: (tokens 0..7, 8..15) x (first, second pair of elements)
    row = 8 * (i >> 1) + 2 * ((2 * x + (m >> 1) + (i >> 1)) & 3) + (i & 1);
    chunk += m & 1;
  }
  const uint32_t swizzle = row_bytes == 128 ? row & 7 : row_bytes == 64 ? (row >> 1) & 3 : 0;
  return row * row_bytes + ((chunk ^ swizzle) << 4);
}
template <int KF>
__device__ __forceinline__ void load_key_block(const uint32_t (&at)[2], uint32_t offset, uint32_t (&af)[2][4]) {
  if (KF == KF_E4M3) {
    uint32_t r[4];
    ldmatrix_x4_trans(r, at[0] + offset);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      // bytes (token 2g, 2g + 1) of row 2t, then of row 2t + 1 -> (d, d + 1) of token 2g, then of token 2g + 1
      const uint32_t b = prmt(r[x], 0, 0x3120);
      af[x >> 1][2 * (x & 1)] = e4m3x2_to_f16x2_lo(b);
      af[x >> 1][2 * (x & 1) + 1] = e4m3x2_to_f16x2_hi(b);
    }
  } else {
    ldmatrix_x4_trans(af[0], at[0] + offset);
    ldmatrix_x4_trans(af[1], at[1] + offset);
  }
}

// fp32 rows of the queries of 8 columns, in f16: the row times 2^(14 - exponent of its largest element) keeps every bit of a
// bf16 element down to 2^-30 of the largest; fp32 elements as hi + lo / 2^11.  `inv` undoes the power of two.
template <int D, int QT, int NQ>
__device__ __forceinline__ void load_rows_scaled(const void* q, size_t at, bool live, int t, uint32_t (&w)[NQ][D / 32][4], float (&inv)[2]) {
  float f[D / 32][8], top = 0.f;
#pragma unroll
  for (int p = 0; p < D / 32; ++p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[p][e] = 0.f;
    if (live && QT == CUDA_LLM_BF16) {
      const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(q) + at + p * 32 + 8 * t);
      const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[p][2 * e] = __uint_as_float(vv[e] << 16);
        f[p][2 * e + 1] = __uint_as_float(vv[e] & 0xffff0000u);
      }
    } else if (live) {
      const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(q) + at + p * 32 + 8 * t);
      const float4 x = src[0], y = src[1];
      f[p][0] = x.x; f[p][1] = x.y; f[p][2] = x.z; f[p][3] = x.w; f[p][4] = y.x; f[p][5] = y.y; f[p][6] = y.z; f[p][7] = y.w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[p][e]));
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const uint32_t e2 = min(max(__float_as_uint(top) >> 23, 15u), 253u);
  const float up = __uint_as_float(min(268u - e2, 254u) << 23), down = __uint_as_float((e2 - 14u) << 23);
  inv[0] = __shfl_sync(0xffffffffu, down, 8 * t);      // columns 2t and 2t + 1 are the rows of lanes 8t and 8t + 4
  inv[1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
  for (int p = 0; p < D / 32; ++p) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = f[p][2 * e] * up, y = f[p][2 * e + 1] * up;
      w[0][p][e] = pack_f16x2(x, y);
      if (NQ == 2) w[NQ - 1][p][e] = pack_f16x2((x - f16x2_lo(w[0][p][e])) * 2048.f, (y - f16x2_hi(w[0][p][e])) * 2048.f);
    }
    rotate_words(w[0][p], t);
    if (NQ == 2) rotate_words(w[NQ - 1][p], t);
  }
}

// Producer warp: lane 0 issues the copies; the block-table entries of the next 32 / pages stages are fetched by all lanes.
// Beside a stage lies a mask of the pages that were copied (bad block-table entries are not).
__device__ __forceinline__ void produce(const WeightsArgs& a, const WeightsGeom& gm, const WeightsMap& map, const WeightsPlan& pl, uint32_t full, uint32_t empty, uint32_t live_at,
                                        uint32_t ring, volatile int* fail_ptr) {
  const int lane = threadIdx.x & 31, batch = 32 / gm.pages, pg_mask = gm.pages - 1, pg_shift = __popc(pg_mask);
  bool ok = true;
  int i = 0, s = pl.s0, st = 0;
  uint32_t free_par = 1;  // the first round finds every slot free
  auto entry = [&](int w_first) -> int {
    const int w = w_first + (lane >> pg_shift);
    if (w >= pl.w1) return -1;
    int sq = s;
    while (w >= pl.pre[sq + 1]) ++sq;
    const int per = (pl.pre[sq + 1] - pl.pre[sq]) / gm.n_hg, u = (w - pl.pre[sq]) % per;
    const int page = u * gm.pages + (lane & pg_mask);
    if ((long long)page * a.page >= pl.lens[sq]) return -1;  // behind the last token: nothing to copy
    int blk = a.bt[(size_t)sq * a.max_blocks + page];
    if (blk < 0 || blk >= a.num_blocks) {
      if (a.status) atomicOr(a.status, CUDA_LLM_ST_BAD_BLOCK);
      blk = -1;
    }
    return blk;
  };
  int next = entry(pl.w0);
  for (int wb = pl.w0; ok && wb < pl.w1; wb += batch) {
    const int mine = next;
    while (wb >= pl.pre[s + 1]) ++s;
    next = entry(wb + batch);
    int sq = s;
    for (int k = 0; k < batch && wb + k < pl.w1; ++k, ++i) {
      const int w = wb + k;
      const unsigned live = __ballot_sync(0xffffffffu, mine >= 0) >> (k << pg_shift) & (gm.pages == 32 ? 0xffffffffu : (1u << gm.pages) - 1);
      ok = mbar_wait(empty + 8 * st, free_par, 0);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      while (w >= pl.pre[sq + 1]) ++sq;
      const int per = (pl.pre[sq + 1] - pl.pre[sq]) / gm.n_hg, h0 = (w - pl.pre[sq]) / per * gm.hg;
      if (lane == 0) {
        sts32(live_at + 4 * st, (int)live);
        mbar_arrive_expect_tx(full + 8 * st, (uint32_t)__popc(live) * (gm.k_bytes + gm.s_bytes));
      }
      __syncwarp();
      // the lanes that hold the stage's entries issue its copies
      if ((lane >> pg_shift) == k && mine >= 0) {
        const int pg = lane & pg_mask;
        const size_t slab = (size_t)mine * a.Hkv + h0;
        const uint32_t to = ring + st * gm.stage_bytes;
        if (gm.box_rows) {
          const int rows = gm.hg * a.D;
          for (int r = 0; r < rows; r += gm.box_rows)
            tma_box_3d(to + pg * gm.k_bytes + r * (gm.k_head / a.D), &map.k, 0, h0 * a.D + r, mine, full + 8 * st);
        } else {
          bulk_g2s(to + pg * gm.k_bytes, a.kc + slab * gm.k_head, gm.k_bytes, full + 8 * st);
        }
        if (gm.s_bytes) bulk_g2s(to + gm.pages * gm.k_bytes + pg * gm.s_bytes, a.ks + slab * gm.s_head, gm.s_bytes, full + 8 * st);
      }
      if (++st == gm.n_stages) {
        st = 0;
        free_par ^= 1;
      }
    }
  }
  if (lane == 0) {
    for (int x = max(0, i - gm.n_stages); x < i; ++x)  // copies in flight land before the CTA ends
      if (!mbar_wait(full + 8 * (x % gm.n_stages), (x / gm.n_stages) & 1, 0)) ok = false;
    if (a.status && (!ok || *fail_ptr)) atomicOr(a.status, CUDA_LLM_ST_TIMEOUT);
  }
}

// Four units per warp and stage share more of what a stage costs a warp, where three such stages fit and the fragments leave
// registers: 8-bit caches, or 16-bit ones of head_dim 64.  (64 sequences: one unit 86 us, two 84, four 77, at that state.)
template <int D, int KF, int QT>
constexpr bool kFourUnits = QT != CUDA_LLM_F32 && (KF == KF_E4M3 || D == 64);

// One stage is one task per computing warp: head warp % hg of the group, a run of 16-token units.
// NT > 0: the query fragments of 8 NT rows stay in registers from stage to stage (a decode step: all rows of a KV head); a
// sequence with more rows than that is right but reloads them.
// NT == 0: many rows per KV head (a window of a prompt): the warp holds the keys and the rows pass eight at a time, from shared
// memory up to kWgtRows of them, else (and as fp32) from L2.
template <int D, int KF, int QT, int NT, bool MX, int U>
__global__ void __launch_bounds__(32 * ((NT ? kWgtWarps : 2 * kWgtWarps) + 1), 1)
kv_weights_kernel(const __grid_constant__ WeightsArgs a, const __grid_constant__ WeightsGeom gm, const __grid_constant__ WeightsMap map) {
  constexpr bool F8 = KF == KF_E4M3;
  constexpr int WARPS = NT ? kWgtWarps : 2 * kWgtWarps, ROWS = NT ? 8 * NT : 8;  // a stage has 16 units at least
  // operand type of the products: f16, unless the cache or (streamed rows) the queries are bf16 / fp32
  constexpr bool BF = KF == KF_BF16 || (NT == 0 && QT != CUDA_LLM_F16);
  constexpr bool SCALED = NT > 0 && F8 && QT != CUDA_LLM_F16;
  constexpr int TERMS = QT != CUDA_LLM_F32 ? 1 : NT ? 2 : 3;  // of an fp32 query: f16 hi + lo, or three bf16
  constexpr int QN = NT ? NT : 1;
  // Block scales of streamed rows go into the keys: bf16 holds code x 2^(block exponent - the token's largest) exactly down to
  // 2^-117 of the largest block; the largest exponent scales the whole dot product.
  constexpr bool FOLD = MX && NT == 0 && BF;
  constexpr bool KEPT = NT == 0 && QT != CUDA_LLM_F32;  // up to kWgtRows streamed rows lie in shared memory
  constexpr int QCH = D / 8;                            // 16-byte chunks of a row there
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t full = base, empty = base + 8 * kWgtMaxStages, live_at = base + 128, ring = base + kWgtHeader;
  int* pre = reinterpret_cast<int*>(smem + 192);  // [S + 1] stages before each sequence
  int* lens = pre + kWgtSeqs + 4;                 // [S] context lengths
  volatile int* fail_ptr = reinterpret_cast<volatile int*>(smem + 160);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < gm.n_stages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, WARPS);
    }
    *fail_ptr = 0;
    mbar_fence_init();
  }
  const WeightsPlan pl = make_plan<32 * (WARPS + 1)>(a, gm.tok_stage, gm.n_hg, pre, lens);
  if (pl.w0 >= pl.w1) return;
  if (warp == WARPS) {
    produce(a, gm, map, pl, full, empty, live_at, ring, fail_ptr);
    return;
  }

  const int g = lane >> 2, t = lane & 3;
  const int groups = a.page >> 4;  // 16-token groups of a page
  const int hl = warp & (gm.hg - 1), tg0 = warp / gm.hg * U, pg0 = tg0 / groups, sub0 = tg0 % groups;
  const uint32_t row_bytes = a.page * (F8 ? 1 : 2);
  // this lane's places in a stage: rows for ldmatrix, scales, page bit; a warp's units are neighbouring groups of one head
  uint32_t key_at[U][2], scale_at[U];
  int pg[U];
#pragma unroll
  for (int x = 0; x < U; ++x) {
    const int sub = (sub0 + x) % groups;
    pg[x] = pg0 + (sub0 + x) / groups;
    const uint32_t slab = ring + pg[x] * gm.k_bytes + hl * gm.k_head;
    key_at[x][0] = slab + key_row<KF>(lane, row_bytes, sub * (F8 ? 1 : 2), 0);
    key_at[x][1] = slab + key_row<KF>(lane, row_bytes, sub * (F8 ? 1 : 2), 1);
    scale_at[x] = ring + gm.pages * gm.k_bytes + pg[x] * gm.s_bytes + hl * gm.s_head + (sub * 16 + 2 * g) * (MX ? 1 : 4);
  }
  const int lane_tok = tg0 * 16 + (F8 ? 2 * g + (t & 1) : g + 8 * (t & 1));  // lanes t = 0, 1 keep the scores of two tokens of a unit
  uint32_t qf[QN][TERMS][D / 32][4];
  RowPair rp[QN];

  // the task one stage ahead: where it is, and its old scores, on their way while the stage in hand is worked on
  int s = pl.s0, ctx = 0, per = 1, hgi = 0, u = 0, left = 0, q0 = 0, n_q = 0, seq = -1, no_old = 0;
  float* sp = nullptr;
  float old[U];
  auto locate = [&](int w) {
    if (left == 0) {  // another sequence or head group
      while (w >= pl.pre[s + 1]) ++s;
      if (s != seq) {
        seq = s;
        ctx = pl.lens[s];
        per = (pl.pre[s + 1] - pl.pre[s]) / gm.n_hg;
        q0 = a.cuq ? a.cuq[s] : a.q_first + s;
        const int q1 = a.cuq ? a.cuq[s + 1] : q0 + 1;
        n_q = q1 - q0;
        if (q0 < 0 || q1 < q0 || q1 > a.total_q) {
          if (a.status && lane == 0) atomicOr(a.status, CUDA_LLM_ST_BAD_QLEN);
          q0 = n_q = 0;
        }
        no_old = (t < 2 && a.decay != 0.f) ? ctx - (a.keep_old ? 0 : n_q) : 0;  // scores from here on start at zero
      }
      hgi = (w - pl.pre[s]) / per;
      u = w - pl.pre[s] - hgi * per;
      left = per - u;
      sp = a.scores + s * a.st_seq + (hgi * gm.hg + hl) * a.st_head + u * gm.tok_stage + lane_tok;
    } else {
      ++u;
      sp += gm.tok_stage;
    }
    --left;
    const int tok = u * gm.tok_stage + lane_tok;
#pragma unroll
    for (int x = 0; x < U; ++x) old[x] = tok + 16 * x < no_old ? sp[16 * x] : 0.f;
  };
  locate(pl.w0);
  int cur_s = -1, cur_h = -1, cur_r = -1, st = 0;
  uint32_t par = 0, ring_off = 0;
  bool dead = false;
  for (int w = pl.w0; w < pl.w1; ++w) {
    const int my_s = s, h = hgi * gm.hg + hl, tok0 = u * gm.tok_stage + tg0 * 16, my_ctx = ctx, my_q0 = q0, my_nq = n_q, rows = n_q * a.group;
    float* const my_sp = sp;
    float my_old[U];
#pragma unroll
    for (int x = 0; x < U; ++x) my_old[x] = old[x];
    if (w + 1 < pl.w1) locate(w + 1);
    if (KEPT && rows <= kWgtRows && (my_s != cur_s || h != cur_h)) {
      // another sequence or head (of all warps alike): its rows, words already rotated for the lanes that will read them, and
      // {log-sum-exp, first token not seen} of every row
      cur_s = my_s;
      cur_h = h;
      asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
      for (int e = tid; e < ((rows + 7) & ~7) * QCH; e += 32 * WARPS) {
        const int r = e / QCH, c = e % QCH, from = min(r, rows - 1), j = from / a.group;
        const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + ((size_t)(my_q0 + j) * a.Hq + h * a.group + (from - j * a.group)) * D + c * 8);
        uint32_t x[4] = {v.x, v.y, v.z, v.w};
        rotate_words(x, c & 3);
        sts128(base + gm.q_off + (r * QCH + (c ^ ((r & 1) << 2))) * 16, x[0], x[1], x[2], x[3]);
      }
      for (int r = tid; r < ((rows + 7) & ~7); r += 32 * WARPS) {
        RowPair x;
        row_pair(a, r, rows, my_q0, my_nq, my_ctx, h, 0, x);
        sts32(base + gm.q_off + kWgtRows * QCH * 16 + r * 8, __float_as_int(x.lse2[0]));
        sts32(base + gm.q_off + kWgtRows * QCH * 16 + r * 8 + 4, x.limit[0]);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
    }
    if (!dead && !mbar_wait(full + 8 * st, par, 0)) {  // the warp goes on without work: others may wait for it at the barrier above
      dead = true;
      *fail_ptr = 1;
    }
    if (tok0 < my_ctx && !dead) {
      auto fetch_rows = [&](int r0) {
        cur_s = my_s;
        cur_h = h;
        cur_r = r0;
#pragma unroll
        for (int nt = 0; nt < QN; ++nt) {
          // rows that pad a block repeat the last one, with a weight of zero: an infinity in K then meets no zero
          const int r = min(r0 + nt * 8 + g, rows - 1), j = a.group_shift >= 0 ? r >> a.group_shift : r / a.group;
          const size_t at = ((size_t)(my_q0 + j) * a.Hq + h * a.group + (r - j * a.group)) * D;
          row_pair(a, r0 + nt * 8, rows, my_q0, my_nq, my_ctx, h, t, rp[nt]);
          if constexpr (SCALED) load_rows_scaled<D, QT, TERMS>(a.q, at, rows > 0, t, qf[nt], rp[nt].inv);
          else load_rows<D, QT>(a.q, at, rows > 0, t, qf[nt]);
        }
      };
      if (NT > 0 && (my_s != cur_s || h != cur_h || cur_r != 0)) fetch_rows(0);
      const uint32_t live = lds32(live_at + 4 * st);
      float f_tok[U][2], sum[U][2];
      uint32_t mx[U][MX ? D / 32 : 1];
#pragma unroll
      for (int x = 0; x < U; ++x) {
        f_tok[x][0] = f_tok[x][1] = a.scale_log2;
        sum[x][0] = sum[x][1] = 0.f;
        if (MX) {
#pragma unroll
          for (int p = 0; p < D / 32; ++p) mx[x][p] = lds16(scale_at[x] + ring_off + p * a.page);
          if (FOLD) {
            uint32_t ea = 0, eb = 0;
#pragma unroll
            for (int p = 0; p < D / 32; ++p) {
              ea = max(ea, mx[x][p] & 0xffu);
              eb = max(eb, mx[x][p] >> 8);
            }
            f_tok[x][0] *= e8m0_to_f32(ea);
            f_tok[x][1] *= e8m0_to_f32(eb);
#pragma unroll
            for (int p = 0; p < D / 32; ++p)  // biased exponents of 2^(block - largest), 0 (a factor of zero) below 2^-126
              mx[x][p] = (uint32_t)max(0, 127 + (int)(mx[x][p] & 0xffu) - (int)ea) | (uint32_t)max(0, 127 + (int)(mx[x][p] >> 8) - (int)eb) << 8;
          }
        } else if (F8) {
          float fa, fb;
          if (a.scale_mode == CUDA_LLM_SCALE_PER_TOKEN) {
            const uint2 v = lds64(scale_at[x] + ring_off);
            fa = __uint_as_float(v.x);
            fb = __uint_as_float(v.y);
          } else {
            const float* ks = reinterpret_cast<const float*>(a.ks);
            fa = 0.f;
            if (a.scale_mode == CUDA_LLM_SCALE_PER_HEAD) fa = ks[h];
            else if (live >> pg[x] & 1) fa = ks[(size_t)a.bt[(size_t)my_s * a.max_blocks + (tok0 + 16 * x) / a.page] * a.Hkv + h];
            fb = fa;
          }
          f_tok[x][0] *= fa;
          f_tok[x][1] *= fb;
        }
      }
      // Every token is compared with the row's limit: a flag for "all rows see all tokens" saves less than it costs (two sequences of 20001 and
      // 32768 tokens, 8 KV heads, 32 rows each: 39 us like this, 43-45 us with a flag that also covers rows that saw nothing).
      auto add_weights = [&](int x, const float (&c)[4], const RowPair& r) {
        const int tok_a = tok0 + 16 * x + (F8 ? 2 * g : g), tok_b = tok_a + (F8 ? 1 : 8);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float wa = fast_exp2(fmaf(c[y], f_tok[x][0] * r.inv[y], -r.lse2[y])), wb = fast_exp2(fmaf(c[2 + y], f_tok[x][1] * r.inv[y], -r.lse2[y]));
          sum[x][0] += tok_a < r.limit[y] ? wa : 0.f;
          sum[x][1] += tok_b < r.limit[y] ? wb : 0.f;
        }
      };
      // c += K block p of one unit times the rows of one 8-column block
      auto dot_block = [&](float (&c)[4], const uint32_t (&af)[2][4], const uint32_t (&q)[TERMS][D / 32][4], int x, int p) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
        if ((!MX || FOLD) && !(NT > 0 && TERMS == 2)) {
#pragma unroll
          for (int e = 0; e < 4; ++e) part[e] = c[e];
        }
        if (NT > 0 && TERMS == 2) {
          mma_any<BF>(part, af[0], q[TERMS - 1][p][0], q[TERMS - 1][p][1]);
          mma_any<BF>(part, af[1], q[TERMS - 1][p][2], q[TERMS - 1][p][3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) part[e] = MX ? part[e] * (1.f / 2048.f) : fmaf(part[e], 1.f / 2048.f, c[e]);
        }
#pragma unroll
        for (int term = (NT > 0 ? 1 : TERMS) - 1; term >= 0; --term) {
          mma_any<BF>(part, af[0], q[term][p][0], q[term][p][1]);
          mma_any<BF>(part, af[1], q[term][p][2], q[term][p][3]);
        }
        if (MX && !FOLD) {
          const float ea = e8m0_to_f32(mx[x][p] & 0xffu), eb = e8m0_to_f32(mx[x][p] >> 8);
          c[0] = fmaf(part[0], ea, c[0]);
          c[1] = fmaf(part[1], ea, c[1]);
          c[2] = fmaf(part[2], eb, c[2]);
          c[3] = fmaf(part[3], eb, c[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] = part[e];
        }
      };
      if constexpr (NT > 0) {
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += ROWS) {
          if (r0 > 0) fetch_rows(r0);
          float c[U][NT][4] = {};
#pragma unroll
          for (int p = 0; p < D / 32; ++p)
#pragma unroll
            for (int x = 0; x < U; ++x) {
              uint32_t af[2][4];
              load_key_block<KF>(key_at[x], ring_off + p * 32 * row_bytes, af);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) dot_block(c[x][nt], af, qf[nt], x, p);
            }
#pragma unroll
          for (int x = 0; x < U; ++x)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) add_weights(x, c[x][nt], rp[nt]);
        }
      } else {
        uint32_t af[U][D / 32][2][4];
#pragma unroll
        for (int x = 0; x < U; ++x)
#pragma unroll
          for (int p = 0; p < D / 32; ++p) {
            load_key_block<KF>(key_at[x], ring_off + p * 32 * row_bytes, af[x][p]);
            if (F8 && BF) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t v = af[x][p][e >> 2][e & 3];
                const float up = !FOLD ? 1.f : __uint_as_float((e & 1 ? mx[x][p] >> 8 : mx[x][p] & 0xffu) << 23);
                af[x][p][e >> 2][e & 3] = pack_bf16x2(f16x2_lo(v) * up, f16x2_hi(v) * up);
              }
            }
          }
        auto add_rows = [&](const uint32_t (&q)[TERMS][D / 32][4], const RowPair& r) {
          float c[U][2][4] = {};  // two chains of products per unit
#pragma unroll
          for (int p = 0; p < D / 32; ++p)
#pragma unroll
            for (int x = 0; x < U; ++x) dot_block(c[x][p & 1], af[x][p], q, x, p);
#pragma unroll
          for (int x = 0; x < U; ++x) {
#pragma unroll
            for (int e = 0; e < 4; ++e) c[x][0][e] += c[x][1][e];
            add_weights(x, c[x][0], r);
          }
        };
        if (KEPT && rows <= kWgtRows) {
#pragma unroll 2
          for (int r0 = 0; r0 < rows; r0 += 8) {
            const uint8_t* const row = smem + gm.q_off + (r0 + g) * QCH * 16;
            uint32_t q[TERMS][D / 32][4];
#pragma unroll
            for (int p = 0; p < D / 32; ++p) {
              const uint4 v = *reinterpret_cast<const uint4*>(row + (((p * 4 + t) ^ ((g & 1) << 2)) << 4));
              q[0][p][0] = v.x; q[0][p][1] = v.y; q[0][p][2] = v.z; q[0][p][3] = v.w;
            }
            const uint4 v = *reinterpret_cast<const uint4*>(smem + gm.q_off + kWgtRows * QCH * 16 + (r0 + 2 * t) * 8);
            RowPair r;
            r.lse2[0] = __uint_as_float(v.x); r.limit[0] = (int)v.y;
            r.lse2[1] = __uint_as_float(v.z); r.limit[1] = (int)v.w;
            r.inv[0] = r.inv[1] = 1.f;
            add_rows(q, r);
          }
        } else {
#pragma unroll 1
          for (int r0 = 0; r0 < rows; r0 += 8) {
            fetch_rows(r0);
            add_rows(qf[0], rp[0]);
          }
        }
      }
#pragma unroll
      for (int x = 0; x < U; ++x) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sum[x][e] += __shfl_xor_sync(0xffffffffu, sum[x][e], 1);
          sum[x][e] += __shfl_xor_sync(0xffffffffu, sum[x][e], 2);
        }
        if (t < 2 && (live >> pg[x] & 1) && tok0 - tg0 * 16 + lane_tok + 16 * x < my_ctx)
          my_sp[16 * x] = fmaf(my_old[x], a.decay, (t & 1) ? sum[x][1] : sum[x][0]);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + 8 * st);
    ring_off += gm.stage_bytes;
    if (++st == gm.n_stages) {
      st = 0;
      ring_off = 0;
      par ^= 1;
    }
  }
}

template <int D, int KF, int QT, int NT, bool MX, int U>
static cudaError_t go(const WeightsArgs& a, const WeightsGeom& gm, const WeightsMap& map, int grid, cudaStream_t st) {
  auto kern = kv_weights_kernel<D, KF, QT, NT, MX, U>;
  static int configured[64] = {0};
  cudaError_t e = allow_shared_memory((const void*)kern, (int)kWgtBudget, configured);
  if (e != cudaSuccess) return e;
  kern<<<grid, 32 * ((NT ? kWgtWarps : 2 * kWgtWarps) + 1), gm.smem, st>>>(a, gm, map);
  return cudaGetLastError();
}

template <int D, int KF, int QT, bool MX>
static cudaError_t go_rows(const WeightsArgs& a, const WeightsGeom& gm, const WeightsMap& map, int grid, int nt, cudaStream_t st) {
  if constexpr (kFourUnits<D, KF, QT>)
    if (nt == 1 && gm.units == 4 * kWgtWarps) return go<D, KF, QT, 1, MX, 4>(a, gm, map, grid, st);
  if (nt == 1) return go<D, KF, QT, 1, MX, 2>(a, gm, map, grid, st);
  if constexpr (QT != CUDA_LLM_F32)
    if (nt == 2) return go<D, KF, QT, 2, MX, 2>(a, gm, map, grid, st);
  return go<D, KF, QT, 0, MX, 1>(a, gm, map, grid, st);
}
template <int D, int KF, int QT>
static cudaError_t go_scales(const WeightsArgs& a, const WeightsGeom& gm, const WeightsMap& map, int grid, int nt, cudaStream_t st) {
  if constexpr (KF == KF_E4M3)
    if (a.scale_mode == CUDA_LLM_SCALE_MX_E8M0) return go_rows<D, KF, QT, true>(a, gm, map, grid, nt, st);
  return go_rows<D, KF, QT, false>(a, gm, map, grid, nt, st);
}
template <int D>
static cudaError_t go_types(const WeightsArgs& a, const WeightsGeom& gm, const WeightsMap& map, int grid, int nt, cudaStream_t st) {
  if (a.k_format == CUDA_LLM_KV_F16) return go_scales<D, KF_F16, CUDA_LLM_F16>(a, gm, map, grid, nt, st);
  if (a.k_format == CUDA_LLM_KV_BF16) return go_scales<D, KF_BF16, CUDA_LLM_BF16>(a, gm, map, grid, nt, st);
  if (a.q_dtype == CUDA_LLM_F32) return go_scales<D, KF_E4M3, CUDA_LLM_F32>(a, gm, map, grid, nt, st);
  if (a.q_dtype == CUDA_LLM_F16) return go_scales<D, KF_E4M3, CUDA_LLM_F16>(a, gm, map, grid, nt, st);
  return go_scales<D, KF_E4M3, CUDA_LLM_BF16>(a, gm, map, grid, nt, st);
}

static cudaError_t launch_kv_weights(WeightsArgs a, int max_q_len, int sms, cudaStream_t st) {
  const long long declared = (long long)a.group * (max_q_len < 1 ? 1 : max_q_len);
  // rows that stay in registers: 8, 16 (16-bit queries), or none
  const int nt = declared <= 8 ? 1 : declared <= 16 && a.q_dtype != CUDA_LLM_F32 ? 2 : 0;
  const int eb = a.k_format == CUDA_LLM_KV_FP8_E4M3 ? 1 : 2, groups = a.page / 16;
  const long long cap = (long long)a.max_blocks * a.page < a.max_tokens ? (long long)a.max_blocks * a.page : a.max_tokens;
  // units of a stage; the larger stage only where there are several of them for every SM (1000 tokens of one sequence would keep
  // 16 SMs busy instead of 32)
  const bool four = nt == 1 && a.q_dtype != CUDA_LLM_F32 && (eb == 1 || a.D == 64) && cap * a.Hkv * a.S / 16 >= 4ll * 4 * kWgtWarps * sms;
  // Many rows (16-bit queries): on tcgen05.  us here / there, E4M3 keys: 20 rows 162 / 219, 64 rows 68 / 68, 128 rows 76 / 54, 256
  // rows 360 / 66, 1024 rows 434 / 82; 16-bit keys: 64 rows 31 / 37, 128 rows 39 / 49.  8 heads of 1000 tokens, fewer tiles than
  // SMs, 128 rows: 14.5 / 16.4.  fp32 queries and fp16 queries on block scales have no form there (20001 and 32768 tokens x 8 heads, 128
  // rows 374 and 137 us, 1024 rows 2650 and 1635, where bf16 queries take 53 and 255).
  const bool fills = cap * a.Hkv * a.S >= 256ll * sms;
  const bool window = (declared > kWgtRows || (declared > 64 && eb == 1 && fills)) && a.q_dtype != CUDA_LLM_F32 &&
                      !(a.q_dtype == CUDA_LLM_F16 && eb == 1 && a.scale_mode == CUDA_LLM_SCALE_MX_E8M0);
  const int want = (four ? 4 : 2) * kWgtWarps;
  WeightsGeom gm;
  gm.hg = nt ? 8 : 1;
  while (a.Hkv % gm.hg || gm.hg * groups > want) gm.hg >>= 1;
  gm.n_hg = a.Hkv / gm.hg;
  gm.pages = want / (gm.hg * groups);
  gm.tok_stage = gm.pages * a.page;
  gm.units = gm.pages * groups * gm.hg;
  gm.k_head = (uint32_t)a.D * a.page * eb;
  gm.s_head = eb == 2 ? 0u : a.scale_mode == CUDA_LLM_SCALE_PER_TOKEN ? (uint32_t)a.page * 4
              : a.scale_mode == CUDA_LLM_SCALE_MX_E8M0 ? (uint32_t)(a.D / 32) * a.page : 0u;
  gm.k_bytes = gm.hg * gm.k_head;
  gm.s_bytes = gm.hg * gm.s_head;
  gm.stage_bytes = ((gm.k_bytes + gm.s_bytes) * gm.pages + 1023) / 1024 * 1024;
  const uint32_t q_bytes = nt || a.q_dtype == CUDA_LLM_F32 ? 0u : (uint32_t)kWgtRows * (a.D * 2 + 8);
  gm.n_stages = (int)((kWgtBudget - kWgtHeader - q_bytes) / gm.stage_bytes);
  if (gm.n_stages > kWgtMaxStages) gm.n_stages = kWgtMaxStages;
  gm.q_off = kWgtHeader + gm.n_stages * gm.stage_bytes;
  gm.smem = gm.q_off + q_bytes;
  WeightsMap map = {};
  gm.box_rows = 0;
  if (a.page * eb >= 64) {
    EncodeTiledFn enc = tensor_map_encoder();
    if (!enc) return cudaErrorNotSupported;
    gm.box_rows = gm.hg * a.D < 256 ? gm.hg * a.D : 256;
    const cuuint64_t dims[3] = {(cuuint64_t)a.page, (cuuint64_t)a.Hkv * a.D, (cuuint64_t)a.num_blocks};
    const cuuint64_t strides[2] = {(cuuint64_t)a.page * eb, (cuuint64_t)a.Hkv * a.D * a.page * eb};
    const cuuint32_t box[3] = {(cuuint32_t)a.page, (cuuint32_t)gm.box_rows, 1}, estr[3] = {1, 1, 1};
    if (enc(&map.k, eb == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(a.kc), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, a.page * eb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  a.group_shift = (a.group & (a.group - 1)) ? -1 : __builtin_ctz(a.group);
  const int S = a.S;
  for (int s0 = 0; s0 < S; s0 += kWgtSeqs) {
    WeightsArgs x = a;
    x.S = S - s0 < kWgtSeqs ? S - s0 : kWgtSeqs;
    x.bt += (size_t)s0 * a.max_blocks;
    x.ctx += s0;
    if (x.cuq) x.cuq += s0;
    x.q_first = s0;
    x.scores += s0 * a.st_seq;
    const long long most = (cap + gm.tok_stage - 1) / gm.tok_stage * gm.n_hg * x.S;
    const int grid = (int)(most < sms ? most : sms);
    const cudaError_t e = window ? launch_kv_weights_window(x, cap, sms, st) : a.D == 64 ? go_types<64>(x, gm, map, grid, nt, st) : go_types<128>(x, gm, map, grid, nt, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
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
  if (p->max_tokens > (1 << 30)) return refuse(CUDA_LLM_EINVAL, "score rows of more than 2^30 entries");
  if (!rows_apart(p->score_strides[0], p->num_seqs, p->score_strides[1], p->num_kv_heads, p->max_tokens))
    return refuse(CUDA_LLM_EINVAL, "score rows overlap");
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
  a.causal = p->is_causal ? 1 : 0; a.keep_old = p->keep_old ? 1 : 0; a.scale_log2 = p->softmax_scale * 1.4426950408889634f; a.decay = p->decay;
  a.q_first = 0;
  return cuda_result(launch_kv_weights(a, p->max_q_len, current_sm_count(), reinterpret_cast<cudaStream_t>(stream)), "kv_weights_kernel launch");
}
