// Accumulated attention weight, windows of a prompt: many query rows per KV head, on the 5th-generation tensor cores.
//
//   S = K Q^T (256 tokens x 128 rows, as two accumulators), weight = sum over the rows that see the token of 2^(S f_token - lse2_row)
//
// Tokens are the M side, so that one thread owns one token: its weight is a sum over its own TMEM lane, its scale and its score
// are its own, and nothing crosses lanes.  A persistent CTA per SM walks an equal range of (sequence, KV head, 256 tokens):
//   warps 0..3, 4..7  weights of one half of the tile each (two S buffers each): tcgen05.ld, exponentials, the score
//   warps 8..15       K: 16 tokens of a row per load, one tile ahead in registers, widened to the queries' type and stored as the
//                     MN-major operand (a page's rows are tokens, so no transposition); blocks of 128 query rows
//                     and their log-sum-exps into a ring
//   warp 8            also allocates TMEM and issues the MMAs
// E4M3 codes are exact in f16 and bf16.  Block scales go into the keys (bf16 queries): bf16 holds code x 2^(block exponent - the
// token's largest) exactly down to 2^-117 of the largest block; the largest exponent and other scales multiply S.
// Measured (events around single calls; E4M3 keys with block scales, 32 queries x 4 heads against 52769 tokens of 8 heads of 128):
// 54 us, where the warp-level kernel takes 76; 256 rows of 4 sequences of 8000-16384 tokens 66 us (387 TFLOP/s) against 360, 1024
// rows against 2 of 5000-8192 82 us against 434.  About 7700 cycles a tile of 128 rows, of which the exponentials need 2048; no
// pipe is full (exponentials 29 %, tensor 16 %, issue 41 %), so it is latency that bounds it.
// Slower: 128 tokens a tile (68 us), an issuing warp of its own (68, it leaves too few registers), MMAs issued by the weighing
// warps (61).
// The rows of a head stay in shared memory while its tokens pass, up to kWinBlocks blocks of 128; with more each tile loads
// them again.  Rows that pad a block repeat the last row with a weight of zero, so that an infinity in K meets no zero.
#include "kv_weights.cuh"
#include "softmax_math.cuh"
#include "tcgen05_primitives.cuh"

namespace b200 {

constexpr int kWinThreads = 512, kWinTokens = 256, kWinRows = 128, kWinBlocks = 2, kWinTiles = 2;
constexpr uint32_t kWinHeader = 9 * 1024;
constexpr uint32_t kWinBlind = 192 + 4 * (2 * kWgtSeqs + 4);  // of every block and loading warp: one of its rows saw nothing
static_assert(kWinBlind % 16 == 0 && kWinBlind + 16 * kWinBlocks <= kWinHeader, "header");

__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {  // read once: past the L1 cache
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <int D>
constexpr uint32_t win_smem() {
  return kWinHeader + kWinBlocks * (kWinRows * D * 2 + kWinRows * 8) + kWinTiles * kWinTokens * D * 2 + 1024;
}

// Where a role is in the CTA's range of tiles.  All roles walk alike.
struct WinWalk {
  int s, h, u, per, ctx, q0, n_q, rows, blocks;
  int entry, first;  // of the ring of row blocks: the segment's first entry; its first tile in this CTA
  bool kept;         // the segment's blocks stay until its end

  __device__ __forceinline__ void sequence(const WeightsArgs& a, const WeightsPlan& pl, bool report) {
    while (pl.pre[s + 1] <= pl.pre[s]) ++s;
    ctx = pl.lens[s];
    per = (ctx + kWinTokens - 1) / kWinTokens;
    q0 = a.cuq ? a.cuq[s] : a.q_first + s;
    const int q1 = a.cuq ? a.cuq[s + 1] : q0 + 1;
    n_q = q1 - q0;
    if (q0 < 0 || q1 < q0 || q1 > a.total_q) {
      if (report && a.status) atomicOr(a.status, CUDA_LLM_ST_BAD_QLEN);
      q0 = n_q = 0;
    }
    rows = n_q * a.group;
    blocks = (rows + kWinRows - 1) / kWinRows;
    kept = blocks <= kWinBlocks;
  }
  __device__ __forceinline__ void start(const WeightsArgs& a, const WeightsPlan& pl, bool report) {
    s = pl.s0;
    sequence(a, pl, report);
    const int w = pl.w0 - pl.pre[s];
    h = w / per;
    u = first = w - h * per;
    entry = 0;
  }
  __device__ __forceinline__ bool last(int w, const WeightsPlan& pl) const { return u == per - 1 || w == pl.w1 - 1; }
  __device__ __forceinline__ int block_entry(int rb) const { return entry + rb + (kept ? 0 : (u - first) * blocks); }
  __device__ __forceinline__ void next(const WeightsArgs& a, const WeightsPlan& pl, int w, bool report) {
    if (w + 1 >= pl.w1) return;
    if (++u < per) return;
    entry += kept ? blocks : (u - first) * blocks;
    u = first = 0;
    if (++h == a.Hkv) {
      h = 0;
      ++s;
      sequence(a, pl, report);
    }
  }
};

// QT: type of the queries and of the products; F8: E4M3 keys; MX: with block scales
template <int D, int QT, bool F8, bool MX>
__global__ void __launch_bounds__(kWinThreads, 1) kv_weights_window_kernel(const __grid_constant__ WeightsArgs a) {
  constexpr bool BF = QT == CUDA_LLM_BF16;
  constexpr uint32_t QCH = kWinRows * 128, QBLK = D / 64 * QCH, KCH = D * 128, KTILE = kWinTokens / 64 * KCH, KHALF = KTILE / 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t k_full = base, k_empty = base + 16, s_full = base + 32, s_free = base + 64, q_full = base + 96, q_empty = base + 128, done = base + 160,
                 tmem_slot = base + 168;
  volatile uint32_t* fail_ptr = reinterpret_cast<volatile uint32_t*>(smem + 172);
  int* pre = reinterpret_cast<int*>(smem + 192);
  int* lens = pre + kWgtSeqs + 4;
  const uint32_t sQ = base + kWinHeader, sK = sQ + kWinBlocks * QBLK;
  const uint32_t row_at = kWinHeader + kWinBlocks * QBLK + kWinTiles * KTILE;  // of every block: 128 x -lse2, 128 x first token not seen
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, page_shift = 31 - __clz(a.page);
  const WeightsPlan pl = make_plan<kWinThreads>(a, kWinTokens, a.Hkv, pre, lens);
  if (pl.w0 >= pl.w1) return;
  if (tid == 0) {
    for (int i = 0; i < kWinTiles; ++i) {
      mbar_init(k_full + 8 * i, 8);
      mbar_init(k_empty + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(s_free + 8 * i, 4);
    }
    for (int i = 0; i < kWinBlocks; ++i) {
      mbar_init(q_full + 8 * i, 8);
      mbar_init(q_empty + 8 * i, 9);  // the MMAs that read it and eight weighing warps
    }
    mbar_init(done, 1);
    *fail_ptr = 0;
    mbar_fence_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + 168);
  // Waits of whole warps suspend, so that they take no issue slots; the issuing thread's, on the path of every tile, poll.
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (mbar_wait(bar, parity, 0)) return true;
    *fail_ptr = 1;
    return false;
  };
  auto poll = [&](uint32_t bar, uint32_t parity) {
    if (tc_wait(bar, parity)) return true;
    *fail_ptr = 1;
    return false;
  };
  WinWalk at;
  at.start(a, pl, tid == 0);

  if (warp >= 8) {
    // ---- keys and query rows
    // A thread takes 16 tokens of some rows of one 32-row block (its scale), such that eight neighbours store to all banks.
    constexpr int N = D / 16, PIECES = F8 ? 1 : 2, EB = F8 ? 1 : 2;
    const int ltid = tid - 256, grp = ltid >> 4, d0 = ltid & 15;
    const int part = D == 128 ? d0 >> 2 : d0 >> 3;
    auto row_of = [&](int i) { return part * 32 + (D == 128 ? (d0 & 3) + 4 * (i ^ (part & 1)) : (d0 & 7) + 8 * i); };
    int tiles = 0;
    bool ok = true;
    uint4 key[N][PIECES], sc[MX ? D / 32 : 1];
    // the tile after the one in hand: where its keys and scales lie (null: nowhere); the one after that, and its page
    const uint8_t *p_ahead = nullptr, *sc_ahead = nullptr;
    WinWalk then = at;
    int then_w = pl.w0, blk_then = -1;
    auto block_of = [&](const WinWalk& x) -> int {
      const int t = x.u * kWinTokens + grp * 16;
      return x.blocks == 0 || t >= x.ctx ? -1 : a.bt[(size_t)x.s * a.max_blocks + (t >> page_shift)];
    };
    auto go_on = [&]() {
      p_ahead = sc_ahead = nullptr;
      if (blk_then >= 0 && blk_then < a.num_blocks) {
        const int off = (then.u * kWinTokens + grp * 16) & (a.page - 1);
        const size_t slab = (size_t)blk_then * a.Hkv + then.h;
        p_ahead = a.kc + (slab * D * a.page + off) * EB;
        if (MX) sc_ahead = a.ks + slab * (D / 32) * a.page + off;
      }
      blk_then = -1;
      if (then_w + 1 < pl.w1) {
        then.next(a, pl, then_w, false);
        blk_then = block_of(then);
      }
      ++then_w;
    };
    auto fetch_row = [&](int i) {
#pragma unroll
      for (int y = 0; y < PIECES; ++y) {
        key[i][y] = make_uint4(0, 0, 0, 0);
        if (p_ahead) key[i][y] = ld_stream(p_ahead + row_of(i) * a.page * EB + y * 16);
      }
    };
    auto fetch_scales = [&]() {
#pragma unroll
      for (int i = 0; i < (MX ? D / 32 : 0); ++i) {
        sc[i] = make_uint4(0, 0, 0, 0);
        if (sc_ahead) sc[i] = __ldg(reinterpret_cast<const uint4*>(sc_ahead + i * a.page));
      }
    };
    auto query_of = [&](int r) { return a.group_shift >= 0 ? r >> a.group_shift : r / a.group; };
    auto load_block = [&](int e, int rb) -> bool {  // 128 query rows
      const int qs = e % kWinBlocks;
      if (!wait(q_empty + 8 * qs, ((e / kWinBlocks) & 1) ^ 1)) return false;
      {  // all loads at once: one after another they would cost a latency each
        uint4 v[D / 16];
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          const int at_x = x * 256 + ltid, row = at_x / (D / 8), c = at_x % (D / 8), r = min(rb * kWinRows + row, at.rows - 1), j = query_of(r);
          v[x] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + ((size_t)(at.q0 + j) * a.Hq + at.h * a.group + (r - j * a.group)) * D + c * 8));
        }
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          const int at_x = x * 256 + ltid, row = at_x / (D / 8), c = at_x % (D / 8);
          sts128(sQ + qs * QBLK + (c >> 3) * QCH + row * 128 + (((c & 7) ^ (row & 7)) << 4), v[x].x, v[x].y, v[x].z, v[x].w);
        }
      }
      const int r = rb * kWinRows + ltid;
      float nl = -__builtin_huge_valf();  // no such row, or a row that saw nothing: weights of zero
      int limit = 0;
      bool blind = false;
      if (ltid < kWinRows && r < at.rows) {
        const int j = query_of(r);
        const float v = a.lse[(size_t)(at.q0 + j) * a.Hq + at.h * a.group + (r - j * a.group)];
        if (v != -__builtin_huge_valf()) {
          nl = v * -1.4426950408889634f;
          limit = a.causal ? at.ctx - at.n_q + 1 + j : at.ctx;
        } else {
          blind = true;  // its products may be NaN, and only the comparison with its limit keeps them out
        }
      }
      blind = __any_sync(0xffffffffu, blind);
      if (ltid < kWinRows) {
        reinterpret_cast<float*>(smem + row_at + qs * 1024)[ltid] = nl;
        reinterpret_cast<int*>(smem + row_at + qs * 1024 + 512)[ltid] = limit;
        if (lane == 0) reinterpret_cast<int*>(smem + kWinBlind + qs * 16)[ltid >> 5] = blind;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full + 8 * qs);
      return true;
    };
    const uint32_t idesc = instr_desc_f16(BF ? 1 : 0, 0, 128, kWinRows) | (1u << 15);  // the keys MN-major
    const uint32_t hi = smem_desc_hi_sw128(1024), k_lo = smem_desc_lo(sK, KCH), q_lo = smem_desc_lo(sQ, 16);
    int items = 0;  // (tile, block of rows) so far
    // one block of rows times the tile in hand, by one thread
    auto multiply = [&](int e, int kb) -> bool {
      const int qs = e % kWinBlocks, buf = items & 1, par = (items >> 1) & 1;
      ++items;
      if (!poll(q_full + 8 * qs, (e / kWinBlocks) & 1)) return false;
#pragma unroll
      for (int team = 0; team < 2; ++team) {
        const int slot = 2 * team + buf;
        if (!poll(s_free + 8 * slot, par ^ 1)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16_parts(tmem + slot * 128, k_lo + ((kb * KTILE + team * KHALF + kk * 2048) >> 4), hi,
                         q_lo + ((qs * QBLK + (kk >> 2) * QCH + (kk & 3) * 32) >> 4), hi, idesc, kk > 0 ? 1u : 0u);
        umma_commit(s_full + 8 * slot);
      }
      return true;
    };
    blk_then = block_of(then);
    go_on();
#pragma unroll
    for (int i = 0; i < N; ++i) fetch_row(i);
    fetch_scales();
    go_on();
    for (int w = pl.w0; ok && w < pl.w1; ++w) {
      const bool work = at.blocks > 0;
      const int kb = tiles % kWinTiles;
      if (work) {
        if (at.kept && at.u == at.first)
          for (int rb = 0; ok && rb < at.blocks; ++rb) ok = load_block(at.block_entry(rb), rb);
        ok = ok && wait(k_empty + 8 * kb, ((tiles / kWinTiles) & 1) ^ 1);
        if (!ok) break;
        const uint32_t to = sK + kb * KTILE + (grp >> 2) * KCH;
        uint32_t up[8];  // 2^(block - largest) of two tokens, bf16; zero below 2^-126
        if (MX) {
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            uint32_t top = 0, own = 0;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
              const uint32_t e = (&sc[i].x)[y];
              top = __vmaxu4(top, e);
              if (i == part) own = e;
            }
            const uint32_t f = __vsubus4(0x7f7f7f7fu, __vsub4(top, own));
            up[2 * y] = prmt(f, 0, 0x4140) << 7;
            up[2 * y + 1] = prmt(f, 0, 0x4342) << 7;
          }
          fetch_scales();
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {  // a row of the next tile is fetched where one of this is done
          const int d = row_of(i);
          uint32_t o[8];
          if (F8) {
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t code = (&key[i][0].x)[y];
              o[2 * y] = e4m3x2_to_f16x2_lo(code);
              o[2 * y + 1] = e4m3x2_to_f16x2_hi(code);
#pragma unroll
              for (int z = 2 * y; BF && z < 2 * y + 2; ++z) {
                o[z] = pack_bf16x2(f16x2_lo(o[z]), f16x2_hi(o[z]));
                if (MX) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(o[z]) : "r"(up[z]));
              }
            }
          } else {
#pragma unroll
            for (int y = 0; y < 8; ++y) o[y] = (&key[i][y >> 2].x)[y & 3];
          }
          fetch_row(i);
          const int j = (grp & 3) * 2;
          sts128(to + d * 128 + ((j ^ (d & 7)) << 4), o[0], o[1], o[2], o[3]);
          sts128(to + d * 128 + (((j + 1) ^ (d & 7)) << 4), o[4], o[5], o[6], o[7]);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(k_full + 8 * kb);
        if (tid == 256) {
          ok = poll(k_full + 8 * kb, (tiles / kWinTiles) & 1);
          if (at.kept) {
            for (int rb = 0; ok && rb < at.blocks; ++rb) ok = multiply(at.block_entry(rb), kb);
            umma_commit(k_empty + 8 * kb);
            for (int rb = 0; at.last(w, pl) && rb < at.blocks; ++rb) umma_commit(q_empty + 8 * (at.block_entry(rb) % kWinBlocks));
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        ++tiles;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) fetch_row(i);
        fetch_scales();
      }
      go_on();
      if (work && !at.kept) {
        for (int rb = 0; ok && rb < at.blocks; ++rb) {
          const int e = at.block_entry(rb);
          ok = load_block(e, rb);
          if (ok && tid == 256) {
            ok = multiply(e, kb);
            umma_commit(q_empty + 8 * (e % kWinBlocks));
          }
        }
        if (tid == 256) umma_commit(k_empty + 8 * kb);
        ok = __all_sync(0xffffffffu, ok);
      }
      at.next(a, pl, w, false);
    }
    if (tid == 256) {
      umma_commit(done);
      tc_wait(done, 0);  // nothing runs on when the tensor memory is given back
    }
    __syncwarp();
  } else {
    // ---- weights
    const int team = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    int items = 0;
    bool ok = true;
    // the next tile: its scales and old score; the page of the one after it
    uint32_t ahead_e[MX ? D / 32 : 1] = {};
    float ahead_f = 1.f, ahead_old = 0.f;
    int ahead_blk = -1, blk_then = -1, ahead_w = pl.w0;
    WinWalk ahead = at;
    auto block_of = [&](const WinWalk& x) -> int {
      const int tok = x.u * kWinTokens + tid;
      if (tok >= x.ctx) return -1;
      const int blk = a.bt[(size_t)x.s * a.max_blocks + (tok >> page_shift)];
      if (blk >= 0 && blk < a.num_blocks) return blk;
      if (a.status) atomicOr(a.status, CUDA_LLM_ST_BAD_BLOCK);
      return -1;
    };
    auto fetch = [&]() {  // of tile `ahead`, whose page is known; then on to the page of the next
      ahead_blk = blk_then;
      ahead_old = 0.f;
      if (ahead_blk >= 0) {
        const int tok = ahead.u * kWinTokens + tid;
        const size_t slab = (size_t)ahead_blk * a.Hkv + ahead.h;
        if (a.decay != 0.f && (a.keep_old || tok < ahead.ctx - ahead.n_q)) ahead_old = a.scores[ahead.s * a.st_seq + ahead.h * a.st_head + tok];
        if (MX) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) ahead_e[i] = __ldg(a.ks + (slab * (D / 32) + i) * a.page + (tok & (a.page - 1)));
        } else if (F8) {
          const float* ks = reinterpret_cast<const float*>(a.ks);
          ahead_f = __ldg(a.scale_mode == CUDA_LLM_SCALE_PER_TOKEN ? ks + slab * a.page + (tok & (a.page - 1))
                          : a.scale_mode == CUDA_LLM_SCALE_PER_HEAD ? ks + ahead.h : ks + slab);
        }
      }
      blk_then = -1;
      if (ahead_w + 1 < pl.w1) {
        ahead.next(a, pl, ahead_w, false);
        blk_then = block_of(ahead);
      }
      ++ahead_w;
    };
    blk_then = block_of(ahead);
    fetch();
    for (int w = pl.w0; ok && w < pl.w1; ++w) {
      const int tok = at.u * kWinTokens + tid, blk = ahead_blk;
      float* const sp = a.scores + at.s * a.st_seq + at.h * a.st_head + tok;
      const float old = ahead_old;
      float f = a.scale_log2;
      if (MX) {
        uint32_t e = 0;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) e = max(e, ahead_e[i]);
        f *= e8m0_to_f32(e);
      } else if (F8) {
        f *= ahead_f;
      }
      fetch();
      const bool edge = (at.u + 1) * kWinTokens > at.ctx - at.n_q;  // some row may not see some token
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      for (int rb = 0; rb < at.blocks; ++rb, ++items) {
        const int e = at.block_entry(rb), qs = e % kWinBlocks, slot = 2 * team + (items & 1);
        ok = wait(q_full + 8 * qs, (e / kWinBlocks) & 1) && wait(s_full + 8 * slot, (items >> 1) & 1);
        if (!ok) break;
        __syncwarp();
        tc_fence_after();
        const float* nl = reinterpret_cast<const float*>(smem + row_at + qs * 1024);
        const int* limit = reinterpret_cast<const int*>(nl + kWinRows);
        const int cols = min(kWinRows, at.rows - rb * kWinRows);
        const int4 blind = *reinterpret_cast<const int4*>(smem + kWinBlind + qs * 16);
        const bool cut = edge || (blind.x | blind.y | blind.z | blind.w);
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) {
          uint32_t x[32];
          tmem_ld32(tmem + lanes + slot * 128 + c, x);
          tc_wait_ld();
          if (cut || c + 32 > cols) {
#pragma unroll
            for (int y = 0; y < 32; ++y) {
              const float p = fast_exp2(fmaf(__uint_as_float(x[y]), f, nl[c + y]));
              sum[y & 3] += tok < limit[c + y] ? p : 0.f;
            }
          } else {
#pragma unroll
            for (int y = 0; y < 32; y += 4) {
              const float4 n4 = *reinterpret_cast<const float4*>(nl + c + y);
              float p0, p1, p2, p3;
              ffma2(p0, p1, __uint_as_float(x[y]), __uint_as_float(x[y + 1]), f, f, n4.x, n4.y);
              ffma2(p2, p3, __uint_as_float(x[y + 2]), __uint_as_float(x[y + 3]), f, f, n4.z, n4.w);
              fadd2(sum[0], sum[1], sum[0], sum[1], fast_exp2(p0), fast_exp2(p1));
              fadd2(sum[2], sum[3], sum[2], sum[3], fast_exp2(p2), fast_exp2(p3));
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free + 8 * slot);
        if (!at.kept && lane == 0) mbar_arrive(q_empty + 8 * qs);
      }
      if (!ok) break;
      if (blk >= 0) *sp = fmaf(old, a.decay, (sum[0] + sum[1]) + (sum[2] + sum[3]));
      if (ok && at.kept && at.last(w, pl)) {
        __syncwarp();
        for (int rb = 0; ok && rb < at.blocks; ++rb) {
          const int e = at.block_entry(rb), qs = e % kWinBlocks;
          if (lane == 0) mbar_arrive(q_empty + 8 * qs);
        }
      }
      at.next(a, pl, w, false);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
  if (tid == 0 && *fail_ptr && a.status) atomicOr(a.status, CUDA_LLM_ST_TIMEOUT);
}

template <int D, int QT, bool F8, bool MX>
static cudaError_t go(const WeightsArgs& a, int grid, cudaStream_t st) {
  auto kern = kv_weights_window_kernel<D, QT, F8, MX>;
  static int configured[64] = {0};
  cudaError_t e = allow_shared_memory((const void*)kern, (int)win_smem<D>(), configured);
  if (e != cudaSuccess) return e;
  kern<<<grid, kWinThreads, win_smem<D>(), st>>>(a);
  return cudaGetLastError();
}
template <int D>
static cudaError_t go_types(const WeightsArgs& a, int grid, cudaStream_t st) {
  if (a.k_format == CUDA_LLM_KV_F16) return go<D, CUDA_LLM_F16, false, false>(a, grid, st);
  if (a.k_format == CUDA_LLM_KV_BF16) return go<D, CUDA_LLM_BF16, false, false>(a, grid, st);
  if (a.q_dtype == CUDA_LLM_F16) return go<D, CUDA_LLM_F16, true, false>(a, grid, st);
  if (a.scale_mode == CUDA_LLM_SCALE_MX_E8M0) return go<D, CUDA_LLM_BF16, true, true>(a, grid, st);
  return go<D, CUDA_LLM_BF16, true, false>(a, grid, st);
}

cudaError_t launch_kv_weights_window(const WeightsArgs& a, long long cap, int sms, cudaStream_t st) {
  const long long most = (cap + kWinTokens - 1) / kWinTokens * a.Hkv * a.S;
  const int grid = (int)(most < sms ? most : sms);
  return a.D == 64 ? go_types<64>(a, grid, st) : go_types<128>(a, grid, st);
}

}  // namespace b200
