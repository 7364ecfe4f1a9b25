// Eviction from a paged KV cache: which tokens stay (a selection by rank per sequence and KV head), and their move to the
// front of the same or of other pages.
//
// Measured, both kernels: 32 sequences x 8 heads of 2500-8000 tokens of 128 E4M3 values, in place down to 2048: 20 + 103 us; one
// sequence x 8 heads of 131072 bf16 tokens, 16384 of them into other pages: 28 + 109 us; one of 700 tokens down to 512: 18 us.
// A kept token is one element of every row, so DRAM moves whole slabs: 0.48 and 0.54 GB here (4.6 and 5.0 TB/s), where the
// kept tokens alone are 0.27 and 0.13 GB.  In place, few long rows are slow: two sequences of 4 heads, the longer cut from 51333 to
// 33301 tokens, take 566 us, since the 17 runs of a head follow one another.
#include <type_traits>

#include "host_common.cuh"
#include "tcgen05_primitives.cuh"

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

// Scores as unsigned integers of the same order: NaN lowest, then -inf .. +inf, -0 as +0; and back.
__device__ __forceinline__ uint32_t rank_key(float x) {
  const uint32_t u = x != x ? 0xffffffffu : __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_score(uint32_t k) { return __uint_as_float(k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u)); }

// ---- selection ------------------------------------------------------------------------------------------------------
// A thread-block cluster per (KV head, sequence); each CTA holds its part of the score row in shared memory.  The budget-th
// largest key comes from three passes over 11, 11 and 10 of its bits (the first, sign, exponent and two bits of the fraction,
// spreads scores of similar size over enough bins for plain atomics): a histogram per CTA, summed over the cluster
// through distributed shared memory.  Then each warp counts, and afterwards writes, the kept tokens of its own run
// of positions, so that the order needs one prefix sum.  The row is read once, before anything is written: new_scores may be
// scores.
constexpr int kSelMaxPart = 49152;  // scores per CTA: 192 KB

__device__ __forceinline__ uint32_t sel_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t sel_parts() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void sel_cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t sel_remote(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %1, %2;\n\tld.shared::cluster.u32 %0, [ra];\n\t}"
               : "=r"(v) : "r"(smem_u32(p)), "r"(rank) : "memory");
  return v;
}

constexpr int kSelBins = 2048;

// PER consecutive words of CTA `rank`
template <int PER>
__device__ __forceinline__ void sel_remote_vec(const uint32_t* p, uint32_t rank, uint32_t (&v)[PER]) {
  static_assert(PER == 2 || PER == 4, "");
  if constexpr (PER == 4)
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %4, %5;\n\tld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [ra];\n\t}"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(smem_u32(p)), "r"(rank) : "memory");
  else
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %2, %3;\n\tld.shared::cluster.v2.u32 {%0, %1}, [ra];\n\t}"
                 : "=r"(v[0]), "=r"(v[1]) : "r"(smem_u32(p)), "r"(rank) : "memory");
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const EvictArgs a) {
  constexpr int WARPS = THREADS / 32, PER = kSelBins / THREADS;
  extern __shared__ uint32_t row[];          // keys of this CTA's part
  __shared__ __align__(16) uint32_t hist[3][kSelBins];
  __shared__ uint32_t counts[2];             // kept for sure, on the edge: of this CTA
  __shared__ uint32_t warp_gt[WARPS], warp_eq[WARPS], found[2];
  asm volatile("griddepcontrol.launch_dependents;");
  const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = sel_rank(), parts = sel_parts();
  const int ctx = evict_ctx(a, s, h == 0 && rank == 0 && tid == 0);
  const int n_keep = min(ctx, a.budget);
  const float* sc = a.scores + s * a.st_seq + h * a.st_head;
  float* ns = a.new_scores ? a.new_scores + s * a.nst_seq + h * a.nst_head : nullptr;
  int32_t* kept = a.kept + ((size_t)s * a.Hkv + h) * a.budget;
  if (h == 0 && rank == 0 && tid == 0) a.new_ctx[s] = n_keep;
  for (int i = n_keep + (int)rank * THREADS + tid; i < a.budget; i += parts * THREADS) kept[i] = -1;
  if (ctx <= a.budget) {  // of the whole cluster
    for (int t = (int)rank * THREADS + tid; t < ctx; t += parts * THREADS) {
      kept[t] = t;
      if (ns && ns != sc) ns[t] = sc[t];
    }
    return;
  }
  const int t0 = (int)((long long)ctx * rank / parts), n = (int)((long long)ctx * (rank + 1) / parts) - t0;
#pragma unroll 4
  for (int i = tid; i < 3 * kSelBins; i += THREADS) (&hist[0][0])[i] = 0;
#pragma unroll 8
  for (int i = tid; i < n; i += THREADS) row[i] = rank_key(sc[t0 + i]);
  __syncthreads();
  const int m0 = max(0, a.sink - t0), m1 = min(n, ctx - a.recent - t0);  // tokens that are ranked
  uint32_t prefix = 0, left = (uint32_t)(n_keep - a.sink - a.recent);    // of them stay
#pragma unroll 1
  for (int pass = 0; pass < 3 && left > 0; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
#pragma unroll 4
    for (int i = m0 + tid; i < m1; i += THREADS) {
      const uint32_t k = row[i];
      if ((k & mask) == prefix) atomicAdd(&hist[pass][(k >> shift) & (kSelBins - 1) & (pass == 2 ? 1023u : 2047u)], 1u);
    }
    if (parts > 1) sel_cluster_sync();
    else __syncthreads();
    // a thread's bins from the top down, and how many keys lie above them
    uint32_t c[PER], mine = 0;
#pragma unroll
    for (int x = 0; x < PER; ++x) c[x] = 0;
    for (uint32_t q = 0; q < parts; ++q) {
      uint32_t y[PER];
      sel_remote_vec<PER>(&hist[pass][kSelBins - PER * (tid + 1)], q, y);
#pragma unroll
      for (int x = 0; x < PER; ++x) c[x] += y[PER - 1 - x];
    }
#pragma unroll
    for (int x = 0; x < PER; ++x) mine += c[x];
    uint32_t above = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, above, o);
      if (lane >= o) above += y;
    }
    if (lane == 31) warp_gt[warp] = above;
    __syncthreads();
    above += __reduce_add_sync(0xffffffffu, lane < warp && lane < WARPS ? warp_gt[lane] : 0u) - mine;
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      if (above < left && left <= above + c[x]) {  // one bin of one thread
        found[0] = (uint32_t)(kSelBins - 1 - (tid * PER + x));
        found[1] = left - above;
      }
      above += c[x];
    }
    __syncthreads();
    prefix |= found[0] << shift;
    left = found[1];
  }
  // keep all ranked keys above `edge` and the first `left` that equal it (none at all if no ranked token stays)
  const uint32_t edge = left > 0 ? prefix : 0xffffffffu;
  const int per = ((n + WARPS - 1) / WARPS + 31) & ~31, b0 = min(n, warp * per), b1 = min(n, b0 + per);
  auto above_at = [&](int i) { return i < m0 || i >= m1 || row[i] > edge; };
  auto edge_at = [&](int i) { return i >= m0 && i < m1 && row[i] == edge; };
  uint32_t gt = 0, eq = 0;
#pragma unroll 4
  for (int i0 = b0; i0 < b1; i0 += 32) {
    const int i = i0 + lane;
    gt += __popc(__ballot_sync(0xffffffffu, i < b1 && above_at(i)));
    eq += __popc(__ballot_sync(0xffffffffu, i < b1 && edge_at(i)));
  }
  if (lane == 0) {
    warp_gt[warp] = gt;
    warp_eq[warp] = eq;
  }
  __syncthreads();
  if (warp == 0) {  // exclusive prefix sums over the warps, totals of the CTA
    uint32_t x = lane < WARPS ? warp_gt[lane] : 0u, y = lane < WARPS ? warp_eq[lane] : 0u;
    const uint32_t x0 = x, y0 = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += u;
        y += v;
      }
    }
    if (lane < WARPS) {
      warp_gt[lane] = x - x0;
      warp_eq[lane] = y - y0;
    }
    if (lane == 31) {
      counts[0] = x;
      counts[1] = y;
    }
  }
  if (parts > 1) sel_cluster_sync();
  else __syncthreads();
  uint32_t at_gt = warp_gt[warp], at_eq = warp_eq[warp];
  for (uint32_t q = 0; q < rank; ++q) {
    at_gt += sel_remote(&counts[0], q);
    at_eq += sel_remote(&counts[1], q);
  }
  for (int i0 = b0; i0 < b1; i0 += 32) {
    const int i = i0 + lane;
    const bool is_gt = i < b1 && above_at(i), is_eq = i < b1 && edge_at(i);
    const uint32_t bg = __ballot_sync(0xffffffffu, is_gt), be = __ballot_sync(0xffffffffu, is_eq), below = (1u << lane) - 1;
    const uint32_t e = at_eq + __popc(be & below);
    if (is_gt || (is_eq && e < left)) {
      const uint32_t to = at_gt + __popc(bg & below) + min(e, left);
      kept[to] = t0 + i;
      if (ns) ns[to] = key_score(row[i]);
    }
    at_gt += __popc(bg);
    at_eq += __popc(be);
  }
  if (parts > 1) sel_cluster_sync();  // nobody leaves while its counts may still be read
}

// ---- move -----------------------------------------------------------------------------------------------------------
// A (page, head) is a slab of rows (head_dim rows of K, ..) of `page` elements, contiguous in memory; a kept token is one element
// in every row.  A CTA owns some rows of K and V of one (sequence, KV head) and walks the new positions in groups of 16 bytes of
// a row: loading warps bring in the slabs that hold kept tokens, each once, by bulk copies into a ring that always holds
// all slabs a group can need; each warp gathers the group's elements from them, a lane one 32-bit
// word of a row, and writes the words out.  Bound by DRAM: whole slabs are read for the tokens kept in them.
//
// In place: a kept token never moves upwards, so every page that is still to be read, however far ahead the copies run, lies
// above the group that is written, or is in the ring already; rows belong to warps, so no other order matters.  The tokens of a head are then one
// CTA's work, and with few (sequence, head) pairs the rows are split over more CTAs; into other pages every run of new
// positions is a CTA of its own.
constexpr int kMoveWarps = 8, kMoveLoaders = 4, kMoveThreads = 32 * (kMoveWarps + kMoveLoaders + 1), kMoveRun = 2048, kMoveMaxRing = 32;

struct MoveTensor {
  uint8_t* p;
  int rows;  // rows of a (page, head)
};
struct MoveArgs {
  EvictArgs e;
  MoveTensor t[2];   // K, V
  MoveTensor sc[2];  // their scales: 1 row of 4 bytes or head_dim / 32 rows of 1 byte; 0 rows: none
  int split;         // CTAs that share the rows of a KV head
  int run;           // new positions that a CTA plans at a time
  int ring;          // slabs in flight
  int teams;         // of warps, which take the groups in turn
  uint32_t slot_bytes, ring_at, smem;
};

template <int EB>
struct MovePlan {                 // of one run of new positions
  uint16_t tok[kMoveRun + 16];    // a token's ring slot << 8 | its place in its page
  uint16_t page[kMoveRun];        // its page in the list below
  int page_blk[kMoveRun];         // pages that hold kept tokens, in order; -1: not in the pool
  int4 group[kMoveRun * EB / 16]; // 16 bytes of a row: last page needed, pages done with it, new page, tokens that there are
  int to[kMoveRun / 16];          // new pages, -1: not in the pool
  uint32_t there[kMoveRun / 32];  // which new positions have a token to move
  uint32_t scan[kMoveThreads / 32];
  int n_pages;
};

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}

// `slot0`: ring slot of the run's first page
template <int EB>
__device__ void plan_run(const MoveArgs& m, MovePlan<EB>& pl, const int32_t* kept, const int32_t* bt, const int32_t* nbt, int p0, int n, int ctx, int slot0) {
  constexpr int G = 16 / EB;
  const EvictArgs& a = m.e;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, shift = 31 - __clz(a.page);
  int* const tokens = pl.page_blk;  // until the step that writes a page's entry, which no step ahead reads as a token
  for (int j = tid; j < n; j += kMoveThreads) tokens[j] = kept[p0 + j];
  __syncthreads();
  uint32_t base = 0;
  int t = -1, prev = -1, blk_ahead = -1, to_ahead = -1, t_ahead = -1, prev_ahead = -1;
  auto look_ahead = [&](int j) {
    t_ahead = j < n ? tokens[j] : -1;
    prev_ahead = j > 0 && j < n ? tokens[j - 1] : -1;
    blk_ahead = (t_ahead >= 0 && t_ahead < ctx) ? bt[t_ahead >> shift] : -1;
    to_ahead = j < n ? nbt[(p0 + j) >> shift] : -1;
  };
  look_ahead(tid);
  for (int j0 = 0; j0 < n; j0 += kMoveThreads) {
    const int j = j0 + tid;
    t = t_ahead;
    prev = prev_ahead;
    int blk = blk_ahead, to = to_ahead;
    look_ahead(j + kMoveThreads);
    const bool first = j < n && (j == 0 || (t >> shift) != (prev >> shift));
    if (blk >= a.num_blocks) blk = -1;
    if (to >= a.num_blocks) to = -1;
    if (j < n && (blk < 0 || to < 0) && a.status) atomicOr(a.status, CUDA_LLM_ST_BAD_BLOCK);
    const uint32_t there = __ballot_sync(0xffffffffu, blk >= 0 && to >= 0);
    const uint32_t starts = __ballot_sync(0xffffffffu, first);
    if (lane == 0) {
      pl.scan[warp] = __popc(starts);
      if (j < n) pl.there[j >> 5] = there;
    }
    __syncthreads();
    uint32_t u = base + __popc(starts & ((2u << lane) - 1)) - 1;
#pragma unroll
    for (int w = 0; w < kMoveThreads / 32; ++w) {
      if (w < warp) u += pl.scan[w];
      base += pl.scan[w];
    }
    if (j < n) {
      pl.tok[j] = (uint16_t)((slot0 + u) % (uint32_t)m.ring << 8 | (uint32_t)(t & (a.page - 1)));
      pl.page[j] = (uint16_t)u;
      if (first) pl.page_blk[u] = blk;
      if ((j & (a.page - 1)) == 0) pl.to[j >> shift] = to;
    }
    __syncthreads();
  }
  if (tid < 16) pl.tok[n + tid] = 0;  // the last group is read whole
  if (tid == 0) pl.n_pages = (int)base;
  for (int g = tid; g * G < n; g += kMoveThreads) {
    const int j = g * G;
    pl.group[g] = make_int4(pl.page[min(j + G, n) - 1], j + G < n ? pl.page[j + G] : (int)base, pl.to[j >> shift],
                            (int)(pl.there[j >> 5] >> (j & 31) & ((1u << G) - 1)));
  }
  __syncthreads();
}

// One row of the scales of K or of V: a lane takes 8 tokens at a time, and the next 8 are on their way while these are stored
// (4 at a time, both tensors by one warp: 4 x 8 heads of 64, 9000 -> 4096 tokens in place, 114 us for 91).
// In place that is safe: a token's old position is no lower than its new one, so what later tokens are loaded from lies
// above what these are stored to; and these have all been loaded.
template <typename E, int EB>
__device__ __forceinline__ void move_scale_row(const EvictArgs& a, const MovePlan<EB>& pl, const MoveTensor& mt, int r, int h, int n, int p0) {
  constexpr int U = 8, STEP = 32 * U;
  const int lane = threadIdx.x & 31, shift = 31 - __clz(a.page);
  E* const p = reinterpret_cast<E*>(mt.p) + r * a.page;
  auto there = [&](int j) { return j < n && (pl.there[j >> 5] >> (j & 31) & 1); };
  auto load = [&](int j0, E (&v)[U]) {
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int j = j0 + x * 32 + lane;
      v[x] = 0;
      if (there(j)) v[x] = p[((long long)pl.page_blk[pl.page[j]] * a.Hkv + h) * mt.rows * a.page + (pl.tok[j] & 255)];
    }
  };
  E v[U], next[U];
  load(0, v);
  for (int j0 = 0; j0 < n; j0 += STEP) {
    load(j0 + STEP, next);
    __syncwarp();
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int j = j0 + x * 32 + lane;
      if (there(j)) p[((long long)pl.to[j >> shift] * a.Hkv + h) * mt.rows * a.page + ((p0 + j) & (a.page - 1))] = v[x];
      v[x] = next[x];
    }
    __syncwarp();
  }
}

// 4 bytes of a new row, `AT` bytes behind the first: 4, 2 or 1 elements from their places in the ring
template <int EB, int AT>
__device__ __forceinline__ uint32_t gather_word(const uint32_t (&from)[4 / EB]) {
  uint32_t x[4 / EB];
#pragma unroll
  for (int k = 0; k < 4 / EB; ++k) {
    if constexpr (EB == 4) asm volatile("ld.shared.b32 %0, [%1 + %2];" : "=r"(x[k]) : "r"(from[k]), "n"(AT));
    else if constexpr (EB == 1) asm volatile("ld.shared.u8 %0, [%1 + %2];" : "=r"(x[k]) : "r"(from[k]), "n"(AT));
    else asm volatile("{\n\t.reg .u16 h;\n\tld.shared.u16 h, [%1 + %2];\n\tcvt.u32.u16 %0, h;\n\t}" : "=r"(x[k]) : "r"(from[k]), "n"(AT));
  }
  if constexpr (EB == 4) return x[0];
  else if constexpr (EB == 2) return prmt(x[0], x[1], 0x5410);
  else return prmt(prmt(x[0], x[1], 0x0040), prmt(x[2], x[3], 0x0040), 0x5410);
}
// ITER rows, eight apart, of one tensor into one new group
template <typename E, int ROW, int ITER>
__device__ __forceinline__ void move_words(const uint32_t (&from)[4 / sizeof(E)], uint8_t* to, uint32_t mine) {
  constexpr int EB = sizeof(E), WT = 4 / EB;
  auto put = [&](uint8_t* at, uint32_t word) {
    if (mine == (1u << WT) - 1) {
      *reinterpret_cast<uint32_t*>(at) = word;
    } else {
#pragma unroll
      for (int k = 0; k < WT; ++k)
        if (mine >> k & 1) reinterpret_cast<E*>(at)[k] = (E)(word >> (8 * EB * k));
    }
  };
  put(to, gather_word<EB, 0>(from));
  if constexpr (ITER > 1) put(to + 8 * ROW, gather_word<EB, 8 * ROW>(from));
}
template <typename E, int ROW, int ITER>
__device__ __forceinline__ void move_words_2(const uint32_t (&fa)[4 / sizeof(E)], const uint32_t (&fb)[4 / sizeof(E)], uint8_t* a, uint8_t* b) {
  constexpr int EB = sizeof(E);
  const uint32_t x = gather_word<EB, 0>(fa), y = gather_word<EB, 0>(fb);
  if constexpr (ITER > 1) {
    const uint32_t u = gather_word<EB, 8 * ROW>(fa), v = gather_word<EB, 8 * ROW>(fb);
    *reinterpret_cast<uint32_t*>(a + 8 * ROW) = u;
    *reinterpret_cast<uint32_t*>(b + 8 * ROW) = v;
  }
  *reinterpret_cast<uint32_t*>(a) = x;
  *reinterpret_cast<uint32_t*>(b) = y;
}

// E: an element of K and V, ES: of their scales.  KI, VI: rows of a lane, K and V (a warp has 8 KI rows of K, or fewer).
template <typename E, typename ES, int PAGE, int KI, int VI>
__global__ void __launch_bounds__(kMoveThreads, 2) evict_move_kernel(const __grid_constant__ MoveArgs m) {
  constexpr int EB = sizeof(E), G = 16 / EB, WT = 4 / EB;  // tokens of a group, of a word
  constexpr int ROW = PAGE * EB;                           // bytes of a row
  extern __shared__ __align__(128) uint8_t smem[];
  MovePlan<EB>& pl = *reinterpret_cast<MovePlan<EB>*>(smem + 1024);
  const EvictArgs& a = m.e;
  const uint32_t base = smem_u32(smem), full = base, empty = base + 8 * kMoveMaxRing, ring = base + m.ring_at;
  volatile int* fail_ptr = reinterpret_cast<volatile int*>(smem + 16 * kMoveMaxRing);
  const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the selection is complete, and with it all that came before it
  const int part = blockIdx.x % m.split, run0 = blockIdx.x / m.split;
  const int ctx = evict_ctx(a, s, false), total = min(ctx, a.budget);
  if (a.in_place ? ctx <= a.budget : run0 * m.run >= total) return;
  const int32_t* kept = a.kept + ((size_t)s * a.Hkv + h) * a.budget;
  const int32_t* bt = a.bt + (size_t)s * a.max_blocks;
  const int32_t* nbt = a.new_bt + (size_t)s * a.new_max_blocks;
  if (tid == 0) {
    for (int i = 0; i < m.ring; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, kMoveWarps);
    }
    *fail_ptr = 0;
    mbar_fence_init();
  }
  const int k_rows = m.t[0].rows / m.split, v_rows = m.t[1].rows / m.split;  // of this CTA
  const long long k_page = (long long)a.Hkv * m.t[0].rows * ROW, v_page = (long long)a.Hkv * m.t[1].rows * ROW;
  uint8_t* const k_base = m.t[0].p + ((long long)h * m.t[0].rows + part * k_rows) * ROW;
  uint8_t* const v_base = m.t[1].p + ((long long)h * m.t[1].rows + part * v_rows) * ROW;
  int st = 0, slot0 = 0;  // ring slot and its phase, carried on from run to run by producer and warps alike
  uint32_t par = 0;
  auto step = [&]() {
    if (++st == m.ring) {
      st = 0;
      par ^= 1;
    }
  };
  bool dead = false;      // a wait ran out: nothing is moved any more, but the barriers of the block are kept
  // in place: all runs of the head, one after another; else one
  for (int p0 = run0 * m.run; p0 < total; p0 += a.in_place ? m.run : total) {
    const int n = min(m.run, total - p0);
    plan_run<EB>(m, pl, kept, bt, nbt, p0, n, ctx, slot0);
    const int n_pages = pl.n_pages;
    slot0 = (slot0 + n_pages) % m.ring;
    if (warp >= kMoveWarps && warp < kMoveWarps + kMoveLoaders) {
      // pages in turn with the other loading warps: alone, one would spend longer on a page than its copies take
      const int mine = warp - kMoveWarps;
      for (int u = 0; u < n_pages; ++u, step()) {
        if (u % kMoveLoaders != mine) continue;
        if (!mbar_wait(empty + 8 * st, par ^ 1, 0)) {
          dead = true;
          *fail_ptr = 1;
          break;
        }
        const int blk = pl.page_blk[u];
        if (lane == 0) {
          mbar_arrive_expect_tx(full + 8 * st, blk >= 0 ? (uint32_t)(k_rows + v_rows) * ROW : 0u);
          if (blk >= 0) {
            bulk_g2s(ring + st * m.slot_bytes, k_base + blk * k_page, (uint32_t)k_rows * ROW, full + 8 * st);
            bulk_g2s(ring + st * m.slot_bytes + k_rows * ROW, v_base + blk * v_page, (uint32_t)v_rows * ROW, full + 8 * st);
          }
        }
        __syncwarp();
      }
    } else if (warp == kMoveWarps + kMoveLoaders) {
      // the rows of the scales go round the CTAs of the head
      for (int r = part; r < m.sc[0].rows + m.sc[1].rows; r += m.split) {
        const bool of_v = r >= m.sc[0].rows;
        move_scale_row<ES>(a, pl, m.sc[of_v ? 1 : 0], of_v ? r - m.sc[0].rows : r, h, n, p0);
      }
    } else {
      // a team's warps share the rows, K and V alike; a lane owns one word of one or two rows of each
      const int row = lane >> 2, w = lane & 3, crew = kMoveWarps / m.teams, team = warp / crew, at = warp % crew;
      const int kr = k_rows / crew * at + row, vr = v_rows / crew * at + row;
      const bool k_live = KI > 1 || row < k_rows / crew, v_live = VI > 1 || row < v_rows / crew;
      uint8_t* const k_row = k_base + kr * ROW + 4 * w;
      uint8_t* const v_row = v_base + vr * ROW + 4 * w;
      const uint32_t k_slab = kr * ROW, v_slab = (k_rows + vr) * ROW;
      int ready = 0, first = 0, first_st = st;  // pages that have arrived; the first one still held, its slot and phase
      uint32_t first_par = par;
      auto wait_upto = [&](int page_last) {  // a lane per page: page_last - first < ring
        if (dead || ready > page_last) return;
        const int page = ready + lane, slot = first_st + page - first;
        const bool wrap = slot >= m.ring;
        bool open = page <= page_last;
        for (uint32_t polls = 0; __any_sync(0xffffffffu, open); ++polls) {
          if (open && mbar_test(full + 8 * (wrap ? slot - m.ring : slot), first_par ^ (wrap ? 1u : 0u))) open = false;
          if (polls > (1u << 22)) {
            dead = true;
            *fail_ptr = 1;
            break;
          }
        }
        ready = page_last + 1;
      };
      // All pages before `next` have been read as far as this warp reads them.  A page is waited for before it is released, also
      // one that only other teams read: its slot's earlier use is then over for everybody.
      auto release = [&](int next) {
        while (first < next) {
          const int done = min(next - first, m.ring);
          wait_upto(first + done - 1);
          __syncwarp();
          const int slot = first_st + lane;
          if (lane < done) mbar_arrive(empty + 8 * (slot >= m.ring ? slot - m.ring : slot));
          first += done;
          first_st += done;
          if (first_st >= m.ring) {
            first_st -= m.ring;
            first_par ^= 1;
          }
        }
      };
      int turn = 0;  // pairs of groups go round the teams
      for (int j0 = 0; j0 < n;) {
        // two groups at a time where the ring can hold all their pages: what a group costs a warp is latency
        const int4 ga = pl.group[j0 / G];
        int4 gb = j0 + G < n ? pl.group[j0 / G + 1] : ga;
        const int page0 = pl.page[j0];
        const bool two = j0 + G < n && gb.x - page0 < m.ring;
        if (!two) gb = ga;
        const bool ours = turn == team;
        if (++turn == m.teams) turn = 0;
        if (!ours) {
          j0 += two ? 2 * G : G;
          continue;
        }
        uint32_t fa[WT], fb[WT];
#pragma unroll
        for (int k = 0; k < WT; ++k) {
          const uint32_t ta = pl.tok[j0 + w * WT + k], tb = pl.tok[j0 + (two ? G : 0) + w * WT + k];
          fa[k] = ring + (ta >> 8) * m.slot_bytes + (ta & 255u) * EB;
          fb[k] = ring + (tb >> 8) * m.slot_bytes + (tb & 255u) * EB;
        }
        release(page0);
        wait_upto(gb.x);  // and with it for all before: nothing is written that is still to be read
        if (!dead) {
          const uint32_t in_a = ((uint32_t)j0 & (PAGE - 1)) * EB, in_b = ((uint32_t)(j0 + G) & (PAGE - 1)) * EB;
          const bool whole = two && ga.w == (1 << G) - 1 && gb.w == (1 << G) - 1;
          auto tensor = [&](auto iter, uint32_t slab, uint8_t* base_row, long long page_bytes) {
            constexpr int ITER = decltype(iter)::value;
            uint32_t xa[WT], xb[WT];
#pragma unroll
            for (int k = 0; k < WT; ++k) {
              xa[k] = fa[k] + slab;
              xb[k] = fb[k] + slab;
            }
            uint8_t* const to_a = base_row + ga.z * page_bytes + in_a;
            uint8_t* const to_b = base_row + gb.z * page_bytes + in_b;
            if (whole) {
              move_words_2<E, ROW, ITER>(xa, xb, to_a, to_b);
            } else {  // one group, the end of a sequence, or a page that is not in the pool
              move_words<E, ROW, ITER>(xa, to_a, (uint32_t)ga.w >> (w * WT) & ((1u << WT) - 1));
              if (two) move_words<E, ROW, ITER>(xb, to_b, (uint32_t)gb.w >> (w * WT) & ((1u << WT) - 1));
            }
          };
          if (k_live) tensor(std::integral_constant<int, KI>{}, k_slab, k_row, k_page);
          if (v_live) tensor(std::integral_constant<int, VI>{}, v_slab, v_row, v_page);
        }
        j0 += two ? 2 * G : G;
        release(gb.y);
      }
      release(n_pages);
      st = first_st;
      par = first_par;
    }
    __syncthreads();
    if (*fail_ptr) break;  // uniform: written before the barrier
  }
  if (tid == kMoveWarps * 32 && *fail_ptr) {
    for (int i = 0; i < m.ring; ++i) mbar_wait(full + 8 * i, par ^ (i < st ? 0 : 1), 1);  // copies in flight land before the CTA ends
    if (a.status) atomicOr(a.status, CUDA_LLM_ST_TIMEOUT);
  }
}

template <typename E, typename ES, int PAGE, int KI, int VI>
static cudaError_t launch_move(const MoveArgs& m, bool overlap, cudaStream_t st) {
  auto kern = evict_move_kernel<E, ES, PAGE, KI, VI>;
  static int configured[64] = {0};
  cudaError_t e = allow_shared_memory((const void*)kern, 227 * 1024, configured);
  if (e != cudaSuccess) return e;
  const unsigned runs = m.e.in_place ? 1u : (unsigned)((m.e.budget + m.run - 1) / m.run);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(runs * m.split, m.e.Hkv, m.e.S);
  cfg.blockDim = dim3(kMoveThreads);
  cfg.dynamicSmemBytes = m.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // its CTAs start while the selection ends, and wait for it
  attr[0].val.programmaticStreamSerializationAllowed = overlap ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, m);
}
template <typename E, typename ES, int PAGE>
static cudaError_t launch_move_rows(const MoveArgs& m, bool overlap, cudaStream_t st) {
  const int crew = kMoveWarps / m.teams, k = m.t[0].rows / m.split / crew, v = m.t[1].rows / m.split / crew;  // rows of a warp
  if (k == 16 && v == 16) return launch_move<E, ES, PAGE, 2, 2>(m, overlap, st);
  if constexpr (sizeof(E) == 1)
    if (k == 16) return launch_move<E, ES, PAGE, 2, 1>(m, overlap, st);
  return launch_move<E, ES, PAGE, 1, 1>(m, overlap, st);
}
template <typename E, typename ES>
static cudaError_t launch_move_page(const MoveArgs& m, bool overlap, cudaStream_t st) {
  return m.e.page == 16 ? launch_move_rows<E, ES, 16>(m, overlap, st) : m.e.page == 32 ? launch_move_rows<E, ES, 32>(m, overlap, st) : launch_move_rows<E, ES, 64>(m, overlap, st);
}

template <int THREADS>
static cudaError_t launch_select(const EvictArgs& a, int parts, int most, cudaStream_t st) {
  auto kern = evict_select_kernel<THREADS>;
  const int smem = ((most + parts - 1) / parts + 1) * 4;
  static int configured[64] = {0};
  cudaError_t e = allow_shared_memory((const void*)kern, kSelMaxPart * 4 + 4, configured);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts, a.Hkv, a.S);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
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
  if (p->budget > (1 << 30)) return refuse(CUDA_LLM_EINVAL, "a budget of more than 2^30 tokens");
  if (p->max_tokens > CUDA_LLM_EVICT_MAX_TOKENS) return refuse(CUDA_LLM_EINVAL, "score rows of more than CUDA_LLM_EVICT_MAX_TOKENS entries");
  if (p->num_seqs == 0) return CUDA_LLM_OK;
  if (p->max_blocks_per_seq < 0 || p->new_max_blocks_per_seq < 0 || p->num_blocks <= 0)
    return refuse(CUDA_LLM_EINVAL, "block tables and pool must not be empty");
  if (p->num_seqs > 65535 || p->num_kv_heads > 65535) return refuse(CUDA_LLM_EINVAL, "more than 65535 sequences or KV heads");
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
  const long long readable = most;  // of a score row
  if (most > p->budget) most = p->budget;
  if (p->new_scores && !rows_apart(p->new_score_strides[0], p->num_seqs, p->new_score_strides[1], p->num_kv_heads, most))
    return refuse(CUDA_LLM_EINVAL, "new score rows overlap");
  if (p->new_scores == p->scores &&
      ((p->num_seqs > 1 && p->new_score_strides[0] != p->score_strides[0]) || (p->num_kv_heads > 1 && p->new_score_strides[1] != p->score_strides[1])))
    return refuse(CUDA_LLM_EINVAL, "new_scores is scores with other strides");
  // a row is read to the end of its context while another may be written already
  if (p->new_scores == p->scores && !rows_apart(p->score_strides[0], p->num_seqs, p->score_strides[1], p->num_kv_heads, readable))
    return refuse(CUDA_LLM_EINVAL, "new_scores is scores and its rows overlap");
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
  // the score row over as many CTAs as leave each at least 4096 scores
  long long row_most = (long long)a.max_blocks * a.page;
  if (row_most > a.max_tokens) row_most = a.max_tokens;
  int parts = 1;
  while (parts < 8 && row_most > 8192ll * parts) parts *= 2;
  rc = cuda_result(row_most > 8192 ? launch_select<1024>(a, parts, (int)row_most, st) : launch_select<512>(a, parts, (int)row_most, st),
                   "evict_select_kernel launch");
  if (rc != CUDA_LLM_OK) return rc;
  const int D = p->head_dim, v_rows = p->v_format == CUDA_LLM_KV_FP4_E2M1 ? D / 2 : D;
  const int sc_rows = !scaled ? 0 : p->scale_mode == CUDA_LLM_SCALE_PER_TOKEN ? 1 : D / 32;
  m.t[0] = MoveTensor{(uint8_t*)p->key_cache, D};
  m.t[1] = MoveTensor{(uint8_t*)p->value_cache, v_rows};
  m.sc[0] = MoveTensor{(uint8_t*)p->k_scale, sc_rows};
  m.sc[1] = MoveTensor{(uint8_t*)p->v_scale, sc_rows};
  const int eb = format_bytes(p->k_format), row_bytes = a.page * eb;
  const long long pairs = (long long)a.S * a.Hkv;
  const int sms = current_sm_count(), group = 16 / eb;
  auto slot = [&](int split) { return (uint32_t)(((D + v_rows) / split * row_bytes + 127) / 128 * 128); };
  m.ring_at = (1024 + (eb == 1 ? sizeof(MovePlan<1>) : eb == 2 ? sizeof(MovePlan<2>) : sizeof(MovePlan<4>)) + 127) / 128 * 128;
  // The ring holds one slab more than a group has tokens, and as many as leave room for two CTAs on an SM.  Rows are split so that this is
  // up to 32 slabs (the window in which the teams work) and, in place, until every SM has work; elsewhere there are runs of
  // positions for that, as long as pays for their plan.
  m.split = 1;
  while (m.split < 8 && slot(m.split) > 8192) m.split *= 2;
  m.run = kMoveRun;
  if (in_place) {
    while (m.split < 8 && pairs * m.split * 2 <= 2 * sms) m.split *= 2;
  } else {
    while (m.run > 256 && pairs * m.split * ((a.budget + m.run - 1) / m.run) < 2 * sms) m.run /= 2;
  }
  m.slot_bytes = slot(m.split);
  m.ring = (int)((113 * 1024 - m.ring_at) / m.slot_bytes);
  if (m.ring < group + 1) m.ring = group + 1;
  if (m.ring > kMoveMaxRing) m.ring = kMoveMaxRing;
  m.smem = m.ring_at + m.ring * m.slot_bytes;
  m.teams = 1;  // a warp has 16 rows of K, or the 8 of an eighth of head_dim 64
  while (m.teams < kMoveWarps && D / m.split / (kMoveWarps / m.teams) < 16) m.teams *= 2;
  // The move's CTAs may start early only where the selection leaves SMs free: 32 x 8 rows of 8000 scores take 126 us without and
  // 129 us with it, 8 rows of 700 scores 27 and 24 us.
  const bool overlap = pairs * parts <= sms;
  const cudaError_t e = eb == 4 ? launch_move_page<uint32_t, uint32_t>(m, overlap, st) : eb == 2 ? launch_move_page<uint16_t, uint32_t>(m, overlap, st)
                        : p->scale_mode == CUDA_LLM_SCALE_PER_TOKEN ? launch_move_page<uint8_t, uint32_t>(m, overlap, st) : launch_move_page<uint8_t, uint8_t>(m, overlap, st);
  return cuda_result(e, "evict_move_kernel launch");
}
