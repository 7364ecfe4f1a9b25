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

// ---- selection ------------------------------------------------------------------------------------------------------
// A thread-block cluster per (KV head, sequence); each CTA holds its part of the score row in shared memory.  The budget-th
// largest key comes from four passes over its bytes: a histogram per CTA (lanes with the same byte add once), summed over the
// cluster through distributed shared memory.  Then each warp counts, and afterwards writes, the kept tokens of its own run
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

template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const EvictArgs a) {
  constexpr int WARPS = THREADS / 32;
  extern __shared__ float row[];
  __shared__ uint32_t hist[4][256], digit_sum[256];
  __shared__ uint32_t counts[2];             // kept for sure, on the edge: of this CTA
  __shared__ uint32_t warp_gt[WARPS], warp_eq[WARPS], found[2];
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
  for (int i = tid; i < 4 * 256; i += THREADS) (&hist[0][0])[i] = 0;
#pragma unroll 4
  for (int i = tid; i < n; i += THREADS) row[i] = sc[t0 + i];
  __syncthreads();
  auto key_at = [&](int i) { return rank_key(row[i], t0 + i < a.sink || t0 + i >= ctx - a.recent); };
  uint32_t prefix = 0, left = (uint32_t)n_keep;
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    const uint32_t mask = pass == 0 ? 0u : 0xffffffffu << (shift + 8);
    for (int i0 = 0; i0 < n; i0 += THREADS) {
      const int i = i0 + tid;
      const uint32_t k = i < n ? key_at(i) : 0u;
      const bool in = i < n && (k & mask) == prefix;
      const uint32_t digit = (k >> shift) & 255;
      const uint32_t same = __match_any_sync(0xffffffffu, in ? digit : 256u);
      if (in && lane == __ffs(same) - 1) atomicAdd(&hist[pass][digit], (uint32_t)__popc(same));
    }
    if (parts > 1) sel_cluster_sync();
    else __syncthreads();
    if (tid < 256) {
      uint32_t sum = hist[pass][tid];
      if (parts > 1) {
        sum = 0;
        for (uint32_t q = 0; q < parts; ++q) sum += sel_remote(&hist[pass][tid], q);
      }
      digit_sum[tid] = sum;
    }
    __syncthreads();
    if (warp == 0) {  // the largest digit d with (keys above d) < left <= (keys from d up)
      uint32_t c[8], mine = 0;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        c[x] = digit_sum[255 - (lane * 8 + x)];
        mine += c[x];
      }
      uint32_t before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
      }
      before -= mine;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        if (before < left && left <= before + c[x]) {
          found[0] = 255 - (lane * 8 + x);
          found[1] = left - before;
        }
        before += c[x];
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    left = found[1];
  }
  // keep all keys above `prefix` and the first `left` that equal it
  const uint32_t edge = prefix;
  const int per = ((n + WARPS - 1) / WARPS + 31) & ~31, b0 = min(n, warp * per), b1 = min(n, b0 + per);
  uint32_t gt = 0, eq = 0;
  for (int i0 = b0; i0 < b1; i0 += 32) {
    const uint32_t k = i0 + lane < b1 ? key_at(i0 + lane) : 0u;
    gt += __popc(__ballot_sync(0xffffffffu, i0 + lane < b1 && k > edge));
    eq += __popc(__ballot_sync(0xffffffffu, i0 + lane < b1 && k == edge));
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
    const uint32_t k = i < b1 ? key_at(i) : 0u;
    const bool is_gt = i < b1 && k > edge, is_eq = i < b1 && k == edge;
    const uint32_t bg = __ballot_sync(0xffffffffu, is_gt), be = __ballot_sync(0xffffffffu, is_eq), below = (1u << lane) - 1;
    const uint32_t e = at_eq + __popc(be & below);
    if (is_gt || (is_eq && e < left)) {
      const uint32_t to = at_gt + __popc(bg & below) + min(e, left);
      kept[to] = t0 + i;
      if (ns) ns[to] = row[i];
    }
    at_gt += __popc(bg);
    at_eq += __popc(be);
  }
  if (parts > 1) sel_cluster_sync();  // nobody leaves while its counts may still be read
}

// ---- move -----------------------------------------------------------------------------------------------------------
// A (page, head) is rows of `page` elements (head_dim rows of K, ..), so a kept token is one element in every row and moving it
// shifts bytes inside rows.  The unit is 16 bytes of a row (a group of 16, 8 or 4 tokens): a lane owns a row, loads the old
// groups that hold kept tokens one after another (each once) and assembles the new groups with byte permutes.  Which bytes go
// where is the same for every row of the KV head: a CTA works that out once for a run of new positions, as a list of old
// groups ("entries") and, for every 32-bit word of a new group, the pieces it takes from them.  Bound by DRAM: whole
// groups are read for the tokens kept in them.
//
// In place: a kept token never moves upwards, so when a lane writes new group g, every old group that it still has to read
// lies above g; rows are owned by lanes, so no other order matters.  One CTA then takes all positions of a KV head in
// turn; into other pages every run of positions is a CTA of its own.
constexpr int kMoveThreads = 256, kMoveRun = 2048, kMoveRing = 16;

struct MoveTensor {
  void* p;
  int rows;  // rows of a (page, head)
};
struct MoveArgs {
  EvictArgs e;
  MoveTensor t[2];      // K, V
  MoveTensor sc[2];     // their scales: rows 1 of 4 bytes, or head_dim / 32 of 1 byte; rows 0: none
  int slices[2];        // 32-row slices of K and V
  int run;              // new positions a CTA works out at a time
};

struct MovePlan {           // of one run of new positions, in shared memory
  int2 entry[kMoveRun + kMoveRing];  // page (or -1) and 16-byte group of the page of an old group
  uint2 piece[kMoveRun + 2];  // selectors {of the low 8 source bytes | high 8 << 16, which of the two | keep or take << 16} + flags
  int to[kMoveRun / 4];     // new page of every new group
  uint32_t have[kMoveRun / 4];  // which of a group's tokens there are
  int kept[kMoveRun];
  uint32_t scan[2][kMoveThreads / 32];
  int n_entries, n_pieces;
};
// flags of a piece, in bits that no selector uses
constexpr uint32_t kNewEntry = 0x80000000u, kWordEnd = 0x8000u;

template <int EB>
__device__ void plan_run(const EvictArgs& a, MovePlan& pl, const int32_t* kept, const int32_t* bt, const int32_t* nbt, int p0, int n, int ctx) {
  constexpr int G = 16 / EB, WT = 4 / EB;  // tokens of a group, of a word
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int j = tid; j < n; j += kMoveThreads) pl.kept[j] = kept[p0 + j];
  __syncthreads();
  uint32_t base_e = 0, base_p = 0;
  for (int j0 = 0; j0 < n; j0 += kMoveThreads) {
    const int j = j0 + tid;
    const int t = j < n ? pl.kept[j] : -1, prev = j > 0 && j < n ? pl.kept[j - 1] : -1;
    const bool first_e = j < n && (j % G == 0 || t / G != prev / G);
    const bool first_p = j < n && (first_e || j % WT == 0);
    int blk = (t >= 0 && t < ctx) ? bt[t / a.page] : -1;
    int to = j < n ? nbt[(p0 + j) / a.page] : -1;
    if (blk >= a.num_blocks || to >= a.num_blocks || ((blk < 0 || to < 0) && j < n)) {
      if (a.status) atomicOr(a.status, CUDA_LLM_ST_BAD_BLOCK);
      if (blk >= a.num_blocks) blk = -1;
      if (to >= a.num_blocks) to = -1;
    }
    const uint32_t there = __ballot_sync(0xffffffffu, blk >= 0 && to >= 0);
    if (j < n && j % G == 0) {
      pl.to[j / G] = to;
      pl.have[j / G] = there >> lane & ((1u << G) - 1);
    }
    uint32_t e = first_e, p = first_p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, e, o), y = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) {
        e += x;
        p += y;
      }
    }
    if (lane == 31) {
      pl.scan[0][warp] = e;
      pl.scan[1][warp] = p;
    }
    __syncthreads();
    uint32_t be = base_e, bp = base_p;
#pragma unroll
    for (int w = 0; w < kMoveThreads / 32; ++w) {
      if (w < warp) {
        be += pl.scan[0][w];
        bp += pl.scan[1][w];
      }
      base_e += pl.scan[0][w];
      base_p += pl.scan[1][w];
    }
    if (first_e) pl.entry[e + be - 1] = make_int2(blk, t % a.page / G);
    if (first_p) {  // the tokens of this piece: same word, same old group
      uint32_t lo = 0, hi = 0, pick = 0, take = 0x3210;
      int k = j;
      do {
        const int from0 = pl.kept[k] % G * EB, to0 = k % WT * EB;
#pragma unroll
        for (int x = 0; x < EB; ++x) {
          const int from = from0 + x, at = 4 * (to0 + x);
          if (from < 8) lo |= (uint32_t)from << at;
          else hi |= (uint32_t)(from - 8) << at;
          pick |= (uint32_t)((from < 8 ? 0 : 4) + to0 + x) << at;
          take |= 4u << at;
        }
        ++k;
      } while (k < n && k % WT != 0 && pl.kept[k] / G == t / G);
      pl.piece[p + bp - 1] = make_uint2(lo | hi << 16, pick | take << 16 | (first_e ? kNewEntry : 0u) | (k % WT == 0 || k == n ? kWordEnd : 0u));
    }
    __syncthreads();
  }
  if (tid == 0) {
    pl.n_entries = (int)base_e;
    pl.n_pieces = (int)base_p;
  }
  for (int x = tid; x < kMoveRing; x += kMoveThreads) pl.entry[base_e + x] = make_int2(-1, 0);
  if (tid < 2) pl.piece[base_p + tid] = make_uint2(0, 0);
  __syncthreads();
}

template <int EB>
__device__ __forceinline__ void move_slice(const EvictArgs& a, const MovePlan& pl, const MoveTensor& mt, int row, int h, int p0, uint32_t ring) {
  constexpr int G = 16 / EB;
  const int n_pieces = pl.n_pieces;
  const bool live = row < mt.rows;
  const uint32_t row_bytes = a.page * EB;
  const long long head_bytes = (long long)mt.rows * row_bytes, page_bytes = head_bytes * a.Hkv;
  uint8_t* const base = static_cast<uint8_t*>(mt.p) + h * head_bytes + (long long)row * row_bytes;
  const uint32_t mine = ring + (threadIdx.x & 31) * 16;
  auto request = [&](int e, int slot) {  // (behind the last entry lie kMoveRing that copy nothing)
    const int2 src = pl.entry[e];
    if (live && src.x >= 0)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(mine + slot * 512), "l"(base + src.x * page_bytes + src.y * 16) : "memory");
    cp_async_commit();
  };
#pragma unroll 1
  for (int e = 0; e < kMoveRing - 1; ++e) request(e < pl.n_entries ? e : pl.n_entries, e);
  int e = -1, slot = kMoveRing - 1, words = 0, g = 0;  // `slot`: where entry e + kMoveRing goes
  uint4 src = make_uint4(0, 0, 0, 0), ahead;
  cp_async_wait<kMoveRing - 2>();
  ahead = lds128(mine);
  uint32_t cur = 0, o0 = 0, o1 = 0, o2 = 0, o3 = 0;
  uint2 next = pl.piece[0];
#pragma unroll 1
  for (int q = 0; q < n_pieces; ++q) {
    const uint2 pc = next;
    next = pl.piece[q + 1];
    if (pc.y & kNewEntry) {
      ++e;
      src = ahead;
      // the slot of the entry before this one is free; the entry after this one is needed next
      const int want = e + kMoveRing - 1;
      request(want < pl.n_entries ? want : pl.n_entries, slot);
      slot = (slot + 1) & (kMoveRing - 1);
      cp_async_wait<kMoveRing - 2>();
      ahead = lds128(mine + ((slot + 1) & (kMoveRing - 1)) * 512);
    }
    const uint32_t lo = prmt(src.x, src.y, pc.x), hi = prmt(src.z, src.w, pc.x >> 16);
    cur = prmt(cur, prmt(lo, hi, pc.y & 0x7777u), (pc.y >> 16) & 0x7777u);
    if (pc.y & kWordEnd) {
      o0 = o1;
      o1 = o2;
      o2 = o3;
      o3 = cur;
      if (++words == 4 || q + 1 == n_pieces) {
        while (words < 4) {  // the last group of a sequence may end early
          o0 = o1;
          o1 = o2;
          o2 = o3;
          o3 = 0;
          ++words;
        }
        words = 0;
        const uint32_t have = pl.have[g];
        if (live && have) {
          uint8_t* dst = base + pl.to[g] * page_bytes + ((p0 + g * G) & (a.page - 1)) * EB;
          if (have == (1u << G) - 1) {
            *reinterpret_cast<uint4*>(dst) = make_uint4(o0, o1, o2, o3);
          } else {
            const uint32_t out[4] = {o0, o1, o2, o3};
#pragma unroll
            for (int k = 0; k < G; ++k)
              if (have >> k & 1) {
                if (EB == 1) dst[k] = (uint8_t)(out[k >> 2] >> (8 * (k & 3)));
                else if (EB == 2) reinterpret_cast<uint16_t*>(dst)[k] = (uint16_t)(out[k >> 1] >> (16 * (k & 1)));
                else reinterpret_cast<uint32_t*>(dst)[k] = out[k & 3];
              }
          }
        }
        ++g;
      }
    }
  }
  cp_async_wait<0>();
  __syncwarp();
}

// scales: a lane takes a token
template <typename E>
__device__ __forceinline__ void move_scales(const EvictArgs& a, const MoveTensor& mt, const int32_t* kept, const int32_t* bt, const int32_t* nbt, int h,
                                            int n, int p0, int ctx) {
  const int lane = threadIdx.x & 31;
  E* const p = static_cast<E*>(mt.p);
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int j = j0 + lane;
    const int t = j < n ? kept[p0 + j] : -1;
    const int blk = (t >= 0 && t < ctx) ? bt[t / a.page] : -1, to = j < n ? nbt[(p0 + j) / a.page] : -1;
    const bool fine = blk >= 0 && blk < a.num_blocks && to >= 0 && to < a.num_blocks;
    for (int r = 0; r < mt.rows; ++r) {
      E x = 0;
      if (fine) x = p[(((size_t)blk * a.Hkv + h) * mt.rows + r) * a.page + t % a.page];
      __syncwarp();
      if (fine) p[(((size_t)to * a.Hkv + h) * mt.rows + r) * a.page + (p0 + j) % a.page] = x;
      __syncwarp();
    }
  }
}

template <int EB, typename ES>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const MoveArgs m) {
  extern __shared__ __align__(16) uint8_t smem[];
  MovePlan& pl = *reinterpret_cast<MovePlan*>(smem);
  const EvictArgs& a = m.e;
  const int h = blockIdx.y, s = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctx = evict_ctx(a, s, false), total = min(ctx, a.budget);
  if (a.in_place && ctx <= a.budget) return;
  const uint32_t ring = smem_u32(smem) + (uint32_t)((sizeof(MovePlan) + 15) & ~15) + warp * (kMoveRing * 512);
  const int32_t* kept = a.kept + ((size_t)s * a.Hkv + h) * a.budget;
  const int32_t* bt = a.bt + (size_t)s * a.max_blocks;
  const int32_t* nbt = a.new_bt + (size_t)s * a.new_max_blocks;
  for (int p0 = blockIdx.x * m.run; p0 < total; p0 += gridDim.x * m.run) {
    const int n = min(m.run, total - p0);
    plan_run<EB>(a, pl, kept, bt, nbt, p0, n, ctx);
    const int slices = m.slices[0] + m.slices[1];
    for (int task = warp; task < slices + 2; task += kMoveThreads / 32) {
      if (task < m.slices[0]) move_slice<EB>(a, pl, m.t[0], task * 32 + lane, h, p0, ring);
      else if (task < slices) move_slice<EB>(a, pl, m.t[1], (task - m.slices[0]) * 32 + lane, h, p0, ring);
      else if (m.sc[task - slices].rows) move_scales<ES>(a, m.sc[task - slices], kept, bt, nbt, h, n, p0, ctx);
    }
    __syncthreads();
  }
}

template <int EB, typename ES>
static cudaError_t launch_move(const MoveArgs& m, cudaStream_t st) {
  auto kern = evict_move_kernel<EB, ES>;
  const int smem = (int)((sizeof(MovePlan) + 15) & ~15) + kMoveThreads / 32 * kMoveRing * 512;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const unsigned runs = m.e.in_place ? 1u : (unsigned)((m.e.budget + m.run - 1) / m.run);
  kern<<<dim3(runs, m.e.Hkv, m.e.S), kMoveThreads, smem, st>>>(m);
  return cudaGetLastError();
}

template <int THREADS>
static cudaError_t launch_select(const EvictArgs& a, int parts, int most, cudaStream_t st) {
  auto kern = evict_select_kernel<THREADS>;
  const int smem = ((most + parts - 1) / parts + 1) * 4;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelMaxPart * 4 + 64);
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
  // the score row over as many CTAs as leave each at least 4096 scores
  long long row_most = (long long)a.max_blocks * a.page;
  if (row_most > a.max_tokens) row_most = a.max_tokens;
  int parts = 1;
  while (parts < 8 && row_most > 8192ll * parts) parts *= 2;
  rc = cuda_result(row_most > 4096 ? launch_select<1024>(a, parts, (int)row_most, st) : launch_select<256>(a, parts, (int)row_most, st),
                   "evict_select_kernel launch");
  if (rc != CUDA_LLM_OK) return rc;
  const int D = p->head_dim, v_rows = p->v_format == CUDA_LLM_KV_FP4_E2M1 ? D / 2 : D;
  const int sc_rows = !scaled ? 0 : p->scale_mode == CUDA_LLM_SCALE_PER_TOKEN ? 1 : D / 32;
  m.t[0] = MoveTensor{p->key_cache, D};
  m.t[1] = MoveTensor{p->value_cache, v_rows};
  m.sc[0] = MoveTensor{p->k_scale, sc_rows};
  m.sc[1] = MoveTensor{p->v_scale, sc_rows};
  m.slices[0] = D / 32;
  m.slices[1] = v_rows / 32;
  m.run = in_place ? kMoveRun : 256;
  const int eb = format_bytes(p->k_format);
  const cudaError_t e = eb == 4 ? launch_move<4, uint32_t>(m, st) : eb == 2 ? launch_move<2, uint32_t>(m, st)
                        : p->scale_mode == CUDA_LLM_SCALE_PER_TOKEN ? launch_move<1, uint32_t>(m, st) : launch_move<1, uint8_t>(m, st);
  return cuda_result(e, "evict_move_kernel launch");
}
