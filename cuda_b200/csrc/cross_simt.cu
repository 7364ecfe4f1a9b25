// Cross attention in fp32 arithmetic on the FMA pipes: fp32 tensors need it (their tolerance is far below what a
// 16-bit operand keeps).
//
//   S = scale Q K^T over a tile of 64 states, running row maximum m and sum l, O = O 2^(m_old - m) + 2^(S - m) V,
//   out = O / l, lse = ln2 (m + log2 l)        (S, m in units of log2)
//
// One CTA of 256 threads takes 64 query rows (head-major: the rows of the heads that share a KV head) and walks the
// states of its sequence; thread (ty, tx) of a 16 x 16 grid holds 4 rows x 4 states of S and 4 rows x D/16 columns of O.
// Q, K and P sit transposed in shared memory, so that each step of a product reads two 16-byte fragments for 16 FMAs; a cluster
// shares the states of a block of rows where blocks are few.  Bound by those shared-memory reads (of this tile: 8 x 8 scores a thread would
// halve them and is not tried): 28 TFLOP/s of the 70 of the FMA
// pipes (4 x 16 heads of 128, 512 positions, 1024 states: 603 us); 2 x 8 heads of 64, 129 positions, 300-577 states: 23 us.
#include "cross_attention.cuh"

namespace b200 {

constexpr int kSimtRows = 64, kSimtKeys = 64;

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }

template <int D>
__global__ void __launch_bounds__(256, 2) cross_simt_kernel(const CrossArgs a) {
  constexpr int LD = kSimtRows + 4;  // padded leading dimension of the transposed tiles
  constexpr float NEG_INF = -__builtin_huge_valf();
  extern __shared__ __align__(16) float sm[];
  __shared__ int pick;
  float* sQ = sm;                  // [D][LD]
  float* sK = sQ + D * LD;         // [D][LD]
  float* sV = sK + D * LD;         // [kSimtKeys][D]
  float* sP = sV + kSimtKeys * D;  // [kSimtKeys][LD]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int kvh = blockIdx.y, b = longest_first<256>(a, blockIdx.z, &pick);
  const int rank = (int)cluster_rank(), parts = (int)cluster_size();
  const int rows = a.group * a.Sq, r0 = blockIdx.x / parts * kSimtRows;
  const int len = cross_kv_len(a, b), tiles = (len + kSimtKeys - 1) / kSimtKeys;
  const int key0 = (int)((long long)tiles * rank / parts) * kSimtKeys, key1 = min(len, (int)((long long)tiles * (rank + 1) / parts) * kSimtKeys);
  const float* kp = static_cast<const float*>(a.k) + b * a.k_st[0] + kvh * a.k_st[1];
  const float* vp = static_cast<const float*>(a.v) + b * a.v_st[0] + kvh * a.v_st[1];
  auto row_head = [&](int r) { return kvh * a.group + r / a.Sq; };
  auto row_pos = [&](int r) { return r % a.Sq; };

#pragma unroll
  for (int i0 = 0; i0 < kSimtRows * (D / 4); i0 += 256) {
    const int i = i0 + tid, r = i & 63, c = i >> 6;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r < rows)
      x = load4(static_cast<const float*>(a.q) + b * a.q_st[0] + row_head(r0 + r) * a.q_st[1] + row_pos(r0 + r) * a.q_st[2] + 4 * c);
    sQ[(4 * c) * LD + r] = x.x;
    sQ[(4 * c + 1) * LD + r] = x.y;
    sQ[(4 * c + 2) * LD + r] = x.z;
    sQ[(4 * c + 3) * LD + r] = x.w;
  }
  float o[4][D / 16], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = NEG_INF;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[i][j] = 0.f;
  }
  for (int t0 = key0; t0 < key1; t0 += kSimtKeys) {
    constexpr int N = kSimtKeys * (D / 4) / 256;  // 16-byte pieces of K and of V per thread: all on their way before the first is stored
    float4 kx[N], vx[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = u * 256 + tid, r = i & 63, c = i >> 6, vr = i / (D / 4), vc = i % (D / 4);
      kx[u] = vx[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t0 + r < len) kx[u] = load4(kp + (t0 + r) * a.k_st[2] + 4 * c);
      if (t0 + vr < len) vx[u] = load4(vp + (t0 + vr) * a.v_st[2] + 4 * vc);
    }
    __syncthreads();  // the tiles of the step before are read
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = u * 256 + tid, r = i & 63, c = i >> 6, vr = i / (D / 4), vc = i % (D / 4);
      sK[(4 * c) * LD + r] = kx[u].x;
      sK[(4 * c + 1) * LD + r] = kx[u].y;
      sK[(4 * c + 2) * LD + r] = kx[u].z;
      sK[(4 * c + 3) * LD + r] = kx[u].w;
      *reinterpret_cast<float4*>(sV + vr * D + 4 * vc) = vx[u];
    }
    __syncthreads();
    float s[4][4] = {};
#pragma unroll 8
    for (int d = 0; d < D; ++d) {
      const float4 x = *reinterpret_cast<const float4*>(sQ + d * LD + ty * 4);
      const float4 y = *reinterpret_cast<const float4*>(sK + d * LD + tx * 4);
      const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = fmaf(xs[i], ys[j], s[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = NEG_INF;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = t0 + tx * 4 + j < len ? s[i][j] * a.scale_log2 : NEG_INF;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int x = 8; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float m_new = fmaxf(m[i], mx);
      const float ref = m_new == NEG_INF ? 0.f : m_new;  // every score so far -inf: weights of zero, not NaN
      const float alpha = exp2f(m[i] - ref);
      m[i] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - ref);
        sum += s[i][j];
      }
      l[i] = l[i] * alpha + sum;  // this thread's share of the row sum
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[i][j] *= alpha;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<float4*>(sP + (tx * 4 + j) * LD + ty * 4) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
    __syncthreads();
#pragma unroll 4
    for (int t = 0; t < kSimtKeys; ++t) {
      const float4 p = *reinterpret_cast<const float4*>(sP + t * LD + ty * 4);
      const float ps[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const float4 y = *reinterpret_cast<const float4*>(sV + t * D + c * 64 + tx * 4);
        const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][c * 4 + j] = fmaf(ps[i], ys[j], o[i][c * 4 + j]);
      }
    }
  }
  // join the parts: every CTA leaves its rows in shared memory, and each writes a share of the rows
  float* po = sK;                                        // [kSimtRows][D]
  float2* pml = reinterpret_cast<float2*>(sV);           // [kSimtRows] {m, l}
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float sum = l[i];
#pragma unroll
    for (int x = 8; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (tx == 0) pml[ty * 4 + i] = make_float2(m[i], sum);
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      *reinterpret_cast<float4*>(po + (ty * 4 + i) * D + c * 64 + tx * 4) = make_float4(o[i][c * 4], o[i][c * 4 + 1], o[i][c * 4 + 2], o[i][c * 4 + 3]);
  }
  if (parts > 1) cluster_sync_all();
  else __syncthreads();
  const uint32_t o_at = smem_u32(po), ml_at = smem_u32(pml);
  for (int e = rank * 256 + tid; e < kSimtRows * (D / 4); e += parts * 256) {
    const int i = e / (D / 4), c = e % (D / 4), r = r0 + i;
    if (r >= rows) break;
    const JoinedWord w = join_parts(ml_at + i * 8, o_at + (i * D + 4 * c) * 4, parts);
    const float4 x = w.x;
    const float M = w.M, L = w.L;
    const float inv = L == 0.f ? 0.f : 1.f / L;  // nothing seen: zeros
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + b * a.o_st[0] + row_head(r) * a.o_st[1] + row_pos(r) * a.o_st[2] + 4 * c) =
        make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    if (a.lse && c == 0) a.lse[((size_t)b * a.Hq + row_head(r)) * a.Sq + row_pos(r)] = L == 0.f ? NEG_INF : kLn2 * (M + log2f(L));
  }
  if (parts > 1) cluster_sync_all();  // no CTA leaves while another still reads its part
}

static cudaError_t launch_clusters(const void* kern, dim3 grid, int threads, size_t smem, int parts, const CrossArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[1] = {const_cast<CrossArgs*>(&a)};
  return cudaLaunchKernelExC(&cfg, kern, args);
}

// Clusters of `parts` CTAs of the tile kernel that the current device runs at once.
template <int D>
static cudaError_t clusters_at_once(const void* kern, size_t smem, int parts, int* count) {
  static int known[64][kMaxParts + 1] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && known[dev][parts]) {
    *count = known[dev][parts];
    return cudaSuccess;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaOccupancyMaxActiveClusters(count, kern, &cfg);
  if (e == cudaSuccess && dev < 64) known[dev][parts] = *count;
  return e;
}

template <int D>
static cudaError_t go_tiles(const CrossArgs& a, cudaStream_t st) {
  constexpr size_t smem = (2 * D * (kSimtRows + 4) + kSimtKeys * D + kSimtKeys * (kSimtRows + 4)) * sizeof(float);
  auto kern = cross_simt_kernel<D>;
  static int configured[64] = {0};
  cudaError_t e = allow_shared_memory((const void*)kern, (int)smem, configured);
  if (e != cudaSuccess) return e;
  const long long rows = (long long)a.group * a.Sq, blocks = (rows + kSimtRows - 1) / kSimtRows;
  // The split with the shortest run: waves of clusters times tiles of a part, and one more for its start and join.  How many
  // clusters run at once depends on their size, as a cluster lies within one group of SMs (38 blocks of 63 tiles: 6 parts take 117 us,
  // 7, which need a second wave, 150).  us here / with powers of two up to a wave of single CTAs: 48 blocks of 10 tiles 27 / 35
  // (64 elements, 5 parts / 4), 62 / 68 (128 elements), 38 of 63 tiles 117 / 162, 512 blocks of 16 tiles 603 / 652 (128 elements, 2 / 1).
  const long long tiles = (a.Skv + kSimtKeys - 1) / kSimtKeys, all = blocks * a.Hkv * a.B;
  int parts = 1;
  long long best = 0;
  for (int p = 1; p <= kMaxParts && (p == 1 || p <= tiles); ++p) {
    int at_once = 0;
    e = clusters_at_once<D>((const void*)kern, smem, p, &at_once);
    if (e != cudaSuccess) return e;
    if (at_once < 1) continue;
    const long long cost = (all + at_once - 1) / at_once * ((tiles + p - 1) / p + 1);
    if (best == 0 || cost < best) {
      best = cost;
      parts = p;
    }
  }
  return launch_clusters((const void*)kern, dim3((unsigned)(blocks * parts), a.Hkv, a.B), 256, smem, parts, a, st);
}

cudaError_t launch_cross_simt(const CrossArgs& a, int D, cudaStream_t st) { return D == 64 ? go_tiles<64>(a, st) : go_tiles<128>(a, st); }

// ---- few query rows: the states are streamed once, HBM-bound -----------------------------------------------------------
// A warp takes 8 states at a time: a lane holds D / LPK elements of a state (LPK lanes per state), so K and V arrive as whole
// 16-byte loads with no shared memory in between.  Partial dot products of R rows x 8 states are summed over the lanes by
// a transposing butterfly: 32 of them need 31 exchanges instead of 160, and leave one score in each lane, where the softmax
// weight is computed once; for the second product the weights go back by broadcast.  Measured: 55 sequences, 8 query and 4 KV
// heads of 64, 1846-6643 states: 89 us = 5.4 TB/s; 16 sequences, 32 and 8 heads of 128, 1000-4096 states: 94 us = 3.6 TB/s
// (four rows: issue-bound).
constexpr int kStreamWarps = 8, kStreamKeys = 8;

template <int D, int R>
__global__ void __launch_bounds__(32 * kStreamWarps) cross_stream_kernel(const CrossArgs a) {
  constexpr int LPK = D / 4;           // lanes per state: 32, or 16 (two states side by side)
  constexpr int SIDE = 32 / LPK;       // states side by side
  constexpr int STEPS = kStreamKeys / SIDE;
  constexpr float NEG_INF = -__builtin_huge_valf();
  extern __shared__ __align__(16) float sm[];
  __shared__ int pick;
  float* part_o = sm;                                                  // [warps][R][D]
  float2* part_ml = reinterpret_cast<float2*>(sm + kStreamWarps * R * D);  // [warps][R]
  float* cta_o = reinterpret_cast<float*>(part_ml + kStreamWarps * R);     // [R][D]
  float2* cta_ml = reinterpret_cast<float2*>(cta_o + R * D);               // [R]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane / LPK, dl = lane % LPK;
  const int kvh = blockIdx.y, b = longest_first<32 * kStreamWarps>(a, blockIdx.z, &pick);
  const int rank = (int)cluster_rank(), parts = (int)cluster_size();
  const int rows = a.group * a.Sq, r0 = blockIdx.x / parts * R;
  const int len = cross_kv_len(a, b), tiles = (len + kStreamKeys - 1) / kStreamKeys;
  const int j0 = (int)((long long)tiles * rank / parts), j1 = (int)((long long)tiles * (rank + 1) / parts);
  const float* kp = static_cast<const float*>(a.k) + b * a.k_st[0] + kvh * a.k_st[1] + 4 * dl;
  const float* vp = static_cast<const float*>(a.v) + b * a.v_st[0] + kvh * a.v_st[1] + 4 * dl;
  auto row_head = [&](int r) { return kvh * a.group + r / a.Sq; };
  auto row_pos = [&](int r) { return r % a.Sq; };
  float4 q[R], o[R];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    q[r] = o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r < rows) q[r] = load4(static_cast<const float*>(a.q) + b * a.q_st[0] + row_head(r0 + r) * a.q_st[1] + row_pos(r0 + r) * a.q_st[2] + 4 * dl);
    m[r] = NEG_INF;
    l[r] = 0.f;
  }
  for (int j = j0 + warp; j < j1; j += kStreamWarps) {
    float4 k[STEPS], v[STEPS];
#pragma unroll
    for (int x = 0; x < STEPS; ++x) {
      const int t = j * kStreamKeys + x * SIDE + sub;
      k[x] = v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t < len) {
        k[x] = load4(kp + t * a.k_st[2]);
        v[x] = load4(vp + t * a.v_st[2]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      // 8 partial sums per row: over the lanes of a state by halving: each exchange halves the number of sums a lane holds
      float s[STEPS];
#pragma unroll
      for (int x = 0; x < STEPS; ++x) s[x] = fmaf(q[r].x, k[x].x, fmaf(q[r].y, k[x].y, fmaf(q[r].z, k[x].z, q[r].w * k[x].w)));
      int bit = LPK / 2;
#pragma unroll
      for (int half = STEPS / 2; half >= 1; half /= 2) {
        const bool up = dl & bit;
#pragma unroll
        for (int x = 0; x < STEPS / 2; ++x)
          if (x < half) {
            const float give = up ? s[x] : s[x + half], keep = up ? s[x + half] : s[x];
            s[x] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
          }
        bit /= 2;
      }
      float sum = s[0];
#pragma unroll
      for (int o2 = LPK / STEPS / 2; o2 >= 1; o2 /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o2);
      // lanes with the same high bits of dl now hold the score of state (those bits) * SIDE + sub
      const int t = j * kStreamKeys + (dl / (LPK / STEPS)) * SIDE + sub;
      const float sc = t < len ? sum * a.scale_log2 : NEG_INF;
      float mx = sc;
#pragma unroll
      for (int o2 = 16; o2 >= LPK / STEPS; o2 /= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o2));
      const float m_new = fmaxf(m[r], mx), ref = m_new == NEG_INF ? 0.f : m_new;
      const float alpha = exp2f(m[r] - ref), p = exp2f(sc - ref);
      m[r] = m_new;
      // every score sits in LPK / STEPS lanes; one of them counts
      l[r] = l[r] * alpha + (dl % (LPK / STEPS) == 0 ? p : 0.f);
      o[r].x *= alpha;
      o[r].y *= alpha;
      o[r].z *= alpha;
      o[r].w *= alpha;
#pragma unroll
      for (int x = 0; x < STEPS; ++x) {
        const float w = __shfl_sync(0xffffffffu, p, sub * LPK + x * (LPK / STEPS));
        o[r].x = fmaf(w, v[x].x, o[r].x);
        o[r].y = fmaf(w, v[x].y, o[r].y);
        o[r].z = fmaf(w, v[x].z, o[r].z);
        o[r].w = fmaf(w, v[x].w, o[r].w);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int x = 16; x; x >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
    if (SIDE == 2) {  // the two states side by side
      o[r].x += __shfl_xor_sync(0xffffffffu, o[r].x, 16);
      o[r].y += __shfl_xor_sync(0xffffffffu, o[r].y, 16);
      o[r].z += __shfl_xor_sync(0xffffffffu, o[r].z, 16);
      o[r].w += __shfl_xor_sync(0xffffffffu, o[r].w, 16);
    }
    if (sub == 0) *reinterpret_cast<float4*>(part_o + (warp * R + r) * D + 4 * dl) = o[r];
    if (lane == 0) part_ml[warp * R + r] = make_float2(m[r], l[r]);
  }
  __syncthreads();
  auto emit = [&](int i, int c, float4 x, float M, float L) {
    const int r = r0 + i;
    if (r >= rows) return;
    const float inv = L == 0.f ? 0.f : 1.f / L;  // nothing seen: zeros
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + b * a.o_st[0] + row_head(r) * a.o_st[1] + row_pos(r) * a.o_st[2] + 4 * c) =
        make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    if (a.lse && c == 0) a.lse[((size_t)b * a.Hq + row_head(r)) * a.Sq + row_pos(r)] = L == 0.f ? NEG_INF : kLn2 * (M + log2f(L));
  };
  for (int e = tid; e < R * (D / 4); e += 32 * kStreamWarps) {
    const int i = e / (D / 4), c = e % (D / 4);
    float M = NEG_INF, L = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kStreamWarps; ++w) M = fmaxf(M, part_ml[w * R + i].x);
    const float ref = M == NEG_INF ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kStreamWarps; ++w) {
      const float2 ml = part_ml[w * R + i];
      const float4 y = *reinterpret_cast<const float4*>(part_o + (w * R + i) * D + 4 * c);
      const float f = exp2f(ml.x - ref);
      L = fmaf(ml.y, f, L);
      x.x = fmaf(y.x, f, x.x);
      x.y = fmaf(y.y, f, x.y);
      x.z = fmaf(y.z, f, x.z);
      x.w = fmaf(y.w, f, x.w);
    }
    if (parts == 1) {
      emit(i, c, x, M, L);
    } else {
      *reinterpret_cast<float4*>(cta_o + i * D + 4 * c) = x;
      if (c == 0) cta_ml[i] = make_float2(M, L);
    }
  }
  if (parts > 1) {
    cluster_sync_all();
    const uint32_t o_at = smem_u32(cta_o), ml_at = smem_u32(cta_ml);
    for (int e = rank * 32 * kStreamWarps + tid; e < R * (D / 4); e += parts * 32 * kStreamWarps) {
      const int i = e / (D / 4), c = e % (D / 4);
      const JoinedWord w = join_parts(ml_at + i * 8, o_at + (i * D + 4 * c) * 4, parts);
      emit(i, c, w.x, w.M, w.L);
    }
    cluster_sync_all();  // no CTA leaves while another still reads its part
  }
}

template <int D, int R>
static cudaError_t go_stream(const CrossArgs& a, cudaStream_t st) {
  constexpr size_t smem = ((size_t)kStreamWarps * R * (D + 2) + R * (D + 2)) * sizeof(float);
  auto kern = cross_stream_kernel<D, R>;
  static int configured[64] = {0};
  cudaError_t e = allow_shared_memory((const void*)kern, (int)smem, configured);
  if (e != cudaSuccess) return e;
  const int rows = a.group * a.Sq, blocks = (rows + R - 1) / R;
  const int parts = cross_parts((long long)blocks * a.Hkv * a.B, (a.Skv + 8 * kStreamKeys - 1) / (8 * kStreamKeys));
  return launch_clusters((const void*)kern, dim3((unsigned)(blocks * parts), a.Hkv, a.B), 32 * kStreamWarps, smem, parts, a, st);
}
template <int D>
static cudaError_t go_stream_rows(const CrossArgs& a, cudaStream_t st) {
  const int rows = a.group * a.Sq;
  return rows <= 1 ? go_stream<D, 1>(a, st) : rows <= 2 ? go_stream<D, 2>(a, st) : rows <= 4 ? go_stream<D, 4>(a, st) : go_stream<D, 8>(a, st);
}
cudaError_t launch_cross_stream(const CrossArgs& a, int D, cudaStream_t st) { return D == 64 ? go_stream_rows<64>(a, st) : go_stream_rows<128>(a, st); }

}  // namespace b200
