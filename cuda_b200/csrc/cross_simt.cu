// Cross attention in fp32 arithmetic on the FMA pipes: fp32 tensors need it (their tolerance is far below what a
// 16-bit operand keeps).
//
//   S = scale Q K^T over a tile of 64 states, running row maximum m and sum l, O = O 2^(m_old - m) + 2^(S - m) V,
//   out = O / l, lse = ln2 (m + log2 l)        (S, m in units of log2)
//
// One CTA of 256 threads takes 64 query rows (head-major: the rows of the heads that share a KV head) and walks the
// states of its sequence; thread (ty, tx) of a 16 x 16 grid holds 4 rows x 4 states of S and 4 rows x D/16 columns of O.
// Q, K and P sit transposed in shared memory, so that each step of a product reads two 16-byte fragments for 16 FMAs.
#include "cross_attention.cuh"

namespace b200 {

constexpr int kSimtRows = 64, kSimtKeys = 64;

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <>
__device__ __forceinline__ float4 load4<__half>(const __half* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(f16x2_lo(u.x), f16x2_hi(u.x), f16x2_lo(u.y), f16x2_hi(u.y));
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 x);
template <>
__device__ __forceinline__ void store4<float>(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
template <>
__device__ __forceinline__ void store4<__half>(__half* p, float4 x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_f16x2(x.x, x.y), pack_f16x2(x.z, x.w));
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, float4 x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
}

template <typename T, int D>
__global__ void __launch_bounds__(256) cross_simt_kernel(const CrossArgs a) {
  constexpr int LD = kSimtRows + 4;  // padded leading dimension of the transposed tiles
  constexpr float NEG_INF = -__builtin_huge_valf();
  extern __shared__ __align__(16) float sm[];
  float* sQ = sm;                  // [D][LD]
  float* sK = sQ + D * LD;         // [D][LD]
  float* sV = sK + D * LD;         // [kSimtKeys][D]
  float* sP = sV + kSimtKeys * D;  // [kSimtKeys][LD]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int rows = a.group * a.Sq, r0 = blockIdx.x * kSimtRows;
  const int len = cross_kv_len(a, b);
  const T* kp = static_cast<const T*>(a.k) + b * a.k_st[0] + kvh * a.k_st[1];
  const T* vp = static_cast<const T*>(a.v) + b * a.v_st[0] + kvh * a.v_st[1];
  auto row_head = [&](int r) { return kvh * a.group + r / a.Sq; };
  auto row_pos = [&](int r) { return r % a.Sq; };

  for (int i = tid; i < kSimtRows * (D / 4); i += 256) {
    const int r = i & 63, c = i >> 6;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r < rows)
      x = load4(static_cast<const T*>(a.q) + b * a.q_st[0] + row_head(r0 + r) * a.q_st[1] + row_pos(r0 + r) * a.q_st[2] + 4 * c);
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
  for (int t0 = 0; t0 < len; t0 += kSimtKeys) {
    __syncthreads();  // the tiles of the step before are read
    for (int i = tid; i < kSimtKeys * (D / 4); i += 256) {
      const int r = i & 63, c = i >> 6;
      const float4 x = t0 + r < len ? load4(kp + (t0 + r) * a.k_st[2] + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
      sK[(4 * c) * LD + r] = x.x;
      sK[(4 * c + 1) * LD + r] = x.y;
      sK[(4 * c + 2) * LD + r] = x.z;
      sK[(4 * c + 3) * LD + r] = x.w;
      const int vr = i / (D / 4), vc = i % (D / 4);
      *reinterpret_cast<float4*>(sV + vr * D + 4 * vc) =
          t0 + vr < len ? load4(vp + (t0 + vr) * a.v_st[2] + 4 * vc) : make_float4(0.f, 0.f, 0.f, 0.f);
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
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float sum = l[i];
#pragma unroll
    for (int x = 8; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    const int r = r0 + ty * 4 + i;
    if (r >= rows) continue;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // nothing seen: zeros
    T* op = static_cast<T*>(a.out) + b * a.o_st[0] + row_head(r) * a.o_st[1] + row_pos(r) * a.o_st[2];
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      store4(op + c * 64 + tx * 4, make_float4(o[i][c * 4] * inv, o[i][c * 4 + 1] * inv, o[i][c * 4 + 2] * inv, o[i][c * 4 + 3] * inv));
    if (a.lse && tx == 0)
      a.lse[((size_t)b * a.Hq + row_head(r)) * a.Sq + row_pos(r)] = sum == 0.f ? NEG_INF : kLn2 * (m[i] + log2f(sum));
  }
}

template <typename T, int D>
static cudaError_t go(const CrossArgs& a, cudaStream_t st) {
  constexpr size_t smem = (2 * D * (kSimtRows + 4) + kSimtKeys * D + kSimtKeys * (kSimtRows + 4)) * sizeof(float);
  auto kern = cross_simt_kernel<T, D>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const long long rows = (long long)a.group * a.Sq;
  kern<<<dim3((unsigned)((rows + kSimtRows - 1) / kSimtRows), a.Hkv, a.B), 256, smem, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_cross_simt(const CrossArgs& a, int D, cudaStream_t st) {
  if (a.dtype == CUDA_LLM_F32) return D == 64 ? go<float, 64>(a, st) : go<float, 128>(a, st);
  if (a.dtype == CUDA_LLM_F16) return D == 64 ? go<__half, 64>(a, st) : go<__half, 128>(a, st);
  return D == 64 ? go<__nv_bfloat16, 64>(a, st) : go<__nv_bfloat16, 128>(a, st);
}

}  // namespace b200
