// Packed fp32 arithmetic and exponentials of the softmax warps of the tcgen05 attention kernels.
#pragma once
#include <cstdint>

namespace b200 {

// 2^x for x <= 0 on the FMA / ALU pipes instead of the special-function unit, which is the busiest
// unit of the softmax warps (one MUFU.EX2 per score is as many cycles per tile as the MMAs): round x
// to the nearest integer n with the 1.5 * 2^23 trick, evaluate a cubic fit of 2^f on f = x - n in
// [-0.5, 0.5] (relative error 8e-5, below what a 16-bit P keeps), add n to the exponent field.
__device__ __forceinline__ float exp2_poly(float x) {
  x = fmaxf(x, -126.f);  // masked scores (-inf) and anything below 2^-126 end up at ~1e-38
  const float r = x + 12582912.f;
  const float f = x - (r - 12582912.f);
  float p = fmaf(f, 0.05508868396282196f, 0.24260404706001282f);
  p = fmaf(f, p, 0.6932762265205383f);
  p = fmaf(f, p, 0.9999289512634277f);
  return __int_as_float(__float_as_int(p) + (__float_as_int(r) << 23));
}

// Packed fp32 arithmetic of sm_100 (two lanes per instruction) and the three-input maximum: the softmax
// warps are bound by the number of instructions they issue per tile, and these halve the scale / subtract,
// the row sum, the polynomial and the row maximum.
__device__ __forceinline__ void ffma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.ftz.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void fadd2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.ftz.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.ftz.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// exp2_poly on two values at once
__device__ __forceinline__ void exp2_poly2(float x0, float x1, float& p0, float& p1) {
  x0 = fmaxf(x0, -126.f);
  x1 = fmaxf(x1, -126.f);
  float r0, r1, t0, t1, f0, f1;
  fadd2(r0, r1, x0, x1, 12582912.f, 12582912.f);
  fadd2(t0, t1, r0, r1, -12582912.f, -12582912.f);
  ffma2(f0, f1, t0, t1, -1.f, -1.f, x0, x1);
  ffma2(p0, p1, f0, f1, 0.05508868396282196f, 0.05508868396282196f, 0.24260404706001282f, 0.24260404706001282f);
  ffma2(p0, p1, f0, f1, p0, p1, 0.6932762265205383f, 0.6932762265205383f);
  ffma2(p0, p1, f0, f1, p0, p1, 0.9999289512634277f, 0.9999289512634277f);
  p0 = __int_as_float(__float_as_int(p0) + (__float_as_int(r0) << 23));
  p1 = __int_as_float(__float_as_int(p1) + (__float_as_int(r1) << 23));
}

}  // namespace b200
