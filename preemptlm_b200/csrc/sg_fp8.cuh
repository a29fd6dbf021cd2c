// 8-bit (e4m3) rows with one fp32 scale per 128 consecutive values.
#pragma once

#include <cuda_fp8.h>

#include "sg_common.cuh"

namespace sg {

constexpr int FP8_BLOCK = 128;     // values that share a scale
constexpr float FP8_MAX = 448.0f;  // largest finite e4m3 value

// Scale of a block whose largest magnitude is amax: the smallest normal fp32
// for a block of zeros (or of values below it), so that no division is by zero
// and the values come back as they were.
__device__ __forceinline__ float fp8_block_scale(float amax) {
  return fmaxf(__fdiv_rn(amax, FP8_MAX), 1.17549435e-38f);
}

// Two values in e4m3, round to nearest even, saturating at +-448 (NaN stays
// NaN); lo in the low byte.
__device__ __forceinline__ uint32_t fp8_pair(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ uint2 fp8_pack8(const float (&v)[8]) {
  return make_uint2(fp8_pair(v[0], v[1]) | fp8_pair(v[2], v[3]) << 16, fp8_pair(v[4], v[5]) | fp8_pair(v[6], v[7]) << 16);
}
// Eight values divided by s (true division: the codes then equal the
// definition's on every input).
__device__ __forceinline__ uint2 fp8_pack8(const float (&v)[8], float s) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(v[i], s);
  return fp8_pack8(q);
}

__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
  v[0] = lo_bf16(w.x); v[1] = hi_bf16(w.x); v[2] = lo_bf16(w.y); v[3] = hi_bf16(w.y);
  v[4] = lo_bf16(w.z); v[5] = hi_bf16(w.z); v[6] = lo_bf16(w.w); v[7] = hi_bf16(w.w);
}

// Pairs of fp32 values in one register pair: one instruction for two operations.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 f2_get(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ void unpack8(const uint4& w, uint64_t (&v)[4]) {
  v[0] = f2(lo_bf16(w.x), hi_bf16(w.x));
  v[1] = f2(lo_bf16(w.y), hi_bf16(w.y));
  v[2] = f2(lo_bf16(w.z), hi_bf16(w.z));
  v[3] = f2(lo_bf16(w.w), hi_bf16(w.w));
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
}

__device__ __forceinline__ uint4 pack8(const uint64_t (&v)[4]) {
  const float2 a = f2_get(v[0]), b = f2_get(v[1]), c = f2_get(v[2]), d = f2_get(v[3]);
  return make_uint4(bf16_pair(a.x, a.y), bf16_pair(b.x, b.y), bf16_pair(c.x, c.y), bf16_pair(d.x, d.y));
}
__device__ __forceinline__ uint2 fp8_pack8(const uint64_t (&v)[4], float s) {
  const float2 a = f2_get(v[0]), b = f2_get(v[1]), c = f2_get(v[2]), d = f2_get(v[3]);
  return fp8_pack8({a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y}, s);
}

}  // namespace sg
