// The 8-bit paged KV cache: layout constants and conversions shared by the kernels that fill and
// read it.
//
// k_cache / v_cache [num_blocks, hkv, 256, 128] hold e4m3 codes, k_scale / v_scale
// [num_blocks, hkv, 4] one fp32 scale per block of 64 tokens and head: value = code * scale.  The
// 64 tokens of a block and head are 8 KB in a row, so one bulk copy brings a tile.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace {

constexpr int KV8_D = 128;      // head width
constexpr int KV8_PAGE = 256;   // tokens of a page
constexpr int KV8_BLOCK = 64;   // tokens that share a scale
constexpr int KV8_SUBS = KV8_PAGE / KV8_BLOCK;
constexpr int KV8_TILE = KV8_BLOCK * KV8_D;  // bytes of one block's codes of one head

// Four e4m3 codes as halves, two to a word: exact, every code is a half value (NaN stays NaN).
QB_DEVICE void e4m3x4_to_half2x2(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
QB_DEVICE void e4m3x4_to_float4(uint32_t codes, float (&f)[4]) {
  uint32_t lo, hi;
  e4m3x4_to_half2x2(codes, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
// Four values as e4m3 codes, round to nearest even; beyond +-448 saturates, NaN stays NaN.
QB_DEVICE uint32_t float4_to_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Two fp32 products, sums, multiply-adds in one instruction.
QB_DEVICE float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
QB_DEVICE float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
QB_DEVICE float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

}  // namespace
