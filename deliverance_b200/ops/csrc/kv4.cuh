// Rows of a KV cache in 4 bits. A row of D numbers is D / 2 bytes of codes (byte i: element 2 i in the low half, 2 i + 1 in the high one) and then, per block
// of 32 elements, its step and its minimum in fp16: 5 bits a number. value = code * step + minimum.
//   m = fp16(min), s = (max - m) / 15 rounded up to 7 significant bits (to multiples of 2^-20 below 2^-14), code = rint((x - m) / s); magnitudes end at 472.
// With 7 bits code * step has 11 and is a number of fp16, as are 1024 s and 64 s (s < 64): reading codes by way of 1024 + code needs one FMA that rounds nothing.
// A block with a NaN in it is NaN.
#pragma once
#include "common.cuh"
#include "kv4_api.h"

namespace dlv {

constexpr float kKv4Limit = 472.f;

// two products or sums, each rounded by itself (mul.rn.f32x2 followed by add.rn.f32x2 comes back from the assembler with one rounding)
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return make_float2(__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y)); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return make_float2(__fsub_rn(a.x, b.x), __fsub_rn(a.y, b.y)); }
__device__ __forceinline__ float fmin3(float a, float b, float c) {
  float y;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {  // NaN if one of them is
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// step and minimum of a block whose (clamped) numbers lie in [lo, hi], and the reciprocal of the step; every operation rounds by itself
struct Kv4Block {
  __half s, m;
  float mf, inv;
  __device__ __forceinline__ Kv4Block(float lo, float hi, bool nan) {
    m = __float2half_rn(lo + 0.f);  // (no negative zero)
    mf = __half2float(m);
    const float s0 = __fmul_rn(fmaxf(__fsub_rn(hi, mf), 0.f), 1.f / 15.f);
    float sf = __int_as_float((__float_as_int(s0) + 0x1FFFF) & ~0x1FFFF);
    if (s0 < 0x1p-14f) sf = ceilf(s0 * 0x1p20f) * 0x1p-20f;
    s = __float2half_rn(sf);
    inv = sf > 0.f ? __frcp_rn(sf) : 0.f;
    if (nan) {
      s = __ushort_as_half(0);
      m = __ushort_as_half(0x7E00);
      mf = inv = 0.f;
    }
  }
  // Eight codes. The sum with 1.5 2^23 rounds halves to even, as rint does, and leaves the integer in its last bits: the products with 16^i put the codes side by side, above a constant. No code is above
  // 15: the step is no less than a fifteenth of the range.
  __device__ __forceinline__ uint32_t codes(const float2* x) const {
    uint32_t r = 0u - 0x4B400000u * 0x11111111u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 c = mul2(add2(x[i], make_float2(-mf, -mf)), make_float2(inv, inv));
      c = add2(make_float2(fmaxf(c.x, 0.f), fmaxf(c.y, 0.f)), make_float2(12582912.f, 12582912.f));
      r += __float_as_uint(c.x) * (1u << (8 * i)) + __float_as_uint(c.y) * (16u << (8 * i));
    }
    return r;
  }
  __device__ __forceinline__ uint32_t side() const { return static_cast<uint32_t>(__half_as_ushort(s)) | static_cast<uint32_t>(__half_as_ushort(m)) << 16; }
};

// eight neighbouring codes and their block's step and minimum -> values: a masked pair of codes under the exponent of 1024 is 1024 + c or 1024 + 16 c, fp16 takes that off exactly, and one fp32 FMA rounds
__device__ __forceinline__ void kv4_values(uint32_t codes, uint32_t side, float* v) {
  const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(side))), m = __half2float(__ushort_as_half(static_cast<unsigned short>(side >> 16)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (i < 2 ? codes : codes >> 8) & (i % 2 ? 0x00F000F0u : 0x000F000Fu) | 0x64006400u;
    const __half2 x = *reinterpret_cast<const __half2*>(&w);
    const float2 c = __half22float2(i % 2 ? __hfma2(x, __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-64.f, -64.f)) : __hadd2(x, __floats2half2_rn(-1024.f, -1024.f)));
    v[i] = fmaf(c.x, s, m);
    v[i + 4] = fmaf(c.y, s, m);
  }
}

}  // namespace dlv
