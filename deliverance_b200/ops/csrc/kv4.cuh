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
    inv = sf > 0.f ? __fdiv_rn(1.f, sf) : 0.f;
    if (nan) {
      s = __ushort_as_half(0);
      m = __ushort_as_half(0x7E00);
      mf = inv = 0.f;
    }
  }
  __device__ __forceinline__ uint32_t code(float x) const {
    const float c = rintf(__fmul_rn(__fsub_rn(x, mf), inv));
    return static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f));  // (a NaN: 0)
  }
  __device__ __forceinline__ uint32_t side() const { return static_cast<uint32_t>(__half_as_ushort(s)) | static_cast<uint32_t>(__half_as_ushort(m)) << 16; }
};

// eight neighbouring codes and their block's step and minimum -> values
__device__ __forceinline__ void kv4_values(uint32_t codes, uint32_t side, float* v) {
  const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(side))), m = __half2float(__ushort_as_half(static_cast<unsigned short>(side >> 16)));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fmaf(static_cast<float>((codes >> (4 * i)) & 15u), s, m);
}

}  // namespace dlv
