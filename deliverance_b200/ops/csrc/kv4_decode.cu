// Decode attention over a KV cache in 4 bits (format: kv4.cuh).
#include "kv4.cuh"
#include "kv4_api.h"

namespace dlv {

// grid (B, H), 4 warps. A warp takes every fourth key: lane l has elements l * D / 32 .. of the row, scores by a warp sum, running maximum and sum, values unpacked the same way.
template <int D>
__global__ void __launch_bounds__(128) kv4_decode_kernel(const Kv4DecodeArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int PER = D / 32, RB = kv4_row_bytes(D);
  __shared__ float so[4][D], sm[4], sl[4];
  const int b = blockIdx.x, h = blockIdx.y, kvh = h / (a.H / a.KV), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int ctx = a.ctx[b];
  if ((ctx < 0 || ctx > a.width * a.page) && threadIdx.x == 0) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
  ctx = max(0, min(ctx, a.width * a.page));
  const int first = a.window > 0 && ctx > a.window ? ctx - a.window : 0;
  float q[PER], o[PER] = {}, m = -INFINITY, l = 0.f;
  const __nv_bfloat16* qr = static_cast<const __nv_bfloat16*>(a.q) + b * a.q_stride + h * D + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; ++i) q[i] = bf2f(qr[i]);
  for (int j = first + warp; j < ctx; j += 4) {
    int page = a.tables[static_cast<long long>(b) * a.width + j / a.page];
    if (page < 0 || page >= a.pages) {
      if (lane == 0) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
      page = 0;
    }
    const long long at = ((static_cast<long long>(page) * a.KV + kvh) * a.page + j % a.page) * RB;
    auto get = [&](const uint8_t* row, int i) {
      const int e = lane * PER + i;
      const uint32_t side = *reinterpret_cast<const uint32_t*>(row + D / 2 + e / 32 * 4);
      const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(side))), lo = __half2float(__ushort_as_half(static_cast<unsigned short>(side >> 16)));
      return fmaf(static_cast<float>((row[e / 2] >> (e % 2 * 4)) & 15), s, lo);
    };
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) x = fmaf(q[i], get(a.k + at, i), x);
    x = warp_sum(x) * a.scale;
    if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
    const float top = fmaxf(m, x), f = m == -INFINITY ? 0.f : __expf(m - top), p = __expf(x - top);
    m = top;
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = o[i] * f + p * get(a.v + at, i);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) so[warp][lane * PER + i] = o[i];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float f[4], sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.f : __expf(sm[w] - top);
    sum += f[w] * sl[w];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    const float v = f[0] * so[0][d] + f[1] * so[1][d] + f[2] * so[2][d] + f[3] * so[3][d];
    static_cast<__nv_bfloat16*>(a.out)[(static_cast<long long>(b) * a.H + h) * D + d] = f2bf(sum > 0.f ? v / sum : 0.f);
  }
}

int launch_kv4_decode(const Kv4DecodeArgs& a, cudaStream_t st) {
  const dim3 grid(a.B, a.H);
  if (a.D == 64) launch_pdl(kv4_decode_kernel<64>, grid, dim3(128), 0, st, a);
  else if (a.D == 128) launch_pdl(kv4_decode_kernel<128>, grid, dim3(128), 0, st, a);
  else launch_pdl(kv4_decode_kernel<256>, grid, dim3(128), 0, st, a);
  return 1;
}

}  // namespace dlv
