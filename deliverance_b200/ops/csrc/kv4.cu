// Writing and unpacking a KV cache in 4 bits (format: kv4.cuh).
#include "kv4.cuh"
#include "kv4_api.h"
#include "io.cuh"

namespace dlv {

// Head norms, rotation, queries out, keys and values quantised into their rows. A thread has 8 neighbouring numbers of a head, D / 8 threads a head, four a block; what it is rotated
// with it reads (and norms) once more, from cache. grid (T, threads of a row / 256).
// The cache holds codes, which change by whole steps: every operation in front of them rounds by itself (no contraction), and sums of squares are in 64 bits (exact for bf16
// numbers within 2^18 of one another), so that the codes do not depend on who computes them.
template <int D, bool PAIRS>
__global__ void __launch_bounds__(256) kv4_write_kernel(const Kv4WriteArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int TPH = D / 8;  // threads of a head
  const int t = blockIdx.x, unit = blockIdx.y * 256 + threadIdx.x, h = unit / TPH, e0 = unit % TPH * 8;
  const bool live = h < a.H + 2 * a.KV;
  const bool is_q = h < a.H, is_k = !is_q && h < a.H + a.KV;
  const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(a.qkv) + t * a.pitch + static_cast<long long>(live ? h : 0) * D;
  float x[8];
  io_ld8(row + e0, x);
  if (is_q || is_k) {
    const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(is_q ? a.q_norm : a.k_norm);
    float inv = 1.f;
    if (w != nullptr) {  // (whole heads, and the same in all threads: the shuffles below are for full groups of a head)
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fma(static_cast<double>(x[i]), static_cast<double>(x[i]), ss);
      const uint32_t group = TPH == 32 ? 0xffffffffu : ((1u << TPH) - 1u) << ((threadIdx.x & 31) / TPH * TPH);
#pragma unroll
      for (int o = 1; o < TPH; o <<= 1) ss += __shfl_xor_sync(group, ss, o);
      inv = static_cast<float>(1.0 / sqrt(ss / D + a.eps));
    }
    auto normed = [&](float v, int e) { return w == nullptr ? v : __fmul_rn(__fmul_rn(v, inv), __fadd_rn(bf2f(w[e]), a.offset)); };
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = normed(x[i], e0 + i);
    const int half = a.half;
    if (e0 < 2 * half) {
      int pos = a.positions[t];
      pos = pos < 0 ? 0 : (pos >= a.max_pos ? a.max_pos - 1 : pos);
      const float *cs = a.cos_t + static_cast<long long>(pos) * half, *sn = a.sin_t + static_cast<long long>(pos) * half;
      if constexpr (PAIRS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int p = e0 / 2 + i;
          if (p < half) {
            const float c = cs[p], n = sn[p], u = y[2 * i], v = y[2 * i + 1];
            y[2 * i] = __fsub_rn(__fmul_rn(u, c), __fmul_rn(v, n));
            y[2 * i + 1] = __fadd_rn(__fmul_rn(v, c), __fmul_rn(u, n));
          }
        }
      } else {
        float z[8], c[8], n[8];
        if (half % 8 == 0) {  // the partners are 8 neighbours too
          const int other = e0 < half ? e0 + half : e0 - half, p = e0 < half ? e0 : e0 - half;
          io_ld8(row + other, z);
          const bool wide = ((reinterpret_cast<uintptr_t>(cs + p) | reinterpret_cast<uintptr_t>(sn + p)) & 15) == 0;
          if (wide) {
            io_ld8(cs + p, c);
            io_ld8(sn + p, n);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (!wide) {
              c[i] = cs[p + i];
              n[i] = sn[p + i];
            }
            z[i] = normed(z[i], other + i);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int e = e0 + i, other = e < half ? e + half : e - half, p = e < half ? e : e - half;
            const bool in = e < 2 * half;
            z[i] = in ? normed(bf2f(row[other]), other) : 0.f;
            c[i] = in ? cs[p] : 1.f;
            n[i] = in ? sn[p] : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float m = __fmul_rn(z[i], n[i]);
          if (e0 + i < half) y[i] = __fsub_rn(__fmul_rn(y[i], c[i]), m);
          else if (e0 + i < 2 * half) y[i] = __fadd_rn(__fmul_rn(y[i], c[i]), m);
        }
      }
    }
    if (is_q) {
      io_st8(static_cast<__nv_bfloat16*>(a.q) + (static_cast<long long>(t) * a.H + h) * D + e0, y);
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
  }
  if (!live) return;
  float lo = INFINITY, hi = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    nan = nan || x[i] != x[i];
    x[i] = fminf(fmaxf(x[i], -kKv4Limit), kKv4Limit);
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
  const uint32_t four = 0xfu << (threadIdx.x & 28);  // the threads of a block
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(four, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(four, hi, o));
    nan = __shfl_xor_sync(four, static_cast<int>(nan), o) || nan;
  }
  const Kv4Block b(lo, hi, nan);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) codes |= b.code(x[i]) << (4 * i);
  const long long slot = a.slots[t];
  if (slot < 0) return;
  if (slot >= a.rows) {
    if (unit % TPH == 0) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
    return;
  }
  const int kvh = is_k ? h - a.H : h - a.H - a.KV;
  const bool narrow = slot <= 0xffffffffll;
  const long long page = narrow ? static_cast<unsigned>(slot) / static_cast<unsigned>(a.page) : slot / a.page;
  uint8_t* dst = (is_k ? a.k : a.v) + ((page * a.KV + kvh) * a.page + (slot - page * a.page)) * kv4_row_bytes(D);
  *reinterpret_cast<uint32_t*>(dst + e0 / 2) = codes;
  if (e0 % 32 == 0) *reinterpret_cast<uint32_t*>(dst + D / 2 + e0 / 8) = b.side();
}

void launch_kv4_write(const Kv4WriteArgs& a, cudaStream_t st) {
  if (a.T == 0) return;
  const dim3 grid(static_cast<unsigned>(a.T), static_cast<unsigned>(((a.H + 2 * a.KV) * (a.D / 8) + 255) / 256));
#define DLV_KV4_WRITE(DD) (a.pairs ? launch_pdl(kv4_write_kernel<DD, true>, grid, dim3(256), 0, st, a) : launch_pdl(kv4_write_kernel<DD, false>, grid, dim3(256), 0, st, a))
  if (a.D == 64) DLV_KV4_WRITE(64);
  else if (a.D == 128) DLV_KV4_WRITE(128);
  else DLV_KV4_WRITE(256);
#undef DLV_KV4_WRITE
}

// Pages -> bf16 or fp32 pages: what prompt attention reads, and what shows a cache's contents. 8 numbers per thread; grid (8-number units of a page / 256, n, keys | values).
template <int D, typename TO>
__global__ void __launch_bounds__(256) kv4_expand_kernel(const Kv4ExpandArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int TPR = D / 8, RB = kv4_row_bytes(D);
  const int unit = blockIdx.x * 256 + threadIdx.x, row = unit / TPR, e0 = unit % TPR * 8, rows = a.KV * a.page;
  if (row >= rows) return;
  int page = a.list[blockIdx.y];
  if (page < 0 || page >= a.pages) {
    if (unit == 0) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
    page = 0;
  }
  const uint8_t* src = (blockIdx.z ? a.v : a.k) + (static_cast<long long>(page) * rows + row) * RB;
  float v[8];
  kv4_values(*reinterpret_cast<const uint32_t*>(src + e0 / 2), *reinterpret_cast<const uint32_t*>(src + D / 2 + e0 / 32 * 4), v);
  io_st8(static_cast<TO*>(blockIdx.z ? a.vo : a.ko) + (static_cast<long long>(blockIdx.y) * rows + row) * D + e0, v);
}

void launch_kv4_expand(const Kv4ExpandArgs& a, cudaStream_t st) {
  if (a.n == 0) return;
  for (int at = 0; at < a.n; at += 65535) {
    Kv4ExpandArgs b = a;
    b.n = a.n - at < 65535 ? a.n - at : 65535;
    b.list += at;
    const long long skip = static_cast<long long>(at) * a.KV * a.page * a.D * (a.f32 ? 4 : 2);
    b.ko = static_cast<uint8_t*>(a.ko) + skip;
    b.vo = static_cast<uint8_t*>(a.vo) + skip;
    const dim3 grid(static_cast<unsigned>((static_cast<long long>(a.KV) * a.page * (a.D / 8) + 255) / 256), static_cast<unsigned>(b.n), 2);
#define DLV_KV4_EXPAND(DD) \
  (a.f32 ? launch_pdl(kv4_expand_kernel<DD, float>, grid, dim3(256), 0, st, b) : launch_pdl(kv4_expand_kernel<DD, __nv_bfloat16>, grid, dim3(256), 0, st, b))
    if (a.D == 64) DLV_KV4_EXPAND(64);
    else if (a.D == 128) DLV_KV4_EXPAND(128);
    else DLV_KV4_EXPAND(256);
#undef DLV_KV4_EXPAND
  }
}

// The pages of a step's sequences -> fp16 pages next to one another (sequence by sequence), for prompt attention, with block tables that name them; a page becomes page / out_page of them.
// Rows behind a sequence's end are zeros there. fp16, because a value is the sum of two fp16 numbers: 2^-12 of it are lost, where bf16 would lose 2^-9. A thread takes four units of 8 numbers, keys and values; grid (units of a page / 1024, pages of the longest sequence, S).
template <int D>
__global__ void __launch_bounds__(256) kv4_expand_seqs_kernel(const Kv4SeqsArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int TPR = D / 8, RB = kv4_row_bytes(D);
  const int s = blockIdx.z, j = blockIdx.y, lane = threadIdx.x & 31, rows = a.KV * a.page;
  auto pages_of = [&](int i) {
    const int n = max(0, min(a.ctx[i], a.width * a.page));
    return (n + a.page - 1) / a.page;
  };
  const int given = a.ctx[s], ctx = max(0, min(given, a.width * a.page)), own = (ctx + a.page - 1) / a.page;
  const bool first = blockIdx.x == 0 && j == 0;  // writes the sequence's block table
  if (j >= own && !first) return;
  int base = 0;
  for (int i = lane; i < s; i += 32) base += pages_of(i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) base += __shfl_xor_sync(0xffffffffu, base, o);
  if (first) {
    const bool bad = given != ctx || own > a.longest || base + own > a.total || (s == a.S - 1 && base + own != a.total);
    if (bad && threadIdx.x == 0) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
    const int cut = a.page / a.out_page;
    for (int c = threadIdx.x; c < a.width * cut; c += 256) a.out_tables[static_cast<long long>(s) * a.width * cut + c] = c < own * cut && base + c / cut < a.total ? base * cut + c : 0;
    if (j >= own) return;
  }
  if (base + j >= a.total) return;
  int page = a.tables[static_cast<long long>(s) * a.width + j];
  if (page < 0 || page >= a.pages) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
    page = 0;
  }
  const long long src = static_cast<long long>(page) * rows, dst = static_cast<long long>(base + j) * rows;
  const int left = ctx - j * a.page;  // rows of this page in use
  uint32_t codes[4][2], side[4][2];
  const int u0 = blockIdx.x * 1024 + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = u0 + 256 * i, row = u / TPR, e0 = u % TPR * 8;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      codes[i][kv] = side[i][kv] = 0;
      if (row < rows && row % a.page < left) {
        const uint8_t* p = (kv ? a.v : a.k) + (src + row) * RB;
        codes[i][kv] = *reinterpret_cast<const uint32_t*>(p + e0 / 2);
        side[i][kv] = *reinterpret_cast<const uint32_t*>(p + D / 2 + e0 / 32 * 4);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = u0 + 256 * i, row = u / TPR, e0 = u % TPR * 8;
    if (row >= rows) break;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float v[8];
      kv4_values(codes[i][kv], side[i][kv], v);
      const int head = row / a.page, at = row % a.page, part = at / a.out_page;  // row of the page -> part, head, row of the part
      const long long to = (dst + (part * a.KV + head) * a.out_page + at % a.out_page) * D + e0;
      __half2 h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<uint4*>(static_cast<__half*>(kv ? a.vo : a.ko) + to) = *reinterpret_cast<const uint4*>(h);
    }
  }
}

void launch_kv4_expand_seqs(const Kv4SeqsArgs& a, cudaStream_t st) {
  if (a.S == 0) return;
  const int units = a.KV * a.page * (a.D / 8);
  const dim3 grid(static_cast<unsigned>((units + 1023) / 1024), static_cast<unsigned>(a.longest < 1 ? 1 : a.longest), static_cast<unsigned>(a.S));
  if (a.D == 64) launch_pdl(kv4_expand_seqs_kernel<64>, grid, dim3(256), 0, st, a);
  else if (a.D == 128) launch_pdl(kv4_expand_seqs_kernel<128>, grid, dim3(256), 0, st, a);
  else launch_pdl(kv4_expand_seqs_kernel<256>, grid, dim3(256), 0, st, a);
}

}  // namespace dlv
