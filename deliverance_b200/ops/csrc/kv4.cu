// Writing and unpacking a KV cache in 4 bits (format: kv4.cuh).
#include "kv4.cuh"
#include "kv4_api.h"
#include "io.cuh"
#include "mma_pair.cuh"

namespace dlv {

// Head norms, rotation, queries out, keys and values quantised into their rows. The cache holds codes, which change by whole steps: every operation in front of them rounds by itself (no contraction), and the
// statistics are in 64 bits (sums of squares exact for bf16 numbers within 2^18 of one another), so that the codes do not depend on who computes them.
//
// A thread has two times 8 neighbouring numbers of one head: what is rotated together is in one thread, and four neighbouring threads have a block of either half. A CTA has all heads of a token, or a part of them, and
// goes through further tokens with the same heads: a thread reads its norm weights once, and copies what it needs of the next two tokens ahead into shared memory, each warp the tables' rows for itself. Bound by
// instructions (some 440 per thread and token): 8,192 rows of 32 + 2 x 8 heads of 128 62 us (177 MB: 27 at the copy rate), 121 with 8 numbers per thread, a partner's numbers read and normed again, and nothing ahead.
template <int D>
constexpr int kWriteHead = D / 16;  // threads of a head
constexpr int kWriteStages = 3;

// what is written of 8 numbers of a key or value
template <int D>
__device__ __forceinline__ void kv4_store(const Kv4WriteArgs& a, float2 (&y)[4], int e, uint32_t group, uint8_t* dst) {
  float lo = fmin3(fmin3(y[0].x, y[0].y, y[1].x), fmin3(y[1].y, y[2].x, y[2].y), fminf(y[3].x, y[3].y));
  float hi = fmax3_nan(fmax3_nan(y[0].x, y[0].y, y[1].x), fmax3_nan(y[1].y, y[2].x, y[2].y), fmax3_nan(y[3].x, y[3].y, y[3].y));
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {  // the threads of a block
    const float other = __shfl_xor_sync(group, hi, o);
    lo = fminf(lo, __shfl_xor_sync(group, lo, o));
    hi = fmax3_nan(hi, other, other);
  }
  const bool nan = hi != hi;
  if (nan || hi > kKv4Limit || lo < -kKv4Limit) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = make_float2(fminf(fmaxf(y[i].x, -kKv4Limit), kKv4Limit), fminf(fmaxf(y[i].y, -kKv4Limit), kKv4Limit));
    lo = fminf(fmaxf(lo, -kKv4Limit), kKv4Limit);
    hi = fminf(fmaxf(hi, -kKv4Limit), kKv4Limit);
  }
  const Kv4Block b(lo, hi, nan);
  const uint32_t codes = b.codes(y);
  if (dst == nullptr) return;
  *reinterpret_cast<uint32_t*>(dst + e / 2) = codes;
  if (e % 32 == 0) *reinterpret_cast<uint32_t*>(dst + D / 2 + e / 8) = b.side();
}
// the row of KV head 0 that a slot names (-1: none)
__device__ __forceinline__ int kv4_row(const Kv4WriteArgs& a, long long slot) {
  if (slot >= a.rows) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
  if (slot < 0 || slot >= a.rows) return -1;
  const int s = static_cast<int>(slot), block = a.by_page.of(s);  // (a cache has fewer than 2^31 rows)
  return block * a.KV * a.page + (s - block * a.page);
}

template <int D, bool PAIRS>
__global__ void __launch_bounds__(512) kv4_write_kernel(const Kv4WriteArgs a) {
  pdl_trigger();
  constexpr int TPH = kWriteHead<D>, STAGES = kWriteStages;
  extern __shared__ __align__(16) uint4 pieces[];  // [STAGES][2][threads] a thread's own, then [STAGES][warps][64] the position's cosines and sines
  const int threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = threadIdx.x % TPH, h = blockIdx.y * (threads / TPH) + threadIdx.x / TPH, half = a.half;
  const bool live = h < a.H + 2 * a.KV, norm = live && a.q_norm != nullptr && h < a.H + a.KV, is_q = h < a.H;
  const uint32_t group = ((1u << TPH) - 1u) << (lane / TPH * TPH);  // the lanes of this head: heads of one warp may be of different kinds
  // halves: element e with e + half, what is not rotated cut in two; pairs: neighbours, the head cut in two
  const bool turns = !PAIRS && 8 * j < half;
  const int ea = PAIRS || turns ? 8 * j : 8 * j + half, eb = PAIRS ? D / 2 + 8 * j : turns ? half + 8 * j : D / 2 + 8 * j;
  const bool wide = half % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.cos_t) | reinterpret_cast<uintptr_t>(a.sin_t)) & 15) == 0;  // (whole pieces of the tables)
  const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(a.qkv) + static_cast<long long>(live ? h : 0) * D;
  float* tables = reinterpret_cast<float*>(pieces + STAGES * 2 * threads + warp * 64);
  const int table_stage = threads / 32 * 256;
  auto place = [&](int t) { return t < a.T ? a.positions[t] : 0; };  // (brought into the tables where it is used: what looks at it here would wait for it)
  auto inside = [&](int pos) { return max(0, min(pos, a.max_pos - 1)); };
  auto fetch = [&](int t, int pos, int stage) {
    if (t < a.T) {
      const __nv_bfloat16* src = row + t * a.pitch;
      const uint32_t dst = smem_u32(pieces + stage * 2 * threads + threadIdx.x);
      cp16(dst, src + ea, true);
      cp16(dst + threads * 16, src + eb, true);
      if (wide && lane * 4 < half) {
        const long long at = static_cast<long long>(inside(pos)) * half + lane * 4;
        const uint32_t tab = smem_u32(tables + stage * table_stage) + lane * 16;
        cp16(tab, a.cos_t + at, true);
        cp16(tab + 512, a.sin_t + at, true);
      }
    }
    cp_commit();
  };
  pdl_wait();
  const int step = gridDim.x;
  int t = blockIdx.x, pos_here = place(t), pos_next = place(t + step), pos_after = place(t + 2 * step);
  long long slot_next = a.slots[t];
  fetch(t, pos_here, 0);
  fetch(t + step, pos_next, 1);
  float2 w[8];  // norm weights
  if (norm) {
    const __nv_bfloat16* weights = static_cast<const __nv_bfloat16*>(is_q ? a.q_norm : a.k_norm);
    io_ld8(weights + ea, reinterpret_cast<float*>(w));
    io_ld8(weights + eb, reinterpret_cast<float*>(w + 4));
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = make_float2(__fadd_rn(w[i].x, a.offset), __fadd_rn(w[i].y, a.offset));
  }
  const int kvh = h - a.H - (h < a.H + a.KV ? 0 : a.KV);
  uint8_t* cache = (h < a.H + a.KV ? a.k : a.v) + static_cast<long long>(kvh) * a.page * kv4_row_bytes(D);
  for (int stage = 0; t < a.T; t += step, stage = stage + 1 == STAGES ? 0 : stage + 1) {
    const int pos = inside(pos_here);
    const long long slot = slot_next;
    fetch(t + 2 * step, pos_after, stage == 0 ? STAGES - 1 : stage - 1);
    pos_here = pos_next;
    pos_next = pos_after;
    pos_after = place(t + 3 * step);
    slot_next = t + step < a.T ? a.slots[t + step] : -1;
    cp_wait<STAGES - 1>();
    __syncwarp();
    if (live) {
      float2 x[8];
      const uint4 ra = pieces[stage * 2 * threads + threadIdx.x], rb = pieces[(stage * 2 + 1) * threads + threadIdx.x];
      x[0] = unpack_bf162(ra.x);
      x[1] = unpack_bf162(ra.y);
      x[2] = unpack_bf162(ra.z);
      x[3] = unpack_bf162(ra.w);
      x[4] = unpack_bf162(rb.x);
      x[5] = unpack_bf162(rb.y);
      x[6] = unpack_bf162(rb.z);
      x[7] = unpack_bf162(rb.w);
      if (norm) {
        double ss = 0.0, s2 = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss = fma(static_cast<double>(x[i].x), static_cast<double>(x[i].x), ss);
          s2 = fma(static_cast<double>(x[i].y), static_cast<double>(x[i].y), s2);
        }
        ss += s2;
#pragma unroll
        for (int o = 1; o < TPH; o <<= 1) ss += __shfl_xor_sync(group, ss, o);
        const float inv = static_cast<float>(rsqrt(ss / D + a.eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = mul2(mul2(x[i], make_float2(inv, inv)), w[i]);
      }
      if (h < a.H + a.KV && half > 0) {
        const float* tab = tables + stage * table_stage;
        const long long at = static_cast<long long>(pos) * half;
        if constexpr (PAIRS) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int k = (i < 4 ? ea / 2 : eb / 2 - 4) + i;
            if (k < half) {
              const float c = wide ? tab[k] : a.cos_t[at + k], n = wide ? tab[128 + k] : a.sin_t[at + k];
              x[i] = add2(mul2(x[i], make_float2(c, c)), mul2(make_float2(x[i].y, x[i].x), make_float2(-n, n)));
            }
          }
        } else if (turns) {
          float2 c[4], n[4];
          if (wide) {
            io_ld8(tab + 8 * j, reinterpret_cast<float*>(c));
            io_ld8(tab + 128 + 8 * j, reinterpret_cast<float*>(n));
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              c[i] = make_float2(a.cos_t[at + 8 * j + 2 * i], a.cos_t[at + 8 * j + 2 * i + 1]);
              n[i] = make_float2(a.sin_t[at + 8 * j + 2 * i], a.sin_t[at + 8 * j + 2 * i + 1]);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 u = x[i], v = x[4 + i];
            x[i] = sub2(mul2(u, c[i]), mul2(v, n[i]));
            x[4 + i] = add2(mul2(v, c[i]), mul2(u, n[i]));
          }
        }
      }
      if (is_q) {
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.q) + (static_cast<long long>(t) * a.H + h) * D;
        *reinterpret_cast<uint4*>(dst + ea) = make_uint4(pack_bf162(x[0].x, x[0].y), pack_bf162(x[1].x, x[1].y), pack_bf162(x[2].x, x[2].y), pack_bf162(x[3].x, x[3].y));
        *reinterpret_cast<uint4*>(dst + eb) = make_uint4(pack_bf162(x[4].x, x[4].y), pack_bf162(x[5].x, x[5].y), pack_bf162(x[6].x, x[6].y), pack_bf162(x[7].x, x[7].y));
      } else {
        const int at = kv4_row(a, slot);
        uint8_t* dst = at < 0 ? nullptr : cache + static_cast<long long>(at) * kv4_row_bytes(D);
        kv4_store<D>(a, reinterpret_cast<float2(&)[4]>(x[0]), ea, group, dst);
        kv4_store<D>(a, reinterpret_cast<float2(&)[4]>(x[4]), eb, group, dst);
      }
    }
    __syncwarp();  // (the tables have been read)
  }
}

// The same where halves are rotated whose blocks lie otherwise (half no multiple of 32): 8 numbers per thread, partners by shuffles. grid (T, threads of a row / 256).
template <int D>
__global__ void __launch_bounds__(256) kv4_write_odd_kernel(const Kv4WriteArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int TPH = D / 8;  // threads of a head
  const int t = blockIdx.x, lane = threadIdx.x & 31, h = (blockIdx.y * 256 + threadIdx.x) / TPH, e0 = threadIdx.x % TPH * 8, half = a.half;
  if (h >= a.H + 2 * a.KV) return;  // (whole heads)
  const uint32_t group = TPH == 32 ? 0xffffffffu : ((1u << (TPH & 31)) - 1u) << (lane / TPH * TPH);
  float2 x[4];
  io_ld8(static_cast<const __nv_bfloat16*>(a.qkv) + t * a.pitch + static_cast<long long>(h) * D + e0, reinterpret_cast<float*>(x));
  if (h < a.H + a.KV) {
    if (a.q_norm != nullptr) {
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss = fma(static_cast<double>(x[i].y), static_cast<double>(x[i].y), fma(static_cast<double>(x[i].x), static_cast<double>(x[i].x), ss));
#pragma unroll
      for (int o = 1; o < TPH; o <<= 1) ss += __shfl_xor_sync(group, ss, o);
      const float inv = static_cast<float>(rsqrt(ss / D + a.eps));
      float2 w[4];
      io_ld8(static_cast<const __nv_bfloat16*>(h < a.H ? a.q_norm : a.k_norm) + e0, reinterpret_cast<float*>(w));
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = mul2(mul2(x[i], make_float2(inv, inv)), make_float2(__fadd_rn(w[i].x, a.offset), __fadd_rn(w[i].y, a.offset)));
    }
    const long long at = static_cast<long long>(max(0, min(a.positions[t], a.max_pos - 1))) * half;
    float v[8], r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = x[i].x;
      v[2 * i + 1] = x[i].y;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // element e0 + i with e0 + i + half or - half: of one thread or of two
      const int e = e0 + i, other = e < half ? e + half : e < 2 * half ? e - half : e;
      float z = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float theirs = __shfl_sync(group, v[k], lane / TPH * TPH + other / 8);
        z = other % 8 == k ? theirs : z;
      }
      const int k = e < half ? e : e - half;
      r[i] = v[i];
      if (e < 2 * half) r[i] = __fadd_rn(__fmul_rn(v[i], a.cos_t[at + k]), __fmul_rn(z, e < half ? -a.sin_t[at + k] : a.sin_t[at + k]));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = make_float2(r[2 * i], r[2 * i + 1]);
  }
  if (h < a.H) {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.q) + (static_cast<long long>(t) * a.H + h) * D + e0) =
        make_uint4(pack_bf162(x[0].x, x[0].y), pack_bf162(x[1].x, x[1].y), pack_bf162(x[2].x, x[2].y), pack_bf162(x[3].x, x[3].y));
    return;
  }
  const int at = kv4_row(a, a.slots[t]), kvh = h - a.H - (h < a.H + a.KV ? 0 : a.KV);
  kv4_store<D>(a, x, e0, group, at < 0 ? nullptr : (h < a.H + a.KV ? a.k : a.v) + static_cast<long long>(at + kvh * a.page) * kv4_row_bytes(D));
}

template <int D, bool PAIRS>
static void launch_write_t(const Kv4WriteArgs& a, cudaStream_t st) {
  constexpr int TPH = kWriteHead<D>, most = 512;
  static PerDeviceOnce once;
  if (once.first()) cudaFuncSetAttribute(kv4_write_kernel<D, PAIRS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWriteStages * (2 * most + most * 2) * 16);
  // a token's heads in one CTA where there are tokens for all SMs, otherwise in parts of 128 threads
  const int heads = a.H + 2 * a.KV, want = heads * TPH < (a.T < 148 ? 128 : most) ? heads * TPH : (a.T < 148 ? 128 : most), threads = (want + 31) / 32 * 32, y = (heads * TPH + threads - 1) / threads;
  const int smem = kWriteStages * (2 * threads + threads * 2) * 16, per_sm = 1024 / threads < 8 ? (1024 / threads < 1 ? 1 : 1024 / threads) : 8, room = 148 * per_sm / y < 1 ? 1 : 148 * per_sm / y;
  launch_pdl(kv4_write_kernel<D, PAIRS>, dim3(a.T < room ? a.T : room, y), dim3(threads), smem, st, a);
}
template <int D>
static void launch_write_d(const Kv4WriteArgs& a, cudaStream_t st) {
  if (a.pairs) launch_write_t<D, true>(a, st);
  else if (a.half % 32 == 0) launch_write_t<D, false>(a, st);
  else launch_pdl(kv4_write_odd_kernel<D>, dim3(a.T, ((a.H + 2 * a.KV) * (D / 8) + 255) / 256), dim3(256), 0, st, a);
}
void launch_kv4_write(const Kv4WriteArgs& a, cudaStream_t st) {
  if (a.T == 0) return;
  if (a.D == 64) launch_write_d<64>(a, st);
  else if (a.D == 128) launch_write_d<128>(a, st);
  else launch_write_d<256>(a, st);
}

// Pages -> bf16 or fp32 pages: what shows a cache's contents. A thread takes four units of 8 numbers, keys and values; grid (units of a page / 1024, n).
template <int D, typename TO>
__global__ void __launch_bounds__(256) kv4_expand_kernel(const Kv4ExpandArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int TPR = D / 8, RB = kv4_row_bytes(D);
  const int rows = a.KV * a.page, u0 = blockIdx.x * 1024 + threadIdx.x;
  int page = a.list[blockIdx.y];
  if (page < 0 || page >= a.pages) {
    if (u0 == 0) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
    page = 0;
  }
  uint32_t codes[4][2], side[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = u0 + 256 * i, row = u / TPR, e0 = u % TPR * 8;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      codes[i][kv] = side[i][kv] = 0;
      if (row < rows) {
        const uint8_t* p = (kv ? a.v : a.k) + (static_cast<long long>(page) * rows + row) * RB;
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
      io_st8(static_cast<TO*>(kv ? a.vo : a.ko) + (static_cast<long long>(blockIdx.y) * rows + row) * D + e0, v);
    }
  }
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
    const dim3 grid(static_cast<unsigned>((static_cast<long long>(a.KV) * a.page * (a.D / 8) + 1023) / 1024), static_cast<unsigned>(b.n));
#define DLV_KV4_EXPAND(DD) \
  (a.f32 ? launch_pdl(kv4_expand_kernel<DD, float>, grid, dim3(256), 0, st, b) : launch_pdl(kv4_expand_kernel<DD, __nv_bfloat16>, grid, dim3(256), 0, st, b))
    if (a.D == 64) DLV_KV4_EXPAND(64);
    else if (a.D == 128) DLV_KV4_EXPAND(128);
    else DLV_KV4_EXPAND(256);
#undef DLV_KV4_EXPAND
  }
}

// The pages of a step's sequences -> fp16 pages next to one another (sequence by sequence), for prompt attention, with block tables that name them; a page becomes page / out_page of them.
// Rows behind a sequence's end, and rows that no window reaches, are zeros there: what stands in them does not matter, not even NaN. fp16, because a value is the sum of two fp16 numbers: up to 2^-11 of it are lost, where bf16 would lose 2^-8. A thread takes four units of 8 numbers, keys and values; grid (units of a page / 1024, pages of the longest sequence, S).
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
    const int qs = a.q_start[s], ql = a.q_len[s];
    const bool bad = given != ctx || own > a.longest || base + own > a.total || (s == a.S - 1 && base + own != a.total) || ql < 0 || ql > ctx || qs < 0 || static_cast<long long>(qs) + ql > a.T;
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
  // rows of this page in use, and those in front of all query rows' windows
  const int left = ctx - j * a.page, front = a.window > 0 ? ctx - max(0, min(a.q_len[s], ctx)) + 1 - a.window - j * a.page : 0;
  uint32_t codes[4][2], side[4][2];
  const int u0 = blockIdx.x * 1024 + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = u0 + 256 * i, row = u / TPR, e0 = u % TPR * 8;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      codes[i][kv] = side[i][kv] = 0;
      if (row < rows && row % a.page < left && row % a.page >= front) {
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
