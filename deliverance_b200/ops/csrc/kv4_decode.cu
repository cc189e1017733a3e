// Decode attention over a KV cache in 4 bits (format: kv4.cuh).
//
// What bounds it: the rows of the cache, 5 bits a number, behind two launches: 12 us and 1.19 of the copy time for 64 sequences of 544 to 4,352 keys, 8 KV heads of 4 x 128 (heads of 64: 14 us and 1.43). At the copy rate an
// SM gets 22 bytes a cycle, 35 numbers, for its 128 lanes: 3.6 lane instructions per number for everything. They do not fill it (56 % of the issue slots); a warp takes scores, softmax and values one behind the other.
//   Keys: a code c under the mask 0x000f is, as an fp16 number, 2^-24 c, under 0x00f0 2^-20 c: operands of a matrix product as they stand (queries of the second kind are divided by 16). The products of a block
//   are multiplied by its step in fp32, q . (c s + m) = sum over blocks of s (q . c) + m (sum of q): the minima are one more product with a column per block.
//   Values: the step belongs to the key, which the product sums over. With the exponent of 1024 a masked code is 1024 + c or 1024 + 16 c, and c s = (1024 + c) s - 1024 s = (1024 + 16 c) (s / 16) - 64 s: one FMA
//   per pair, and exact, because s has 7 bits. sum p (c s + m) = sum p c s + sum p m, one more product with a row per word of codes.
//
// Products are mma.sync m16n8k16 in fp16 with the cache as the 16-row operand and the (up to 8) query heads of a KV head as the 8 columns (two such column tiles for 9 to 16 heads): with heads as rows half
// of every product would be wasted on groups of 4 or 8, and so would the exponentials. Scores S^T [keys x heads] = K Q^T, O^T [D x heads] = V^T P^T.
//   K operand: row = key, k = elements; which element stands at which k is free as long as Q agrees. Lane (g, t) = (lane / 4, lane % 4) takes word t of every block of key g's codes, 8 of them.
//   V operand: row = element, k = keys; lane (g, t) takes the words (8 codes) g and g + 8 of keys 2 t and 2 t + 1, put side by side by two byte permutes per word pair; row g of product i is code i of word g.
//   P^T: a score tile transposed by movmatrix.
// Queries are multiplied by the power of two that brings a head's largest number to [2^14, 2^15): bf16's range fits fp16 then (what is lost is below 2^-34 of that number). Probabilities are held 2^12 times as large and relative to a maximum that follows when a
// score has outgrown it by 2^3: they stay below 2^15, and 2^-36 of the largest is the smallest that counts.
//
// Work: the 32-key tiles of all sequences and KV heads in a row, cut into equal shares, one per warp, in order. A share may end inside a sequence and hold several; a warp writes the heads of (sequence, KV
// head) pairs that it has seen whole, and partial results (at most two: of the pair its share begins inside, and of the one it ends inside) otherwise, which a second launch merges. The four warps of a CTA merge
// theirs first where all lie inside one pair. No sequence's length decides who waits for whom: batches of unlike lengths need no plan.
// A warp copies its tiles (32 rows lie next to one another) through a ring of its own, one bulk copy each for keys and values, and nothing but the end of the CTA brings the warps together.
#include "kv4.cuh"
#include "kv4_api.h"

namespace dlv {

namespace {

constexpr int kTile = 32;      // keys of a tile
constexpr int kWarps = kKv4Warps;
constexpr int kMinTiles = kKv4MinTiles;
constexpr int kNear = 8;       // partial results of a pair that the second launch fetches at once
constexpr float kShift = 12.f, kSlack = 3.f;
constexpr float kLog2e = 1.44269504088896341f;

enum : int { kFirst = 1, kLast = 2, kOpen = 4, kClose = 8, kPartial = 16 };  // a tile is its pair's first, its last, the first of a pair that a share has, the last, has keys that do not count

template <int D, int NT>
struct Kv4Ring {
  static constexpr int kRow = kv4_row_bytes(D), kCopy = kTile * kRow, kStage = 2 * kCopy;
  static constexpr int kStages = 2;
  static constexpr int kCtas = (D == 64 ? 4 : D == 128 ? 3 : 2) - (NT - 1);  // per SM, as registers allow
  static constexpr int kBytes = kWarps * kStages * kStage;
};

__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(magic));
  return y;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = v.x;
      w[i + 1] = v.y;
      w[i + 2] = v.z;
      w[i + 3] = v.w;
    }
  }
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float tanh_series(float x) {
  const float x2 = x * x;
  float p = fmaf(x2, -1382.f / 155925.f, 62.f / 2835.f);
  p = fmaf(x2, p, -17.f / 315.f);
  p = fmaf(x2, p, 2.f / 15.f);
  p = fmaf(x2, p, -1.f / 3.f);
  p = fmaf(x2, p, 1.f);
  return x * p;
}
// steps of a pair of numbers -> the factors and summands that unpack them
struct Kv4Steps {
  uint32_t s, s16, b, b16;
  __device__ __forceinline__ explicit Kv4Steps(uint32_t steps) : s(steps), s16(hmul2(steps, 0x2C002C00u)), b(hmul2(steps, 0xE400E400u)), b16(hmul2(steps, 0xD400D400u)) {}  // / 16, * -1024, * -64
  __device__ __forceinline__ uint32_t low(uint32_t w) const { return hfma2(and_or(w, 0x000F000Fu, 0x64006400u), s, b); }
  __device__ __forceinline__ uint32_t high(uint32_t w) const { return hfma2(and_or(w, 0x00F000F0u, 0x64006400u), s16, b16); }
};

__device__ __forceinline__ int tiles_of(const Kv4DecodeArgs& a, int ctx, int& first_key, int& first_tile) {
  first_key = a.window > 0 && ctx > a.window ? ctx - a.window : 0;
  first_tile = first_key / kTile;
  return (ctx + kTile - 1) / kTile - first_tile;
}
__device__ __forceinline__ int clamped(const Kv4DecodeArgs& a, int ctx) { return max(0, min(ctx, a.width * a.page)); }

}  // namespace

template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, Kv4Ring<D, NT>::kCtas) kv4_decode_kernel(const Kv4DecodeArgs a) {
  pdl_trigger();
  using R = Kv4Ring<D, NT>;
  constexpr int BLK = D / 32, CH = D == 256 ? 2 : 1;  // blocks, and chunks of up to four of them
  constexpr int OG = D == 256 ? 2 : 1;          // groups of 16 words of a row (D = 64: 8 words, both halves of them)
  constexpr int OT = D == 64 ? 4 : 8;           // products per group
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ __align__(8) uint64_t bars[kWarps][R::kStages];
  __shared__ int4 notes[kWarps][64];  // of the tiles that are copied and those to come: flags, pair, keys of the tile that count (from, to)
  __shared__ long long places[kWarps][64];  // where their rows lie in the caches
  __shared__ int2 spans[kWarps][64];        // the pair's first tile and number of tiles
  __shared__ int abort_word;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  volatile int* abort_flag = &abort_word;
  uint8_t* ring = ring_all + warp * R::kStages * R::kStage;
  if (tid == 0) abort_word = 0;
  if (lane < R::kStages) mbar_init(smem_u32(&bars[warp][lane]), 1);
  mbar_fence_init();
  __syncthreads();
  pdl_wait();

  // ---- where the shares of this CTA and of this warp begin: every warp adds the lengths up by itself, 32 sequences at a time
  auto tiles_at = [&](int b) {
    int fk, ft;
    return b < a.B ? tiles_of(a, clamped(a, a.ctx[b]), fk, ft) : 0;
  };
  int sum_all = 0;
  for (int b = lane; b < a.B; b += 32) sum_all += tiles_at(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum_all += __shfl_xor_sync(0xffffffffu, sum_all, o);
  const Kv4Shares shares(sum_all * a.KV, static_cast<int>(gridDim.x) * kWarps);
  const int worker = blockIdx.x * kWarps + warp;
  const long long cta_lo = static_cast<long long>(blockIdx.x) * kWarps * shares.per, cta_hi = min(static_cast<long long>(shares.total), cta_lo + kWarps * static_cast<long long>(shares.per));
  if (cta_lo >= shares.total && blockIdx.x > 0) return;  // (CTA 0 notes the sums below)
  int cta_b = 0, cta_base = 0, cur_b = 0, cur_base = 0;  // sequences of the CTA's and the warp's first tile, and the tiles in front of them
  for (int b0 = 0, front = 0; b0 < a.B; b0 += 32) {
    const int n = tiles_at(b0 + lane);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    upto += front;
    if (blockIdx.x == 0 && warp == 0 && b0 + lane < a.B) {
      a.sums[b0 + lane + 1] = upto;
      if (a.ctx[b0 + lane] != clamped(a, a.ctx[b0 + lane])) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
      for (int h = 0; n == 0 && a.near > 0 && h < a.KV; ++h) a.counts[(b0 + lane) * a.KV + h] = 0;
    }
    const int from = (upto - n) * a.KV, to = upto * a.KV;
    const uint32_t in_cta = __ballot_sync(0xffffffffu, from <= cta_lo && cta_lo < to), in_warp = __ballot_sync(0xffffffffu, from <= cta_lo + warp * shares.per && cta_lo + warp * shares.per < to);
    if (in_cta) {
      cta_b = b0 + __ffs(in_cta) - 1;
      cta_base = __shfl_sync(0xffffffffu, from, __ffs(in_cta) - 1);
    }
    if (in_warp) {
      cur_b = b0 + __ffs(in_warp) - 1;
      cur_base = __shfl_sync(0xffffffffu, from, __ffs(in_warp) - 1);
    }
    front = __shfl_sync(0xffffffffu, upto, 31);
    if (front * static_cast<long long>(a.KV) > cta_lo + warp * shares.per && blockIdx.x > 0) break;
  }
  if (blockIdx.x == 0 && tid == 0) a.sums[0] = 0;
  const int lo = min(worker * shares.per, shares.total), n_mine = min(shares.per, shares.total - lo);

  // ---- copies: lanes look up the next 32 tiles of the share at a time
  auto load = [&](int j) {
    if ((j & 31) == 0) {
      const int i = lo + j + lane;
      if (j + lane < n_mine) {
        int fk, ft, ctx = clamped(a, a.ctx[cur_b]), n = tiles_of(a, ctx, fk, ft);
        while (i >= cur_base + n * a.KV) {
          cur_base += n * a.KV;
          ++cur_b;
          ctx = clamped(a, a.ctx[cur_b]);
          n = tiles_of(a, ctx, fk, ft);
        }
        const int kvh = (i - cur_base) / n, tile = (i - cur_base) - kvh * n, key = (ft + tile) * kTile, in_page = key / a.page;
        int page = a.tables[static_cast<long long>(cur_b) * a.width + in_page];
        if (page < 0 || page >= a.pages) {
          atomicCAS(a.status, kStatusOk, kStatusBadArgs);
          page = 0;
        }
        const int from = max(0, fk - key), to = min(kTile, ctx - key);
        notes[warp][(j + lane) & 63] = make_int4((tile == 0 ? kFirst : 0) | (tile == n - 1 ? kLast : 0) | (j + lane == 0 || tile == 0 ? kOpen : 0) | (tile == n - 1 || j + lane == n_mine - 1 ? kClose : 0) |
                                                     (from > 0 || to < kTile ? kPartial : 0), cur_b * a.KV + kvh, from, to);
        spans[warp][(j + lane) & 63] = make_int2(cur_base + kvh * n, n);
        places[warp][(j + lane) & 63] = ((static_cast<long long>(page) * a.KV + kvh) * a.page + (key - in_page * a.page)) * R::kRow;
      }
      __syncwarp();
    }
    if (lane == 0) {
      const int stage = j % R::kStages;
      const long long at = places[warp][j & 63];
      const uint32_t bar = smem_u32(&bars[warp][stage]), dst = smem_u32(ring + stage * R::kStage);
      mbar_expect_tx(bar, R::kStage);
      bulk_load_1d(dst, a.k + at, R::kCopy, bar);
      bulk_load_1d(dst + R::kCopy, a.v + at, R::kCopy, bar);
    }
  };
  int issued = 0;
  for (; issued < R::kStages - 1 && issued < n_mine; ++issued) load(issued);

  // ---- the running state of a pair
  const int G = a.H / a.KV;
  uint32_t qf[NT][BLK][2][2];  // Q^T operands: block, half of a word's codes, register
  uint32_t q_sum[NT][CH];      // the sum of q over a block, as two fp16 numbers
  float factor[NT][2], to_tanh[NT][2];  // product of heads 2 t4 and 2 t4 + 1 -> exponent of two; softcap: product -> argument of tanh -> exponent
  float o[OG][OT][NT][4], om[OG][NT][4], ol[NT][4], top[NT][2];
  int pair = 0;
  bool from_start = false;
  auto open = [&](int new_pair) {
    pair = new_pair;
    const int b = pair / a.KV, kvh = pair - b * a.KV;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool real = nt * 8 + g < G;
      const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(a.q) + b * a.q_stride + (static_cast<long long>(kvh) * G + (real ? nt * 8 + g : 0)) * D;
      alignas(16) uint32_t raw[BLK][4];  // 8 numbers of every block
      uint32_t most = 0;
#pragma unroll
      for (int blk = 0; blk < BLK; ++blk) {
        *reinterpret_cast<uint4*>(raw[blk]) = *reinterpret_cast<const uint4*>(row + blk * 32 + t4 * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!real) raw[blk][i] = 0u;
          most = max(most, max(raw[blk][i] << 16 & 0x7FFF0000u, raw[blk][i] & 0x7FFF0000u));
        }
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const uint32_t e = min(max(most >> 23, 1u), 253u);
      // (a negative scale turns the queries around, so that the largest product is the largest score; one of zero must not make NaN of -inf)
      const float down = copysignf(__uint_as_float((254u - e) << 23), a.scale), up = __uint_as_float(e << 23) * fabsf(a.scale);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = __shfl_sync(0xffffffffu, up, t4 * 8 + i * 4);
        factor[nt][i] = a.softcap > 0.f ? a.softcap * kLog2e : fmaxf(f * kLog2e, 1e-37f);
        to_tanh[nt][i] = a.softcap > 0.f ? f / a.softcap : 0.f;
      }
      float sums[BLK];
#pragma unroll
      for (int blk = 0; blk < BLK; ++blk) {
        float v[8];
        sums[blk] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack_bf162(raw[blk][i]);
          v[2 * i] = f.x * down;
          v[2 * i + 1] = f.y * down;
          sums[blk] += v[2 * i] + v[2 * i + 1];
        }
        sums[blk] += __shfl_xor_sync(0xffffffffu, sums[blk], 1);
        sums[blk] += __shfl_xor_sync(0xffffffffu, sums[blk], 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // codes under the mask 0x00F0 are 16 times as large
          qf[nt][blk][h][0] = pack_h2(v[2 * h] * 0x1p14f, v[2 * h + 4] * 0x1p14f);
          qf[nt][blk][h][1] = pack_h2(v[2 * h + 1] * 0x1p10f, v[2 * h + 5] * 0x1p10f);
        }
      }
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {  // lane t's block of the chunk
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < BLK / CH; ++i) sum = t4 == i ? sums[ch * (BLK / CH) + i] : sum;  // (D = 64: lanes 2 and 3 have none)
        const float hi = __half2float(__float2half_rn(sum));
        q_sum[nt][ch] = pack_h2(hi, sum - hi);
      }
      top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) ol[nt][i] = 0.f;
#pragma unroll
      for (int og = 0; og < OG; ++og) {
#pragma unroll
        for (int i = 0; i < 4; ++i) om[og][nt][i] = 0.f;
#pragma unroll
        for (int ot = 0; ot < OT; ++ot) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[og][ot][nt][i] = 0.f;
        }
      }
    }
  };
  // word `half` (0: g, 1: g + 8) of group og as eight numbers of head 2 t4 + i, with the minima's share
  auto word_of = [&](int og, int half, int nt, int i, float* v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (D == 64) v[e] = e < 4 ? o[og][e][nt][i] + om[og][nt][i] : o[og][e - 4][nt][2 + i] + om[og][nt][2 + i];
      else v[e] = half == 0 ? o[og][e][nt][i] + om[og][nt][i] : o[og][e][nt][2 + i] + om[og][nt][2 + i];
    }
  };
  constexpr int HALVES = D == 64 ? 1 : 2;
  auto write_out = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int h = nt * 8 + 2 * t4 + i;
        if (h >= G) continue;
        const float inv = 1.f / ol[nt][i];
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (static_cast<long long>(pair) * G + h) * D;
#pragma unroll
        for (int og = 0; og < OG; ++og) {
#pragma unroll
          for (int hf = 0; hf < HALVES; ++hf) {
            float v[8];
            word_of(og, hf, nt, i, v);
            *reinterpret_cast<uint4*>(dst + og * 128 + (hf * 8 + g) * 8) =
                make_uint4(pack_bf162(v[0] * inv, v[1] * inv), pack_bf162(v[2] * inv, v[3] * inv), pack_bf162(v[4] * inv, v[5] * inv), pack_bf162(v[6] * inv, v[7] * inv));
          }
        }
      }
    }
  };
  // unnormalised rows, maximum and sum of every head: dst [G][D], ml [G][2]. Maxima pass NaN over: a NaN in the sum stands as the maximum too, so that no join takes the part for one without keys.
  auto write_part = [&](float* dst, float* ml) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int h = nt * 8 + 2 * t4 + i;
        if (h >= G) continue;
#pragma unroll
        for (int og = 0; og < OG; ++og) {
#pragma unroll
          for (int hf = 0; hf < HALVES; ++hf) {
            float v[8];
            word_of(og, hf, nt, i, v);
            float4* at = reinterpret_cast<float4*>(dst + h * D + og * 128 + (hf * 8 + g) * 8);
            at[0] = make_float4(v[0], v[1], v[2], v[3]);
            at[1] = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
        if (g == 0) {
          ml[2 * h] = ol[nt][i] == ol[nt][i] ? top[nt][i] : ol[nt][i];
          ml[2 * h + 1] = ol[nt][i];
        }
      }
    }
  };
  // do several shares of this CTA, all that it has, lie inside one pair? (every thread gets the same answer; kv4_merge_kernel asks the same)
  bool together = false;
  if (cta_hi > cta_lo) {
    const int n = tiles_at(cta_b), kvh = static_cast<int>((cta_lo - cta_base) / n);
    together = cta_hi - cta_lo > shares.per && cta_hi <= cta_base + static_cast<long long>(kvh + 1) * n;
  }

  bool ok = true;
  for (int j = 0; j < n_mine; ++j) {
    if (issued < n_mine) {
      load(issued);
      ++issued;
    }
    const int stage = j % R::kStages;
    const int flags = notes[warp][j & 63].x;
    if (flags & kOpen) {  // (in front of the wait: the queries' way from memory passes under that of the rows)
      open(notes[warp][j & 63].y);
      from_start = flags & kFirst;
    }
    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars[warp][stage]), (j / R::kStages) & 1, abort_flag, a.status));
    if (!ok) break;
    uint8_t *sk = ring + stage * R::kStage, *sv = sk + R::kCopy;
    if (flags & kPartial) {  // what stands in rows that do not count may be anything: steps and minima of zero make zeros of it
      const int live_lo = notes[warp][j & 63].z, live_hi = notes[warp][j & 63].w;
      if (lane < live_lo || lane >= live_hi) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          *reinterpret_cast<uint32_t*>(sk + lane * R::kRow + D / 2 + 4 * i) = 0u;
          *reinterpret_cast<uint32_t*>(sv + lane * R::kRow + D / 2 + 4 * i) = 0u;
        }
      }
      fence_proxy_async_smem();  // (in front of the next copy into this stage)
      __syncwarp();
    }

    // ---- scores of two times 16 keys: per block of elements the products with the codes, times its step, and the minima's share
    float s[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint8_t *r0 = sk + (mt * 16 + g) * R::kRow, *r1 = r0 + 8 * R::kRow;
      uint32_t side0[BLK], side1[BLK], low[2][CH];
      float low_s[NT][4];
      lds_words<BLK>(r0 + D / 2, side0);
      lds_words<BLK>(r1 + D / 2, side1);
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {  // (lane t has block t of every chunk: its minimum twice)
        const int blk = D == 64 ? t4 & 1 : ch * 4 + t4;
        const uint32_t m0 = *reinterpret_cast<const uint32_t*>(r0 + D / 2 + blk * 4), m1 = *reinterpret_cast<const uint32_t*>(r1 + D / 2 + blk * 4);
        low[0][ch] = __byte_perm(m0, m0, 0x3232);
        low[1][ch] = __byte_perm(m1, m1, 0x3232);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_f16_first(low_s[nt], low[0][0], low[1][0], CH == 2 ? low[0][CH - 1] : 0u, CH == 2 ? low[1][CH - 1] : 0u, q_sum[nt][0], CH == 2 ? q_sum[nt][CH - 1] : 0u);
        s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
      }
#pragma unroll
      for (int blk = 0; blk < BLK; ++blk) {
        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(r0 + blk * 16 + t4 * 4), w1 = *reinterpret_cast<const uint32_t*>(r1 + blk * 16 + t4 * 4);
        const uint32_t x0 = w0 >> 8, x1 = w1 >> 8;
        const float s0 = __half2float(__ushort_as_half(static_cast<unsigned short>(side0[blk]))), s1 = __half2float(__ushort_as_half(static_cast<unsigned short>(side1[blk])));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float c[4];
          mma_f16_first(c, w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[nt][blk][0][0], qf[nt][blk][0][1]);
          mma_f16(c, x0 & 0x000F000Fu, x1 & 0x000F000Fu, x0 & 0x00F000F0u, x1 & 0x00F000F0u, qf[nt][blk][1][0], qf[nt][blk][1][1]);
          s[mt][nt][0] = fmaf(s0, c[0], s[mt][nt][0]);
          s[mt][nt][1] = fmaf(s0, c[1], s[mt][nt][1]);
          s[mt][nt][2] = fmaf(s1, c[2], s[mt][nt][2]);
          s[mt][nt][3] = fmaf(s1, c[3], s[mt][nt][3]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[mt][nt][i] = fmaf(s[mt][nt][i], 1024.f, low_s[nt][i]);  // (codes are 2^-24 c, queries 2^14 times as large)
      }
    }
    // ---- probabilities
    if (a.softcap > 0.f) {
      float largest = 0.f;
#pragma unroll
      for (int i = 0; i < 8 * NT; ++i) {
        s[i / 4 & 1][i / 8][i & 3] *= to_tanh[i / 8][i & 1];
        largest = fmaxf(largest, fabsf(s[i / 4 & 1][i / 8][i & 3]));
      }
      // The series up to x^11 where all of the warp's arguments are below 0.35 (what it leaves out is 1.2e-8 of the value there), otherwise tanhf: 128 x 1920 keys of 256-wide heads, cap 50, in a captured stream of
      // calls, 124 us with scores of unit size, 132 with sixteen times as large ones, 119 without a cap.
      if (__all_sync(0xffffffffu, largest < 0.35f)) {
#pragma unroll
        for (int i = 0; i < 8 * NT; ++i) s[i / 4 & 1][i / 8][i & 3] = tanh_series(s[i / 4 & 1][i / 8][i & 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 8 * NT; ++i) s[i / 4 & 1][i / 8][i & 3] = tanhf(s[i / 4 & 1][i / 8][i & 3]);
      }
    }
    if (flags & kPartial) {
      const int live_lo = notes[warp][j & 63].z, live_hi = notes[warp][j & 63].w;
#pragma unroll
      for (int i = 0; i < 8 * NT; ++i) {
        const int key = (i / 4 & 1) * 16 + g + (i >> 1 & 1) * 8;
        if (key < live_lo || key >= live_hi) s[i / 4 & 1][i / 8][i & 3] = -INFINITY;
      }
    }
    uint32_t pf[2][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float most[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) most[i] = factor[nt][i] * fmaxf(fmax3(s[0][nt][i], s[0][nt][2 + i], s[1][nt][i]), s[1][nt][2 + i]);
      if (__any_sync(0xffffffffu, most[0] > top[nt][0] + kSlack || most[1] > top[nt][1] + kSlack)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], d));
          const float up = fmaxf(top[nt][i], most[i]), f = top[nt][i] == -INFINITY ? 0.f : ex2(top[nt][i] - up);
          top[nt][i] = up;
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            ol[nt][r + i] *= f;
#pragma unroll
            for (int og = 0; og < OG; ++og) {
              om[og][nt][r + i] *= f;
#pragma unroll
              for (int ot = 0; ot < OT; ++ot) o[og][ot][nt][r + i] *= f;
            }
          }
        }
      }
      const float down[2] = {kShift - top[nt][0], kShift - top[nt][1]};
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          pf[mt][nt][r] = transpose8(pack_h2(ex2(fmaf(s[mt][nt][2 * r], factor[nt][0], down[0])), ex2(fmaf(s[mt][nt][2 * r + 1], factor[nt][1], down[1]))));
      }
    }
    // ---- values
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint8_t* r0 = sv + (mt * 16 + 2 * t4) * R::kRow;  // keys 2 t4, 2 t4 + 1 and 8 behind them
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_f16(ol[nt], 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, pf[mt][nt][0], pf[mt][nt][1]);
#pragma unroll
      for (int og = 0; og < OG; ++og) {
        uint32_t lows[4], lo16[4], hi16[4];  // [half of the group's words][keys 2 t4 .. | 2 t4 + 8 ..] as a0, a1, a2, a3 take them: half + 2 * keys
        Kv4Steps steps[4] = {Kv4Steps(0u), Kv4Steps(0u), Kv4Steps(0u), Kv4Steps(0u)};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
          for (int hf = 0; hf < HALVES; ++hf) {
            const int word = og * 16 + hf * 8 + g;
            const uint8_t *ra = r0 + ks * 8 * R::kRow, *rb = ra + R::kRow;
            const uint32_t wa = *reinterpret_cast<const uint32_t*>(ra + word * 4), wb = *reinterpret_cast<const uint32_t*>(rb + word * 4);
            const uint32_t sa = *reinterpret_cast<const uint32_t*>(ra + D / 2 + (word >> 2) * 4), sb = *reinterpret_cast<const uint32_t*>(rb + D / 2 + (word >> 2) * 4);
            const int at = ks * 2 + hf;
            lo16[at] = __byte_perm(wa, wb, 0x5410);
            hi16[at] = __byte_perm(wa, wb, 0x7632);
            lows[at] = __byte_perm(sa, sb, 0x7632);
            steps[at] = Kv4Steps(__byte_perm(sa, sb, 0x5410));
          }
        }
        if constexpr (D == 64) {  // row g: codes 0..3 of word g, row g + 8: codes 4..7
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x0 = lo16[0] >> (8 * h), x1 = hi16[0] >> (8 * h), x2 = lo16[2] >> (8 * h), x3 = hi16[2] >> (8 * h);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(o[og][2 * h][nt], steps[0].low(x0), steps[0].low(x1), steps[2].low(x2), steps[2].low(x3), pf[mt][nt][0], pf[mt][nt][1]);
              mma_f16(o[og][2 * h + 1][nt], steps[0].high(x0), steps[0].high(x1), steps[2].high(x2), steps[2].high(x3), pf[mt][nt][0], pf[mt][nt][1]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(om[og][nt], lows[0], lows[0], lows[2], lows[2], pf[mt][nt][0], pf[mt][nt][1]);
        } else {
#pragma unroll
          for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t x[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) x[i] = (part ? hi16[i] : lo16[i]) >> (8 * h);
              const uint32_t a0 = steps[0].low(x[0]), a1 = steps[1].low(x[1]), a2 = steps[2].low(x[2]), a3 = steps[3].low(x[3]);
              const uint32_t b0 = steps[0].high(x[0]), b1 = steps[1].high(x[1]), b2 = steps[2].high(x[2]), b3 = steps[3].high(x[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_f16(o[og][part * 4 + 2 * h][nt], a0, a1, a2, a3, pf[mt][nt][0], pf[mt][nt][1]);
                mma_f16(o[og][part * 4 + 2 * h + 1][nt], b0, b1, b2, b3, pf[mt][nt][0], pf[mt][nt][1]);
              }
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(om[og][nt], lows[0], lows[1], lows[2], lows[3], pf[mt][nt][0], pf[mt][nt][1]);
        }
      }
    }
    __syncwarp();  // (the stage has been read)
    if (flags & kClose) {
      const bool all = from_start && (flags & kLast);
      if (all) write_out();
      long long at = worker * 2 + (from_start ? 1 : 0);
      if (a.near > 0 && (all || !together)) {
        const int2 span = spans[warp][j & 63];
        const Kv4Parts parts(shares, span.x, span.y);
        at = kv4_place(a.B * a.KV, a.near, pair, parts.number(worker), at);
        if (from_start && lane == 0) a.counts[pair] = all ? -1 : parts.parts;
      }
      if (!all && !together) write_part(a.part_o + at * G * D, a.part_ml + at * G * 2);
    }
  }
  if (!ok) {  // a wait ran out: the copies in flight land first (bounded)
    for (int j = max(0, issued - R::kStages); j < issued; ++j) {
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(smem_u32(&bars[warp][j % R::kStages]), (j / R::kStages) & 1) && globaltimer_ns() - t0 < 20000000ull) {
      }
    }
  }
  if (!together) return;
  // ---- one partial result of the whole CTA (every warp's ring is its own, and read out by now)
  float *po = reinterpret_cast<float*>(ring_all), *ml = po + kWarps * G * D;
  __syncthreads();
  if (n_mine > 0 && ok) write_part(po + warp * G * D, ml + warp * G * 2);
  else if (lane < G) {
    ml[warp * G * 2 + 2 * lane] = -INFINITY;
    ml[warp * G * 2 + 2 * lane + 1] = 0.f;
  }
  __syncthreads();
  long long slot = blockIdx.x * kWarps * 2;
  if (a.near > 0) {
    const int n = tiles_at(cta_b), kvh = static_cast<int>((cta_lo - cta_base) / n), first = cta_base + kvh * n, cta_pair = cta_b * a.KV + kvh;
    const Kv4Parts parts(shares, first, n);
    slot = kv4_place(a.B * a.KV, a.near, cta_pair, parts.number(blockIdx.x * kWarps), slot);
    if (tid == 0 && first == cta_lo) a.counts[cta_pair] = parts.parts;
  }
  for (int i = tid; i < G * (D / 4); i += kWarps * 32) {
    const int h = i / (D / 4), d = i % (D / 4) * 4;
    float up = -INFINITY, f[kWarps], sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) up = fmaxf(up, ml[(w * G + h) * 2]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float m = ml[(w * G + h) * 2];
      f[w] = m == -INFINITY ? 0.f : ex2(m - up);
      sum += f[w] * ml[(w * G + h) * 2 + 1];
      if (f[w] == 0.f) continue;
      const float4 p = *reinterpret_cast<const float4*>(po + (w * G + h) * D + d);
      v.x += f[w] * p.x;
      v.y += f[w] * p.y;
      v.z += f[w] * p.z;
      v.w += f[w] * p.w;
    }
    *reinterpret_cast<float4*>(a.part_o + slot * G * D + h * D + d) = v;
    if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * G + h) * 2) = make_float2(sum == sum ? up : sum, sum);
  }
}

// Partial results of a pair -> its heads: sum of exp2(maximum - largest) rows / the same of sums; zeros for sequences without keys. Many pairs of few parts each: a warp per pair and 256 / D heads, which fetches
// what a pair has on average while it reads how many there are (a CTA per pair and head, which looks that up first, takes 2.3 us longer: 64 x 2176 keys 46.7 -> 44.4 us, 64 x 544 22.7 -> 20.0).
template <int D>
__global__ void __launch_bounds__(128) kv4_merge_kernel(const Kv4DecodeArgs a, int workers) {
  pdl_trigger();
  constexpr int DQ = D / 4, ITEMS = 2, HEADS = ITEMS * 32 / DQ, AHEAD = kNear;
  const int G = a.H / a.KV, chunks = (G + HEADS - 1) / HEADS, unit = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, pair = unit / chunks, h0 = (unit - pair * chunks) * HEADS;
  if (pair >= a.B * a.KV) return;
  const int b = pair / a.KV, kvh = pair - b * a.KV;
  float2 ml[AHEAD][ITEMS];
  float4 x[AHEAD][ITEMS];
  auto fetch = [&](int i, long long at) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int h = h0 + (k * 32 + lane) / DQ;
      if (h < G) {
        ml[i][k] = *reinterpret_cast<const float2*>(a.part_ml + (at * G + h) * 2);
        x[i][k] = *reinterpret_cast<const float4*>(a.part_o + (at * G + h0) * D + (k * 32 + lane) * 4);
      }
    }
  };
  pdl_wait();
  const int count = a.counts[pair], before = a.sums[b], behind = a.sums[b + 1], total = a.sums[a.B];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    if (i < a.near) fetch(i, static_cast<long long>(pair) * a.near + i);  // (what is not there is not looked at)
  }
  if (count < 0) return;
  float up[ITEMS], sum[ITEMS];
  float4 v[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    up[k] = -INFINITY;
    sum[k] = 0.f;
    v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  auto add = [&](int i) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      if (h0 + (k * 32 + lane) / DQ < G && ml[i][k].x != -INFINITY) {  // (NaN goes into everything)
        const float top = fmaxf(up[k], ml[i][k].x), f = ex2(up[k] - top), w = ex2(ml[i][k].x - top);
        up[k] = top;
        sum[k] = sum[k] * f + w * ml[i][k].y;
        v[k].x = v[k].x * f + w * x[i][k].x;
        v[k].y = v[k].y * f + w * x[i][k].y;
        v[k].z = v[k].z * f + w * x[i][k].z;
        v[k].w = v[k].w * f + w * x[i][k].w;
      }
    }
  };
  const int near = min(count, a.near);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    if (i < near) add(i);
  }
  if (count > near) {
    // (a warp whose wait ran out has left no count: what stands there is anything, and the parts that there can be are the limit)
    const int n = behind - before;
    const Kv4Parts p(Kv4Shares(total * a.KV, workers), before * a.KV + kvh * n, n);
    const int most = p.most(count);
    for (int i0 = near; i0 < most; i0 += AHEAD) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (i0 + i < most) fetch(i, kv4_place(a.B * a.KV, a.near, pair, i0 + i, p.maker(i0 + i)));
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (i0 + i < most) add(i);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int h = h0 + (k * 32 + lane) / DQ;
    if (h >= G) continue;
    const float inv = count == 0 ? 0.f : 1.f / sum[k];
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (static_cast<long long>(pair) * G + h0) * D + (k * 32 + lane) * 4) =
        make_uint2(pack_bf162(v[k].x * inv, v[k].y * inv), pack_bf162(v[k].z * inv, v[k].w * inv));
  }
}

// The same for few pairs of many parts: grid (B * KV, G), D / 4 threads per group of parts. A thread's first parts are on their way while the weights are worked out (1 x 4000 keys: 9.9 us, with the other kernel 10.7).
template <int D>
__global__ void __launch_bounds__(128) kv4_merge_long_kernel(const Kv4DecodeArgs a, int workers) {
  pdl_trigger();
  constexpr int DQ = D / 4, GROUPS = 128 / DQ, MAX = kKv4MaxCtas + 2 * kWarps, AHEAD = 8;
  __shared__ float weight[MAX];
  __shared__ float red[2][4];
  __shared__ float4 acc[GROUPS][DQ];
  const int G = a.H / a.KV, pair = blockIdx.x, b = pair / a.KV, kvh = pair - b * a.KV, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const int before = a.sums[b], n = a.sums[b + 1] - before;
  const Kv4Shares shares(a.sums[a.B] * a.KV, workers);
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (static_cast<long long>(pair) * G + h) * D;
  if (n == 0) {
    for (int d = tid; d < D; d += 128) dst[d] = f2bf(0.f);
    return;
  }
  const Kv4Parts q(shares, before * a.KV + kvh * n, n);
  const int parts = q.parts;
  if (parts == 1 && !q.j0) return;  // one warp has seen the pair whole
  auto slot_of = [&](int i) { return static_cast<long long>(q.maker(i)); };
  const int group = tid / DQ, d = tid % DQ * 4;
  float4 p[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    if (group + i * GROUPS < parts) p[i] = *reinterpret_cast<const float4*>(a.part_o + (slot_of(group + i * GROUPS) * G + h) * D + d);
  }
  float up = -INFINITY, sum = 0.f, m0 = -INFINITY, l0 = 0.f;
  for (int i = tid; i < parts; i += 128) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (slot_of(i) * G + h) * 2);
    weight[i] = ml.x;
    if (ml.x > m0) {  // (this thread's own sums, relative to their maximum)
      l0 *= ex2(m0 - ml.x);
      m0 = ml.x;
    }
    if (ml.x > -INFINITY) l0 += ml.y * ex2(ml.x - m0);
  }
  up = warp_max(m0);
  if (lane == 0) red[0][warp] = up;
  __syncthreads();
  up = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  sum = warp_sum(m0 > -INFINITY ? l0 * ex2(m0 - up) : 0.f);
  if (lane == 0) red[1][warp] = sum;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](int i, const float4& x) {
    const float w = ex2(weight[i] - up);
    v.x = fmaf(w, x.x, v.x);
    v.y = fmaf(w, x.y, v.y);
    v.z = fmaf(w, x.z, v.z);
    v.w = fmaf(w, x.w, v.w);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    if (group + i * GROUPS < parts) add(group + i * GROUPS, p[i]);
  }
#pragma unroll 4
  for (int i = group + AHEAD * GROUPS; i < parts; i += GROUPS) add(i, *reinterpret_cast<const float4*>(a.part_o + (slot_of(i) * G + h) * D + d));
  acc[group][tid % DQ] = v;
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    const float4 x = acc[i][tid];
    v.x += x.x;
    v.y += x.y;
    v.z += x.z;
    v.w += x.w;
  }
  const float inv = 1.f / (red[1][0] + red[1][1] + red[1][2] + red[1][3]);
  *reinterpret_cast<uint2*>(dst + d) = make_uint2(pack_bf162(v.x * inv, v.y * inv), pack_bf162(v.z * inv, v.w * inv));
}

template <int D, int NT>
static void launch_decode_t(const Kv4DecodeArgs& a, int ctas, cudaStream_t st) {
  using R = Kv4Ring<D, NT>;
  static PerDeviceOnce once;
  if (once.first()) cudaFuncSetAttribute(kv4_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, R::kBytes);
  launch_pdl(kv4_decode_kernel<D, NT>, dim3(ctas), dim3(kWarps * 32), R::kBytes, st, a);
  const int G = a.H / a.KV, pairs = a.B * a.KV, units = pairs * ((G * D + 255) / 256);
  if (a.near > 0) launch_pdl(kv4_merge_kernel<D>, dim3((units + 3) / 4), dim3(128), 0, st, a, ctas * kWarps);
  else launch_pdl(kv4_merge_long_kernel<D>, dim3(pairs, G), dim3(128), 0, st, a, ctas * kWarps);
}

int kv4_decode_ctas(int B, int KV, int G, int D, long long rows, int sms) {
  const int per_sm[3][2] = {{Kv4Ring<64, 1>::kCtas, Kv4Ring<64, 2>::kCtas}, {Kv4Ring<128, 1>::kCtas, Kv4Ring<128, 2>::kCtas}, {Kv4Ring<256, 1>::kCtas, Kv4Ring<256, 2>::kCtas}};
  const int room = sms * per_sm[D == 64 ? 0 : D == 128 ? 1 : 2][G > 8];
  const long long most = (static_cast<long long>(B) * KV * ((rows + kTile - 1) / kTile) + kWarps * kMinTiles - 1) / (kWarps * kMinTiles);
  const int ctas = room < kKv4MaxCtas ? room : kKv4MaxCtas;
  return most < ctas ? static_cast<int>(most < 1 ? 1 : most) : ctas;
}
// As many as a pair has on average, and one at either end (what is fetched for nothing costs as much as the rest); 0 where that is too many, and a pair is worth more than a warp.
int kv4_decode_near(int ctas, int pairs) {
  const int n = ctas * kWarps / pairs + 2;
  return n <= kNear ? n : 0;
}

void launch_kv4_decode(const Kv4DecodeArgs& a, int ctas, cudaStream_t st) {
  const bool two = a.H / a.KV > 8;
  if (a.D == 64) two ? launch_decode_t<64, 2>(a, ctas, st) : launch_decode_t<64, 1>(a, ctas, st);
  else if (a.D == 128) two ? launch_decode_t<128, 2>(a, ctas, st) : launch_decode_t<128, 1>(a, ctas, st);
  else two ? launch_decode_t<256, 2>(a, ctas, st) : launch_decode_t<256, 1>(a, ctas, st);
}

}  // namespace dlv
