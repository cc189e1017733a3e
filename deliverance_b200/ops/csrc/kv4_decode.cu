// Decode attention over a KV cache in 4 bits (format: kv4.cuh).
//
// What bounds it: the rows of the cache, 5 bits a number, and right behind them the instructions that unpack them. At the copy rate an SM gets 22 bytes a cycle, 35 numbers, for its 128 lanes: 3.6
// lane instructions per number for everything. So numbers are unpacked in pairs, straight into the registers of tensor-core operands, by one mask and one fp16 FMA per pair:
//   a code c under the mask 0x000f is the fp16 number 1024 + c, under 0x00f0 it is 1024 + 16 c;  c s = (1024 + c) s - 1024 s = (1024 + 16 c) (s / 16) - 64 s,
// one FMA each, and exact, because s has 7 bits. The minima stay out of it: q . (c s + m) = q . c s + sum over blocks of m (sum of q in the block), one more matrix product with one column per block,
// and sum p (c s + m) = sum p c s + (sum p m), one more with one row per word of codes.
//
// Products are mma.sync m16n8k16 in fp16 with the cache as the 16-row operand and the (up to 8) query heads of a KV head as the 8 columns (two such column tiles for 9 to 16 heads): with heads as rows half
// of every product would be wasted on groups of 4 or 8, and so would the exponentials. Scores S^T [keys x heads] = K Q^T, O^T [D x heads] = V^T P^T.
//   K operand: row = key, k = elements; which element stands at which k is free as long as Q agrees. Lane (g, t) = (lane / 4, lane % 4) takes 16 neighbouring bytes of key g's codes, so that they have one step.
//   V operand: row = element, k = keys; lane (g, t) takes the words (8 codes) g and g + 8 of keys 2 t and 2 t + 1, put side by side by two byte permutes per word pair; row g of product i is code i of word g.
//   P^T: a score tile transposed by movmatrix.
// Queries are divided by the power of two that brings a head's largest number to [1, 2): bf16's range fits fp16 then. Probabilities are held 2^12 times as large and relative to a maximum that follows when a
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
constexpr int kWarps = 4;
constexpr int kMinTiles = 2;   // of a share
constexpr float kShift = 12.f, kSlack = 3.f;
constexpr float kLog2e = 1.44269504088896341f;

template <int D, int NT>
struct Kv4Ring {
  static constexpr int kRow = kv4_row_bytes(D), kCopy = kTile * kRow, kStage = 2 * kCopy;
  static constexpr int kStages = D == 64 ? 4 : D == 128 ? 3 : 2;
  static constexpr int kCtas = (D == 64 ? 4 : D == 128 ? 3 : 2) - (NT - 1);  // per SM, as registers allow
  static constexpr int kBytes = kWarps * kStages * kStage;
};

// A share of the tiles: tile i of the step belongs to warp i / per.
struct Kv4Shares {
  int total, per;
  __device__ Kv4Shares(int total_, int workers) : total(total_), per(max(kMinTiles, (total_ + workers - 1) / workers)) {}
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
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
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
  pdl_wait();
  using R = Kv4Ring<D, NT>;
  constexpr int CH = D == 256 ? 2 : 1;          // chunks of codes that a lane takes of a key
  constexpr int CW = D == 64 ? 2 : 4;           // words of a chunk
  constexpr int OG = D == 256 ? 2 : 1;          // groups of 16 words of a row (D = 64: 8 words, both halves of them)
  constexpr int OT = D == 64 ? 4 : 8;           // products per group
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ __align__(8) uint64_t bars[kWarps][R::kStages];
  __shared__ int4 notes[kWarps][64];  // of the tiles that are copied and those to come: pair, first key of the tile, length, flags (1: the pair's first tile, 2: its last)
  __shared__ long long places[kWarps][64];  // where their rows lie in the caches
  __shared__ int scan[kWarps], begin[kWarps][2], sum_all, abort_word;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  volatile int* abort_flag = &abort_word;
  uint8_t* ring = ring_all + warp * R::kStages * R::kStage;
  if (tid == 0) {
    abort_word = 0;
    sum_all = 0;
  }
  if (lane < R::kStages) mbar_init(smem_u32(&bars[warp][lane]), 1);
  mbar_fence_init();
  __syncthreads();

  // ---- where this warp's share begins
  int mine = 0;
  for (int b = tid; b < a.B; b += kWarps * 32) {
    const int given = a.ctx[b], ctx = clamped(a, given);
    if (given != ctx) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
    int fk, ft;
    mine += tiles_of(a, ctx, fk, ft);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) atomicAdd(&sum_all, mine);
  __syncthreads();
  const Kv4Shares shares(sum_all * a.KV, static_cast<int>(gridDim.x) * kWarps);
  const int worker = blockIdx.x * kWarps + warp;
  if (static_cast<long long>(blockIdx.x) * kWarps * shares.per >= shares.total && blockIdx.x > 0) return;  // (CTA 0 notes the sums below)
  for (int b0 = 0, front = 0; b0 < a.B; b0 += kWarps * 32) {
    const int b = b0 + tid;
    int fk, ft;
    const int n = b < a.B ? tiles_of(a, clamped(a, a.ctx[b]), fk, ft) : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) upto += scan[w];
    }
    upto += front;
    if (blockIdx.x == 0 && b < a.B) {
      a.sums[b + 1] = upto;
      if (b == 0) a.sums[0] = 0;
    }
    const long long from = static_cast<long long>(upto - n) * a.KV, to = static_cast<long long>(upto) * a.KV;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const long long lo = static_cast<long long>(blockIdx.x * kWarps + w) * shares.per;
      if (from <= lo && lo < to) {
        begin[w][0] = b;
        begin[w][1] = static_cast<int>(from);
      }
    }
    front += scan[0] + scan[1] + scan[2] + scan[3];
    __syncthreads();
  }
  const int lo = min(worker * shares.per, shares.total), n_mine = min(shares.per, shares.total - lo);

  // ---- copies: lanes look up the next 32 tiles of the share at a time
  int cur_b = 0, cur_base = 0;
  if (n_mine > 0) {
    cur_b = begin[warp][0];
    cur_base = begin[warp][1];
  }
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
        notes[warp][(j + lane) & 63] = make_int4(cur_b * a.KV + kvh, key, ctx, (tile == 0 ? 1 : 0) | (tile == n - 1 ? 2 : 0));
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
  uint32_t qf[NT][CH][CW][2][2];  // Q^T operands: word, half of its codes, register
  uint32_t q_sum[NT][CH];         // a lane's part of the sums of q, as two fp16 numbers
  float factor[NT][2];            // score of heads 2 t4 and 2 t4 + 1 -> exponent of two (softcap: -> argument of tanh)
  float o[OG][OT][NT][4], om[OG][NT][4], ol[NT][4], top[NT][2];
  int pair = -1;
  bool from_start = false;
  auto open = [&](int new_pair) {
    pair = new_pair;
    const int b = pair / a.KV, kvh = pair - b * a.KV;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool real = nt * 8 + g < G;
      const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(a.q) + b * a.q_stride + (static_cast<long long>(kvh) * G + (real ? nt * 8 + g : 0)) * D;
      alignas(16) uint32_t raw[CH][CW * 4];
      uint32_t most = 0;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
#pragma unroll
        for (int i = 0; i < CW * 4; ++i) {
          if (i % 4 == 0) *reinterpret_cast<uint4*>(&raw[ch][i]) = *reinterpret_cast<const uint4*>(row + ch * 128 + t4 * CW * 8 + 2 * i);
          if (!real) raw[ch][i] = 0u;
          most = max(most, max(raw[ch][i] << 16 & 0x7FFF0000u, raw[ch][i] & 0x7FFF0000u));
        }
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const uint32_t e = min(max(most >> 23, 1u), 253u);
      const float down = __uint_as_float((254u - e) << 23), up = __uint_as_float(e << 23) * (a.softcap > 0.f ? a.scale / a.softcap : a.scale * kLog2e);
#pragma unroll
      for (int i = 0; i < 2; ++i) factor[nt][i] = __shfl_sync(0xffffffffu, up, t4 * 8 + i * 4);
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < CW; ++w) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_bf162(raw[ch][w * 4 + i]);
            v[2 * i] = f.x * down;
            v[2 * i + 1] = f.y * down;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            qf[nt][ch][w][h][0] = pack_h2(v[2 * h], v[2 * h + 4]);
            qf[nt][ch][w][h][1] = pack_h2(v[2 * h + 1], v[2 * h + 5]);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qf[nt][ch][w][h][r]));
              sum += f.x + f.y;
            }
          }
        }
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
  // unnormalised rows, maximum and sum of every head: dst [G][D], ml [G][2]
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
          ml[2 * h] = top[nt][i];
          ml[2 * h + 1] = ol[nt][i];
        }
      }
    }
  };
  // do several shares of this CTA, all that it has, lie inside one pair? (every thread gets the same answer; kv4_merge_kernel asks the same)
  const long long cta_lo = static_cast<long long>(blockIdx.x) * kWarps * shares.per, cta_hi = min(static_cast<long long>(shares.total), cta_lo + kWarps * static_cast<long long>(shares.per));
  bool together = false;
  if (cta_hi > cta_lo) {
    const int b = begin[0][0], base = begin[0][1];
    int fk, ft;
    const int n = tiles_of(a, clamped(a, a.ctx[b]), fk, ft), kvh = static_cast<int>((cta_lo - base) / n);
    together = cta_hi - cta_lo > shares.per && cta_hi <= base + static_cast<long long>(kvh + 1) * n;
  }

  bool ok = true;
  for (int j = 0; j < n_mine; ++j) {
    if (issued < n_mine) {
      load(issued);
      ++issued;
    }
    const int stage = j % R::kStages;
    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars[warp][stage]), (j / R::kStages) & 1, abort_flag, a.status));
    if (!ok) break;
    const int4 note = notes[warp][j & 63];
    if (note.x != pair) {
      open(note.x);
      from_start = note.w & 1;
    }
    uint8_t *sk = ring + stage * R::kStage, *sv = sk + R::kCopy;
    const int first_key = a.window > 0 && note.z > a.window ? note.z - a.window : 0;
    const int live_lo = first_key - note.y, live_hi = note.z - note.y;  // keys of the tile that count
    const bool whole = live_lo <= 0 && live_hi >= kTile;
    if (!whole) {  // what stands in rows that do not count may be anything: steps and minima of zero make zeros of it
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

    // ---- scores of two times 16 keys
    float s[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint8_t *r0 = sk + (mt * 16 + g) * R::kRow, *r1 = r0 + 8 * R::kRow;
      uint32_t low[2][CH];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        uint32_t w0[4], w1[4];
        if constexpr (D == 64) {
          const uint2 u0 = *reinterpret_cast<const uint2*>(r0 + t4 * 8), u1 = *reinterpret_cast<const uint2*>(r1 + t4 * 8);
          w0[0] = u0.x; w0[1] = u0.y;
          w1[0] = u1.x; w1[1] = u1.y;
        } else {
          const uint4 u0 = *reinterpret_cast<const uint4*>(r0 + ch * 64 + t4 * 16), u1 = *reinterpret_cast<const uint4*>(r1 + ch * 64 + t4 * 16);
          w0[0] = u0.x; w0[1] = u0.y; w0[2] = u0.z; w0[3] = u0.w;
          w1[0] = u1.x; w1[1] = u1.y; w1[2] = u1.z; w1[3] = u1.w;
        }
        const int blk = D == 64 ? t4 >> 1 : ch * 4 + t4;
        const uint32_t side0 = *reinterpret_cast<const uint32_t*>(r0 + D / 2 + blk * 4), side1 = *reinterpret_cast<const uint32_t*>(r1 + D / 2 + blk * 4);
        const Kv4Steps k0(__byte_perm(side0, side0, 0x1010)), k1(__byte_perm(side1, side1, 0x1010));
        low[0][ch] = __byte_perm(side0, side0, 0x3232);
        low[1][ch] = __byte_perm(side1, side1, 0x3232);
#pragma unroll
        for (int w = 0; w < CW; ++w) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x0 = h ? w0[w] >> 8 : w0[w], x1 = h ? w1[w] >> 8 : w1[w];
            const uint32_t a0 = k0.low(x0), a1 = k1.low(x1), a2 = k0.high(x0), a3 = k1.high(x1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(s[mt][nt], a0, a1, a2, a3, qf[nt][ch][w][h][0], qf[nt][ch][w][h][1]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        mma_f16(s[mt][nt], low[0][0], low[1][0], CH == 2 ? low[0][CH - 1] : 0u, CH == 2 ? low[1][CH - 1] : 0u, q_sum[nt][0], CH == 2 ? q_sum[nt][CH - 1] : 0u);
    }
    // ---- probabilities
#pragma unroll
    for (int i = 0; i < 8 * NT; ++i) s[i / 4 & 1][i / 8][i & 3] *= factor[i / 8][i & 1];
    if (a.softcap > 0.f) {
#pragma unroll
      for (int i = 0; i < 8 * NT; ++i) s[i / 4 & 1][i / 8][i & 3] = tanhf(s[i / 4 & 1][i / 8][i & 3]) * (a.softcap * kLog2e);
    }
    if (!whole) {
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
      for (int i = 0; i < 2; ++i) most[i] = fmaxf(fmaxf(s[0][nt][i], s[0][nt][2 + i]), fmaxf(s[1][nt][i], s[1][nt][2 + i]));
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
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          pf[mt][nt][r] = transpose8(pack_h2(ex2(s[mt][nt][2 * r] - (top[nt][0] - kShift)), ex2(s[mt][nt][2 * r + 1] - (top[nt][1] - kShift))));
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
    const bool end = note.w & 2;
    if (from_start && end) write_out();
    else if ((end || j == n_mine - 1) && !together) {
      const long long slot = static_cast<long long>(worker) * 2 + (from_start ? 1 : 0);
      write_part(a.part_o + slot * G * D, a.part_ml + slot * G * 2);
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
  const long long slot = static_cast<long long>(blockIdx.x) * kWarps * 2;
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
    if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * G + h) * 2) = make_float2(up, sum);
  }
}

// Partial results of a pair -> its heads: sum of exp2(maximum - largest) rows / the same of sums. grid (B * KV, G), D / 4 threads per group of parts. Pairs that one warp has seen whole are finished, those of
// sequences without keys get zeros.
template <int D>
__global__ void __launch_bounds__(128) kv4_merge_kernel(const Kv4DecodeArgs a, int workers) {
  pdl_trigger();
  pdl_wait();
  constexpr int DQ = D / 4, GROUPS = 128 / DQ, MAX = kKv4MaxCtas + 2 * kWarps;
  __shared__ float weight[MAX];
  __shared__ float red[8];
  __shared__ float4 acc[GROUPS][DQ];
  const int G = a.H / a.KV, pair = blockIdx.x, b = pair / a.KV, kvh = pair - b * a.KV, h = blockIdx.y, tid = threadIdx.x;
  const Kv4Shares shares(a.sums[a.B] * a.KV, workers);
  const int before = a.sums[b], n = a.sums[b + 1] - before, first = before * a.KV + kvh * n, last = first + n - 1, per = shares.per, cta = kWarps * per;
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (static_cast<long long>(pair) * G + h) * D;
  if (n == 0) {
    for (int d = tid; d < D; d += 128) dst[d] = f2bf(0.f);
    return;
  }
  const int w0 = first / per, w1 = last / per, c0 = first / cta, c1 = last / cta;
  if (w0 == w1) return;
  auto joined = [&](int c) {  // the CTA's shares are one part
    const int lo = c * cta, hi = min(shares.total, lo + cta);
    return hi - lo > per && first <= lo && hi <= last + 1;
  };
  // parts in order: of the first CTA, one of each in the middle, of the last
  const bool j0 = joined(c0), j1 = joined(c1);
  const int n0 = j0 ? 1 : min(w1, c0 * kWarps + kWarps - 1) - w0 + 1, mid = max(0, c1 - c0 - 1), n1 = c1 == c0 ? 0 : j1 ? 1 : w1 - c1 * kWarps + 1, parts = n0 + mid + n1;
  auto slot_of = [&](int i) {
    int w;
    bool own = false;  // a warp's own part
    if (i < n0) {
      w = j0 ? c0 * kWarps : w0 + i;
      own = !j0;
    } else if (i < n0 + mid) {
      w = (c0 + 1 + i - n0) * kWarps;
    } else {
      w = c1 * kWarps + (i - n0 - mid);
      own = !j1;
    }
    return static_cast<long long>(w) * 2 + (own && first >= w * per ? 1 : 0);
  };
  float up = -INFINITY, sum = 0.f;
  for (int i = tid; i < parts; i += 128) {
    weight[i] = a.part_ml[(slot_of(i) * G + h) * 2];
    up = fmaxf(up, weight[i]);
  }
  up = block_max(up, red);
  for (int i = tid; i < parts; i += 128) {
    weight[i] = weight[i] == -INFINITY ? 0.f : ex2(weight[i] - up);
    sum += weight[i] * a.part_ml[(slot_of(i) * G + h) * 2 + 1];
  }
  sum = block_sum(sum, red);
  const int group = tid / DQ, d = tid % DQ * 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = group; i < parts; i += GROUPS) {
    const float4 p = *reinterpret_cast<const float4*>(a.part_o + (slot_of(i) * G + h) * D + d);
    const float w = weight[i];
    v.x += w * p.x;
    v.y += w * p.y;
    v.z += w * p.z;
    v.w += w * p.w;
  }
  acc[group][tid % DQ] = v;
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    const float4 p = acc[i][tid];
    v.x += p.x;
    v.y += p.y;
    v.z += p.z;
    v.w += p.w;
  }
  const float inv = 1.f / sum;
  *reinterpret_cast<uint2*>(dst + d) = make_uint2(pack_bf162(v.x * inv, v.y * inv), pack_bf162(v.z * inv, v.w * inv));
}

template <int D, int NT>
static void launch_decode_t(const Kv4DecodeArgs& a, int ctas, cudaStream_t st) {
  using R = Kv4Ring<D, NT>;
  static PerDeviceOnce once;
  if (once.first()) cudaFuncSetAttribute(kv4_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, R::kBytes);
  launch_pdl(kv4_decode_kernel<D, NT>, dim3(ctas), dim3(kWarps * 32), R::kBytes, st, a);
  launch_pdl(kv4_merge_kernel<D>, dim3(a.B * a.KV, a.H / a.KV), dim3(128), 0, st, a, ctas * kWarps);
}

int kv4_decode_ctas(int B, int KV, int G, int D, long long rows, int sms) {
  const int per_sm[3][2] = {{Kv4Ring<64, 1>::kCtas, Kv4Ring<64, 2>::kCtas}, {Kv4Ring<128, 1>::kCtas, Kv4Ring<128, 2>::kCtas}, {Kv4Ring<256, 1>::kCtas, Kv4Ring<256, 2>::kCtas}};
  const int room = sms * per_sm[D == 64 ? 0 : D == 128 ? 1 : 2][G > 8];
  const long long most = (static_cast<long long>(B) * KV * ((rows + kTile - 1) / kTile) + kWarps * kMinTiles - 1) / (kWarps * kMinTiles);
  const int ctas = room < kKv4MaxCtas ? room : kKv4MaxCtas;
  return most < ctas ? static_cast<int>(most < 1 ? 1 : most) : ctas;
}
long long kv4_decode_room(int ctas, int G, int D) { return static_cast<long long>(ctas) * kWarps * 2 * G * (D + 2); }

void launch_kv4_decode(const Kv4DecodeArgs& a, int ctas, cudaStream_t st) {
  const bool two = a.H / a.KV > 8;
  if (a.D == 64) two ? launch_decode_t<64, 2>(a, ctas, st) : launch_decode_t<64, 1>(a, ctas, st);
  else if (a.D == 128) two ? launch_decode_t<128, 2>(a, ctas, st) : launch_decode_t<128, 1>(a, ctas, st);
  else two ? launch_decode_t<256, 2>(a, ctas, st) : launch_decode_t<256, 1>(a, ctas, st);
}

}  // namespace dlv
