// Beam search: selection over beams and vocabulary, and the moves of beam states that follow it.
//
// Selection: value[w, v] = scores[w] + z[w, v] - log sum_u exp z[w, u], the K largest finite ones of a request's W rows, ties to the lowest w * V + v.
// The order inside a row is the order of the raw logits (soft-capping and positive scaling are monotone), so rows are cut into splits that each keep
// their K best logits, their maximum and their sum of exponentials from one pass; a second kernel compares the candidates of all rows in 64 bits.
// What bounds it: the logits, read once.
#include <cfloat>

#include "beam_api.h"
#include "common.cuh"

namespace dlv {

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 16;                   // logits per thread and tile
constexpr int kTile = kThreads * kPerThread;     // logits per tile
constexpr int kSoft = 512;                       // the list is cut back to K when it is longer than this behind a tile
constexpr int kList = kSoft + kTile;             // so that a whole tile always fits
constexpr int kShort = kThreads;                 // candidates that are put in order by counting

// larger key = better candidate: the logit's order, then the lower token
__device__ __forceinline__ uint32_t float_order(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float float_from_order(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ unsigned long long candidate_key(float x, int i) {
  return (static_cast<unsigned long long>(float_order(x + 0.f)) << 32) | (0xffffffffu - static_cast<uint32_t>(i));  // (-0 and 0 are equal)
}
__device__ __forceinline__ float key_logit(unsigned long long k) { return float_from_order(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int key_token(unsigned long long k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }

// (-inf is a masked token and stays one)
__device__ __forceinline__ float post(float x, float softcap, float inv_scale) {
  x *= inv_scale;
  return softcap > 0.f && x > -INFINITY ? softcap * tanhf(x / softcap) : x;
}

template <typename T>
struct Vec {
  static constexpr int N = 16 / static_cast<int>(sizeof(T));
};
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[4]) {
  x[0] = __uint_as_float(u.x);
  x[1] = __uint_as_float(u.y);
  x[2] = __uint_as_float(u.z);
  x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[8]) {
  const float2 a = unpack_bf162(u.x), b = unpack_bf162(u.y), c = unpack_bf162(u.z), d = unpack_bf162(u.w);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return bf2f(v); }

struct SelectShared {
  unsigned long long list[kList];
  unsigned long long shorter[kShort];
  unsigned long long group[64];
  unsigned long long edge;
  double sum[kThreads / 32];
  float max[kThreads / 32];
  int count, n_short;
};

// K-th largest of the 64 group maxima (a group: four neighbouring threads): K entries of the list at least are not below it. All keys of a thread are
// 0 where it has none.
__device__ __forceinline__ unsigned long long group_edge(SelectShared& sh, unsigned long long best, int K) {
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
    best = other > best ? other : best;
  }
  const int t = threadIdx.x;
  if ((t & 3) == 0) sh.group[t >> 2] = best;
  __syncthreads();
  if (t < 64) {
    const unsigned long long mine = sh.group[t];
    int rank = 0;
#pragma unroll 8
    for (int u = 0; u < 64; ++u) {
      const unsigned long long other = sh.group[u];
      rank += other > mine || (other == mine && u < t) ? 1 : 0;  // (equal only where groups are empty)
    }
    if (rank == K - 1) sh.edge = mine;
  }
  __syncthreads();
  return sh.edge;
}

// Cuts the list back to its K best, in order. Returns how many there are.
__device__ int cut_list(SelectShared& sh, int K) {
  const int t = threadIdx.x, n = sh.count;
  if (t == 0) sh.n_short = 0;
  unsigned long long edge = 0;
  if (n > kShort) {
    unsigned long long best = 0;
    for (int i = t; i < n; i += kThreads) best = sh.list[i] > best ? sh.list[i] : best;
    edge = group_edge(sh, best, K);
    int above = 0;
    for (int i = t; i < n; i += kThreads) above += sh.list[i] >= edge ? 1 : 0;
    // (a list in an unlucky order: many entries above the edge; keys differ, so a search over the bits finds the K-th largest itself)
    int rough = 0;
    for (int b = 0; b < 5; ++b) rough += __syncthreads_count((above >> b) & 1) << b;
    if (rough > kShort) {
      edge = 0;
      for (int b = 63; b >= 0; --b) {
        const unsigned long long probe = edge | (1ull << b);
        int c = 0, total = 0;
        for (int i = t; i < n; i += kThreads) c += sh.list[i] >= probe ? 1 : 0;
        for (int q = 0; q < 5; ++q) total += __syncthreads_count((c >> q) & 1) << q;
        if (total >= K) edge = probe;
      }
    }
  }
  __syncthreads();
  for (int i = t; i < n; i += kThreads)
    if (sh.list[i] >= edge) sh.shorter[atomicAdd(&sh.n_short, 1)] = sh.list[i];
  __syncthreads();
  const int m = sh.n_short;
  if (t < m) {
    const unsigned long long mine = sh.shorter[t];
    int rank = 0;
    for (int u = 0; u < m; ++u) rank += sh.shorter[u] > mine ? 1 : 0;
    if (rank < K) sh.list[rank] = mine;
  }
  const int left = min(m, K);
  if (t == 0) sh.count = left;
  __syncthreads();
  return left;
}

// grid: B * W * splits. A thread reads 16 logits of a tile in groups of 16 bytes (one by one where the row does not start on 16 bytes: the same logits in the
// same thread, so that equal rows have equal sums and their candidates tie), keeps a running maximum and sum, and lists what beats the K-th best found so far.
// Later tiles hold higher tokens, so an equal logit never does.
template <typename T, bool MASK>
__global__ void __launch_bounds__(kThreads) beam_part_kernel(const __grid_constant__ BeamSelectArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ SelectShared sh;
  constexpr int N = Vec<T>::N, NV = kPerThread / N;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, K = a.K;
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const int lo = min(a.V, split * a.per), hi = min(a.V, lo + a.per);
  const T* x_row = static_cast<const T*>(a.logits) + static_cast<long long>(row) * a.ld;
  const uint32_t* bits = MASK ? a.mask + static_cast<long long>(row) * a.mask_ld : nullptr;
  const bool whole = (reinterpret_cast<uintptr_t>(x_row) & 15) == 0;  // (splits start at multiples of 64 logits)
  const bool plain = a.softcap <= 0.f && a.inv_scale == 1.f;
  if (t == 0) sh.count = 0;
  float m = -FLT_MAX, edge = -INFINITY;
  double sum = 0.0;
  bool first = true;
  __syncthreads();
  for (int at = lo; at < hi; at += kTile) {
    float x[NV][N];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = at + (v * kThreads + t) * N;
      if (i + N <= hi) {
        if (whole) {
          unpack(__ldg(reinterpret_cast<const uint4*>(x_row + i)), x[v]);
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) x[v][e] = to_float(__ldg(x_row + i + e));
        }
        if constexpr (MASK) {
          const uint32_t word = bits[i >> 5] >> (i & 31);
#pragma unroll
          for (int e = 0; e < N; ++e) x[v][e] = (word >> e) & 1u ? x[v][e] : -INFINITY;
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          x[v][e] = -INFINITY;
          if (i + e < hi && (!MASK || ((bits[(i + e) >> 5] >> ((i + e) & 31)) & 1u))) x[v][e] = to_float(x_row[i + e]);
        }
      }
    }
    // maximum and sum of exponentials (NaN and +inf make the sum NaN: such a row has no candidates)
    float top = -INFINITY, top_z;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) top = fmaxf(top, x[j / N][j % N]);
    top_z = plain ? top : post(top, a.softcap, a.inv_scale);
    if (top_z > m) {
      sum *= static_cast<double>(expf(m - top_z));
      m = top_z;
    }
    float part = 0.f;
    if (plain) {
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) part += expf(x[j / N][j % N] - m);
    } else {
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) part += expf(post(x[j / N][j % N], a.softcap, a.inv_scale) - m);
    }
    sum += static_cast<double>(part);
    // candidates
    unsigned long long least = 0;
    if (first) {
      first = false;
      unsigned long long best = 0;
#pragma unroll
      for (int v = NV - 1; v >= 0; --v) {
#pragma unroll
        for (int e = N - 1; e >= 0; --e) {
          const float y = x[v][e];
          if (y > -INFINITY) {
            const unsigned long long k = candidate_key(y, at + (v * kThreads + t) * N + e);
            best = k > best ? k : best;
          }
        }
      }
      least = group_edge(sh, best, K);
    }
    bool over = false;
    if (top > edge) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float y = x[v][e];
          if (y > edge) {
            const unsigned long long k = candidate_key(y, at + (v * kThreads + t) * N + e);
            if (k >= least) {
              const int p = atomicAdd(&sh.count, 1);
              sh.list[p] = k;
              over = over || p >= kSoft;
            }
          }
        }
      }
    }
    if (__syncthreads_or(over)) {
      cut_list(sh, K);
      edge = key_logit(sh.list[K - 1]);
    } else if (least != 0) {
      edge = key_logit(least);
    }
  }
  const int n = cut_list(sh, K);
  const long long out = static_cast<long long>(blockIdx.x) * K;
  if (t < K) {
    a.cand_x[out + t] = t < n ? key_logit(sh.list[t]) : -INFINITY;
    a.cand_i[out + t] = t < n ? key_token(sh.list[t]) : 0;
  }
  // the split's maximum and sum, threads in a fixed order
  const float wm = warp_max(m);
  sum *= static_cast<double>(expf(m - wm));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) {
    sh.max[warp] = wm;
    sh.sum[warp] = sum;
  }
  __syncthreads();
  if (t == 0) {
    float top = sh.max[0];
    for (int w = 1; w < kThreads / 32; ++w) top = fmaxf(top, sh.max[w]);
    double total = 0.0;
    for (int w = 0; w < kThreads / 32; ++w) total += sh.sum[w] * static_cast<double>(expf(sh.max[w] - top));
    a.part_m[blockIdx.x] = top;
    a.part_sum[blockIdx.x] = total;
  }
}

__device__ __forceinline__ unsigned long long double_order(double v) {
  const long long u = __double_as_longlong(v);
  return u < 0 ? ~static_cast<unsigned long long>(u) : static_cast<unsigned long long>(u) | 0x8000000000000000ull;
}
__device__ __forceinline__ double double_from_order(unsigned long long o) {
  return __longlong_as_double(static_cast<long long>(o & 0x8000000000000000ull ? o ^ 0x8000000000000000ull : ~o));
}

// best (largest value, lowest place) of a warp: every lane gets it; value 0: none
__device__ __forceinline__ void warp_best(unsigned long long& value, uint32_t& place) {
  const uint32_t hi = static_cast<uint32_t>(value >> 32), top = __reduce_max_sync(0xffffffffu, hi);
  const uint32_t lo = hi == top ? static_cast<uint32_t>(value) : 0u, low = __reduce_max_sync(0xffffffffu, lo);
  place = __reduce_min_sync(0xffffffffu, hi == top && static_cast<uint32_t>(value) == low ? place : 0xffffffffu);
  value = (static_cast<unsigned long long>(top) << 32) | low;
}

// one CTA per request: W * splits * K <= 8 * NT candidates in registers, K rounds of "take the best"
template <int NT>
__global__ void __launch_bounds__(NT) beam_merge_kernel(const __grid_constant__ BeamSelectArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int PER = kBeamMaxMerge / 1024, NW = NT / 32;
  __shared__ double base[kBeamMaxBeams];
  __shared__ float top[kBeamMaxBeams];
  __shared__ unsigned long long best_value[2][NW];
  __shared__ uint32_t best_place[2][NW];
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int S = a.splits, K = a.K, W = a.W, n = W * S * K;
  for (int w = warp; w < W; w += NW) {
    const long long at = (static_cast<long long>(b) * W + w) * S;
    float m = -FLT_MAX;
    for (int s = lane; s < S; s += 32) m = fmaxf(m, a.part_m[at + s]);
    m = warp_max(m);
    double sum = 0.0;
    for (int s = lane; s < S; s += 32) sum += a.part_sum[at + s] * exp(static_cast<double>(a.part_m[at + s]) - static_cast<double>(m));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      top[w] = m;
      base[w] = static_cast<double>(a.scores[static_cast<long long>(b) * W + w]) - log(sum);
    }
  }
  __syncthreads();
  unsigned long long value[PER];
  uint32_t place[PER];
  const long long first = static_cast<long long>(b) * n;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = j * NT + t;
    value[j] = 0;
    place[j] = 0xffffffffu;
    if (i < n) {
      const int w = i / (S * K);
      const float x = a.cand_x[first + i];
      if (x > -INFINITY) {
        double z = static_cast<double>(x) * static_cast<double>(a.inv_scale);
        if (a.softcap > 0.f) z = static_cast<double>(a.softcap) * tanh(z / static_cast<double>(a.softcap));
        const double v = base[w] + (z - static_cast<double>(top[w]));
        if (isfinite(v)) {
          value[j] = double_order(v);
          place[j] = static_cast<uint32_t>(w) * static_cast<uint32_t>(a.V) + static_cast<uint32_t>(a.cand_i[first + i]);
        }
      }
    }
  }
  const long long out = static_cast<long long>(b) * K;
  for (int k = 0; k < K; ++k) {
    unsigned long long mine = 0;
    uint32_t at = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (value[j] > mine || (value[j] == mine && place[j] < at)) {
        mine = value[j];
        at = place[j];
      }
    }
    unsigned long long v = mine;
    uint32_t p = at;
    warp_best(v, p);
    if (lane == 0) {
      best_value[k & 1][warp] = v;
      best_place[k & 1][warp] = p;
    }
    __syncthreads();
    v = lane < NW ? best_value[k & 1][lane] : 0;
    p = lane < NW ? best_place[k & 1][lane] : 0xffffffffu;
    warp_best(v, p);
    if (v == 0) {  // (the same for all threads)
      for (int r = k + t; r < K; r += NT) {
        a.out_value[out + r] = -INFINITY;
        a.out_parent[out + r] = -1;
        a.out_token[out + r] = -1;
      }
      return;
    }
    if (v == mine && p == at) {
      a.out_value[out + k] = static_cast<float>(double_from_order(v));
      a.out_parent[out + k] = p / static_cast<uint32_t>(a.V);
      a.out_token[out + k] = p % static_cast<uint32_t>(a.V);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (place[j] == p) value[j] = 0, place[j] = 0xffffffffu;
    }
  }
}

}  // namespace

int beam_select_splits(int rows, int W, int K, int V) {
  const int tiles = (V + kTile - 1) / kTile;
  int s = (4 * 148 + rows - 1) / rows;
  s = s < tiles ? s : tiles;
  const int most = kBeamMaxMerge / (W * K);
  s = s < most ? s : most;
  return s > 1 ? s : 1;
}

void launch_beam_select(const BeamSelectArgs& a, bool f32, cudaStream_t st) {
  if (a.B == 0) return;
  const dim3 grid(static_cast<unsigned>(a.B) * a.W * a.splits);
  if (f32) {
    if (a.mask != nullptr) launch_pdl(beam_part_kernel<float, true>, grid, dim3(kThreads), 0, st, a);
    else launch_pdl(beam_part_kernel<float, false>, grid, dim3(kThreads), 0, st, a);
  } else {
    if (a.mask != nullptr) launch_pdl(beam_part_kernel<__nv_bfloat16, true>, grid, dim3(kThreads), 0, st, a);
    else launch_pdl(beam_part_kernel<__nv_bfloat16, false>, grid, dim3(kThreads), 0, st, a);
  }
  if (a.W * a.splits * a.K <= kBeamMaxMerge / 4) launch_pdl(beam_merge_kernel<256>, dim3(a.B), dim3(256), 0, st, a);
  else launch_pdl(beam_merge_kernel<1024>, dim3(a.B), dim3(1024), 0, st, a);
}

// =====================================================================================================================
// Moves of beam states
// =====================================================================================================================
// slot[j] takes over what slot[parent[j]] held, in place: a thread owns the same few bytes of all of a request's slots, reads what every moved beam will
// hold before it writes any of it, and nobody else touches them. No second buffer, one launch for all tensors. Parents outside 0 .. W - 1 leave their
// beam as it is. What bounds it: the bytes of distinct parents read and of moved beams written (a parent that several beams read comes from L1).
template <int UNIT>
struct MoveUnit;
template <>
struct MoveUnit<16> {
  using type = uint4;
};
template <>
struct MoveUnit<4> {
  using type = uint32_t;
};
template <>
struct MoveUnit<2> {
  using type = unsigned short;
};

// grid (units of a slot / 256, tensors, requests)
template <int UNIT, int MAXW>
__global__ void __launch_bounds__(256) beam_move_kernel(const __grid_constant__ BeamMoveArgs a) {
  using U = typename MoveUnit<UNIT>::type;
  pdl_trigger();
  pdl_wait();
  __shared__ long long from[MAXW], to[MAXW];  // slots; to < 0: the beam stays
  const int b = blockIdx.z, t = threadIdx.x;
  const BeamMoveTensor& d = a.t[blockIdx.y];
  const int rows = a.rows != nullptr ? max(0, min(a.rows[b], a.max_rows)) : a.max_rows;
  const long long part = static_cast<long long>(rows) * d.row_bytes / UNIT;  // units of one segment that move
  const long long u = static_cast<long long>(blockIdx.x) * 256 + t;
  if (static_cast<long long>(blockIdx.x) * 256 >= part * d.segments) return;
  if (t < MAXW) {
    long long s = -1, r = -1;
    if (t < a.W) {
      const long long p = a.parents[static_cast<long long>(b) * a.W + t];
      if (p >= 0 && p < a.W && p != t) {
        r = a.slots[static_cast<long long>(b) * a.W + t];
        s = a.slots[static_cast<long long>(b) * a.W + p];
        if (r < 0 || r >= a.num_slots || s < 0 || s >= a.num_slots) {
          atomicCAS(a.status, kStatusOk, kStatusBadArgs);
          r = -1;
        }
      }
    }
    from[t] = s;
    to[t] = r;
  }
  __syncthreads();
  if (u >= part * d.segments) return;
  const long long seg = u / part;
  uint8_t* base = static_cast<uint8_t*>(d.base) + seg * (d.slot_bytes / d.segments) + (u - seg * part) * UNIT;
  U v[MAXW];
#pragma unroll
  for (int j = 0; j < MAXW; ++j)
    if (to[j] >= 0) v[j] = *reinterpret_cast<const U*>(base + from[j] * d.slot_bytes);
#pragma unroll
  for (int j = 0; j < MAXW; ++j)
    if (to[j] >= 0) *reinterpret_cast<U*>(base + to[j] * d.slot_bytes) = v[j];
}

template <int UNIT>
static void move_by_width(const BeamMoveArgs& a, dim3 grid, cudaStream_t st) {
  if (a.W <= 4) launch_pdl(beam_move_kernel<UNIT, 4>, grid, dim3(256), 0, st, a);
  else if (a.W <= 8) launch_pdl(beam_move_kernel<UNIT, 8>, grid, dim3(256), 0, st, a);
  else if (a.W <= 16) launch_pdl(beam_move_kernel<UNIT, 16>, grid, dim3(256), 0, st, a);
  else launch_pdl(beam_move_kernel<UNIT, 32>, grid, dim3(256), 0, st, a);
}

void launch_beam_move(const BeamMoveArgs& a, int B, int unit, cudaStream_t st) {
  long long units = 0;
  for (int i = 0; i < a.n; ++i) {
    const long long u = static_cast<long long>(a.max_rows) * a.t[i].row_bytes / unit * a.t[i].segments;
    units = u > units ? u : units;
  }
  if (B == 0 || a.n == 0 || units == 0) return;
  const dim3 grid(static_cast<unsigned>((units + 255) / 256), a.n, B);
  if (unit == 16) move_by_width<16>(a, grid, st);
  else if (unit == 4) move_by_width<4>(a, grid, st);
  else move_by_width<2>(a, grid, st);
}

}  // namespace dlv
