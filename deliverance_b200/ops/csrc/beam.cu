// Beam search: selection over beams and vocabulary, and the moves of beam states that follow it.
//
// Selection: value[w, v] = scores[w] + z[w, v] - log sum_u exp z[w, u], the K largest finite ones of a request's W rows, ties to the lowest w * V + v.
// The order inside a row is the order of the raw logits (soft-capping and positive scaling are monotone). The first kernel reads every logit once and leaves, per
// row, maxima and sums of exponentials, and the largest logit of every group of 128 (bf16: 256) neighbours. The K best candidates lie in the K groups with the largest
// maxima (equal ones: the first), so the second kernel compares those maxima over all rows, in 64 bits because rows differ by their log-sum-exp, and reads only
// the few groups that can matter again. Inside a row the order is exact. What is compared across rows is exact but for the log-sum-exps, sums of 32-bit exponentials (each off by 2^-22 + 1.5 * 2^-23 times its
// distance from the maximum, 16 at a time added in 32 bits, the rest in 64): candidates of different beams within 8e-6 of each other may change places. What bounds it: the logits, read once.
#include <cfloat>

#include "beam_api.h"
#include "common.cuh"

namespace dlv {

namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kPerLane = 16;                      // logits per lane and tile
constexpr int kTile = kThreads * kPerLane;        // logits of a CTA's tile
constexpr int kMergeThreads = 512, kMergeWarps = kMergeThreads / 32;
constexpr int kClusters = 64;                     // threads of the second kernel, eight by eight: K of their best are the first bound
constexpr int kMostGroups = 1024, kMostListed = 512;  // groups and candidates that are looked at without a closer bound

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

// 16 bytes of a row (element by element where rows do not start on 16 bytes: the same logits in the same lane, so that equal rows have equal sums and their
// candidates tie); -inf at and behind hi
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 load_vector(const T* row, int i, int hi) {
  constexpr int N = Vec<T>::N;
  if (ALIGNED && i + N <= hi) return __ldg(reinterpret_cast<const uint4*>(row + i));
  uint4 u;
  T e[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (sizeof(T) == 4) e[j] = -INFINITY;
    else e[j] = __ushort_as_bfloat16(static_cast<unsigned short>(0xff80u));
    if (i + j < hi) e[j] = row[i + j];
  }
  if constexpr (sizeof(T) == 4) {
    u = make_uint4(__float_as_uint(e[0]), __float_as_uint(e[1]), __float_as_uint(e[2]), __float_as_uint(e[3]));
  } else {
    auto two = [](T a, T b) { return static_cast<uint32_t>(__bfloat16_as_ushort(a)) | static_cast<uint32_t>(__bfloat16_as_ushort(b)) << 16; };
    u = make_uint4(two(e[0], e[1]), two(e[2], e[3]), two(e[4], e[5]), two(e[6], e[7]));
  }
  return u;
}

// exp(x - m) of two logits for x <= m, relative error 2^-22 + |x - m| 2^-22: exactly 1 at x = m, so that what weighs most is exact
__device__ __forceinline__ uint64_t pair(float a, float b) { return static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a); }
__device__ __forceinline__ uint64_t exp_below(uint64_t x, uint64_t minus_m, uint64_t log2e) {
  uint64_t d;
  float lo, hi;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(minus_m));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(d), "l"(log2e));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(lo) : "f"(__uint_as_float(static_cast<uint32_t>(d))));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(hi) : "f"(__uint_as_float(static_cast<uint32_t>(d >> 32))));
  return pair(lo, hi);
}
// maximum over the warp, NaN left out
__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// grid: B * W * splits. A tile is 16 logits per thread, 16 bytes of a warp's lanes side by side: one group per load. The next tile is on its way while a tile is
// worked on; a running maximum per warp (the groups' maxima are there anyway; one per lane moves in nearly every tile of some lane) and a sum per thread, joined at the end in a fixed
// order. 256 rows of 151,936, the whole selection: 34.7 us, 24 at the copy rate of fp32 (29.0 and 12 in bf16, where some ten instructions per logit and one exponential
// in 16 a cycle hold it). With expf 42; 32 logits per thread 37, 8 logits 38 to 45; two more tiles on their way through shared memory 46 (16-byte asynchronous copies per thread) and
// 57 (bulk copies per warp).
// (Candidates listed in this kernel instead of groups' maxima were 33 of 74 us: every tile has one in some warp, and all lanes wait while it is listed.)
// PLAIN: neither scale nor cap.
template <typename T, bool MASK, bool ALIGNED, bool PLAIN>
__global__ void __launch_bounds__(kThreads, 8) beam_part_kernel(const __grid_constant__ BeamSelectArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ double sums[kWarps];
  __shared__ float tops[kWarps];
  constexpr int N = Vec<T>::N, NV = kPerLane / N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const int lo = min(a.V, split * a.per), hi = min(a.V, lo + a.per);
  const T* x_row = static_cast<const T*>(a.logits) + static_cast<long long>(row) * a.ld;
  const uint32_t* bits = MASK ? a.mask + static_cast<long long>(row) * a.mask_ld : nullptr;
  float* group_max = a.group_max + static_cast<long long>(row) * a.groups;
  float m = -FLT_MAX;  // (the warp's)
  double sum = 0.0;
  uint4 raw[NV];
  uint32_t word[NV];
  auto fetch = [&](int at) {
    const int first = at + (warp * NV * 32 + lane) * N;
    const T* p = x_row + first;
    if (ALIGNED && at + kTile <= hi) {  // (the same for the whole CTA)
#pragma unroll
      for (int v = 0; v < NV; ++v) raw[v] = __ldg(reinterpret_cast<const uint4*>(p + v * 32 * N));
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) raw[v] = load_vector<T, ALIGNED>(x_row, first + v * 32 * N, hi);
    }
    if constexpr (MASK) {
#pragma unroll
      for (int v = 0; v < NV; ++v) word[v] = first + v * 32 * N < hi ? bits[(first + v * 32 * N) >> 5] >> (first & 31) : 0u;
    }
  };
  if (lo < hi) fetch(lo);
#pragma unroll 2
  for (int at = lo; at < hi; at += kTile) {
    float x[NV][N];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      unpack(raw[v], x[v]);
      if constexpr (MASK) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[v][e] = (word[v] >> e) & 1u ? x[v][e] : -INFINITY;
      }
    }
    if (at + kTile < hi) fetch(at + kTile);
    // (NaN is left out of the maxima; NaN and +inf make the sum NaN, and a row with such a sum has no candidates)
    float top = -INFINITY, mine = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float g = x[v][0];
#pragma unroll
      for (int e = 1; e < N; ++e) g = fmaxf(g, x[v][e]);
      g = redux_max(g);
      top = fmaxf(top, g);
      if (lane == v) mine = g;
    }
    const int group = at / (32 * N) + warp * NV + lane;
    if (lane < NV && group * 32 * N < hi) group_max[group] = mine;
    const float top_z = PLAIN ? top : post(top, a.softcap, a.inv_scale);
    if (top_z > m) {  // (the same for the whole warp)
      sum *= static_cast<double>(expf(m - top_z));
      m = top_z;
    }
    uint64_t part2 = 0;
    const uint64_t minus_m = pair(-m, -m), log2e = pair(1.44269504088896341f, 1.44269504088896341f);
#pragma unroll
    for (int j = 0; j < kPerLane; j += 2) {
      const float y0 = PLAIN ? x[j / N][j % N] : post(x[j / N][j % N], a.softcap, a.inv_scale);
      const float y1 = PLAIN ? x[j / N][j % N + 1] : post(x[j / N][j % N + 1], a.softcap, a.inv_scale);
      asm("add.rn.f32x2 %0, %0, %1;" : "+l"(part2) : "l"(exp_below(pair(y0, y1), minus_m, log2e)));
    }
    const float part = __uint_as_float(static_cast<uint32_t>(part2)) + __uint_as_float(static_cast<uint32_t>(part2 >> 32));
    sum += static_cast<double>(part);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) {
    tops[warp] = m;
    sums[warp] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    const float t = lane < kWarps ? tops[lane] : -FLT_MAX, all = warp_max(t);
    double s = lane < kWarps ? sums[lane] * static_cast<double>(expf(t - all)) : 0.0;
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      a.part_m[blockIdx.x] = all;
      a.part_sum[blockIdx.x] = s;
    }
  }
}

__device__ __forceinline__ unsigned long long double_order(double v) {
  const long long u = __double_as_longlong(v + 0.0);
  return u < 0 ? ~static_cast<unsigned long long>(u) : static_cast<unsigned long long>(u) | 0x8000000000000000ull;
}

// (out of line: the second kernel runs once through its code, and fetching copies of the hyperbolic tangent between what always runs takes it 0.4 us)
__device__ __noinline__ double capped(double z, double cap) { return cap * tanh(z / cap); }
__device__ __noinline__ float capped(float z, float cap) { return cap * tanhf(z / cap); }

// Number of threads' set flags over the CTA, for the searches that need many of them
__device__ __forceinline__ int merge_count(int c, int* red, int& turn) {
  c = __reduce_add_sync(0xffffffffu, c);
  const int lane = threadIdx.x & 31;
  int* r = red + turn * kMergeWarps;
  turn ^= 1;
  if (lane == 0) r[threadIdx.x >> 5] = c;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, lane < kMergeWarps ? r[lane] : 0);
}

// The K-th best of n (value, place) pairs, found bit by bit: the value, then the place among equals. at(i, place) gives a pair's value, -inf: none. With fewer than
// K pairs the value is -inf. Places differ.
template <typename At>
__device__ __noinline__ void kth_best(int n, int K, At at, int* red, double& value, uint32_t& place) {
  int turn = 0;
  unsigned long long edge = 0;
  uint32_t p;
  const unsigned long long none = double_order(-INFINITY);
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long probe = edge | (1ull << bit);
    int c = 0;
    for (int i = threadIdx.x; i < n; i += kMergeThreads) {
      const unsigned long long o = double_order(at(i, p));
      c += o > none && o >= probe ? 1 : 0;
    }
    if (merge_count(c, red, turn) >= K) edge = probe;
  }
  value = edge > none ? __longlong_as_double(static_cast<long long>(edge & 0x8000000000000000ull ? edge ^ 0x8000000000000000ull : ~edge)) : -INFINITY;
  place = 0xffffffffu;
  if (edge <= none) return;
  int c = 0;
  for (int i = threadIdx.x; i < n; i += kMergeThreads) c += double_order(at(i, p)) > edge ? 1 : 0;
  const int left = K - merge_count(c, red, turn);  // so many of the equal ones, the lowest places
  uint32_t low = 0;                                // the largest bound below which fewer than `left` equal ones lie
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t probe = low | (1u << bit);
    c = 0;
    for (int i = threadIdx.x; i < n; i += kMergeThreads) c += double_order(at(i, p)) == edge && p < probe ? 1 : 0;
    if (merge_count(c, red, turn) < left) low = probe;
  }
  place = low;
}

// One CTA per request. Bound: K of 64 clusters of threads have seen a group whose maximum reaches it, so K candidates do. The groups that reach it are read
// again, and the candidates that reach it are put in order by counting. Where too many do (long runs of one value), the K-th best itself is searched for.
// What bounds it: latency, 6 us of dependent loads, barriers and one logarithm in 64 bits at 4 beams of 151,936 logits; with 16 beams the 19,000 maxima of a request, 22 us
// (12 or 40 of them per thread in registers: the same).
template <typename T>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const __grid_constant__ BeamSelectArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ double base[kBeamMaxBeams];
  __shared__ float top[kBeamMaxBeams];
  __shared__ double values[kMostListed];
  __shared__ float rough[kBeamMaxBeams], cluster_value[kClusters], edge_value;
  __shared__ uint32_t places[kMostListed];
  __shared__ int groups[kMostGroups], red[2 * kMergeWarps], listed, n_groups;
  constexpr int N = Vec<T>::N, GROUP = 32 * N;
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int K = a.K, W = a.W, n = W * a.groups;
  const float* maxima = a.group_max + static_cast<long long>(b) * n;
  constexpr int AHEAD = 12;
  // Of few groups a cluster has every 64th, so that those of one beam are spread over all clusters: neighbours in one cluster made bounds that thousands of candidates
  // reach (3 requests of 12 beams and 1,300 tokens 33 us instead of 12, 20 of 16 guided beams and 3,000 tokens 54 instead of 19). Many groups spread by themselves, and
  // are read side by side (4 x 16 beams of 151,936 tokens 30 us instead of 32).
  const int own = n <= 8 * kMergeThreads ? (t & 7) * kClusters + (t >> 3) : t;
  float x[AHEAD];  // (on their way while the sums are joined)
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) x[j] = j * kMergeThreads + own < n ? maxima[j * kMergeThreads + own] : -INFINITY;
  if (t == 0) listed = n_groups = 0;
  for (int w = warp; w < W; w += kMergeWarps) {
    const long long at = (static_cast<long long>(b) * W + w) * a.splits;
    const float score = a.scores[static_cast<long long>(b) * W + w];
    float m = -FLT_MAX;
    for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, a.part_m[at + s]);
    m = warp_max(m);
    double sum = 0.0;
    for (int s = lane; s < a.splits; s += 32) sum += a.part_sum[at + s] * static_cast<double>(expf(a.part_m[at + s] - m));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      top[w] = m;
      base[w] = static_cast<double>(score) - log(sum);
      const float r = static_cast<float>(base[w] - static_cast<double>(m));
      rough[w] = isfinite(r) ? r : -INFINITY;
    }
  }
  __syncthreads();
  auto value_of = [&](float y, int w) {
    if (!(y > -INFINITY)) return -static_cast<double>(INFINITY);
    double z = static_cast<double>(y) * static_cast<double>(a.inv_scale);
    if (a.softcap > 0.f) z = capped(z, static_cast<double>(a.softcap));
    const double v = base[w] + (z - static_cast<double>(top[w]));
    return isfinite(static_cast<float>(v)) ? v : -static_cast<double>(INFINITY);  // (as it is returned)
  };
  // in 32 bits: off by less than half of `slack` (roundings of the row's constant, of the sum and of scale and cap)
  auto rough_post = [&](float y) {
    y *= a.inv_scale;
    return a.softcap > 0.f && y > -INFINITY ? capped(y, a.softcap) : y;
  };
  auto rough_of = [&](float y, int i) { return rough_post(y) + rough[a.by_groups.of(i)]; };
  float best = -INFINITY;
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    const int i = j * kMergeThreads + own;
    x[j] = i < n ? rough_of(x[j], i) : -INFINITY;
    best = fmaxf(best, x[j]);
  }
  for (int i0 = AHEAD * kMergeThreads + own; i0 < n; i0 += 8 * kMergeThreads) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = i0 + j * kMergeThreads < n ? maxima[i0 + j * kMergeThreads] : -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * kMergeThreads < n) best = fmaxf(best, rough_of(y[j], i0 + j * kMergeThreads));
  }
  // a value that K at least of the CTA's threads' best reach: the K-th best of 64 clusters of eight threads
  auto bound_of = [&](float mine) {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if ((t & 7) == 0) cluster_value[t >> 3] = mine;
    __syncthreads();
    const int g = t >> 3;  // eight threads count for one cluster
    int rank = 0;
#pragma unroll
    for (int q = 0; q < kClusters / 8; ++q) {
      const int u = q * 8 + (t & 7);
      rank += cluster_value[u] > mine || (cluster_value[u] == mine && u < g) ? 1 : 0;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if ((t & 7) == 0 && rank == K - 1) edge_value = mine;
    __syncthreads();
    return edge_value;
  };
  const float reached = bound_of(best);
  float most = 0.f;
  for (int w = lane; w < W; w += 32) most = fmaxf(most, rough[w] > -INFINITY ? fabsf(rough[w]) : 0.f);
  most = warp_max(most);
  auto below = [&](float v) { return v - (0x1p-20f * (most + fabsf(v)) + 0x1p-18f * a.softcap); };
  const float bound = below(reached);
  double edge = static_cast<double>(bound);  // K candidates at least are not below this
  uint32_t last = 0xffffffffu;               // of the groups (then: candidates) that equal the edge, those up to this place
  auto list_group = [&](int i) {
    const int p = atomicAdd(&n_groups, 1);
    if (p < kMostGroups) groups[p] = i;
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (x[j] > -INFINITY && x[j] >= bound) list_group(j * kMergeThreads + own);
  for (int i0 = AHEAD * kMergeThreads + own; i0 < n; i0 += 8 * kMergeThreads) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = i0 + j * kMergeThreads < n ? maxima[i0 + j * kMergeThreads] : -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * kMergeThreads;
      if (i < n) {
        const float f = rough_of(y[j], i);
        if (f > -INFINITY && f >= bound) list_group(i);
      }
    }
  }
  __syncthreads();
  if (n_groups > kMostGroups) {
    kth_best(n, K, [&](int i, uint32_t& p) { p = static_cast<uint32_t>(i); return value_of(maxima[i], i / a.groups); }, red, edge, last);
    __syncthreads();
    if (t == 0) n_groups = 0;
    __syncthreads();
    for (int i = t; i < n; i += kMergeThreads) {
      const double v = value_of(maxima[i], i / a.groups);
      if (v > -INFINITY && (v > edge || (v == edge && static_cast<uint32_t>(i) <= last))) list_group(i);
    }
    __syncthreads();
  }
  const int m_groups = n_groups;
  // candidate j of the listed groups
  auto logit = [&](int g, int e, int& w, int& v) {
    w = a.by_groups.of(groups[g]);
    v = (groups[g] - w * a.groups) * GROUP + e;
    const long long row = static_cast<long long>(b) * W + w;
    if (v >= a.V || (a.mask != nullptr && !((a.mask[row * a.mask_ld + (v >> 5)] >> (v & 31)) & 1u))) return -INFINITY;
    const T y = static_cast<const T*>(a.logits)[row * a.ld + v];
    if constexpr (sizeof(T) == 4) return static_cast<float>(y);
    else return bf2f(y);
  };
  auto place_of = [&](int w, int v) { return static_cast<uint32_t>(w) * static_cast<uint32_t>(a.V) + static_cast<uint32_t>(v); };
  last = 0xffffffffu;
  const bool loose = m_groups > 4 * K + 16 || reached == -INFINITY;
#pragma unroll 1
  for (int round = loose ? 1 : 0;; ++round) {
    if (round == 1) {  // a closer bound, from the candidates themselves: rows that a mask leaves few tokens, few groups
      float mine = -INFINITY;
#pragma unroll 1
      for (int g = warp; g < m_groups; g += kMergeWarps) {
#pragma unroll
        for (int q = 0; q < N; ++q) {
          int w, v;
          const float y = logit(g, q * 32 + lane, w, v);
          mine = fmaxf(mine, rough_post(y) + rough[w]);
        }
      }
      __syncthreads();
      edge = fmax(edge, static_cast<double>(below(bound_of(mine))));
    } else if (round == 2) {  // long runs of one value
      kth_best(m_groups * GROUP, K, [&](int i, uint32_t& p) {
        int w, v;
        const float y = logit(i / GROUP, i % GROUP, w, v);
        p = place_of(w, v);
        return value_of(y, w);
      }, red, edge, last);
    }
#pragma unroll 1
    for (int g = warp; g < m_groups && *static_cast<volatile int*>(&listed) <= kMostListed; g += kMergeWarps) {
      float y[N];
      int w, v;
#pragma unroll
      for (int q = 0; q < N; ++q) y[q] = logit(g, q * 32 + lane, w, v);
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const double d = value_of(y[q], w);
        const uint32_t p = place_of(w, (groups[g] - w * a.groups) * GROUP + q * 32 + lane);
        if (d > -INFINITY && (d > edge || (d == edge && p <= last))) {
          const int at = atomicAdd(&listed, 1);
          if (at < kMostListed) {
            values[at] = d;
            places[at] = p;
          }
        }
      }
    }
    __syncthreads();
    if (listed <= kMostListed) break;
    __syncthreads();
    if (t == 0) listed = 0;
    __syncthreads();
  }
  const int m = listed;
  const long long out = static_cast<long long>(b) * K;
  for (int j = t; j < m; j += kMergeThreads) {
    const double v = values[j];
    const uint32_t p = places[j];
    int rank = 0;
    for (int u = 0; u < m; ++u) rank += values[u] > v || (values[u] == v && places[u] < p) ? 1 : 0;
    if (rank < K) {
      a.out_value[out + rank] = static_cast<float>(v);
      a.out_parent[out + rank] = p / static_cast<uint32_t>(a.V);
      a.out_token[out + rank] = p % static_cast<uint32_t>(a.V);
    }
  }
  for (int r = m + t; r < K; r += kMergeThreads) {
    a.out_value[out + r] = -INFINITY;
    a.out_parent[out + r] = -1;
    a.out_token[out + r] = -1;
  }
}

}  // namespace

int beam_select_group(bool f32) { return f32 ? 32 * Vec<float>::N : 32 * Vec<__nv_bfloat16>::N; }

// CTAs per row. Much work: four units each, which end at different times and so keep the GPU full (256 rows of 151,936 with 4 / 10 / 13 CTAs each: 36.7 / 34.7 / 35.9 us, in bf16 33.3 / 29.0 / 29.3).
// Little work: a unit each (4 rows of 83,308 with 1 / 21 CTAs each: 17.9 / 9.2 us). Otherwise the fewest that keep the GPU about evenly busy (eight resident per SM), each with a unit at least (256 rows of 32,000 with 4 / 8: 14.4 / 14.7).
int beam_select_splits(int rows, int V) {
  const int tiles = (V + kBeamSplitUnit - 1) / kBeamSplitUnit, slots = 8 * 148;
  if (static_cast<long long>(rows) * tiles <= slots) return tiles;
  const long long quarters = (tiles + 3) / 4;
  if (rows * quarters >= 2 * slots) return static_cast<int>(quarters);
  int best = 1;
  double most = 0.0;
  for (int s = 1; s <= tiles && s <= 64; ++s) {
    const double n = static_cast<double>(rows) * ((tiles + (tiles + s - 1) / s - 1) / ((tiles + s - 1) / s)), waves = n / slots;
    const double even = waves / static_cast<double>(static_cast<long long>(waves + 0.999999));
    if (even > most + 0.1) {
      most = even;
      best = s;
    }
    if (most > 0.85) break;
  }
  return best;
}

template <typename T, bool MASK>
static void launch_part(const BeamSelectArgs& a, dim3 grid, cudaStream_t st) {
  const bool aligned = (reinterpret_cast<uintptr_t>(a.logits) | static_cast<uintptr_t>(a.ld * static_cast<long long>(sizeof(T)))) % 16 == 0;
  const bool plain = a.softcap <= 0.f && a.inv_scale == 1.f;
  if (aligned && plain) launch_pdl(beam_part_kernel<T, MASK, true, true>, grid, dim3(kThreads), 0, st, a);
  else if (aligned) launch_pdl(beam_part_kernel<T, MASK, true, false>, grid, dim3(kThreads), 0, st, a);
  else if (plain) launch_pdl(beam_part_kernel<T, MASK, false, true>, grid, dim3(kThreads), 0, st, a);
  else launch_pdl(beam_part_kernel<T, MASK, false, false>, grid, dim3(kThreads), 0, st, a);
}

void launch_beam_select(const BeamSelectArgs& a, bool f32, cudaStream_t st) {
  if (a.B == 0) return;
  const dim3 grid(static_cast<unsigned>(a.B) * a.W * a.splits);
  if (f32) {
    a.mask != nullptr ? launch_part<float, true>(a, grid, st) : launch_part<float, false>(a, grid, st);
    launch_pdl(beam_merge_kernel<float>, dim3(a.B), dim3(kMergeThreads), 0, st, a);
  } else {
    a.mask != nullptr ? launch_part<__nv_bfloat16, true>(a, grid, st) : launch_part<__nv_bfloat16, false>(a, grid, st);
    launch_pdl(beam_merge_kernel<__nv_bfloat16>, dim3(a.B), dim3(kMergeThreads), 0, st, a);
  }
}

// =====================================================================================================================
// Moves of beam states
// =====================================================================================================================
// slot[j] takes over what slot[parent[j]] held, in place: a thread owns the same few bytes of all of a request's slots, reads what every moved beam will
// hold before it writes any of it, and nobody else touches them. No second buffer, one launch for all tensors. Parents outside 0 .. W - 1 leave their
// beam as it is. What bounds it: the bytes of distinct parents read and of moved beams written (a parent that several beams read comes from L1).
// grid (parts of a slot, tensors, requests): a part takes every gridDim.x-th 256 units
template <int UNIT, int MAXW>
__global__ void __launch_bounds__(256, MAXW <= 4 ? 5 : MAXW <= 8 ? 4 : MAXW <= 16 ? 2 : 1) beam_move_kernel(const __grid_constant__ BeamMoveArgs a) {
  using U = typename CopyUnit<UNIT>::type;
  pdl_trigger();
  pdl_wait();
  __shared__ long long from[MAXW], to[MAXW];  // byte offsets of slots; to < 0: the beam stays
  const int b = blockIdx.z, t = threadIdx.x;
  const BeamMoveTensor& d = a.t[blockIdx.y];
  // (everything that the moves depend on is asked for at once)
  const int filled = a.rows != nullptr ? a.rows[b] : a.max_rows;
  long long slot = -1, parent = -1;
  if (t < a.W) {
    slot = a.slots[static_cast<long long>(b) * a.W + t];
    parent = a.parents[static_cast<long long>(b) * a.W + t];
  }
  const int rows = max(0, min(filled, a.max_rows));
  const long long part = static_cast<long long>(rows) * d.row_bytes / UNIT, all = part * d.segments;  // units of one segment that move, of a slot
  if (static_cast<long long>(blockIdx.x) * 256 >= all) return;
  if (t < 32) {
    const bool moves = parent >= 0 && parent < a.W && parent != t;
    const long long source = __shfl_sync(0xffffffffu, slot, moves ? static_cast<int>(parent) : t);
    const bool good = slot >= 0 && slot < a.num_slots && source >= 0 && source < a.num_slots;
    if (moves && !good) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
    if (t < MAXW) {
      from[t] = source * d.slot_bytes;
      to[t] = moves && good ? slot * d.slot_bytes : -1;
    }
  }
  __syncthreads();
  const long long pitch = d.slot_bytes / d.segments;
  for (long long u = static_cast<long long>(blockIdx.x) * 256 + t; u < all; u += static_cast<long long>(gridDim.x) * 256) {
    const long long seg = all == part ? 0 : u / part;
    uint8_t* base = static_cast<uint8_t*>(d.base) + seg * pitch + (u - seg * part) * UNIT;
    U v[MAXW];
#pragma unroll
    for (int j = 0; j < MAXW; ++j)
      if (to[j] >= 0) v[j] = *reinterpret_cast<const U*>(base + from[j]);
#pragma unroll
    for (int j = 0; j < MAXW; ++j)
      if (to[j] >= 0) *reinterpret_cast<U*>(base + to[j]) = v[j];
  }
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
  // looking the slots up takes a CTA as long as moving a unit, so pages, of which a slot has little, get fewer CTAs (16 x 8 beams, 44 pools: 10.3 us with 16 per SM, 11.3 with 64;
  // 32 x 16 beams 54 and 65; states of 2 MB 363 and 345)
  const long long parts = (units + 255) / 256, room = 148 * (a.paged ? 16 : 64) / (static_cast<long long>(a.n) * B);
  const dim3 grid(static_cast<unsigned>(room < 1 ? 1 : room < parts ? room : parts), a.n, B);
  if (unit == 16) move_by_width<16>(a, grid, st);
  else if (unit == 4) move_by_width<4>(a, grid, st);
  else move_by_width<2>(a, grid, st);
}

}  // namespace dlv
