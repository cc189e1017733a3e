// Bounded cache: which rows of the paged cache stay, and their way to the front.
//
// Of a sequence's n > keep rows the last `recent` stay and of the others the keep - recent with the largest accumulated attention weight (equal weights: the
// earliest), per layer and KV head. The first kernel finds them, writes their list in ascending order and shortens the weights; the second moves K and V rows.
// Row j of the result comes from row list[j] >= j. What bounds it: the kept rows of K and V, read and written once.
#include "beam_api.h"
#include "common.cuh"

namespace dlv {

namespace {

constexpr int kSelectThreads = 512;

// larger = heavier; NaN is the smallest, -0 equals 0
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// sum over the CTA (kSelectThreads threads); `red`: two buffers used in turn, one barrier per call
__device__ __forceinline__ int block_count(int v, int* red, int turn) {
  v = __reduce_add_sync(0xffffffffu, v);
  const int lane = threadIdx.x & 31;
  int* r = red + turn * (kSelectThreads / 32);
  if (lane == 0) r[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, lane < kSelectThreads / 32 ? r[lane] : 0);
}

// Whether this sequence can be worked on: its slot lies inside the weights and no earlier sequence of the call has it.
__device__ __forceinline__ bool slot_ok(const long long* slots, int b, int num_slots) {
  const long long s = slots[b];
  bool bad = s <= 0 || s >= num_slots;
  for (int i = threadIdx.x; i < b; i += blockDim.x) bad = bad || slots[i] == s;
  return !__syncthreads_or(bad);
}

// grid (KV, B, layers)
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ int red[2 * (kSelectThreads / 32)];
  __shared__ int ties[2][kSelectThreads / 32], takes[2][kSelectThreads / 32];
  const int kvh = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int n = max(0, min(a.ctx[b], a.table_width * a.page));
  int* kept = a.kept + ((static_cast<long long>(layer) * a.B + b) * a.KV + kvh) * a.keep;
  const bool ok = n == 0 || slot_ok(a.slots, b, a.num_slots);
  if (layer == 0 && kvh == 0 && t == 0) {
    a.lens[b] = ok ? min(n, a.keep) : n;
    if (!ok) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
  }
  if (!ok || n <= a.keep) {
    for (int j = t; j < a.keep; j += kSelectThreads) kept[j] = ok && j < n ? j : -1;
    return;
  }
  float* w = a.layer[layer].weights + (a.slots[b] * a.KV + kvh) * a.capacity;
  const int counted = min(n, a.capacity), old = n - a.recent, want = a.keep - a.recent;
  auto key_at = [&](int i) { return weight_order(i < counted ? w[i] : 0.f); };
  // edge: the largest value that `want` of the old keys reach; `spare` of those that equal it stay
  uint32_t edge = 0xffffffffu;
  int spare = 0;
  if (want > 0) {
    edge = 0;
    constexpr int R = 8;
    uint32_t mine[R];
#pragma unroll
    for (int r = 0; r < R; ++r) mine[r] = r * kSelectThreads + t < old ? key_at(r * kSelectThreads + t) : 0u;
    int turn = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t probe = edge | (1u << bit);
      int c = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) c += mine[r] >= probe ? 1 : 0;
      for (int i = R * kSelectThreads + t; i < old; i += kSelectThreads) c += key_at(i) >= probe ? 1 : 0;
      c = block_count(c, red, turn);
      turn ^= 1;
      if (c >= want) edge = probe;
    }
    int c = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) c += mine[r] > edge ? 1 : 0;
    for (int i = R * kSelectThreads + t; i < old; i += kSelectThreads) c += key_at(i) > edge ? 1 : 0;
    spare = want - block_count(c, red, turn);
  }
  // the list, in ascending order
  int tie_base = 0, take_base = 0, turn = 0;
  for (int i0 = 0; i0 < n; i0 += kSelectThreads, turn ^= 1) {
    const int i = i0 + t;
    const uint32_t key = i < old ? key_at(i) : 0u;
    const bool tie = i < old && key == edge && spare > 0;
    const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) ties[turn][warp] = __popc(tie_mask);
    __syncthreads();
    int tie_before = tie_base, tie_all = 0;
#pragma unroll
    for (int q = 0; q < kSelectThreads / 32; ++q) {
      if (q < warp) tie_before += ties[turn][q];
      tie_all += ties[turn][q];
    }
    tie_before += __popc(tie_mask & ((1u << lane) - 1u));
    const bool take = i < n && (i >= old || key > edge || (tie && tie_before < spare));
    const uint32_t take_mask = __ballot_sync(0xffffffffu, take);
    if (lane == 0) takes[turn][warp] = __popc(take_mask);
    __syncthreads();
    int at = take_base, take_all = 0;
#pragma unroll
    for (int q = 0; q < kSelectThreads / 32; ++q) {
      if (q < warp) at += takes[turn][q];
      take_all += takes[turn][q];
    }
    at += __popc(take_mask & ((1u << lane) - 1u));
    if (take && at < a.keep) kept[at] = i;
    tie_base += tie_all;
    take_base += take_all;
  }
  __syncthreads();
  // weights: entry j takes over entry kept[j] >= j; a tile is read as a whole before it is written
  for (int j0 = 0; j0 < counted; j0 += kSelectThreads) {
    const int j = j0 + t;
    float v = 0.f;
    if (j < a.keep && j < counted) {
      const int i = kept[j];
      v = i < counted ? w[i] : 0.f;
    }
    __syncthreads();
    if (j < counted) w[j] = v;
  }
}

template <int UNIT>
struct RowUnit;
template <>
struct RowUnit<16> {
  using type = uint4;
};
template <>
struct RowUnit<4> {
  using type = uint32_t;
};
template <>
struct RowUnit<2> {
  using type = unsigned short;
};

// grid (2 * slices, B * KV, layers): a CTA moves a range of columns of all rows of K or V of one head, in ascending batches of rows that are read as a
// whole before they are written. Sources lie at or behind their targets, so no batch reads what an earlier one wrote, and in place is safe.
template <int UNIT>
__global__ void __launch_bounds__(256) evict_move_kernel(const __grid_constant__ EvictArgs a, int slices) {
  using U = typename RowUnit<UNIT>::type;
  constexpr int BATCH = 8;
  pdl_trigger();
  pdl_wait();
  const int value = blockIdx.x & 1, slice = blockIdx.x >> 1, b = blockIdx.y / a.KV, kvh = blockIdx.y % a.KV, layer = blockIdx.z, t = threadIdx.x;
  const EvictLayer& L = a.layer[layer];
  uint8_t* cache = static_cast<uint8_t*>(value ? L.v : L.k);
  const int row_bytes = value ? L.v_bytes : L.k_bytes, units = row_bytes / UNIT;
  const int c0 = static_cast<int>(static_cast<long long>(units) * slice / slices), c1 = static_cast<int>(static_cast<long long>(units) * (slice + 1) / slices);
  const int n = min(max(0, min(a.ctx[b], a.table_width * a.page)), a.keep);
  const int* kept = a.kept + ((static_cast<long long>(layer) * a.B + b) * a.KV + kvh) * a.keep;
  if (n == 0 || c0 == c1 || kept[0] < 0) return;  // (nothing of a sequence on a bad slot moves)
  const int* from = a.tables + static_cast<long long>(b) * a.table_width;
  const int* to = a.out_tables + static_cast<long long>(b) * a.out_width;
  for (int c = c0; c < c1; c += 256) {
    const int width = min(256, c1 - c), lines = 256 / width;  // rows side by side
    const int line = t / width, col = c + t % width;
    const bool on = line < lines;
    for (int j0 = 0; j0 < n; j0 += lines * BATCH) {
      U v[BATCH];
      long long target[BATCH];
#pragma unroll
      for (int q = 0; q < BATCH; ++q) {
        const int j = j0 + q * lines + line;
        target[q] = -1;
        if (on && j < n) {
          const int i = kept[j], ps = from[i / a.page], pd = to[j / a.page];
          if (ps < 0 || ps >= a.pages || pd < 0 || pd >= a.pages) {
            atomicCAS(a.status, kStatusOk, kStatusBadArgs);
          } else {
            const long long s = (static_cast<long long>(ps) * a.KV + kvh) * a.page + i % a.page, d = (static_cast<long long>(pd) * a.KV + kvh) * a.page + j % a.page;
            if (s != d) {
              target[q] = d;
              v[q] = *reinterpret_cast<const U*>(cache + s * row_bytes + static_cast<long long>(col) * UNIT);
            }
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < BATCH; ++q)
        if (target[q] >= 0) *reinterpret_cast<U*>(cache + target[q] * row_bytes + static_cast<long long>(col) * UNIT) = v[q];
    }
  }
}

}  // namespace

void launch_evict(const EvictArgs& a, int unit, cudaStream_t st) {
  if (a.B == 0 || a.layers == 0 || a.KV == 0) return;
  launch_pdl(evict_select_kernel, dim3(a.KV, a.B, a.layers), dim3(kSelectThreads), 0, st, a);
  const dim3 grid(2, a.B * a.KV, a.layers);
  if (unit == 16) launch_pdl(evict_move_kernel<16>, grid, dim3(256), 0, st, a, 1);
  else if (unit == 4) launch_pdl(evict_move_kernel<4>, grid, dim3(256), 0, st, a, 1);
  else launch_pdl(evict_move_kernel<2>, grid, dim3(256), 0, st, a, 1);
}

}  // namespace dlv
