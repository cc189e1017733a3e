// Bounded cache: which rows of the paged cache stay, and their way to the front.
//
// Of a sequence's n > keep rows the last `recent` stay and of the others the keep - recent with the largest accumulated attention weight (equal weights: the
// earliest), per layer and KV head. The first kernel finds them, writes their list in ascending order and shortens the weights; the second moves K and V rows.
// Row j of the result comes from row list[j] >= j. What bounds it: the kept rows of K and V, read and written once.
#include "beam_api.h"
#include "common.cuh"

namespace dlv {

namespace {

// larger = heavier; NaN is the smallest, -0 equals 0
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float weight_of(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order); }

// sum over the CTA's NT threads; `red`: two buffers used in turn, one barrier per call
template <int NT>
__device__ __forceinline__ int block_count(int v, int* red, int turn) {
  v = __reduce_add_sync(0xffffffffu, v);
  const int lane = threadIdx.x & 31;
  int* r = red + turn * (NT / 32);
  if (lane == 0) r[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, lane < NT / 32 ? r[lane] : 0);
}

// Whether this sequence can be worked on: its slot lies inside the weights and no earlier sequence of the call has it.
__device__ __forceinline__ bool slot_ok(const long long* slots, int b, int num_slots) {
  const long long s = slots[b];
  bool bad = s <= 0 || s >= num_slots;
  for (int i = threadIdx.x; i < b; i += blockDim.x) bad = bad || slots[i] == s;
  return !__syncthreads_or(bad);
}

// exclusive sum over the CTA, and the total; `red` as in block_count
template <int NT>
__device__ __forceinline__ int block_scan(int v, int* red, int turn, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, in, o);
    in += lane >= o ? u : 0;
  }
  int* r = red + turn * (NT / 32);
  if (lane == 31) r[warp] = in;
  __syncthreads();
  const int w = lane < NT / 32 ? r[lane] : 0;
  total = __reduce_add_sync(0xffffffffu, w);
  return in - v + __reduce_add_sync(0xffffffffu, lane < warp ? w : 0);
}

// What the selection of one (sequence, KV head, layer) works on; false: there is nothing to choose, and the list is written.
struct EvictTask {
  int n, counted, old, want;
  int* kept;
  float* w;
  __device__ bool open(const EvictArgs& a) {
    const int kvh = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, t = threadIdx.x;
    n = max(0, min(a.ctx[b], a.table_width * a.page));
    kept = a.kept + ((static_cast<long long>(layer) * a.B + b) * a.KV + kvh) * a.keep;
    const bool ok = n == 0 || slot_ok(a.slots, b, a.num_slots);
    if (layer == 0 && kvh == 0 && t == 0) {
      a.lens[b] = ok ? min(n, a.keep) : n;
      if (!ok || a.ctx[b] != n) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
    }
    if (!ok || n <= a.keep) {
      for (int j = t; j < a.keep; j += blockDim.x) kept[j] = ok && j < n ? j : -1;
      return false;
    }
    w = a.layer[layer].weights + (a.slots[b] * a.KV + kvh) * a.capacity;
    counted = min(n, a.capacity);
    old = n - a.recent;
    want = a.keep - a.recent;
    return true;
  }
};

// grid (KV, B, layers). Up to R * NT rows, `rounds` per thread: a warp has neighbouring rows, 32 at a time, and every thread its rows' weights as ordered integers in registers.
// The edge (what the want-th heaviest weighs) is found bit by bit, a count over the CTA each, until exactly `want` keys reach it. Places are counted by ballots,
// and the weights that stay are written from the registers. What bounds it: issue (some 80 instructions per row) and, with 1,024 threads, the barriers of the search.
// 4,608 heads of 2,304 rows 63 us with 256 threads of 10 rows and four CTAs per SM (five 63, six 66; 512 of 5 83; 128 of 20 71; with rows side by side in a thread, by way of shared memory, 109),
// 256 heads of 30,000 rows 44 to 71 us with 1,024 of 36 (512 of 72 76 to 101), 1,024 of 9,000 rows 64 with 512 of 20 (one CTA per SM 76; 1,024 of 10 76; 256 of 40 92).
template <int NT, int R, int CTAS>
__global__ void __launch_bounds__(NT, CTAS) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int WARPS = NT / 32;
  __shared__ int red[2 * WARPS];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  EvictTask k;
  if (!k.open(a)) return;
  const int rounds = (k.n + NT - 1) / NT;  // (at most R: the launcher's choice)
  const int first = warp * rounds * 32 + lane, end = (warp + 1) * rounds * 32;
  // row first + 32 r is one of this thread's, has a weight, can go: for 32 r below
  const int mine = min(k.n, end) - first, weighed = min(k.counted, end) - first, open = min(k.old, end) - first;
  const uint32_t before = (1u << lane) - 1u;
  const float* w = k.w + first;
  uint32_t key[R];  // of the rows that can go, 0 for the others
#pragma unroll
  for (int r = 0; r < R; ++r) key[r] = r * 32 < min(open, weighed) ? __float_as_uint(w[r * 32]) : 0u;  // (a row without a weight: 0.0)
#pragma unroll
  for (int r = 0; r < R; ++r) key[r] = r * 32 < open ? weight_order(__uint_as_float(key[r])) : 0u;
  uint32_t edge = 0xffffffffu;  // keys above the edge stay, and `spare` of those that equal it
  int spare = 0, turn = 0;
  if (k.want > 0) {
    __shared__ uint32_t few[NT];
    __shared__ int n_few;
    if (t == 0) n_few = 0;
    edge = 0;
    int reach = k.old, above = 0, bit = 31;  // keys that reach the edge, and those beyond the range that is still open above it
    bool exact = false;
    for (; bit >= 0 && !exact && reach - above > NT; --bit) {
      const uint32_t probe = edge | (1u << bit);
      int c = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) c += key[r] >= probe ? 1 : 0;
      c = block_count<NT>(c, red, turn);
      turn ^= 1;
      if (c >= k.want) edge = probe, reach = c;
      else above = c;
      exact = c == k.want;
    }
    if (bit >= 0 && !exact) {  // one open key per thread from here on
      const uint32_t range = bit == 31 ? 0xffffffffu : (2u << bit) - 1u;  // keys from edge to edge + range
      int c = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) c += r * 32 < open && key[r] - edge <= range ? 1 : 0;
      int at = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, at, o);
        at += lane >= o ? u : 0;
      }
      __syncthreads();  // (n_few is 0)
      int base = 0;
      if (lane == 31) base = atomicAdd(&n_few, at);
      at += __shfl_sync(0xffffffffu, base, 31) - c;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r * 32 < open && key[r] - edge <= range) few[at++] = key[r];
      __syncthreads();
      const uint32_t own = t < n_few ? few[t] : 0u;
      const int beyond = above;
      for (; bit >= 0 && !exact; --bit) {
        const uint32_t probe = edge | (1u << bit);
        const int c = beyond + __syncthreads_count(own >= probe);
        if (c >= k.want) edge = probe;
        exact = c == k.want;
        if (c < k.want) above = c;
      }
    }
    if (exact) edge -= 1;  // (all that reach the probe: above probe - 1; a probe is not 0)
    else spare = k.want - above;
  }
  // sum over the warps in front of this one of a number that a warp's lanes share
  auto in_front = [&](int v) {
    int* q = red + turn * WARPS;
    turn ^= 1;
    if (lane == 0) q[warp] = v;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, lane < warp ? q[lane] : 0);
  };
  int tie = 0;  // keys that equal the edge in front of a round
  if (spare > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= rounds) break;
      tie += __popc(__ballot_sync(0xffffffffu, r * 32 < open && key[r] == edge));
    }
    tie = in_front(tie);
  }
  uint32_t takes[(R + 31) / 32] = {};
  int place = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rounds) break;
    bool take = r * 32 < mine && (r * 32 >= open || key[r] > edge);
    if (spare > 0) {
      const bool even = r * 32 < open && key[r] == edge;
      const uint32_t all = __ballot_sync(0xffffffffu, even);
      take = take || (even && tie + __popc(all & before) < spare);
      tie += __popc(all);
    }
    takes[r / 32] |= (take ? 1u : 0u) << (r % 32);
    place += __popc(__ballot_sync(0xffffffffu, take));
  }
  if (open < mine) {  // the weights of the recent rows, as they are
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r * 32 >= open && r * 32 < weighed) key[r] = __float_as_uint(w[r * 32]);
  }
  const int own_places = place;
  place = in_front(place);  // (with the barrier behind which all weights are in registers)
  if (t == NT - 1 && place + own_places != a.keep) atomicCAS(a.status, kStatusOk, kStatusBadArgs);  // (a wrong edge would be said; the list never overruns)
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rounds) break;
    const bool take = (takes[r / 32] >> (r % 32)) & 1u;
    const uint32_t all = __ballot_sync(0xffffffffu, take);
    const int j = place + __popc(all & before);
    if (take && j < a.keep) {
      k.kept[j] = first + r * 32;
      if (j < k.counted) k.w[j] = r * 32 < open ? weight_of(key[r]) : __uint_as_float(key[r]);
    }
    place += __popc(all);
  }
  for (int j = a.keep + t; j < k.counted; j += NT) k.w[j] = 0.f;
}

// The same for any length, with the weights read again for every count and the list in global memory.
__global__ void __launch_bounds__(512) evict_select_long_kernel(const __grid_constant__ EvictArgs a) {
  constexpr int NT = 512;
  pdl_trigger();
  pdl_wait();
  __shared__ int red[2 * (NT / 32)];
  const int t = threadIdx.x;
  EvictTask k;
  if (!k.open(a)) return;
  auto key_at = [&](int i) { return weight_order(i < k.counted ? k.w[i] : 0.f); };
  auto count = [&](auto&& test, int turn) {
    int c = 0;
    for (int i = t; i < k.old; i += NT) c += test(key_at(i)) ? 1 : 0;
    return block_count<NT>(c, red, turn);
  };
  uint32_t edge = 0xffffffffu;
  int spare = 0, turn = 0;
  if (k.want > 0) {
    edge = 0;
    for (int bit = 31; bit >= 0; --bit, turn ^= 1) {
      const uint32_t probe = edge | (1u << bit);
      if (count([&](uint32_t u) { return u >= probe; }, turn) >= k.want) edge = probe;
    }
    spare = k.want - count([&](uint32_t u) { return u > edge; }, turn);
    turn ^= 1;
  }
  int tie_base = 0, take_base = 0;
  for (int i0 = 0; i0 < k.n; i0 += NT) {
    const int i = i0 + t;
    const uint32_t key = i < k.old ? key_at(i) : 0u;
    const bool even = i < k.old && key == edge;
    int all;
    const int before = tie_base + block_scan<NT>(even ? 1 : 0, red, turn, all);
    turn ^= 1;
    tie_base += all;
    const bool take = i < k.n && (i >= k.old || key > edge || (even && before < spare));
    const int place = take_base + block_scan<NT>(take ? 1 : 0, red, turn, all);
    turn ^= 1;
    take_base += all;
    if (take && place < a.keep) k.kept[place] = i;
  }
  if (t == 0 && take_base != a.keep) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
  __syncthreads();
  // entry j takes over entry kept[j] >= j: a tile is read as a whole before it is written
  for (int j0 = 0; j0 < k.counted; j0 += NT) {
    const int j = j0 + t;
    float v = 0.f;
    if (j < a.keep && j < k.counted) {
      const int i = k.kept[j];
      v = i < k.counted ? k.w[i] : 0.f;
    }
    __syncthreads();
    if (j < k.counted) k.w[j] = v;
  }
}

// grid (2 * slices, B * KV, layers): a CTA moves a range of columns of all rows of K or V of one head, in ascending batches of rows that are read as a
// whole before they are written. Sources lie at or behind their targets, so no batch reads what an earlier one wrote, and in place is safe. The places of a
// batch's rows are looked up once per row, while the rows of the batch in front are on their way (looked up by every thread for itself: 16 sequences of 2,304 rows in
// 36 layers 2,509 us instead of 1,590). 9.6 GB in 1,470 us, the copy rate; 288 heads of 1,024 rows 50 us, 47 at the copy rate. (Selection and move in one kernel: 1,850 us. Registers
// spill, and while one CTA of an SM selects, only the other moves.)
constexpr int kMoveThreads = 512, kMoveBatch = 8;
template <int UNIT>
__global__ void __launch_bounds__(kMoveThreads, 2) evict_move_kernel(const __grid_constant__ EvictArgs a, int slices, int most_lines) {
  using U = typename CopyUnit<UNIT>::type;
  pdl_trigger();
  pdl_wait();
  extern __shared__ int2 place[];  // [2][rows of a batch]: source and target row in the cache; target -1: the row stays
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
  for (int c = c0; c < c1; c += kMoveThreads) {
    const int width = min(kMoveThreads, c1 - c), lines = min(kMoveThreads / width, most_lines);  // rows side by side
    const int line = t / width, rows = lines * kMoveBatch;                                       // rows of a batch
    uint8_t* column = cache + static_cast<long long>(c + t % width) * UNIT;
    auto look_up = [&](int j0, int2* at) {
      for (int r = t; r < rows; r += kMoveThreads) {
        int2 p = make_int2(0, -1);
        if (j0 + r < n) {
          const int i = kept[j0 + r], j = j0 + r, ps = from[i / a.page], pd = to[j / a.page];
          if (ps < 0 || ps >= a.pages || pd < 0 || pd >= a.pages) {
            atomicCAS(a.status, kStatusOk, kStatusBadArgs);
          } else {
            p = make_int2((ps * a.KV + kvh) * a.page + i % a.page, (pd * a.KV + kvh) * a.page + j % a.page);
            if (p.x == p.y) p.y = -1;
          }
        }
        at[r] = p;
      }
    };
    look_up(0, place);
    __syncthreads();
    for (int j0 = 0, turn = 0; j0 < n; j0 += rows, turn ^= 1) {
      const int2* at = place + turn * rows;
      U v[kMoveBatch];
      int target[kMoveBatch];
#pragma unroll
      for (int q = 0; q < kMoveBatch; ++q) {
        const int2 p = line < lines ? at[q * lines + line] : make_int2(0, -1);
        target[q] = p.y;
        if (p.y >= 0) v[q] = *reinterpret_cast<const U*>(column + static_cast<long long>(p.x) * row_bytes);
      }
      if (j0 + rows < n) look_up(j0 + rows, place + (turn ^ 1) * rows);
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kMoveBatch; ++q)
        if (target[q] >= 0) *reinterpret_cast<U*>(column + static_cast<long long>(target[q]) * row_bytes) = v[q];
    }
    __syncthreads();
  }
}

}  // namespace

void launch_evict(const EvictArgs& a, int unit, cudaStream_t st) {
  if (a.B == 0 || a.layers == 0 || a.KV == 0) return;
  const dim3 heads(a.KV, a.B, a.layers);
  const long long most = static_cast<long long>(a.table_width) * a.page;  // rows of a sequence
  if (most <= 256 * 10) launch_pdl(evict_select_kernel<256, 10, 4>, heads, dim3(256), 0, st, a);
  else if (most <= 512 * 20) launch_pdl(evict_select_kernel<512, 20, 2>, heads, dim3(512), 0, st, a);
  else if (most <= 1024 * 36) launch_pdl(evict_select_kernel<1024, 36, 1>, heads, dim3(1024), 0, st, a);
  else launch_pdl(evict_select_long_kernel, heads, dim3(512), 0, st, a);
  // columns are cut (to 64 bytes at least) where there are too few heads to fill the GPU
  int wide = 0;
  for (int i = 0; i < a.layers; ++i) wide = a.layer[i].k_bytes > wide ? a.layer[i].k_bytes : wide;
  int slices = 1;
  while (slices < 8 && 2ll * slices * a.B * a.KV * a.layers < 2 * 148 && wide / (2 * slices) >= 64) slices *= 2;
  const dim3 grid(2 * slices, a.B * a.KV, a.layers);
  // rows of a batch: at most the threads' units in columns of the narrowest slice
  int narrow = wide;
  for (int i = 0; i < a.layers; ++i) {
    narrow = a.layer[i].k_bytes < narrow ? a.layer[i].k_bytes : narrow;
    narrow = a.layer[i].v_bytes < narrow ? a.layer[i].v_bytes : narrow;
  }
  const int units = narrow / unit / slices > 1 ? narrow / unit / slices : 1;
  const int lines = kMoveThreads / (units < kMoveThreads ? units : kMoveThreads);
  const size_t smem = static_cast<size_t>(2) * lines * kMoveBatch * sizeof(int2);
#define DLV_EVICT_MOVE(UU)                                                                                                                       \
  do {                                                                                                                                           \
    static PerDeviceOnce once;                                                                                                                   \
    if (once.first()) cudaFuncSetAttribute(evict_move_kernel<UU>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kMoveThreads * kMoveBatch * 8); \
    launch_pdl(evict_move_kernel<UU>, grid, dim3(kMoveThreads), smem, st, a, slices, lines);                                                     \
  } while (0)
  if (unit == 16) DLV_EVICT_MOVE(16);
  else if (unit == 4) DLV_EVICT_MOVE(4);
  else DLV_EVICT_MOVE(2);
#undef DLV_EVICT_MOVE
}

}  // namespace dlv
