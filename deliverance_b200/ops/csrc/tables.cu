// Positions, cache slots, block tables, query tiles and last rows of a step, from the requests' lengths and page lists: one launch instead of a host loop over tokens and a copy per
// table.
#include "common.cuh"
#include "kv4_api.h"

namespace dlv {

// Every CTA adds the lengths up by itself (a few KB out of L2) and keeps where each request's rows and tiles begin in shared memory; threads then look up the request of their token, table
// entry or tile. What is inconsistent (negative lengths, rows without a page, tables too narrow, another number of tokens or tiles than announced) is reported, and written as
// slot -1, which the cache writers leave out. Kernels of a step read lengths and tiles in front of their wait for the kernel before them, so this one lets none start early: no trigger, and
// what it wrote is in L2 before a CTA leaves.
__global__ void __launch_bounds__(256) step_tables_kernel(const StepTablesArgs a) {
  pdl_wait();
  extern __shared__ int begin[];  // [2 * (S + 1)]: rows, tiles
  __shared__ int part[2][8], base[2];
  int *rows = begin, *tiles = begin + a.S + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 2) base[tid] = 0;
  bool bad = false;
  for (int s0 = 0; s0 < a.S; s0 += 256) {
    const int s = s0 + tid;
    int n = s < a.S ? a.fresh[s] : 0;
    bad = bad || n < 0 || n > a.T;
    n = max(0, min(n, a.T));
    const int own[2] = {n, (n + a.tile - 1) / a.tile};
    int sum[2] = {own[0], own[1]};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int v = __shfl_up_sync(0xffffffffu, sum[i], o);
        if (lane >= o) sum[i] += v;
      }
    }
    if (lane == 31) {
      part[0][warp] = sum[0];
      part[1][warp] = sum[1];
    }
    __syncthreads();
    int front[2] = {base[0], base[1]};
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < warp) {
        front[0] += part[0][w];
        front[1] += part[1][w];
      }
    }
    if (s < a.S) {
      rows[s] = front[0] + sum[0] - own[0];
      tiles[s] = front[1] + sum[1] - own[1];
    }
    __syncthreads();
    if (tid == 255) {
      base[0] = front[0] + sum[0];
      base[1] = front[1] + sum[1];
    }
    __syncthreads();
  }
  if (tid < 2) (tid == 0 ? rows : tiles)[a.S] = base[tid];
  __syncthreads();
  const int total = rows[a.S], n_tiles = tiles[a.S];
  bad = bad || total != a.T || (a.tiles > 0 && n_tiles != a.tiles);
  // the last request that begins at or in front of i
  auto owner = [&](const int* at, int i) {
    int lo = 0, hi = a.S;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (at[mid] <= i) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  const long long step = static_cast<long long>(gridDim.x) * 256, me = static_cast<long long>(blockIdx.x) * 256 + tid;
  for (long long t = me; t < a.T; t += step) {
    long long slot = -1;
    int pos = 0;
    if (t < total) {
      const int s = owner(rows, static_cast<int>(t)), off = static_cast<int>(t) - rows[s], row = a.cached[s] + off;
      const int p0 = a.page_start[s], p1 = a.page_start[s + 1], p = row / a.page;
      pos = a.start[s] + off;
      const bool ok = row >= 0 && p0 >= 0 && p < p1 - p0 && p1 <= a.n_pages;
      bad = bad || !ok;
      if (ok) slot = static_cast<long long>(a.pages[p0 + p]) * a.page + row % a.page;
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
  for (long long i = me; i < static_cast<long long>(a.S) * a.width; i += step) {
    const int s = static_cast<int>(i / a.width), c = static_cast<int>(i % a.width), p0 = a.page_start[s], p1 = a.page_start[s + 1];
    const bool ok = p0 >= 0 && p0 <= p1 && p1 <= a.n_pages && p1 - p0 <= a.width;
    bad = bad || !ok;
    a.tables[i] = ok && c < p1 - p0 ? a.pages[p0 + c] : 0;
  }
  for (long long i = me; i < a.tiles; i += step) {
    int s = 0, q0 = 0;
    if (i < n_tiles) {
      s = owner(tiles, static_cast<int>(i));
      q0 = (static_cast<int>(i) - tiles[s]) * a.tile;
    }
    a.tile_seq[i] = s;
    a.tile_q0[i] = q0;
  }
  for (long long s = me; s < a.S; s += step) {
    const int n = rows[s + 1] - rows[s];
    a.q_start[s] = rows[s];
    a.ctx_len[s] = a.cached[s] + n;
    a.last[s] = static_cast<long long>(rows[s]) + n - 1;
  }
  if (bad) atomicCAS(a.status, kStatusOk, kStatusBadArgs);
  __threadfence();
}

void launch_step_tables(const StepTablesArgs& a, cudaStream_t st) {
  if (a.S == 0) return;
  long long most = a.T;
  if (static_cast<long long>(a.S) * a.width > most) most = static_cast<long long>(a.S) * a.width;
  const size_t smem = 2 * (static_cast<size_t>(a.S) + 1) * sizeof(int);
  static PerDeviceOnce once;
  if (once.first()) cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * (kStepTablesMaxSeqs + 1) * static_cast<int>(sizeof(int)));
  const long long ctas = (most + 255) / 256;
  launch_pdl(step_tables_kernel, dim3(static_cast<unsigned>(ctas < 1 ? 1 : ctas > 296 ? 296 : ctas)), dim3(256), smem, st, a);
}

}  // namespace dlv
