// How decode attention over a 4-bit cache cuts its work, and where the partial results of its first launch lie for its second (kv4_decode.cu). Arithmetic on sizes only, the same on the host.
#pragma once

#ifdef __CUDACC__
#define DLV_KV4_HD __host__ __device__ __forceinline__
#else
#define DLV_KV4_HD inline
#endif

namespace dlv {

constexpr int kKv4Warps = 4;     // of a CTA
constexpr int kKv4MinTiles = 2;  // of a share

// A share of the tiles: tile i of the step belongs to warp i / per.
struct Kv4Shares {
  int total, per;
  DLV_KV4_HD Kv4Shares(int total_, int workers) : total(total_), per((total_ + workers - 1) / workers) {
    if (per < kKv4MinTiles) per = kKv4MinTiles;
  }
};

// The parts of a pair's result. Parts in order: of the first CTA that has some of it, one of each CTA in the middle, of the last; a CTA whose shares all lie inside the pair makes one of them.
struct Kv4Parts {
  int parts, n0, mid, w0, c0, c1, first, per;
  bool j0, j1;
  DLV_KV4_HD Kv4Parts(const Kv4Shares& shares, int first_, int n) : first(first_), per(shares.per) {
    const int last = first + n - 1, w1 = last / per, cta = kKv4Warps * per;
    w0 = first / per;
    c0 = w0 / kKv4Warps;
    c1 = w1 / kKv4Warps;
    auto joined = [&](int c) {
      const int lo = c * cta, hi = shares.total < lo + cta ? shares.total : lo + cta;
      return hi - lo > per && first <= lo && hi <= last + 1;
    };
    j0 = joined(c0);
    j1 = joined(c1);
    const int w_end = c0 * kKv4Warps + kKv4Warps - 1;
    n0 = j0 ? 1 : (w1 < w_end ? w1 : w_end) - w0 + 1;
    mid = c1 - c0 > 1 ? c1 - c0 - 1 : 0;
    parts = n > 0 ? n0 + mid + (c1 == c0 ? 0 : j1 ? 1 : w1 - c1 * kKv4Warps + 1) : 0;
  }
  DLV_KV4_HD int number(int w) const {  // of the part that warp w (or its CTA) makes
    const int c = w / kKv4Warps;
    return c == c0 ? (j0 ? 0 : w - w0) : c < c1 ? n0 + c - c0 - 1 : n0 + mid + (j1 ? 0 : w - c1 * kKv4Warps);
  }
  DLV_KV4_HD int maker(int i) const {  // the (first) warp that makes part i, and which of its two parts that is
    const bool middle = i >= n0 && i < n0 + mid, own = i < n0 ? !j0 : !middle && !j1;
    const int w = i < n0 ? (j0 ? c0 * kKv4Warps : w0 + i) : middle ? (c0 + 1 + i - n0) * kKv4Warps : c1 * kKv4Warps + (i - n0 - mid);
    return w * 2 + (own && first >= w * per ? 1 : 0);
  }
  DLV_KV4_HD int most(int count) const { return count < parts ? count : parts; }  // parts to look at, of `count` that a pair is said to have
};
// Where part i of a pair lies, in [G, D] rows of the workspace, for kv4_merge_kernel: the first `near` of every pair next to one another, so that the second launch can fetch them before it knows how many there are; the
// others with the warp that makes them (`maker`).
DLV_KV4_HD long long kv4_place(int pairs, int near, int pair, int i, long long maker) {
  return i < near ? static_cast<long long>(pair) * near + i : static_cast<long long>(pairs) * near + maker;
}
// Partial results that have a place.
DLV_KV4_HD long long kv4_decode_parts(int ctas, int pairs, int near) { return static_cast<long long>(ctas) * kKv4Warps * 2 + static_cast<long long>(pairs) * near; }

}  // namespace dlv
