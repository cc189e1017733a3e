// Launchers of the 4-bit KV cache (kv4.cu, kv4_decode.cu) and of step tables (tables.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "divisor.h"
#include "kv4_parts.h"

namespace dlv {

constexpr int kv4_row_bytes(int D) { return D / 2 + D / 8; }

struct Kv4WriteArgs {
  const void* qkv;  // bf16 rows of H + 2 KV heads, `pitch` elements apart
  long long pitch;
  const int* positions;      // [T]
  const long long* slots;    // [T]
  const void *q_norm, *k_norm;  // bf16 [D] or null
  const float *cos_t, *sin_t;   // [max_pos, half] or null
  void* q;                      // bf16 [T, H * D]
  uint8_t *k, *v;               // [pages, KV, page, row bytes]
  int* status;
  long long rows;  // pages * page
  Divisor by_page;
  int T, H, KV, D, page, half, max_pos;
  bool pairs;
  double eps;
  float offset;
};
void launch_kv4_write(const Kv4WriteArgs& a, cudaStream_t st);

struct Kv4ExpandArgs {
  const uint8_t *k, *v;  // [pages, KV, page, row bytes]
  const int* list;       // [n] pages
  void *ko, *vo;         // [n, KV, page, D]
  int* status;
  int n, pages, KV, page, D;
  bool f32;
};
void launch_kv4_expand(const Kv4ExpandArgs& a, cudaStream_t st);

struct Kv4SeqsArgs {
  const uint8_t *k, *v;
  const int* tables;  // [S, width]
  const int *ctx, *q_start, *q_len;  // [S]
  void *ko, *vo;      // fp16 [total * page / out_page, KV, out_page, D]
  int* out_tables;    // [S, width * page / out_page]
  int* status;
  long long T;        // query rows
  int S, width, longest, total, pages, KV, page, out_page, D, window;  // longest: pages of a sequence, at most
};
void launch_kv4_expand_seqs(const Kv4SeqsArgs& a, cudaStream_t st);

struct Kv4DecodeArgs {
  const void* q;  // bf16 [B, H * D], rows q_stride elements apart, 16-byte aligned
  long long q_stride;
  const uint8_t *k, *v;
  const int* tables;  // [B, width]
  const int* ctx;     // [B]
  void* out;          // bf16 [B, H * D]
  int* sums;          // [B + 1] 32-key tiles of a KV head in front of every sequence (written by the first launch for the second)
  int* counts;        // [B * KV] partial results of every (sequence, KV head) pair, -1: finished
  float *part_o, *part_ml;  // partial results, [G, D] and [G, 2]
  int near;           // as many of every pair lie next to one another
  int* status;
  int B, H, KV, D, page, pages, width, window;
  float scale, softcap;
};
constexpr int kKv4MaxCtas = 1024;
int kv4_decode_ctas(int B, int KV, int G, int D, long long rows, int sms);  // CTAs for sequences of up to `rows` keys
int kv4_decode_near(int ctas, int pairs);
void launch_kv4_decode(const Kv4DecodeArgs& a, int ctas, cudaStream_t st);  // two launches

struct StepTablesArgs {
  const int *pages, *page_start, *cached, *start, *fresh;  // [n_pages], [S + 1], [S], [S], [S]
  int *positions, *q_start, *ctx_len, *tables, *tile_seq, *tile_q0;
  long long *slots, *last;
  int* status;
  int S, T, n_pages, width, page, tile, tiles;
};
constexpr int kStepTablesMaxSeqs = 8192;
void launch_step_tables(const StepTablesArgs& a, cudaStream_t st);

}  // namespace dlv
