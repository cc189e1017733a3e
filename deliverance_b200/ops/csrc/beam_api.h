// Launchers of beam search and of the bounded cache (beam.cu, evict.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "divisor.h"

namespace dlv {

constexpr int kBeamMaxBeams = 32;        // beams of one request
constexpr int kBeamMaxPicks = 64;        // candidates returned per request
constexpr int kBeamMoveTensors = 96;     // tensors of one launch of beam_reorder (the table travels as a kernel parameter)

struct BeamSelectArgs {
  const void* logits;  // [B * W, V], fp32 or bf16, rows ld elements apart
  long long ld;
  int V;
  const uint32_t* mask;  // allow-bits [B * W, mask_ld] or null
  int mask_ld;
  float softcap, inv_scale;
  const float* scores;  // [B, W]
  int B, W, K, splits, per;  // per: logits of one split, a multiple of 4,096
  int groups;                // groups of a row
  Divisor by_groups;
  float* part_m;             // [B * W, splits] maximum of the split (of the post-processed logits)
  double* part_sum;          // [B * W, splits] sum of exp(logit - maximum)
  float* group_max;          // [B * W, groups] largest raw logit of every group
  float* out_value;          // [B, K]
  long long *out_parent, *out_token;
};
// logits of fp32 (bf16: 0)
void launch_beam_select(const BeamSelectArgs& a, bool f32, cudaStream_t st);
int beam_select_group(bool f32);              // neighbouring logits of a group
int beam_select_splits(int rows, int V);      // CTAs per row of V logits, when there are `rows` rows
constexpr int kBeamSplitUnit = 4096;

// what one access of a copying kernel moves: 16, 4 or 2 bytes
template <int UNIT>
struct CopyUnit;
template <>
struct CopyUnit<16> {
  using type = uint4;
};
template <>
struct CopyUnit<4> {
  using type = uint32_t;
};
template <>
struct CopyUnit<2> {
  using type = unsigned short;
};

struct BeamMoveTensor {
  void* base;
  long long slot_bytes;  // bytes from one slot (page) to the next
  int segments;          // parts of a slot, slot_bytes / segments apart; of each the first rows * row_bytes bytes move
  int row_bytes;
};
struct BeamMoveArgs {
  BeamMoveTensor t[kBeamMoveTensors];
  const long long* slots;    // [B, W]
  const long long* parents;  // [B, W]
  const int* rows;           // [B], null: max_rows everywhere
  int* status;
  int n, W, num_slots, max_rows;
  bool paged;
};
// unit: bytes that one access moves (16, 4 or 2): all sizes and addresses are multiples of it
void launch_beam_move(const BeamMoveArgs& a, int B, int unit, cudaStream_t st);

// ---- bounded cache ----------------------------------------------------------------------------------------------------
constexpr int kEvictLayers = 96;  // layers of one launch (the table travels as a kernel parameter)

struct EvictLayer {
  void *k, *v;     // [pages, KV, page, D]
  float* weights;  // [slots, KV, capacity]
  int k_bytes, v_bytes;  // bytes of a row
};
struct EvictArgs {
  EvictLayer layer[kEvictLayers];
  const int* tables;      // [B, table_width]
  const int* out_tables;  // [B, out_width]
  const int* ctx;         // [B]
  const long long* slots; // [B]
  int* kept;              // [layers, B, KV, keep]
  int* lens;              // [B]
  int* status;
  int layers, B, KV, page, pages, num_slots, capacity, table_width, out_width, keep, recent;
};
// unit: bytes of one access (16, 4 or 2). Two launches.
void launch_evict(const EvictArgs& a, int unit, cudaStream_t st);

// Decode attention that adds its probabilities to the keys' weights (attention.cu).
constexpr int kWeighMaxSplits = 128;
struct WeighArgs {
  float* scores;          // [B, H, S] scaled and capped, -inf where masked; S: a multiple of 16
  float *part_ml, *part_o;  // [B, H, splits, 2], [B, H, splits, D]: with more than one split
  void* out;              // [B, H * D] bf16
  const int* ctx;
  const int* used;        // the plan's splits per sequence, or null: by length
  const long long* slots;
  float* weights;  // [num_slots, KV, capacity]
  int* status;
  int B, H, KV, D, S, splits, window, min_slices, num_slots, capacity, max_ctx, pages;
};
// 1: unsupported shape
int launch_decode_attention_weighted(const void* q, long long q_stride, const void* kc, const void* vc, const int* bt, int bt_stride, int page, float scale, float cap, WeighArgs a,
                                     cudaStream_t st);

}  // namespace dlv
