// Launchers of beam search and of the bounded cache (beam.cu, evict.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dlv {

constexpr int kBeamMaxBeams = 32;        // beams of one request
constexpr int kBeamMaxPicks = 64;        // candidates returned per request
constexpr int kBeamMaxMerge = 8192;      // candidates of one request that the second kernel takes
constexpr int kBeamMoveTensors = 96;     // tensors of one launch of beam_reorder (the table travels as a kernel parameter)

struct BeamSelectArgs {
  const void* logits;  // [B * W, V], fp32 or bf16, rows ld elements apart
  long long ld;
  int V;
  const uint32_t* mask;  // allow-bits [B * W, mask_ld] or null
  int mask_ld;
  float softcap, inv_scale;
  const float* scores;  // [B, W]
  int B, W, K, splits, per;  // per: logits of one split
  float* part_m;             // [B * W, splits] maximum of the split (of the post-processed logits)
  double* part_sum;          // [B * W, splits] sum of exp(logit - maximum)
  float* cand_x;             // [B * W, splits, K] raw logits of the split's best, -inf: none
  int* cand_i;               // [B * W, splits, K] their tokens
  float* out_value;          // [B, K]
  long long *out_parent, *out_token;
};
// logits of fp32 (bf16: 0)
void launch_beam_select(const BeamSelectArgs& a, bool f32, cudaStream_t st);
// splits of a row of V logits, when there are `rows` rows
int beam_select_splits(int rows, int W, int K, int V);

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

// Adds the probabilities of a decode step to the weights: scores fp32 [B, H, S] (scaled and capped, -inf where masked), part_ml [B, H, splits, 2] of the
// attention kernel, used: its plan or null (then min_slices).
struct WeighArgs {
  const float* scores;
  const float* part_ml;
  const int* ctx;
  const int* used;
  const long long* slots;
  float* weights;  // [num_slots, KV, capacity]
  int* status;
  int B, H, KV, S, splits, window, min_slices, num_slots, capacity, max_ctx;
};
void launch_weigh(const WeighArgs& a, cudaStream_t st);

}  // namespace dlv
