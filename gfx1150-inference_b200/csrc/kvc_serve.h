// Head norms with rotation, shared prefixes and eviction on the paged pool: what their host
// side (kvc_serve_host.cpp) hands to their kernels (kvc_serve.cu; shared prefixes are work
// for the kernels of kvc_tree.cu).
#pragma once

#include <vector>

#include "kvc_spec.h"

namespace kvc {

constexpr int kMaxRopeAxes = 4;    // KVC_MAX_ROPE_AXES

struct NormRopeArgs {
  PagedView p;
  const uint8_t* q;                // (n, num_heads, D), rows q_stride bytes apart; may be null
  uint8_t* q_out;                  // (n, num_heads, D) packed
  const uint8_t* k_new;            // (n, num_kv_heads, D)
  const uint8_t* v_new;
  const uint8_t* q_weight;         // (D) or null: not normalised
  const uint8_t* k_weight;
  size_t q_stride, k_stride, v_stride;
  const int32_t* rows;             // (n) or null (row 0)
  const int32_t* positions;        // (n) slots in the cache; negative: padding, skipped
  const int32_t* rope_positions;   // (n, axes)
  int axes;
  int n;
  int num_heads;                   // 0 without q
  int head_dim;
  int pairs;                       // rotated pairs of a head, from its front
  float eps;
  double turns[kMaxRopePairs];     // inv_freq / 2 pi
  uint8_t axis[kMaxRopePairs];
};
// neox: pair j is dims j and j + pairs, else 2 j and 2 j + 1.
cudaError_t launch_norm_rope(const NormRopeArgs& a, int dtype, bool neox, int sms, cudaStream_t s);

struct EvictArgs {
  PagedView p;                     // layer 0
  size_t layer_bytes;
  int n_layers;
  const int32_t* rows;             // (n) or null (row i)
  const int32_t* ctx;              // (n) cached positions
  const float* weights;            // (n_layers, weight_rows, num_kv_heads, weight_slots)
  float* weights_out;              // the same shape; may be `weights`
  int weight_rows, weight_slots;
  int32_t* kept;                   // (n_layers, n, num_kv_heads, budget)
  int n, budget, recent;
};
cudaError_t launch_evict(const EvictArgs& a, int sms, cudaStream_t s);

}  // namespace kvc

// Work list of one decode step over shared prefixes (kvc_plan_shared), used by every layer.
struct kvc_shared_plan {
  kvc_tree_plan t;                 // its pieces, their partials and its upload
};
