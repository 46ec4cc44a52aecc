// Drafted-token and beam operators of the paged pool: what their host side
// (kvc_spec_host.cpp) hands to their kernels (kvc_spec.cu, kvc_tree.cu, kvc_beam.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <new>
#include <vector>

#include "kvc_common.h"
#include "kvc_internal.h"

struct kvc_tree_plan;

namespace kvc {

constexpr int kMaxTreeNodes = 256;  // KVC_MAX_TREE_NODES
constexpr int kMaxBeams = 16;       // KVC_MAX_BEAMS
constexpr int kMaxBeamOut = 32;     // KVC_MAX_BEAM_OUT

// One layer of a pool and the block tables that name its pages.
struct PagedView {
  uint8_t* k;
  uint8_t* v;
  const int32_t* block_tables;   // (bt_rows, bt_stride)
  int bt_rows;
  int bt_stride;
  int num_kv_heads;
  int page_size;
  int num_pages;
  int row_units;                 // head_dim * elem_size / 16
  int layout;
  size_t page_head_bytes;
  uint32_t* err;                 // device error word
};

struct AppendRopeArgs {
  PagedView p;
  const uint8_t* q;              // (n, num_heads, D), rows q_stride bytes apart; may be null
  uint8_t* q_out;                // (n, num_heads, D) packed
  const uint8_t* k_new;          // (n, num_kv_heads, D)
  const uint8_t* v_new;
  size_t q_stride, k_stride, v_stride;
  const int32_t* rows;           // (n) or null (row 0)
  const int32_t* positions;      // (n) slots in the cache; negative: padding, skipped
  const int32_t* rope_positions; // (n) angles, or null (positions)
  int n;
  int num_heads;                 // 0 without q
  int head_dim;
  int dtype;
  int neox;
  int sms;                       // of the device
  double turns[kMaxRopePairs];   // inv_freq / 2 pi
};

struct CommitArgs {
  PagedView p;                   // layer 0 of the range
  size_t layer_bytes;
  int n_layers;
  const int32_t* rows;           // (n) or null (row i)
  const int32_t* ctx;            // (n) first slot of the drafted rows
  const int32_t* paths;          // (n, path_stride) node numbers, ascending
  const int32_t* path_lens;      // (n)
  int path_stride;
  int n;
};

struct ReorderArgs {
  PagedView p;                   // layer 0
  int32_t* tables;               // p.block_tables, written
  size_t layer_bytes;
  int n_layers;
  const int32_t* parents;        // (n, beams) beam numbers within the sequence
  const int32_t* ctx;            // (n) positions every beam of the sequence has cached
  int n;
  int beams;
};

// ---- tree attention -----------------------------------------------------------------
// One piece of work of one CTA: tiles [tile0, tile1) of the positions of one
// sequence for one KV head and a block of its (node, q-head) rows.  Row r of the
// sequence is node r / group, q-head kvh * group + r % group.
struct alignas(16) TreeSeg {
  int bt_row, ctx, nodes, tok0;
  int kvh, row0, rows, tile0;
  int tile1, part, pad0, pad1;   // part: first row of its partials, -1: writes the output
};
// Rows whose partials are joined: n_parts pieces, `rows` partial rows apart.
struct alignas(16) TreeMerge {
  int part, n_parts, tok0, row0;
  int kvh, rows, pad0, pad1;
};

struct TreeArgs {
  PagedView p;
  const void* q;                 // (tokens, H, D)
  void* out;
  const uint32_t* mask;          // (tokens, mask_words), or null: node i sees nodes 0 .. i
  int mask_words;
  const TreeSeg* segs;
  const int* cta_segs;           // (n_ctas + 1) segments of each CTA
  const TreeMerge* merges;
  int n_ctas, n_merges, max_merge_rows;
  float* part_o;                 // (partial rows, D), unnormalised
  float2* part_ml;               // (partial rows) max (log2 units) and sum
  int num_heads, group, head_dim, dtype;
  float scale_log2;
};

// Tile shape of the kernel a batch takes: positions per tile and rows per block.
struct TreeTile {
  int positions, rows;
  int ctas_per_sm;
  int piece_cost;                // start and end of a piece of work, in tiles
  bool tensor;                   // tcgen05 kernel
};
// small_tiles: how many tiles of 32 rows x 32 positions (kTreeSmall) the batch has.
constexpr int kTreeSmall = 32;
TreeTile tree_tile(const PoolGeom& g, int64_t small_tiles, int sms);
cudaError_t launch_tree(const TreeArgs& a, const TreeTile& t, cudaStream_t s);

// ---- beam selection ---------------------------------------------------------------------
struct BeamArgs {
  const uint8_t* logits;         // (n * beams, vocab), rows row_bytes apart
  size_t row_bytes;
  int dtype;
  const float* cum;              // (n, beams)
  int n, beams, vocab, n_out;
  int sms;                       // of the device
  int32_t* tokens;               // (n, n_out)
  int32_t* parents;
  float* scores;
  // workspace: per (row, chunk) the max, the sum and the n_out best candidates
  int n_chunks, batches;         // set by the launcher: chunks of a row, batches of a warp
  float2* ml;
  uint64_t* cand;
};
int beam_chunks(int vocab);   // at most
cudaError_t launch_beam_select(BeamArgs a, cudaStream_t s);

// A launch that may begin before the one ahead of it has ended.  The kernels launched so
// touch what others do only behind wait_prerequisites(); where each lets its own successor
// begin is said beside them.
template <typename A>
cudaError_t launch_early(void (*kernel)(A), dim3 grid, int threads, size_t smem, cudaStream_t s,
                         const A& args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args);
}

cudaError_t launch_append_rope(const AppendRopeArgs& a, cudaStream_t s);
cudaError_t launch_commit(const CommitArgs& a, cudaStream_t s);
cudaError_t launch_reorder(const ReorderArgs& a, cudaStream_t s);

// Shared by the entry points and the layer pipeline.
int do_append_rope(kvc_pool* pool, int layer, const void* d_q, int q_stride, void* d_q_out,
                   int num_heads, const void* d_k_new, int k_stride, const void* d_v_new,
                   int v_stride, const int32_t* d_bt, int bt_rows, int bt_stride,
                   const int32_t* d_rows, const int32_t* d_positions,
                   const int32_t* d_rope_positions, int n, float freq_base, int neox,
                   cudaStream_t s);
// The plan, the layer and the sizes of a call, before anything of it is launched.
int check_tree_call(const kvc_pool* pool, const kvc_tree_plan* plan, int layer,
                    const int32_t* d_mask, int mask_words, int bt_stride, float scale);
int do_decode_tree(kvc_pool* pool, const kvc_tree_plan* plan, int layer, const void* d_q,
                   const int32_t* d_mask, int mask_words, void* d_out, const int32_t* d_bt,
                   int bt_stride, float scale, cudaStream_t s);

// The device current at construction comes back at the end of the scope.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (cudaGetDevice(&prev_) != cudaSuccess) prev_ = -1;
    if (prev_ == device)
      prev_ = -1;   // nothing to put back
    else
      rc_ = use_device(device);
  }
  ~DeviceScope() {
    if (prev_ >= 0) cudaSetDevice(prev_);
  }
  DeviceScope(const DeviceScope&) = delete;
  int rc() const { return rc_; }

 private:
  int prev_ = -1;
  int rc_ = 0;
};

// Device error word of `device` (which is current); looked up once.
int device_error_word(int device, uint32_t** out);
// SMs of `device`; looked up once.
int sms_of(int device);

}  // namespace kvc

// Work list of one verification step (kvc_plan_tree), used by every layer.
struct kvc_tree_plan {
  bool valid = false;
  int device = -1;
  int n_seqs = 0, n_tokens = 0, num_heads = 0, max_nodes = 0, max_end = 0, max_row = 0;
  kvc::PoolGeom pool_geom;
  kvc::TreeTile tile{};
  int n_ctas = 0, n_merges = 0, max_merge_rows = 0;
  size_t part_rows = 0;
  const kvc::TreeSeg* dev_segs = nullptr;
  const int* dev_cta_segs = nullptr;
  const kvc::TreeMerge* dev_merges = nullptr;
  const int32_t* dev_rows = nullptr;   // (n_tokens) block-table row of each token
  const int32_t* dev_slots = nullptr;  // (n_tokens) cache slot of each token
  kvc::DevBuf d_blob, d_part_o, d_part_ml;
  kvc::DevBuf d_layer;                 // activations of kvc_forward_layer_tree
  kvc::HostBuf h_stage;
  cudaEvent_t upload_done = nullptr;

  void release() {
    d_blob.release();
    d_part_o.release();
    d_part_ml.release();
    d_layer.release();
    h_stage.release();
    if (upload_done) cudaEventDestroy(upload_done);
    upload_done = nullptr;
    valid = false;
  }
};

// Workspace of the beam selection.
struct kvc_beam {
  int device = 0;
  int max_seqs = 0, max_beams = 0, max_vocab = 0, max_out = 0;
  int sms = 0;
  kvc::DevBuf ws;
  size_t ml_bytes = 0;
};
