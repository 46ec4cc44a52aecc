// Drafted-token and beam operators of the paged pool: what their host side
// (kvc_spec_host.cpp) hands to their kernels (kvc_spec.cu, kvc_tree.cu, kvc_beam.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>
#include <exception>
#include <new>
#include <vector>

#include "kvc_common.h"
#include "kvc_internal.h"
#include "kvcache.h"

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
// One piece of work of one CTA: tiles [tile0, tile1) of the positions from `base` (a whole
// number of slabs) to ctx + nodes of one block-table row, for one KV head and a block of
// (node, q-head) rows.  Row r is node r / group, q-head kvh * group + r % group; node n is
// token tok0 + n of the batch.  Every row sees the positions below ctx, the mask names
// those that it sees of the `nodes` behind them.
struct alignas(16) TreeSeg {
  int bt_row, ctx, nodes, tok0;
  int kvh, row0, rows, tile0;
  int tile1, part, base;         // part: first row of its partials, -1: writes the output
  int scores;                    // 16 floats: where row 0's scores start (TreeArgs::scores),
                                 // -1: not kept
};
// Rows whose partials are joined: n_parts pieces, `rows` partial rows apart.
struct alignas(16) TreeMerge {
  int part, n_parts, tok0, row0;
  int kvh, rows, pad0, pad1;
};

// The pieces of one row run: partial rows `part` on, n pieces `rows` partial rows apart, the
// run's first row at `row` of each.  Of the decode kernel: its n splits from `part` on.
struct JoinPieces {
  int part, n, rows, row;
};
// Rows of one sequence and KV head: token, first q-head and number of q-heads.
struct alignas(16) SharedJoin {
  JoinPieces prefix, own;
  int token, head, rows, pad;
};
// Slots of one (sequence, KV head) whose weights are added up: kWeighSlots from slot0 on from
// kept scores, kRecountSlots where they are computed again.
constexpr int kWeighSlots = 1024, kRecountSlots = 128;
struct alignas(16) TreeWeigh {
  int bt_row, ctx, nodes, tok0;
  int kvh, slot0, scores;        // scores: as in TreeSeg
  int chain;                     // of its first row block in TreeArgs::chains
};
constexpr int kMergeThreads = 256;
// (token, q-head) rows up to which a sequence keeps its scores on the tensor cores (measured
// beside recount_mma_kernel).
constexpr int kKeepRows = 32;

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
  const SharedJoin* joins;       // instead of merges, for shared prefixes
  int n_joins;
  // Own positions that the decode kernel attends to: its partial states, (splits, H, D) and
  // (splits, H), and the counter of its work list, which the join re-arms; null: none.
  const float* own_o;
  const float2* own_ml;
  unsigned int* own_queue;
  // Attention that adds its weights up (null otherwise): where the sums go, (table rows, KV
  // heads, weight_slots), every row's final (max, sum), and kept raw scores.
  float* weights;
  unsigned int* gave_up;         // set where a wait gave up: no weights until the plan is built again
  float2* row_ml;                // (tokens, H)
  float* scores;
  const TreeWeigh* weighs;       // those with kept scores, then those without
  int n_weighs, n_recounts;
  // The pieces that a row block's statistics are joined from (none: they are in row_ml), one
  // for each chain_rows rows of a (sequence, KV head); with own_o: one for each token.
  const JoinPieces* chains;
  int chain_rows;
  int weight_slots;
  float score_scale;             // what a kept score is multiplied by, log2 units
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
cudaError_t launch_shared_join(const TreeArgs& a, cudaStream_t s);
// CTAs that take one of a.merges.
inline int merge_ctas(const TreeArgs& a, size_t elem) {
  const int per = a.max_merge_rows * static_cast<int>(a.head_dim * elem / 16);
  return (per + kMergeThreads - 1) / kMergeThreads;
}
// The joins and the weights of what has just been attended to.
cudaError_t launch_weigh(const TreeArgs& a, const TreeTile& t, cudaStream_t s);

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

// Dynamic shared memory opt-in, once per kernel, device and size.
template <auto Kernel>
cudaError_t allow_smem(size_t smem) {
  static std::atomic<size_t> done[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_acquire) >= smem) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem));
  if (e == cudaSuccess && dev >= 0 && dev < 64) {
    size_t cur = done[dev].load(std::memory_order_relaxed);
    while (cur < smem && !done[dev].compare_exchange_weak(cur, smem)) {
    }
  }
  return e;
}

// Asks for the attention kernels' split of shared memory and L1, once per kernel and device.
template <auto Kernel>
cudaError_t prefer_shared() {
  static std::atomic<bool> done[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_acquire))) return e;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                           cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
  return e;
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
// What the attention kernels take of a call, without its mask and its joins.
int tree_args(const kvc_pool* pool, const kvc_tree_plan* plan, int layer, const void* d_q,
              void* d_out, const int32_t* d_bt, int bt_stride, float scale, TreeArgs* out);
// A plan is not built while its stream is being captured.
int refuse_capture(cudaStream_t s, const char* what);
// d_weights: null, or (weight_rows, KV heads, weight_slots) sums that the weights are added to.
int do_decode_tree(kvc_pool* pool, const kvc_tree_plan* plan, int layer, const void* d_q,
                   const int32_t* d_mask, int mask_words, void* d_out, const int32_t* d_bt,
                   int bt_stride, float scale, cudaStream_t s, float* d_weights = nullptr,
                   int weight_rows = 0, int weight_slots = 0);

// Floats that the scores of one plan take at most.
constexpr int64_t kMaxScores = 1ll << 30;
// Cuts whole runs (tile0 0, tile1 their tiles) into the CTAs' shares; by_rows: counting what a
// tile costs by its rows.
void cut_runs(const std::vector<TreeSeg>& runs, const TreeTile& tile, int sms, bool by_rows,
              std::vector<TreeSeg>* segs, std::vector<int>* cta_segs);
// Work for the decode kernel: the positions [base[i], lens[i]) of query i in table row
// rows[i], in pieces that its warps take one after another.
struct UnitList {
  std::vector<int4> recs;            // three records a unit
  std::vector<JoinPieces> splits;    // of each query
  int n_splits = 0;
};
// A query with a base is joined with something else: its splits are partial states, were it
// but one.  longest: positions of a piece at most (rounded to whole pages), 0: as many as
// kvc_plan_decode takes.
void build_units(const PoolGeom& g, int group, int sms, const std::vector<int>& rows,
                 const std::vector<int>& base, const std::vector<int>& lens, int longest,
                 UnitList* out);
// Its arguments for units of `plan`, in a call whose attention takes `a`.  beside: it runs
// beside the launch ahead, an attention kernel that writes nothing that it reads, and which
// began behind everything that does.
DecodeArgs unit_args(const kvc_tree_plan* plan, const TreeArgs& a, bool beside);
// A plan's records go to its device buffer in one copy; dev[i]: where parts[i] will be.
struct PlanPart {
  const void* data;
  size_t bytes;
};
int upload_plan(kvc_tree_plan* p, const PlanPart* parts, int n, const uint8_t** dev, cudaStream_t s);

// No C++ exception leaves a C entry point.
template <typename F>
int guarded(const char* what, F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return set_error(KVC_ERR_RUNTIME, "%s: %s", what, e.what());
  } catch (...) {
    return set_error(KVC_ERR_RUNTIME, "%s: unknown exception", what);
  }
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int check_table(const int32_t* d_bt, int bt_rows, int bt_stride);
// The view of `layer` of a pool (its device is current).
int paged_view(const kvc_pool* pool, int layer, const int32_t* d_bt, int bt_rows, int bt_stride,
               PagedView* v);

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
  // kvc_tree_plan_set_weights: builds make room for the scores; has_scores: the last did
  bool keep_scores = false, has_scores = false;
  int n_weighs = 0, n_recounts = 0;
  const kvc::TreeWeigh* dev_weighs = nullptr;
  const kvc::JoinPieces* dev_chains = nullptr;   // of row blocks, then of single tokens
  int token_weigh0 = 0;
  // Work on the decode kernel: unit records and their counter, and the joins of its splits
  const int4* dev_units = nullptr;
  unsigned int* dev_queue = nullptr;
  unsigned int* dev_gave_up = nullptr;   // TreeArgs::gave_up
  const kvc::SharedJoin* dev_joins = nullptr;
  const int* dev_score_base = nullptr;
  int n_units = 0, n_unit_ctas = 0, n_joins = 0;
  kvc::DevBuf d_own_o, d_own_ml;
  kvc::DevBuf d_blob, d_part_o, d_part_ml, d_scores, d_row_ml;
  kvc::DevBuf d_layer;                 // activations of kvc_forward_layer_tree
  kvc::HostBuf h_stage;
  cudaEvent_t upload_done = nullptr;

  void release() {
    d_blob.release();
    d_part_o.release();
    d_part_ml.release();
    d_scores.release();
    d_row_ml.release();
    d_own_o.release();
    d_own_ml.release();
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
