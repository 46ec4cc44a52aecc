// Host side of the drafted-token and beam operators: argument checks, the tree
// plan, the beam workspace and the C entry points.  Kernels: kvc_spec.cu,
// kvc_tree.cu, kvc_beam.cu.
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <exception>

#include "kvc_common.h"
#include "kvc_internal.h"
#include "kvc_spec.h"
#include "kvcache.h"

namespace kvc {

int device_error_word(int device, uint32_t** out) {
  static std::atomic<uint32_t*> words[64];
  if (device < 0 || device >= 64) return set_error(KVC_ERR_INVALID_ARG, "unknown device %d.", device);
  uint32_t* w = words[device].load(std::memory_order_acquire);
  if (!w) {
    void* p = nullptr;
    const cudaError_t e = device_error_address(&p);
    if (e != cudaSuccess) return cuda_error(e, "device error word");
    w = static_cast<uint32_t*>(p);
    words[device].store(w, std::memory_order_release);
  }
  *out = w;
  return KVC_OK;
}

int sms_of(int device) {
  static std::atomic<int> sms[64];
  if (device < 0 || device >= 64) return device_sms(device);
  int n = sms[device].load(std::memory_order_relaxed);
  if (n == 0) sms[device].store(n = device_sms(device), std::memory_order_relaxed);
  return n;
}

int check_table(const int32_t* d_bt, int bt_rows, int bt_stride) {
  if (!d_bt) return set_error(KVC_ERR_INVALID_ARG, "block tables must not be null.");
  if (bt_rows <= 0 || bt_stride <= 0)
    return set_error(KVC_ERR_INVALID_ARG, "block tables must have rows and columns.");
  return KVC_OK;
}

// The view of `layer` of a pool (its device is current).
int paged_view(const kvc_pool* pool, int layer, const int32_t* d_bt, int bt_rows, int bt_stride,
               PagedView* v) {
  const PoolGeom& g = pool->g;
  v->k = pool->k + static_cast<size_t>(layer) * g.layer_bytes;
  v->v = pool->v + static_cast<size_t>(layer) * g.layer_bytes;
  v->block_tables = d_bt;
  v->bt_rows = bt_rows;
  v->bt_stride = bt_stride;
  v->num_kv_heads = g.num_kv_heads;
  v->page_size = g.page_size;
  v->num_pages = g.num_pages;
  v->row_units = g.head_dim * g.elem_size / 16;
  v->layout = g.layout;
  v->page_head_bytes = g.page_head_bytes;
  return device_error_word(pool->device, &v->err);
}

int do_append_rope(kvc_pool* pool, int layer, const void* d_q, int q_stride, void* d_q_out,
                   int num_heads, const void* d_k_new, int k_stride, const void* d_v_new,
                   int v_stride, const int32_t* d_bt, int bt_rows, int bt_stride,
                   const int32_t* d_rows, const int32_t* d_positions,
                   const int32_t* d_rope_positions, int n, float freq_base, int neox,
                   cudaStream_t s) {
  const PoolGeom& g = pool->g;
  if (layer < 0 || layer >= g.num_layers)
    return set_error(KVC_ERR_OUT_OF_RANGE, "layer_idx out of range for the KV pool.");
  if (n < 0) return set_error(KVC_ERR_INVALID_ARG, "row count must be non-negative.");
  if (g.head_dim % 2 != 0)
    return set_error(KVC_ERR_INVALID_ARG, "head_dim must be a positive even integer for RoPE.");
  if (!(freq_base > 0.0f) || !std::isfinite(freq_base))
    return set_error(KVC_ERR_INVALID_ARG, "freq_base must be positive.");
  if (n == 0) return KVC_OK;
  if (!d_k_new || !d_v_new || !d_positions)
    return set_error(KVC_ERR_INVALID_ARG, "K/V rows and positions must not be null.");
  if (d_q && (!d_q_out || num_heads <= 0))
    return set_error(KVC_ERR_INVALID_ARG, "q needs its output and a positive head count.");
  if (int rc = check_table(d_bt, bt_rows, bt_stride)) return rc;
  if (!aligned16(d_q) || !aligned16(d_q_out) || !aligned16(d_k_new) || !aligned16(d_v_new))
    return set_error(KVC_ERR_INVALID_ARG, "q and K/V row buffers must be 16-byte aligned.");
  const int heads = d_q ? num_heads : 0;
  const int64_t q_row = static_cast<int64_t>(heads) * g.head_dim;
  const int64_t kv_row = static_cast<int64_t>(g.num_kv_heads) * g.head_dim;
  const int64_t qs = q_stride ? q_stride : q_row, ks = k_stride ? k_stride : kv_row;
  const int64_t vs = v_stride ? v_stride : kv_row;
  if ((d_q && qs < q_row) || ks < kv_row || vs < kv_row)
    return set_error(KVC_ERR_INVALID_ARG, "a token stride is smaller than its row.");
  if ((d_q && qs * g.elem_size % 16) || ks * g.elem_size % 16 || vs * g.elem_size % 16)
    return set_error(KVC_ERR_INVALID_ARG, "token strides must be multiples of 16 bytes.");
  if (d_q && d_q_out == d_q && qs != q_row)
    return set_error(KVC_ERR_INVALID_ARG, "q can be rotated in place only when it is packed.");
  AppendRopeArgs a = {};
  if (int rc = paged_view(pool, layer, d_bt, bt_rows, bt_stride, &a.p)) return rc;
  a.q = static_cast<const uint8_t*>(d_q);
  a.q_out = static_cast<uint8_t*>(d_q_out);
  a.k_new = static_cast<const uint8_t*>(d_k_new);
  a.v_new = static_cast<const uint8_t*>(d_v_new);
  a.q_stride = static_cast<size_t>(qs) * g.elem_size;
  a.k_stride = static_cast<size_t>(ks) * g.elem_size;
  a.v_stride = static_cast<size_t>(vs) * g.elem_size;
  a.rows = d_rows;
  a.positions = d_positions;
  a.rope_positions = d_rope_positions ? d_rope_positions : d_positions;
  a.n = n;
  a.num_heads = heads;
  a.head_dim = g.head_dim;
  a.dtype = g.dtype;
  a.neox = neox ? 1 : 0;
  a.sms = sms_of(pool->device);
  for (int i = 0; i < g.head_dim / 2; ++i)
    a.turns[i] = std::pow(static_cast<double>(freq_base), -2.0 * i / g.head_dim) /
                 6.283185307179586476925286766559;
  const cudaError_t e = launch_append_rope(a, s);
  return e == cudaSuccess ? KVC_OK : cuda_error(e, "append + rope kernel");
}

int check_tree_call(const kvc_pool* pool, const kvc_tree_plan* plan, int layer,
                    const int32_t* d_mask, int mask_words, int bt_stride, float scale) {
  const PoolGeom& g = pool->g;
  if (!plan->valid) return set_error(KVC_ERR_INVALID_ARG, "plan has not been built.");
  if (layer < 0 || layer >= g.num_layers)
    return set_error(KVC_ERR_OUT_OF_RANGE, "layer_idx out of range for the KV pool.");
  const PoolGeom& pg = plan->pool_geom;
  if (pg.head_dim != g.head_dim || pg.num_kv_heads != g.num_kv_heads ||
      pg.page_size != g.page_size || pg.dtype != g.dtype || plan->device != pool->device)
    return set_error(KVC_ERR_INVALID_ARG, "plan was built for a pool of another geometry.");
  if (plan->n_tokens == 0) return KVC_OK;
  if (d_mask && mask_words <= 0)
    return set_error(KVC_ERR_INVALID_ARG, "mask_words must be positive.");
  if (!std::isfinite(scale)) return set_error(KVC_ERR_INVALID_ARG, "scale must be finite.");
  if (bt_stride <= 0 || plan->max_end > static_cast<int64_t>(bt_stride) * g.page_size)
    return set_error(KVC_ERR_OUT_OF_RANGE, "a sequence exceeds the block-table width.");
  return KVC_OK;
}

int tree_args(const kvc_pool* pool, const kvc_tree_plan* plan, int layer, const void* d_q,
              void* d_out, const int32_t* d_bt, int bt_stride, float scale, TreeArgs* out) {
  const PoolGeom& g = pool->g;
  if (!d_q || !d_out || !d_bt)
    return set_error(KVC_ERR_INVALID_ARG, "q, out and block tables must not be null.");
  if (!aligned16(d_q) || !aligned16(d_out))
    return set_error(KVC_ERR_INVALID_ARG, "q and out must be 16-byte aligned.");
  TreeArgs& a = *out;
  if (int rc = paged_view(pool, layer, d_bt, plan->max_row + 1, bt_stride, &a.p)) return rc;
  a.q = d_q;
  a.out = d_out;
  a.segs = plan->dev_segs;
  a.cta_segs = plan->dev_cta_segs;
  a.n_ctas = plan->n_ctas;
  a.part_o = static_cast<float*>(plan->d_part_o.ptr);
  a.part_ml = static_cast<float2*>(plan->d_part_ml.ptr);
  a.num_heads = plan->num_heads;
  a.group = plan->num_heads / g.num_kv_heads;
  a.head_dim = g.head_dim;
  a.dtype = g.dtype;
  a.scale_log2 = scale * kLog2e;
  return KVC_OK;
}

int do_decode_tree(kvc_pool* pool, const kvc_tree_plan* plan, int layer, const void* d_q,
                   const int32_t* d_mask, int mask_words, void* d_out, const int32_t* d_bt,
                   int bt_stride, float scale, cudaStream_t s, float* d_weights, int weight_rows,
                   int weight_slots) {
  if (int rc = check_tree_call(pool, plan, layer, d_mask, mask_words, bt_stride, scale)) return rc;
  if (plan->n_tokens == 0) return KVC_OK;
  TreeArgs a = {};
  if (int rc = tree_args(pool, plan, layer, d_q, d_out, d_bt, bt_stride, scale, &a)) return rc;
  a.mask = reinterpret_cast<const uint32_t*>(d_mask);
  a.mask_words = d_mask ? mask_words : 0;
  a.merges = plan->dev_merges;
  a.n_merges = plan->n_merges;
  a.max_merge_rows = plan->max_merge_rows;
  if (d_weights) {
    if (!plan->has_scores)
      return set_error(KVC_ERR_INVALID_ARG, "the plan was built without kvc_tree_plan_set_weights.");
    if (plan->max_row >= weight_rows)
      return set_error(KVC_ERR_OUT_OF_RANGE, "a sequence's row is outside the weights.");
    if (plan->max_end > weight_slots)
      return set_error(KVC_ERR_OUT_OF_RANGE, "a sequence exceeds the weights' slots.");
    const size_t q_bytes = static_cast<size_t>(plan->n_tokens) * plan->num_heads * a.head_dim * pool->g.elem_size;
    const uintptr_t q0 = reinterpret_cast<uintptr_t>(d_q), o0 = reinterpret_cast<uintptr_t>(d_out);
    if (plan->n_recounts > 0 && q0 < o0 + q_bytes && o0 < q0 + q_bytes)
      return set_error(KVC_ERR_INVALID_ARG,
                       "out must not overlap q where rows are counted again from it.");
    a.scores = static_cast<float*>(plan->d_scores.ptr);
    a.row_ml = static_cast<float2*>(plan->d_row_ml.ptr);
    a.weighs = plan->dev_weighs;
    a.n_weighs = plan->n_weighs;
    a.chains = plan->dev_chains;
    a.chain_rows = plan->tile.rows;
    a.n_recounts = plan->n_recounts;
    a.weights = d_weights;
    a.gave_up = plan->dev_gave_up;
    a.weight_slots = weight_slots;
    // (the tensor cores' kernel takes the scale's sign into q)
    a.score_scale = plan->tile.tensor ? std::fabs(a.scale_log2) : a.scale_log2;
    if (plan->n_units > 0 && !d_mask) {
      DecodeArgs d = unit_args(plan, a, false);
      d.scores = a.scores;
      d.score_base = plan->dev_score_base;
      d.row_ml = a.row_ml;
      d.gave_up = a.gave_up;
      a.joins = plan->dev_joins;
      a.n_joins = plan->n_joins;
      a.own_o = d.part_o;
      a.own_ml = d.part_ml;
      a.own_queue = d.queue;
      a.score_scale = 1.0f;   // (that kernel keeps them scaled)
      a.weighs += plan->token_weigh0;
      cudaError_t e = launch_decode(d, a.dtype, a.p.layout, s);
      if (e == cudaSuccess) e = launch_weigh(a, plan->tile, s);
      return e == cudaSuccess ? KVC_OK : cuda_error(e, "weighed decode kernels");
    }
  }
  const cudaError_t e = launch_tree(a, plan->tile, s);
  return e == cudaSuccess ? KVC_OK : cuda_error(e, "tree attention kernel");
}

int refuse_capture(cudaStream_t s, const char* what) {
  // A captured upload would read the staging buffer at every replay, whatever a later build
  // has put there (the capture stays valid).
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  const cudaError_t e = cudaStreamIsCapturing(s, &cap);
  if (e != cudaSuccess) return cuda_error(e, "cudaStreamIsCapturing");
  if (cap != cudaStreamCaptureStatusNone)
    return set_error(KVC_ERR_INVALID_ARG,
                     "%s cannot be built on a stream that is being captured: build it "
                     "before the capture and capture the calls that use it.", what);
  return KVC_OK;
}

// The work list: the runs of position tiles are laid end to end and cut into shares of
// equal cost, one per CTA.  A run that falls into several shares is joined from its pieces'
// partials.
void cut_runs(const std::vector<TreeSeg>& runs, const TreeTile& tile, int sms, bool by_rows,
              std::vector<TreeSeg>* segs, std::vector<int>* cta_segs) {
  segs->clear();
  cta_segs->assign(1, 0);
  // A tile of a block that fills both streams of the tensor-core kernel costs twice one of a
  // block whose tiles the streams share.
  bool small = false, large = false;
  for (const TreeSeg& r : runs) (2 * r.rows > tile.rows ? large : small) = true;
  const int unit = by_rows && tile.tensor && tile.rows > 128 && small && large ? 2 : 1;
  auto weight = [&](const TreeSeg& r) { return 2 * r.rows > tile.rows ? unit : 1; };
  int64_t tiles = 0;
  for (const TreeSeg& r : runs) tiles += static_cast<int64_t>(r.tile1) * weight(r);
  const int64_t ctas = std::min<int64_t>(static_cast<int64_t>(sms) * tile.ctas_per_sm, tiles);
  // A piece costs its tiles and `pc` for its start and end; a CTA's pieces cost at most `limit`
  // together, give or take a pc: a cut that would leave less than that on either side moves
  // to the end of the run or of the share.  pc is tile.piece_cost where CTAs have many tiles
  // (4 against 1 there: 32 ragged trees 115 against 118 us), and less where they have few and
  // short pieces spread the work further (63 drafted tokens at 511: 16 us at 1, 22 at 4).
  // walk() lays the runs out for a limit, calls emit(run, tile, tiles) and close() for each
  // piece and each full share, and returns the number of shares.
  const int64_t pc = std::min<int64_t>(
      tile.piece_cost * unit, std::max<int64_t>(1, ctas > 0 ? tiles / (8 * ctas) : 1));
  auto walk = [&](int64_t limit, auto&& emit, auto&& close) {
    int64_t shares = 0, cost = 0;
    for (const TreeSeg& r : runs) {
      const int run = r.tile1, wt = weight(r);
      for (int t = 0; t < run;) {
        const int64_t room = (limit - cost - pc) / wt;
        if (cost > 0 && room < run - t && room < std::max<int64_t>(1, pc)) {
          close();
          ++shares;
          cost = 0;
          continue;
        }
        int take = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(run - t, room)));
        if (run - t - take < pc) take = run - t;
        emit(r, t, take);
        t += take;
        cost += static_cast<int64_t>(take) * wt + pc;
      }
    }
    return shares + (cost > 0 ? 1 : 0);
  };
  // the smallest limit that needs no more shares than there are CTAs
  auto fits = [&](int64_t limit) {
    return walk(limit, [](const TreeSeg&, int, int) {}, [] {}) <= ctas;
  };
  const int64_t n_runs = static_cast<int64_t>(runs.size());
  int64_t lo = 1, hi = 1;
  if (ctas > 0) {
    lo = std::max<int64_t>(1, (tiles + n_runs * pc) / ctas);
    for (hi = (tiles + (n_runs + ctas) * pc) / ctas + 1; !fits(hi);) hi *= 2;
  }
  while (lo < hi) {
    const int64_t mid = lo + (hi - lo) / 2;
    if (fits(mid))
      hi = mid;
    else
      lo = mid + 1;
  }
  walk(
      hi,
      [&](const TreeSeg& r, int t, int take) {
        TreeSeg sg = r;
        sg.tile0 = t;
        sg.tile1 = t + take;
        segs->push_back(sg);
      },
      [&] { cta_segs->push_back(static_cast<int>(segs->size())); });
  if (cta_segs->back() < static_cast<int>(segs->size()))
    cta_segs->push_back(static_cast<int>(segs->size()));
}

void build_units(const PoolGeom& g, int group, int sms, const std::vector<int>& rows,
                 const std::vector<int>& base, const std::vector<int>& lens, int longest,
                 UnitList* out) {
  const int n = static_cast<int>(lens.size()), chunks = (group + 7) / 8;
  std::vector<int> own(n), refine(n);
  for (int i = 0; i < n; ++i) own[i] = lens[i] - base[i];
  int C = split_partition_sms(g.page_size, own.data(), n, g.num_kv_heads * chunks, sms, refine.data());
  if (longest > 0 && C > longest) {
    C = (longest + g.page_size - 1) / g.page_size * g.page_size;
    std::fill(refine.begin(), refine.end(), 0);
  }
  out->splits.assign(n, JoinPieces{});
  std::vector<int4> items;
  for (int i = 0; i < n; ++i) {
    if (own[i] == 0) continue;
    out->splits[i].part = out->n_splits;
    out->splits[i].n = emit_splits(i, own[i], C, refine[i], [&](int4 it) {
      it.z += base[i];
      it.w += base[i];
      items.push_back(it);
    });
    out->n_splits += out->splits[i].n;
  }
  std::stable_sort(items.begin(), items.end(),
                   [](const int4& x, const int4& y) { return x.w - x.z > y.w - y.z; });
  for (const int4& it : items) {
    const int i = it.x;
    const int pieces = out->splits[i].n + (base[i] > 0 ? 1 : 0);   // (one: writes out itself)
    for (int kvh = 0; kvh < g.num_kv_heads; ++kvh)
      for (int c = 0; c < chunks; ++c) {
        out->recs.push_back(it);
        out->recs.push_back(make_int4(rows[i], lens[i], out->splits[i].part, pieces));
        out->recs.push_back(make_int4(kvh, c, kvh * group + c * 8, std::min(8, group - c * 8)));
      }
  }
}

DecodeArgs unit_args(const kvc_tree_plan* plan, const TreeArgs& a, bool beside) {
  DecodeArgs d = {};
  d.k_layer = a.p.k;
  d.v_layer = a.p.v;
  d.q = a.q;
  d.out = a.out;
  d.block_tables = a.p.block_tables;
  d.bt_stride = a.p.bt_stride;
  d.part_o = static_cast<float*>(plan->d_own_o.ptr);
  d.part_ml = static_cast<float2*>(plan->d_own_ml.ptr);
  d.sched_recs = plan->dev_units;
  d.n_units = d.n_items = d.sched_cap = plan->n_units;
  d.queue = plan->dev_queue;
  d.n_sched_ctas = plan->n_unit_ctas;
  d.early_prefetch = beside ? 2 : 0;
  d.num_heads = a.num_heads;
  d.num_kv_heads = a.p.num_kv_heads;
  d.group = a.group;
  d.n_hchunk = (a.group + 7) / 8;
  d.head_dim = a.head_dim;
  d.page_size = a.p.page_size;
  d.num_pages = a.p.num_pages;
  d.scale_log2 = a.scale_log2;
  d.no_merge = 1;
  return d;
}

int upload_plan(kvc_tree_plan* p, const PlanPart* parts, int n, const uint8_t** dev, cudaStream_t s) {
  cudaError_t e;
  auto al = [](size_t b) { return (b + 255) & ~static_cast<size_t>(255); };
  size_t total = 0;
  for (int i = 0; i < n; ++i) total += al(parts[i].bytes);
  if ((e = p->d_blob.ensure(total))) return cuda_error(e, "plan buffers");
  if (p->upload_done) {  // the staging is free once the previous upload has landed
    if (const int rc = wait_event(p->upload_done, "plan upload")) return rc;
  } else if ((e = cudaEventCreateWithFlags(&p->upload_done, cudaEventDisableTiming))) {
    return cuda_error(e, "cudaEventCreate");
  }
  if ((e = p->h_stage.ensure(total))) return cuda_error(e, "cudaMallocHost(plan)");
  uint8_t* h = static_cast<uint8_t*>(p->h_stage.ptr);
  size_t at = 0;
  for (int i = 0; i < n; ++i) {
    if (parts[i].bytes) memcpy(h + at, parts[i].data, parts[i].bytes);
    dev[i] = static_cast<const uint8_t*>(p->d_blob.ptr) + at;
    at += al(parts[i].bytes);
  }
  if ((e = cudaMemcpyAsync(p->d_blob.ptr, h, total, cudaMemcpyHostToDevice, s)))
    return cuda_error(e, "plan upload");
  if ((e = cudaEventRecord(p->upload_done, s))) return cuda_error(e, "cudaEventRecord(plan)");
  return KVC_OK;
}

namespace {

// Every (sequence, KV head, row block) is a run of position tiles.
int tree_build(kvc_tree_plan* p, const kvc_pool* pool, const int32_t* h_rows,
               const int32_t* h_ctx, const int32_t* h_nodes, int n_seqs, int num_heads,
               cudaStream_t s) {
  const PoolGeom& g = pool->g;
  if (n_seqs < 0) return set_error(KVC_ERR_INVALID_ARG, "n_seqs must be non-negative.");
  if (n_seqs > 0 && (!h_ctx || !h_nodes))
    return set_error(KVC_ERR_INVALID_ARG, "ctx_lens and node_counts must not be null.");
  if (num_heads <= 0 || num_heads % g.num_kv_heads != 0)
    return set_error(KVC_ERR_INVALID_ARG, "num_heads must be divisible by num_kv_heads.");
  p->valid = false;
  const int group = num_heads / g.num_kv_heads, sms = sms_of(pool->device);
  int64_t tokens = 0, tiles = 0, scores = 0, max_end = 0, small = 0;
  int max_row = 0, max_nodes = 0;
  std::vector<int32_t> rows, slots;
  std::vector<int> seen;
  for (int i = 0; i < n_seqs; ++i) {
    const int row = h_rows ? h_rows[i] : i;
    if (h_ctx[i] < 0) return set_error(KVC_ERR_INVALID_ARG, "context length must be non-negative.");
    if (row < 0) return set_error(KVC_ERR_INVALID_ARG, "block-table row must be non-negative.");
    if (h_nodes[i] < 0 || h_nodes[i] > kMaxTreeNodes)
      return set_error(KVC_ERR_INVALID_ARG, "node counts must be in [0, %d].", kMaxTreeNodes);
    const int64_t end = static_cast<int64_t>(h_ctx[i]) + h_nodes[i];
    if (end > (1ll << 30)) return set_error(KVC_ERR_INVALID_ARG, "a sequence is too long.");
    for (int t = 0; t < h_nodes[i]; ++t) {
      rows.push_back(row);
      slots.push_back(h_ctx[i] + t);
    }
    tokens += h_nodes[i];
    if (h_nodes[i] > 0) max_end = std::max(max_end, end);
    max_row = std::max(max_row, row);
    if (p->keep_scores && h_nodes[i] > 0) seen.push_back(row);
    max_nodes = std::max(max_nodes, h_nodes[i]);
    small += (static_cast<int64_t>(h_nodes[i]) * group + kTreeSmall - 1) / kTreeSmall *
             g.num_kv_heads * ((end + kTreeSmall - 1) / kTreeSmall);
  }
  std::sort(seen.begin(), seen.end());
  const bool rows_apart = std::adjacent_find(seen.begin(), seen.end()) == seen.end();
  const TreeTile tile = tree_tile(g, small, sms);
  auto keeps = [&](int nodes) { return p->keep_scores && (!tile.tensor || nodes * group <= kKeepRows); };
  for (int i = 0; i < n_seqs; ++i) {
    const int64_t blocks = (static_cast<int64_t>(h_nodes[i]) * group + tile.rows - 1) / tile.rows;
    const int64_t end = static_cast<int64_t>(h_ctx[i]) + h_nodes[i];
    tiles += blocks * g.num_kv_heads * ((end + tile.positions - 1) / tile.positions);
    if (keeps(h_nodes[i])) scores += static_cast<int64_t>(h_nodes[i]) * num_heads * ((end + 15) / 16);
  }
  if (tokens * num_heads > (1ll << 30) || tiles > (1ll << 30))
    return set_error(KVC_ERR_INVALID_ARG, "the batch is too large for one plan.");
  if (p->keep_scores && scores > kMaxScores / 16)
    return set_error(KVC_ERR_INVALID_ARG, "the batch keeps more scores than one plan holds (2^30).");
  if (p->keep_scores && !rows_apart)
    return set_error(KVC_ERR_INVALID_ARG,
                     "two sequences of one block-table row cannot add their weights up together.");
  std::vector<TreeSeg> runs, segs;
  std::vector<TreeMerge> merges;
  std::vector<TreeWeigh> weighs, recounts;
  std::vector<int> cta_segs;
  int tok0 = 0, score0 = 0;
  for (int i = 0; i < n_seqs; tok0 += h_nodes[i++]) {
    const int n_rows = h_nodes[i] * group, end = h_ctx[i] + h_nodes[i];
    for (int kvh = 0; kvh < g.num_kv_heads && n_rows > 0; ++kvh) {
      TreeSeg sg = {};
      sg.bt_row = h_rows ? h_rows[i] : i;
      sg.ctx = h_ctx[i];
      sg.nodes = h_nodes[i];
      sg.tok0 = tok0;
      sg.kvh = kvh;
      sg.tile1 = (end + tile.positions - 1) / tile.positions;
      sg.part = -1;
      if (p->keep_scores) {
        const bool keep = keeps(h_nodes[i]);
        sg.scores = keep ? score0 : -1;
        if (keep) score0 += n_rows * ((end + 15) / 16);
        std::vector<TreeWeigh>& list = keep ? weighs : recounts;
        for (int slot = 0; slot < end; slot += keep ? kWeighSlots : kRecountSlots)
          list.push_back(TreeWeigh{sg.bt_row, sg.ctx, sg.nodes, sg.tok0, kvh, slot, sg.scores,
                                   static_cast<int>(runs.size())});
      }
      for (int r0 = 0; r0 < n_rows; r0 += tile.rows) {
        sg.row0 = r0;
        sg.rows = std::min(tile.rows, n_rows - r0);
        runs.push_back(sg);
      }
    }
  }
  cut_runs(runs, tile, sms, p->keep_scores, &segs, &cta_segs);
  // Single tokens whose weights are wanted: the decode kernel streams K and V faster for a
  // token's few rows (32 x 1 at 1K-8K, fp16: 92 us, 105 with the kernel for trees) and keeps
  // scores at less cost (98, 125).  The pieces above serve calls with a mask.
  UnitList units;
  std::vector<SharedJoin> joins;
  std::vector<int> score_base;
  if (p->keep_scores && tile.tensor && max_nodes == 1 && group <= kKeepRows) {
    std::vector<int> unit_rows, lens;
    for (int i = 0; i < n_seqs; ++i) {
      if (h_nodes[i] == 0) continue;
      unit_rows.push_back(h_rows ? h_rows[i] : i);
      lens.push_back(h_ctx[i] + 1);
    }
    build_units(g, group, sms, unit_rows, std::vector<int>(lens.size(), 0), lens, 0, &units);
    for (size_t t = 0; t < lens.size(); ++t)
      for (int kvh = 0; kvh < g.num_kv_heads && units.splits[t].n > 1; ++kvh) {
        SharedJoin j = {};
        j.prefix.rows = j.own.rows = 1;
        j.own = units.splits[t];
        j.token = static_cast<int>(t);
        j.head = kvh * group;
        j.rows = group;
        joins.push_back(j);
      }
    for (const TreeWeigh& w : weighs)
      if (w.kvh == 0 && w.slot0 == 0) score_base.push_back(w.scores);
  }
  // runs in several pieces are joined from their partials
  std::vector<JoinPieces> chains(p->keep_scores ? runs.size() : 0);
  size_t part_rows = 0, run = 0;
  int max_merge_rows = 0;
  for (size_t first = 0; first < segs.size(); ++run) {
    size_t next = first + 1;
    while (next < segs.size() && segs[next].tile0 > 0) ++next;
    if (next - first > 1) {
      const TreeSeg& sg = segs[first];
      TreeMerge m = {};
      m.part = static_cast<int>(part_rows);
      m.n_parts = static_cast<int>(next - first);
      m.tok0 = sg.tok0;
      m.row0 = sg.row0;
      m.kvh = sg.kvh;
      m.rows = sg.rows;
      merges.push_back(m);
      max_merge_rows = std::max(max_merge_rows, sg.rows);
      if (p->keep_scores) chains[run] = JoinPieces{m.part, m.n_parts, sg.rows, 0};
      for (size_t k = first; k < next; ++k) {
        segs[k].part = static_cast<int>(part_rows);
        part_rows += sg.rows;
      }
    }
    first = next;
  }
  p->n_seqs = n_seqs;
  p->n_tokens = static_cast<int>(tokens);
  p->num_heads = num_heads;
  p->max_nodes = max_nodes;
  p->max_end = static_cast<int>(max_end);
  p->max_row = max_row;
  p->tile = tile;
  p->n_ctas = static_cast<int>(cta_segs.size()) - 1;
  p->n_merges = static_cast<int>(merges.size());
  p->max_merge_rows = max_merge_rows;
  p->part_rows = part_rows;
  p->n_weighs = static_cast<int>(weighs.size());
  p->n_recounts = static_cast<int>(recounts.size());
  // (those with the most rows first: the last CTAs are short ones)
  std::stable_sort(recounts.begin(), recounts.end(),
                   [](const TreeWeigh& x, const TreeWeigh& y) { return x.nodes > y.nodes; });
  weighs.insert(weighs.end(), recounts.begin(), recounts.end());
  p->has_scores = p->keep_scores;
  p->n_joins = static_cast<int>(joins.size());
  p->n_units = static_cast<int>(units.recs.size() / 3);
  p->n_unit_ctas = std::min(sms * kPersistCtasPerSm, (p->n_units + kPersistWarps - 1) / kPersistWarps);
  p->pool_geom = g;
  p->device = pool->device;
  if (tokens == 0) {
    p->valid = true;
    return KVC_OK;
  }
  cudaError_t e;
  if ((e = p->d_part_o.ensure(sizeof(float) * std::max<size_t>(1, part_rows) * g.head_dim)) ||
      (e = p->d_part_ml.ensure(sizeof(float2) * std::max<size_t>(1, part_rows))))
    return cuda_error(e, "plan buffers");
  if (p->keep_scores &&
      ((e = p->d_scores.ensure(sizeof(float) * 16 * static_cast<size_t>(std::max(1, score0)))) ||
       (e = p->d_row_ml.ensure(sizeof(float2) * static_cast<size_t>(tokens) * num_heads))))
    return cuda_error(e, "plan buffers");
  const size_t split_rows = std::max<size_t>(1, units.n_splits) * num_heads;
  if (!units.recs.empty() && ((e = p->d_own_o.ensure(sizeof(float) * split_rows * g.head_dim)) ||
                              (e = p->d_own_ml.ensure(sizeof(float2) * split_rows))))
    return cuda_error(e, "plan buffers");
  // (single tokens: their weighs again, with the tokens' chains, behind those of the row blocks)
  p->token_weigh0 = static_cast<int>(weighs.size());
  if (!units.recs.empty()) {
    for (int i = 0; i < p->n_weighs; ++i) {
      TreeWeigh w = weighs[i];
      w.chain = static_cast<int>(chains.size()) + w.tok0;
      weighs.push_back(w);
    }
    chains.insert(chains.end(), units.splits.begin(), units.splits.end());
  }
  const unsigned int zero = 0, gave_up = injected_failure(KVC_FAULT_KERNEL_WAIT);
  const PlanPart parts[] = {{segs.data(), sizeof(TreeSeg) * segs.size()},
                            {cta_segs.data(), sizeof(int) * cta_segs.size()},
                            {merges.data(), sizeof(TreeMerge) * merges.size()},
                            {rows.data(), sizeof(int32_t) * rows.size()},
                            {slots.data(), sizeof(int32_t) * slots.size()},
                            {weighs.data(), sizeof(TreeWeigh) * weighs.size()},
                            {joins.data(), sizeof(SharedJoin) * joins.size()},
                            {units.recs.data(), sizeof(int4) * units.recs.size()},
                            {score_base.data(), sizeof(int) * score_base.size()},
                            {&zero, sizeof(zero)},
                            {chains.data(), sizeof(JoinPieces) * chains.size()},
                            {&gave_up, sizeof(gave_up)}};
  const uint8_t* d[12];
  if (const int rc = upload_plan(p, parts, 12, d, s)) return rc;
  p->dev_gave_up = reinterpret_cast<unsigned int*>(const_cast<uint8_t*>(d[11]));
  p->dev_chains = reinterpret_cast<const JoinPieces*>(d[10]);
  p->dev_joins = reinterpret_cast<const SharedJoin*>(d[6]);
  p->dev_units = reinterpret_cast<const int4*>(d[7]);
  p->dev_score_base = reinterpret_cast<const int*>(d[8]);
  p->dev_queue = reinterpret_cast<unsigned int*>(const_cast<uint8_t*>(d[9]));
  p->dev_segs = reinterpret_cast<const TreeSeg*>(d[0]);
  p->dev_cta_segs = reinterpret_cast<const int*>(d[1]);
  p->dev_merges = reinterpret_cast<const TreeMerge*>(d[2]);
  p->dev_rows = reinterpret_cast<const int32_t*>(d[3]);
  p->dev_slots = reinterpret_cast<const int32_t*>(d[4]);
  p->dev_weighs = reinterpret_cast<const TreeWeigh*>(d[5]);
  p->valid = true;
  return KVC_OK;
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_append_rope(kvc_pool_t* pool, int layer, const void* d_q, int q_stride,
                               void* d_q_out, int num_heads, const void* d_k_new, int k_stride,
                               const void* d_v_new, int v_stride, const int32_t* d_block_tables,
                               int bt_rows, int bt_stride, const int32_t* d_rows,
                               const int32_t* d_positions, const int32_t* d_rope_positions, int n,
                               float freq_base, int neox, void* stream) {
  if (!pool) return set_error(KVC_ERR_INVALID_ARG, "pool must not be null.");
  return guarded("kvc_append_rope", [&]() -> int {
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    return do_append_rope(pool, layer, d_q, q_stride, d_q_out, num_heads, d_k_new, k_stride,
                          d_v_new, v_stride, d_block_tables, bt_rows, bt_stride, d_rows,
                          d_positions, d_rope_positions, n, freq_base, neox,
                          static_cast<cudaStream_t>(stream));
  });
}

extern "C" int kvc_tree_plan_create(kvc_tree_plan_t** out) {
  if (!out) return set_error(KVC_ERR_INVALID_ARG, "out must not be null.");
  *out = new (std::nothrow) kvc_tree_plan();
  return *out ? KVC_OK : set_error(KVC_ERR_RUNTIME, "out of host memory.");
}

extern "C" int kvc_tree_plan_destroy(kvc_tree_plan_t* plan) {
  if (!plan) return KVC_OK;
  if (plan->device >= 0) {
    DeviceScope dev(plan->device);
    plan->release();
  }
  delete plan;
  return KVC_OK;
}

extern "C" int kvc_plan_tree(kvc_tree_plan_t* plan, const kvc_pool_t* pool, const int32_t* h_rows,
                             const int32_t* h_ctx_lens, const int32_t* h_node_counts, int n_seqs,
                             int num_heads, void* stream) {
  if (!plan || !pool) return set_error(KVC_ERR_INVALID_ARG, "plan and pool must not be null.");
  return guarded("kvc_plan_tree", [&]() -> int {
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    if (int rc = refuse_capture(static_cast<cudaStream_t>(stream), "a tree plan")) return rc;
    if (plan->device >= 0 && plan->device != pool->device) {  // its buffers are elsewhere
      DeviceScope old(plan->device);
      plan->release();
    }
    return tree_build(plan, pool, h_rows, h_ctx_lens, h_node_counts, n_seqs, num_heads,
                      static_cast<cudaStream_t>(stream));
  });
}

extern "C" int kvc_tree_plan_info(const kvc_tree_plan_t* plan, int* n_tokens, int* n_ctas,
                                  size_t* scratch_bytes) {
  if (!plan) return set_error(KVC_ERR_INVALID_ARG, "plan must not be null.");
  if (n_tokens) *n_tokens = plan->n_tokens;
  if (n_ctas) *n_ctas = plan->n_ctas;
  if (scratch_bytes)
    *scratch_bytes = plan->d_part_o.cap + plan->d_part_ml.cap + plan->d_scores.cap + plan->d_row_ml.cap + plan->d_own_o.cap +
                     plan->d_own_ml.cap;
  return KVC_OK;
}

extern "C" int kvc_tree_plan_set_weights(kvc_tree_plan_t* plan, int on) {
  if (!plan) return set_error(KVC_ERR_INVALID_ARG, "plan must not be null.");
  plan->keep_scores = on != 0;
  return KVC_OK;
}

extern "C" int kvc_decode_tree(kvc_pool_t* pool, const kvc_tree_plan_t* plan, int layer,
                               const void* d_q, const int32_t* d_mask, int mask_words,
                               void* d_out, const int32_t* d_block_tables, int bt_stride,
                               float scale, void* stream) {
  if (!pool || !plan) return set_error(KVC_ERR_INVALID_ARG, "pool and plan must not be null.");
  return guarded("kvc_decode_tree", [&]() -> int {
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    return do_decode_tree(pool, plan, layer, d_q, d_mask, mask_words, d_out, d_block_tables,
                          bt_stride, scale, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int kvc_decode_tree_weights(kvc_pool_t* pool, const kvc_tree_plan_t* plan, int layer,
                                       const void* d_q, const int32_t* d_mask, int mask_words,
                                       float* d_weights, int weight_rows, int weight_slots,
                                       void* d_out, const int32_t* d_block_tables, int bt_stride,
                                       float scale, void* stream) {
  if (!pool || !plan) return set_error(KVC_ERR_INVALID_ARG, "pool and plan must not be null.");
  return guarded("kvc_decode_tree_weights", [&]() -> int {
    if (!d_weights) return set_error(KVC_ERR_INVALID_ARG, "weights must not be null.");
    if (reinterpret_cast<uintptr_t>(d_weights) & 3u)
      return set_error(KVC_ERR_INVALID_ARG, "weights must be 4-byte aligned.");
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    return do_decode_tree(pool, plan, layer, d_q, d_mask, mask_words, d_out, d_block_tables,
                          bt_stride, scale, static_cast<cudaStream_t>(stream), d_weights,
                          weight_rows, weight_slots);
  });
}

extern "C" int kvc_commit_tree(kvc_pool_t* pool, const int32_t* d_block_tables, int bt_rows,
                               int bt_stride, const int32_t* d_rows, const int32_t* d_ctx_lens,
                               const int32_t* d_paths, int path_stride,
                               const int32_t* d_path_lens, int n_seqs, void* stream) {
  if (!pool) return set_error(KVC_ERR_INVALID_ARG, "pool must not be null.");
  return guarded("kvc_commit_tree", [&]() -> int {
    if (n_seqs < 0 || n_seqs > 65535)
      return set_error(KVC_ERR_INVALID_ARG, "n_seqs must be in [0, 65535].");
    if (path_stride < 0 || path_stride > kMaxTreeNodes)
      return set_error(KVC_ERR_INVALID_ARG, "path_stride must be in [0, %d].", kMaxTreeNodes);
    if (n_seqs == 0 || path_stride == 0) return KVC_OK;
    if (!d_ctx_lens || !d_paths || !d_path_lens)
      return set_error(KVC_ERR_INVALID_ARG, "contexts, paths and lengths must not be null.");
    if (int rc = check_table(d_block_tables, bt_rows, bt_stride)) return rc;
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    CommitArgs a = {};
    if (int rc = paged_view(pool, 0, d_block_tables, bt_rows, bt_stride, &a.p)) return rc;
    a.layer_bytes = pool->g.layer_bytes;
    a.n_layers = pool->g.num_layers;
    a.rows = d_rows;
    a.ctx = d_ctx_lens;
    a.paths = d_paths;
    a.path_lens = d_path_lens;
    a.path_stride = path_stride;
    a.n = n_seqs;
    const cudaError_t e = launch_commit(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? KVC_OK : cuda_error(e, "commit kernel");
  });
}

extern "C" int kvc_reorder_beams(kvc_pool_t* pool, int32_t* d_block_tables, int bt_stride,
                                 const int32_t* d_parents, const int32_t* d_ctx_lens, int n_seqs,
                                 int n_beams, void* stream) {
  if (!pool) return set_error(KVC_ERR_INVALID_ARG, "pool must not be null.");
  return guarded("kvc_reorder_beams", [&]() -> int {
    if (n_seqs < 0 || n_seqs > 65535)
      return set_error(KVC_ERR_INVALID_ARG, "n_seqs must be in [0, 65535].");
    if (n_beams <= 0 || n_beams > kMaxBeams)
      return set_error(KVC_ERR_INVALID_ARG, "n_beams must be in [1, %d].", kMaxBeams);
    if (n_seqs == 0) return KVC_OK;
    if (!d_parents || !d_ctx_lens)
      return set_error(KVC_ERR_INVALID_ARG, "parents and contexts must not be null.");
    if (int rc = check_table(d_block_tables, n_seqs * n_beams, bt_stride)) return rc;
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    ReorderArgs a = {};
    if (int rc = paged_view(pool, 0, d_block_tables, n_seqs * n_beams, bt_stride, &a.p)) return rc;
    a.tables = d_block_tables;
    a.layer_bytes = pool->g.layer_bytes;
    a.n_layers = pool->g.num_layers;
    a.parents = d_parents;
    a.ctx = d_ctx_lens;
    a.n = n_seqs;
    a.beams = n_beams;
    const cudaError_t e = launch_reorder(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? KVC_OK : cuda_error(e, "reorder kernel");
  });
}

extern "C" int kvc_beam_create(int max_seqs, int max_beams, int max_vocab, int max_out,
                               int device, kvc_beam_t** out) {
  if (!out) return set_error(KVC_ERR_INVALID_ARG, "out must not be null.");
  *out = nullptr;
  return guarded("kvc_beam_create", [&]() -> int {
    if (max_seqs <= 0 || max_vocab <= 0)
      return set_error(KVC_ERR_INVALID_ARG, "max_seqs and max_vocab must be positive.");
    if (max_beams <= 0 || max_beams > kMaxBeams)
      return set_error(KVC_ERR_INVALID_ARG, "max_beams must be in [1, %d].", kMaxBeams);
    if (max_out <= 0 || max_out > kMaxBeamOut)
      return set_error(KVC_ERR_INVALID_ARG, "max_out must be in [1, %d].", kMaxBeamOut);
    if (max_vocab >= (1 << 27) || static_cast<int64_t>(max_seqs) * max_beams > 65535)
      return set_error(KVC_ERR_INVALID_ARG, "the vocabulary or the batch is too large.");
    const int64_t slots = static_cast<int64_t>(max_seqs) * max_beams *
                          beam_chunks(max_vocab);
    if (slots > (1ll << 30) / max_out)
      return set_error(KVC_ERR_INVALID_ARG, "the beam workspace would be too large.");
    DeviceScope dev(device);
    if (dev.rc()) return dev.rc();
    kvc_beam* b = new kvc_beam();
    b->device = device;
    b->max_seqs = max_seqs;
    b->max_beams = max_beams;
    b->max_vocab = max_vocab;
    b->max_out = max_out;
    b->sms = sms_of(device);
    b->ml_bytes = (sizeof(float2) * slots + 255) & ~static_cast<size_t>(255);
    const cudaError_t e = b->ws.ensure(b->ml_bytes + sizeof(uint64_t) * slots * max_out);
    if (e != cudaSuccess) {
      delete b;
      return cuda_error(e, "cudaMalloc(beam workspace)");
    }
    *out = b;
    return KVC_OK;
  });
}

extern "C" int kvc_beam_destroy(kvc_beam_t* beam) {
  if (!beam) return KVC_OK;
  {
    DeviceScope dev(beam->device);
    beam->ws.release();
  }
  delete beam;
  return KVC_OK;
}

extern "C" int kvc_beam_select(kvc_beam_t* beam, const void* d_logits, int dtype,
                               int64_t row_stride, const float* d_scores_in, int n_seqs,
                               int n_beams, int vocab, int n_out, int32_t* d_tokens,
                               int32_t* d_parents, float* d_scores_out, void* stream) {
  if (!beam) return set_error(KVC_ERR_INVALID_ARG, "beam must not be null.");
  return guarded("kvc_beam_select", [&]() -> int {
    const int es = elem_size_of(dtype);
    if (es == 0) return set_error(KVC_ERR_INVALID_ARG, "unknown dtype %d.", dtype);
    if (n_seqs < 0 || n_beams <= 0 || vocab <= 0 || n_out <= 0)
      return set_error(KVC_ERR_INVALID_ARG, "beam sizes must be positive.");
    if (n_seqs > beam->max_seqs || n_beams > beam->max_beams || vocab > beam->max_vocab ||
        n_out > beam->max_out)
      return set_error(KVC_ERR_INVALID_ARG, "the selection is larger than its workspace.");
    if (static_cast<int64_t>(n_beams) * vocab < n_out)
      return set_error(KVC_ERR_INVALID_ARG, "fewer candidates than results.");
    const int64_t stride = row_stride ? row_stride : vocab;
    if (stride < vocab) return set_error(KVC_ERR_INVALID_ARG, "row_stride is smaller than a row.");
    if (n_seqs == 0) return KVC_OK;
    if (!d_logits || !d_scores_in || !d_tokens || !d_parents || !d_scores_out)
      return set_error(KVC_ERR_INVALID_ARG, "logits, scores and outputs must not be null.");
    if (reinterpret_cast<uintptr_t>(d_logits) % es)
      return set_error(KVC_ERR_INVALID_ARG, "logits must be aligned to their elements.");
    DeviceScope dev(beam->device);
    if (dev.rc()) return dev.rc();
    BeamArgs a = {};
    a.logits = static_cast<const uint8_t*>(d_logits);
    a.row_bytes = static_cast<size_t>(stride) * es;
    a.dtype = dtype;
    a.cum = d_scores_in;
    a.n = n_seqs;
    a.beams = n_beams;
    a.vocab = vocab;
    a.n_out = n_out;
    a.sms = beam->sms;
    a.tokens = d_tokens;
    a.parents = d_parents;
    a.scores = d_scores_out;
    a.ml = static_cast<float2*>(beam->ws.ptr);
    a.cand = reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(beam->ws.ptr) + beam->ml_bytes);
    const cudaError_t e = launch_beam_select(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? KVC_OK : cuda_error(e, "beam selection kernel");
  });
}
