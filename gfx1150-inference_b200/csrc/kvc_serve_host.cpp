// Host side of head norms with rotation, shared prefixes and eviction: argument checks, the
// shared plan and the C entry points.  Kernels: kvc_serve.cu, kvc_tree.cu.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "kvc_serve.h"

namespace kvc {
namespace {

int norm_rope_args(const kvc_pool* pool, int layer, const void* d_q, int q_stride, void* d_q_out,
                   int num_heads, const void* d_q_weight, const void* d_k_new, int k_stride,
                   const void* d_k_weight, const void* d_v_new, int v_stride, float eps,
                   const int32_t* d_bt, int bt_rows, int bt_stride, const int32_t* d_rows,
                   const int32_t* d_positions, const int32_t* d_rope_positions, int n_axes, int n,
                   const double* h_inv_freq, const uint8_t* h_axes, int n_pairs, NormRopeArgs* out) {
  const PoolGeom& g = pool->g;
  if (layer < 0 || layer >= g.num_layers)
    return set_error(KVC_ERR_OUT_OF_RANGE, "layer_idx out of range for the KV pool.");
  if (n < 0) return set_error(KVC_ERR_INVALID_ARG, "row count must be non-negative.");
  if (n_pairs < 0 || 2 * static_cast<int64_t>(n_pairs) > g.head_dim)
    return set_error(KVC_ERR_INVALID_ARG, "a head has at most head_dim / 2 pairs to rotate.");
  if (n_pairs > 0 && !h_inv_freq)
    return set_error(KVC_ERR_INVALID_ARG, "the pairs' frequencies must not be null.");
  if (n_axes < 1 || n_axes > kMaxRopeAxes)
    return set_error(KVC_ERR_INVALID_ARG, "axes must be in [1, %d].", kMaxRopeAxes);
  for (int j = 0; j < n_pairs; ++j) {
    if (!std::isfinite(h_inv_freq[j]))
      return set_error(KVC_ERR_INVALID_ARG, "the pairs' frequencies must be finite.");
    if (h_axes && h_axes[j] >= n_axes)
      return set_error(KVC_ERR_INVALID_ARG, "a pair's axis is out of range.");
  }
  if ((d_q_weight || d_k_weight) && (!(eps > 0.0f) || !std::isfinite(eps)))
    return set_error(KVC_ERR_INVALID_ARG, "eps must be positive.");
  if (n == 0) return KVC_OK;
  if (!d_k_new || !d_v_new || !d_positions)
    return set_error(KVC_ERR_INVALID_ARG, "K/V rows and positions must not be null.");
  if (d_q && (!d_q_out || num_heads <= 0))
    return set_error(KVC_ERR_INVALID_ARG, "q needs its output and a positive head count.");
  if (int rc = check_table(d_bt, bt_rows, bt_stride)) return rc;
  if (!aligned16(d_q) || !aligned16(d_q_out) || !aligned16(d_k_new) || !aligned16(d_v_new) ||
      !aligned16(d_q_weight) || !aligned16(d_k_weight))
    return set_error(KVC_ERR_INVALID_ARG, "q, K/V rows and weights must be 16-byte aligned.");
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
  NormRopeArgs& a = *out;
  if (int rc = paged_view(pool, layer, d_bt, bt_rows, bt_stride, &a.p)) return rc;
  a.q = static_cast<const uint8_t*>(d_q);
  a.q_out = static_cast<uint8_t*>(d_q_out);
  a.k_new = static_cast<const uint8_t*>(d_k_new);
  a.v_new = static_cast<const uint8_t*>(d_v_new);
  a.q_weight = static_cast<const uint8_t*>(d_q_weight);
  a.k_weight = static_cast<const uint8_t*>(d_k_weight);
  a.q_stride = static_cast<size_t>(qs) * g.elem_size;
  a.k_stride = static_cast<size_t>(ks) * g.elem_size;
  a.v_stride = static_cast<size_t>(vs) * g.elem_size;
  a.rows = d_rows;
  a.positions = d_positions;
  // (without positions of their own all axes count the slots)
  a.rope_positions = d_rope_positions ? d_rope_positions : d_positions;
  a.axes = d_rope_positions ? n_axes : 1;
  a.n = n;
  a.num_heads = heads;
  a.head_dim = g.head_dim;
  a.pairs = n_pairs;
  a.eps = eps;
  for (int j = 0; j < n_pairs; ++j) {
    a.turns[j] = h_inv_freq[j] / 6.283185307179586476925286766559;
    a.axis[j] = d_rope_positions && h_axes ? h_axes[j] : 0;
  }
  return KVC_OK;
}

// Every group's prefix is a set of runs of its members' rows, every sequence's own positions
// another; a row's result is joined from its pieces of both.
int shared_build(kvc_shared_plan* sp, const kvc_pool* pool, const int32_t* h_rows,
                 const int32_t* h_lens, int n_seqs, const int32_t* h_sizes,
                 const int32_t* h_prefix, int n_groups, int num_heads, cudaStream_t s) {
  kvc_tree_plan* p = &sp->t;
  const PoolGeom& g = pool->g;
  if (n_seqs < 0 || n_groups < 0)
    return set_error(KVC_ERR_INVALID_ARG, "n_seqs and n_groups must be non-negative.");
  if ((n_seqs > 0 && !h_lens) || (n_groups > 0 && (!h_sizes || !h_prefix)))
    return set_error(KVC_ERR_INVALID_ARG, "lengths, group sizes and prefixes must not be null.");
  if (num_heads <= 0 || num_heads % g.num_kv_heads != 0)
    return set_error(KVC_ERR_INVALID_ARG, "num_heads must be divisible by num_kv_heads.");
  const int group = num_heads / g.num_kv_heads, Hkv = g.num_kv_heads, sms = sms_of(pool->device);
  int64_t members = 0, small = 0;
  int max_end = 0, max_row = 0;
  for (int i = 0; i < n_seqs; ++i) {
    if (h_lens[i] < 0) return set_error(KVC_ERR_INVALID_ARG, "context length must be non-negative.");
    if (h_lens[i] > (1 << 30)) return set_error(KVC_ERR_INVALID_ARG, "a sequence is too long.");
    if (h_rows && h_rows[i] < 0)
      return set_error(KVC_ERR_INVALID_ARG, "block-table row must be non-negative.");
    max_end = std::max(max_end, h_lens[i]);
    max_row = std::max(max_row, h_rows ? h_rows[i] : i);
  }
  for (int k = 0; k < n_groups; ++k) {
    if (h_sizes[k] <= 0) return set_error(KVC_ERR_INVALID_ARG, "a group has at least one member.");
    if (h_prefix[k] < 0 || h_prefix[k] % g.page_size != 0)
      return set_error(KVC_ERR_INVALID_ARG, "a shared prefix is a whole number of pages.");
    if (members + h_sizes[k] > n_seqs)
      return set_error(KVC_ERR_INVALID_ARG, "the groups have more members than the batch.");
    for (int64_t i = members; i < members + h_sizes[k]; ++i)
      if (h_lens[i] < h_prefix[k])
        return set_error(KVC_ERR_INVALID_ARG, "a sequence is shorter than its group's prefix.");
    members += h_sizes[k];
  }
  if (members != n_seqs)
    return set_error(KVC_ERR_INVALID_ARG, "the groups have fewer members than the batch.");
  if (static_cast<int64_t>(n_seqs) * num_heads > (1ll << 30))
    return set_error(KVC_ERR_INVALID_ARG, "the batch is too large for one plan.");
  p->valid = false;
  // tiles of the small fp32 kernel, which are what decides between the two
  for (int k = 0, i = 0; k < n_groups; i += h_sizes[k++]) {
    auto blocks = [&](int64_t rows) { return (rows * group + kTreeSmall - 1) / kTreeSmall * Hkv; };
    small += blocks(h_sizes[k]) * (h_prefix[k] / kTreeSmall);
    for (int j = i; j < i + h_sizes[k]; ++j)
      small += blocks(1) * ((h_lens[j] - h_prefix[k] + kTreeSmall - 1) / kTreeSmall);
  }
  const TreeTile tile = tree_tile(g, small, sms);
  std::vector<TreeSeg> runs, segs;
  std::vector<int> cta_segs;
  std::vector<int> own_run(n_seqs, -1), prefix_run(n_groups, -1);   // of KV head 0, block 0
  std::vector<int> base(n_seqs, 0);
  const int own_blocks = tile.tensor ? 1 : (group + tile.rows - 1) / tile.rows;
  int64_t tiles = 0;
  auto add = [&](int bt_row, int first, int end, int tok0, int n_rows) {
    for (int kvh = 0; kvh < Hkv; ++kvh)
      for (int r0 = 0; r0 < n_rows; r0 += tile.rows) {
        TreeSeg sg = {};
        sg.bt_row = bt_row;
        sg.ctx = end;
        sg.tok0 = tok0;
        sg.kvh = kvh;
        sg.row0 = r0;
        sg.rows = std::min(tile.rows, n_rows - r0);
        sg.tile1 = (end - first + tile.positions - 1) / tile.positions;
        sg.part = -1;
        sg.base = first;
        tiles += sg.tile1;
        runs.push_back(sg);
      }
  };
  for (int k = 0, i = 0; k < n_groups; i += h_sizes[k++]) {
    // A prefix is worth a run of its own from one tile on: below that the members' own first
    // tiles hold it anyway.
    if (h_sizes[k] < 2 || h_prefix[k] < tile.positions) continue;
    prefix_run[k] = static_cast<int>(runs.size());
    add(h_rows ? h_rows[i] : i, 0, h_prefix[k], i, h_sizes[k] * group);
    std::fill(base.begin() + i, base.begin() + i + h_sizes[k], h_prefix[k]);
  }
  // Own positions.  Where the decode kernel runs on the tensor cores it takes them: its eight
  // warps an SM each work on a piece of their own, and a short piece (96 x 30-700 positions, 64 x
  // 128 heads: 39 us) costs it half of what it costs a CTA of the tree kernel (74 us), which
  // is made for many rows.
  std::vector<JoinPieces> splits(tile.tensor ? n_seqs : 0);
  std::vector<int4> units;
  int n_splits = 0;
  if (tile.tensor) {
    std::vector<int> own(n_seqs), refine(n_seqs);
    for (int i = 0; i < n_seqs; ++i) own[i] = h_lens[i] - base[i];
    const int chunks = (group + 7) / 8;
    const int C = split_partition_sms(g.page_size, own.data(), n_seqs, Hkv * chunks, sms, refine.data());
    std::vector<int4> items;
    for (int i = 0; i < n_seqs; ++i) {
      if (own[i] == 0) continue;
      splits[i].part = n_splits;
      splits[i].n = emit_splits(i, own[i], C, refine[i], [&](int4 it) {
        it.z += base[i];
        it.w += base[i];
        items.push_back(it);
      });
      n_splits += splits[i].n;
    }
    std::stable_sort(items.begin(), items.end(),
                     [](const int4& x, const int4& y) { return x.w - x.z > y.w - y.z; });
    for (const int4& it : items) {
      const int i = it.x;
      // (more than one split: the kernel leaves partial states)
      const int n = splits[i].n + (base[i] > 0 ? 1 : 0);
      for (int kvh = 0; kvh < Hkv; ++kvh)
        for (int c = 0; c < chunks; ++c) {
          units.push_back(it);
          units.push_back(make_int4(h_rows ? h_rows[i] : i, h_lens[i], splits[i].part, n));
          units.push_back(make_int4(kvh, c, kvh * group + c * 8, std::min(8, group - c * 8)));
        }
    }
  }
  for (int i = 0; i < n_seqs && !tile.tensor; ++i) {
    if (h_lens[i] <= base[i]) continue;
    own_run[i] = static_cast<int>(runs.size());
    add(h_rows ? h_rows[i] : i, base[i], h_lens[i], i, group);
  }
  if (tiles > (1ll << 30))
    return set_error(KVC_ERR_INVALID_ARG, "the batch is too large for one plan.");
  cut_runs(runs, tile, sms, &segs, &cta_segs);
  // Pieces of a run follow one another.  A run that is a row's only one, in one piece, writes
  // the output itself; the others write partials.
  std::vector<JoinPieces> pieces(runs.size());
  const int first_own = [&] {
    for (int i = 0; i < n_seqs; ++i)
      if (own_run[i] >= 0) return own_run[i];
    return static_cast<int>(runs.size());
  }();
  size_t part_rows = 0;
  int run = -1;
  for (size_t at = 0; at < segs.size();) {
    size_t next = at + 1;
    while (next < segs.size() && segs[next].tile0 > 0) ++next;
    const TreeSeg& sg = segs[at];
    ++run;
    if (next - at > 1 || run < first_own || base[sg.tok0] > 0) {
      pieces[run] = JoinPieces{static_cast<int>(part_rows), static_cast<int>(next - at), sg.rows, 0};
      for (size_t k = at; k < next; ++k) {
        segs[k].part = static_cast<int>(part_rows);
        part_rows += sg.rows;
      }
    }
    at = next;
  }
  if (part_rows > (1u << 30))
    return set_error(KVC_ERR_INVALID_ARG, "the batch is too large for one plan.");
  std::vector<SharedJoin> joins;
  for (int k = 0, i0 = 0; k < n_groups; i0 += h_sizes[k++]) {
    const int prefix_blocks = (h_sizes[k] * group + tile.rows - 1) / tile.rows;
    for (int i = i0; i < i0 + h_sizes[k]; ++i)
      for (int kvh = 0; kvh < Hkv; ++kvh)
        for (int r = 0; r < group;) {
          // the rows up to the end of a block of the prefix or of the own run
          const int row = (i - i0) * group + r;     // within the group
          int rows = tile.tensor ? group - r : std::min(group - r, tile.rows - r % tile.rows);
          SharedJoin j = {};
          j.prefix.rows = j.own.rows = 1;
          if (prefix_run[k] >= 0) {
            rows = std::min(rows, tile.rows - row % tile.rows);
            j.prefix = pieces[prefix_run[k] + kvh * prefix_blocks + row / tile.rows];
            j.prefix.row = row % tile.rows;
          }
          if (tile.tensor) {
            if (base[i] > 0 || splits[i].n > 1) j.own = splits[i];   // (else it is written already)
          } else if (own_run[i] >= 0) {
            j.own = pieces[own_run[i] + kvh * own_blocks + r / tile.rows];
            j.own.row = r % tile.rows;
          }
          j.token = i;
          j.head = kvh * group + r;
          j.rows = rows;
          r += rows;
          if (j.prefix.n + j.own.n > 0 || h_lens[i] == 0) joins.push_back(j);
        }
  }
  p->n_seqs = p->n_tokens = n_seqs;
  p->num_heads = num_heads;
  p->max_end = max_end;
  p->max_row = max_row;
  p->tile = tile;
  p->n_ctas = static_cast<int>(cta_segs.size()) - 1;
  p->part_rows = part_rows;
  p->pool_geom = g;
  p->device = pool->device;
  sp->n_joins = static_cast<int>(joins.size());
  if (n_seqs == 0) {
    p->valid = true;
    return KVC_OK;
  }
  cudaError_t e;
  if ((e = p->d_part_o.ensure(sizeof(float) * std::max<size_t>(1, part_rows) * g.head_dim)) ||
      (e = p->d_part_ml.ensure(sizeof(float2) * std::max<size_t>(1, part_rows))))
    return cuda_error(e, "plan buffers");
  if (tile.tensor &&
      ((e = sp->d_own_o.ensure(sizeof(float) * std::max<size_t>(1, n_splits) * num_heads * g.head_dim)) ||
       (e = sp->d_own_ml.ensure(sizeof(float2) * std::max<size_t>(1, n_splits) * num_heads))))
    return cuda_error(e, "plan buffers");
  const unsigned int zero = 0;
  const PlanPart parts[] = {{segs.data(), sizeof(TreeSeg) * segs.size()},
                            {cta_segs.data(), sizeof(int) * cta_segs.size()},
                            {joins.data(), sizeof(SharedJoin) * joins.size()},
                            {units.data(), sizeof(int4) * units.size()},
                            {&zero, sizeof(zero)}};
  const uint8_t* d[5];
  if (const int rc = upload_plan(p, parts, 5, d, s)) return rc;
  sp->dev_units = reinterpret_cast<const int4*>(d[3]);
  sp->dev_queue = reinterpret_cast<unsigned int*>(const_cast<uint8_t*>(d[4]));
  sp->n_units = static_cast<int>(units.size() / 3);
  sp->n_unit_ctas = std::min(sms * kPersistCtasPerSm, (sp->n_units + kPersistWarps - 1) / kPersistWarps);
  p->dev_segs = reinterpret_cast<const TreeSeg*>(d[0]);
  p->dev_cta_segs = reinterpret_cast<const int*>(d[1]);
  sp->dev_joins = reinterpret_cast<const SharedJoin*>(d[2]);
  p->valid = true;
  return KVC_OK;
}

// The decode kernel's part of a call whose attention takes `a`.
DecodeArgs own_args(const kvc_shared_plan* sp, const TreeArgs& a, bool behind_prefix) {
  DecodeArgs d = {};
  d.k_layer = a.p.k;
  d.v_layer = a.p.v;
  d.q = a.q;
  d.out = a.out;
  d.block_tables = a.p.block_tables;
  d.bt_stride = a.p.bt_stride;
  d.part_o = static_cast<float*>(sp->d_own_o.ptr);
  d.part_ml = static_cast<float2*>(sp->d_own_ml.ptr);
  d.sched_recs = sp->dev_units;
  d.n_units = d.n_items = d.sched_cap = sp->n_units;
  d.queue = sp->dev_queue;
  d.n_sched_ctas = sp->n_unit_ctas;
  d.early_prefetch = behind_prefix ? 1 : 0;
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

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_append_norm_rope(
    kvc_pool_t* pool, int layer, const void* d_q, int q_stride, void* d_q_out, int num_heads,
    const void* d_q_weight, const void* d_k_new, int k_stride, const void* d_k_weight,
    const void* d_v_new, int v_stride, float eps, const int32_t* d_block_tables, int bt_rows,
    int bt_stride, const int32_t* d_rows, const int32_t* d_positions,
    const int32_t* d_rope_positions, int n_axes, int n, const double* h_inv_freq,
    const uint8_t* h_axes, int n_pairs, int neox, void* stream) {
  if (!pool) return set_error(KVC_ERR_INVALID_ARG, "pool must not be null.");
  return guarded("kvc_append_norm_rope", [&]() -> int {
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    NormRopeArgs a = {};
    if (int rc = norm_rope_args(pool, layer, d_q, q_stride, d_q_out, num_heads, d_q_weight, d_k_new,
                                k_stride, d_k_weight, d_v_new, v_stride, eps, d_block_tables, bt_rows,
                                bt_stride, d_rows, d_positions, d_rope_positions, n_axes, n,
                                h_inv_freq, h_axes, n_pairs, &a))
      return rc;
    if (n == 0) return KVC_OK;
    const cudaError_t e = launch_norm_rope(a, pool->g.dtype, neox != 0, sms_of(pool->device),
                                           static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? KVC_OK : cuda_error(e, "append + norm + rope kernel");
  });
}

extern "C" int kvc_shared_plan_create(kvc_shared_plan_t** out) {
  if (!out) return set_error(KVC_ERR_INVALID_ARG, "out must not be null.");
  *out = new (std::nothrow) kvc_shared_plan();
  return *out ? KVC_OK : set_error(KVC_ERR_RUNTIME, "out of host memory.");
}

extern "C" int kvc_shared_plan_destroy(kvc_shared_plan_t* plan) {
  if (!plan) return KVC_OK;
  if (plan->t.device >= 0) {
    DeviceScope dev(plan->t.device);
    plan->release();
  }
  delete plan;
  return KVC_OK;
}

extern "C" int kvc_plan_shared(kvc_shared_plan_t* plan, const kvc_pool_t* pool,
                               const int32_t* h_rows, const int32_t* h_lens, int n_seqs,
                               const int32_t* h_group_sizes, const int32_t* h_prefix_lens,
                               int n_groups, int num_heads, void* stream) {
  if (!plan || !pool) return set_error(KVC_ERR_INVALID_ARG, "plan and pool must not be null.");
  return guarded("kvc_plan_shared", [&]() -> int {
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    if (int rc = refuse_capture(static_cast<cudaStream_t>(stream), "a shared-prefix plan")) return rc;
    if (plan->t.device >= 0 && plan->t.device != pool->device) {  // its buffers are elsewhere
      DeviceScope old(plan->t.device);
      plan->release();
    }
    return shared_build(plan, pool, h_rows, h_lens, n_seqs, h_group_sizes, h_prefix_lens, n_groups,
                        num_heads, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int kvc_shared_plan_info(const kvc_shared_plan_t* plan, int* n_queries, int* n_ctas,
                                    size_t* scratch_bytes) {
  if (!plan) return set_error(KVC_ERR_INVALID_ARG, "plan must not be null.");
  return kvc_tree_plan_info(&plan->t, n_queries, n_ctas, scratch_bytes);
}

extern "C" int kvc_decode_shared(kvc_pool_t* pool, const kvc_shared_plan_t* plan, int layer,
                                 const void* d_q, void* d_out, const int32_t* d_block_tables,
                                 int bt_stride, float scale, void* stream) {
  if (!pool || !plan) return set_error(KVC_ERR_INVALID_ARG, "pool and plan must not be null.");
  return guarded("kvc_decode_shared", [&]() -> int {
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    const kvc_tree_plan& p = plan->t;
    if (int rc = check_tree_call(pool, &p, layer, nullptr, 0, bt_stride, scale)) return rc;
    if (p.n_tokens == 0) return KVC_OK;
    TreeArgs a = {};
    if (int rc = tree_args(pool, &p, layer, d_q, d_out, d_block_tables, bt_stride, scale, &a)) return rc;
    a.joins = plan->dev_joins;
    a.n_joins = plan->n_joins;
    cudaError_t e = launch_tree(a, p.tile, static_cast<cudaStream_t>(stream));
    if (e == cudaSuccess && plan->n_units > 0) {
      // (the prefix's launch writes no KV, and lets this one begin only behind what came before)
      const DecodeArgs own = own_args(plan, a, p.n_ctas > 0);
      a.own_o = own.part_o;
      a.own_ml = own.part_ml;
      a.own_queue = own.queue;
      e = launch_decode(own, a.dtype, a.p.layout, static_cast<cudaStream_t>(stream));
    }
    if (e == cudaSuccess) e = launch_shared_join(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? KVC_OK : cuda_error(e, "shared-prefix attention kernel");
  });
}

extern "C" int kvc_evict(kvc_pool_t* pool, const int32_t* d_block_tables, int bt_rows,
                         int bt_stride, const int32_t* d_rows, const int32_t* d_ctx_lens,
                         int n_seqs, const float* d_weights, float* d_weights_out, int weight_rows,
                         int weight_slots, int budget, int recent, int32_t* d_kept, void* stream) {
  if (!pool) return set_error(KVC_ERR_INVALID_ARG, "pool must not be null.");
  return guarded("kvc_evict", [&]() -> int {
    if (n_seqs < 0 || n_seqs > 65535)
      return set_error(KVC_ERR_INVALID_ARG, "n_seqs must be in [0, 65535].");
    if (budget <= 0) return set_error(KVC_ERR_INVALID_ARG, "budget must be positive.");
    if (recent < 0 || recent > budget)
      return set_error(KVC_ERR_INVALID_ARG, "recent must be in [0, budget].");
    if (weight_rows <= 0 || weight_slots <= 0)
      return set_error(KVC_ERR_INVALID_ARG, "weights must have rows and slots.");
    if (2ll * pool->g.num_layers > 65535)
      return set_error(KVC_ERR_INVALID_ARG, "the pool has too many layers.");
    if (n_seqs == 0) return KVC_OK;
    if (!d_ctx_lens || !d_weights || !d_weights_out || !d_kept)
      return set_error(KVC_ERR_INVALID_ARG, "contexts, weights and kept slots must not be null.");
    if (int rc = check_table(d_block_tables, bt_rows, bt_stride)) return rc;
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    EvictArgs a = {};
    if (int rc = paged_view(pool, 0, d_block_tables, bt_rows, bt_stride, &a.p)) return rc;
    a.layer_bytes = pool->g.layer_bytes;
    a.n_layers = pool->g.num_layers;
    a.rows = d_rows;
    a.ctx = d_ctx_lens;
    a.weights = d_weights;
    a.weights_out = d_weights_out;
    a.weight_rows = weight_rows;
    a.weight_slots = weight_slots;
    a.kept = d_kept;
    a.n = n_seqs;
    a.budget = budget;
    a.recent = recent;
    const cudaError_t e = launch_evict(a, sms_of(pool->device), static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? KVC_OK : cuda_error(e, "eviction kernels");
  });
}
