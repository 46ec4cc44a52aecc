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

int norm_rope_args(const kvc_pool* pool, const kvc_norm_rope_args& in, NormRopeArgs* out) {
  const PoolGeom& g = pool->g;
  if (in.layer < 0 || in.layer >= g.num_layers)
    return set_error(KVC_ERR_OUT_OF_RANGE, "layer_idx out of range for the KV pool.");
  if (in.n < 0) return set_error(KVC_ERR_INVALID_ARG, "row count must be non-negative.");
  if (in.n_pairs < 0 || 2 * static_cast<int64_t>(in.n_pairs) > g.head_dim)
    return set_error(KVC_ERR_INVALID_ARG, "a head has at most head_dim / 2 pairs to rotate.");
  if (in.n_pairs > 0 && !in.h_inv_freq)
    return set_error(KVC_ERR_INVALID_ARG, "the pairs' frequencies must not be null.");
  if (in.n_axes < 1 || in.n_axes > kMaxRopeAxes)
    return set_error(KVC_ERR_INVALID_ARG, "axes must be in [1, %d].", kMaxRopeAxes);
  for (int j = 0; j < in.n_pairs; ++j) {
    if (!std::isfinite(in.h_inv_freq[j]))
      return set_error(KVC_ERR_INVALID_ARG, "the pairs' frequencies must be finite.");
    if (in.h_axes && in.h_axes[j] >= in.n_axes)
      return set_error(KVC_ERR_INVALID_ARG, "a pair's axis is out of range.");
  }
  if ((in.d_q_weight || in.d_k_weight) && (!(in.eps > 0.0f) || !std::isfinite(in.eps)))
    return set_error(KVC_ERR_INVALID_ARG, "eps must be positive.");
  if (in.n == 0) return KVC_OK;
  if (!in.d_k_new || !in.d_v_new || !in.d_positions)
    return set_error(KVC_ERR_INVALID_ARG, "K/V rows and positions must not be null.");
  if (in.d_q && (!in.d_q_out || in.num_heads <= 0))
    return set_error(KVC_ERR_INVALID_ARG, "q needs its output and a positive head count.");
  if (int rc = check_table(in.d_block_tables, in.bt_rows, in.bt_stride)) return rc;
  if (!aligned16(in.d_q) || !aligned16(in.d_q_out) || !aligned16(in.d_k_new) || !aligned16(in.d_v_new) ||
      !aligned16(in.d_q_weight) || !aligned16(in.d_k_weight))
    return set_error(KVC_ERR_INVALID_ARG, "q, K/V rows and weights must be 16-byte aligned.");
  const int heads = in.d_q ? in.num_heads : 0;
  const int64_t q_row = static_cast<int64_t>(heads) * g.head_dim;
  const int64_t kv_row = static_cast<int64_t>(g.num_kv_heads) * g.head_dim;
  const int64_t qs = in.q_stride ? in.q_stride : q_row, ks = in.k_stride ? in.k_stride : kv_row;
  const int64_t vs = in.v_stride ? in.v_stride : kv_row;
  if ((in.d_q && qs < q_row) || ks < kv_row || vs < kv_row)
    return set_error(KVC_ERR_INVALID_ARG, "a token stride is smaller than its row.");
  if ((in.d_q && qs * g.elem_size % 16) || ks * g.elem_size % 16 || vs * g.elem_size % 16)
    return set_error(KVC_ERR_INVALID_ARG, "token strides must be multiples of 16 bytes.");
  if (in.d_q && in.d_q_out == in.d_q && qs != q_row)
    return set_error(KVC_ERR_INVALID_ARG, "q can be rotated in place only when it is packed.");
  NormRopeArgs& a = *out;
  if (int rc = paged_view(pool, in.layer, in.d_block_tables, in.bt_rows, in.bt_stride, &a.p)) return rc;
  a.q = static_cast<const uint8_t*>(in.d_q);
  a.q_out = static_cast<uint8_t*>(in.d_q_out);
  a.k_new = static_cast<const uint8_t*>(in.d_k_new);
  a.v_new = static_cast<const uint8_t*>(in.d_v_new);
  a.q_weight = static_cast<const uint8_t*>(in.d_q_weight);
  a.k_weight = static_cast<const uint8_t*>(in.d_k_weight);
  a.q_stride = static_cast<size_t>(qs) * g.elem_size;
  a.k_stride = static_cast<size_t>(ks) * g.elem_size;
  a.v_stride = static_cast<size_t>(vs) * g.elem_size;
  a.rows = in.d_rows;
  a.positions = in.d_positions;
  // (without positions of their own all axes count the slots)
  a.rope_positions = in.d_rope_positions ? in.d_rope_positions : in.d_positions;
  a.axes = in.d_rope_positions ? in.n_axes : 1;
  a.n = in.n;
  a.num_heads = heads;
  a.head_dim = g.head_dim;
  a.pairs = in.n_pairs;
  a.eps = in.eps;
  for (int j = 0; j < in.n_pairs; ++j) {
    a.turns[j] = in.h_inv_freq[j] / 6.283185307179586476925286766559;
    a.axis[j] = in.d_rope_positions && in.h_axes ? in.h_axes[j] : 0;
  }
  return KVC_OK;
}

// Bytes that sharing saves a layer, from which on it is done.
constexpr double kSharedSaving = 32e6;
// Prefixes and own positions side by side.  An SM needs kFullTile us for 128 positions x 128 dims
// of more than 128 rows, kPartTile for one of fewer rows, kPieceTime for a start and an end, and
// reads kBesideRate bytes a us of own positions, of which a warp takes kBesideSplit at a time.
// (Swept on 96 x 24K, 9 ragged groups and six more shapes: 128, 192 and 256 positions x 28e3 to
// 120e3 bytes; within 5 % of the best on each.)
constexpr double kFullTile = 1.9, kPartTile = 1.6, kPieceTime = 4.0, kBesideRate = 48e3;
constexpr int kBesideSplit = 256;

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
  std::vector<int> prefix(std::max(0, n_groups));   // shared by the members of group k
  for (int k = 0; k < n_groups; ++k) {
    if (h_sizes[k] <= 0) return set_error(KVC_ERR_INVALID_ARG, "a group has at least one member.");
    if (h_prefix[k] < 0)
      return set_error(KVC_ERR_INVALID_ARG, "a prefix has a non-negative length.");
    if (members + h_sizes[k] > n_seqs)
      return set_error(KVC_ERR_INVALID_ARG, "the groups have more members than the batch.");
    prefix[k] = h_sizes[k] > 1 ? h_prefix[k] : 0;   // (without company it does not matter)
    if (prefix[k] % g.page_size != 0)
      return set_error(KVC_ERR_INVALID_ARG, "a shared prefix is a whole number of pages.");
    for (int64_t i = members; i < members + h_sizes[k]; ++i)
      if (h_lens[i] < prefix[k])
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
    small += blocks(h_sizes[k]) * (prefix[k] / kTreeSmall);
    for (int j = i; j < i + h_sizes[k]; ++j)
      small += blocks(1) * ((h_lens[j] - prefix[k] + kTreeSmall - 1) / kTreeSmall);
  }
  const TreeTile tile = tree_tile(g, small, sms);
  std::vector<TreeSeg> runs, segs;
  std::vector<int> cta_segs;
  std::vector<int> own_run(n_seqs, -1), prefix_run(n_groups, -1);   // of KV head 0, block 0
  std::vector<int> base(n_seqs, 0);
  const int own_blocks = (group + tile.rows - 1) / tile.rows;
  int64_t tiles = 0, own_tiles = 0;
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
  // What sharing saves has to pay for a launch and the joins.  Measured over groups of 2-64
  // members, prefixes of 128-8192 positions, 2 x 64 and 8 x 128 dims, 16 bit: below 32 MB of K
  // and V that are not read again it costs 0-5 us (8 x 2 members on 512, 17 MB: 19.3 against
  // 16.3 us), above that it wins (8 x 4 on 512, 50 MB: 18.9 against 21.3; 8 x 16 on 2048, 1 GB: 43
  // against 167).  The CUDA-core kernels, whose tiles cost the same for any number of rows,
  // gain from every tile.
  double saved = 0;
  for (int k = 0; k < n_groups; ++k)
    saved += 2.0 * (h_sizes[k] - 1) * prefix[k] * Hkv * g.head_dim * g.elem_size;
  const bool worth = !tile.tensor || saved >= kSharedSaving;
  for (int k = 0, i = 0; k < n_groups; i += h_sizes[k++]) {
    // (below one tile the members' own first tiles hold the prefix anyway)
    if (!worth || h_sizes[k] < 2 || prefix[k] < tile.positions) continue;
    prefix_run[k] = static_cast<int>(runs.size());
    add(h_rows ? h_rows[i] : i, 0, prefix[k], i, h_sizes[k] * group);
    std::fill(base.begin() + i, base.begin() + i + h_sizes[k], prefix[k]);
  }
  // Own positions.  Where the decode kernel runs on the tensor cores it takes them: its eight
  // warps an SM each work on a piece of their own, and a short piece (96 x 30-700 positions, 64 x
  // 128 heads: 39 us) costs it half of what it costs a CTA of the tree kernel (74 us), which
  // is made for many rows.  That is a launch more: while every tile finds a CTA of its own the
  // tree kernel takes all (4 sequences on 512, 32 x 64 heads: 10 us, 14.7 with both).
  for (int i = 0; i < n_seqs; ++i)
    own_tiles += (h_lens[i] - base[i] + tile.positions - 1) / tile.positions * static_cast<int64_t>(own_blocks) * Hkv;
  if (tiles + own_tiles > (1ll << 30))
    return set_error(KVC_ERR_INVALID_ARG, "the batch is too large for one plan.");
  const bool decode = tile.tensor && tiles + own_tiles > static_cast<int64_t>(sms) * tile.ctas_per_sm;
  UnitList units;
  if (decode) {
    std::vector<int> rows(n_seqs);
    for (int i = 0; i < n_seqs; ++i) rows[i] = h_rows ? h_rows[i] : i;
    build_units(g, group, sms, rows, base, std::vector<int>(h_lens, h_lens + n_seqs),
                tiles > 0 ? kBesideSplit : 0, &units);
  }
  for (int i = 0; i < n_seqs && !decode; ++i) {
    if (h_lens[i] <= base[i]) continue;
    own_run[i] = static_cast<int>(runs.size());
    add(h_rows ? h_rows[i] : i, base[i], h_lens[i], i, group);
  }
  // The two kernels run side by side, the prefixes' on some SMs and the decode kernel on the
  // others: each SM takes one or the other.  The prefixes get their share of the work.  (Decode
  // CTAs follow on SMs that the prefixes leave, and take what is left of their list.)
  int prefix_sms = sms;
  if (decode && tiles > 0) {
    double prefix_us = 0, own_bytes = 0;
    for (const TreeSeg& r : runs)
      prefix_us += (2 * r.rows > tile.rows ? kFullTile : kPartTile) * r.tile1 * tile.positions / 128.0 * g.head_dim / 128.0;
    for (int i = 0; i < n_seqs; ++i)
      own_bytes += 2.0 * (h_lens[i] - base[i]) * Hkv * ((group + 7) / 8) * g.head_dim * g.elem_size;
    const double own_us = own_bytes / kBesideRate;
    // prefix_us / x + kPieceTime = own_us / (sms - x)
    double lo = 1, hi = sms;
    for (int k = 0; k < 20; ++k) {
      const double x = (lo + hi) / 2;
      (prefix_us / x + kPieceTime > own_us / std::max(0.01, sms - x) ? lo : hi) = x;
    }
    prefix_sms = std::max(1, std::min(sms, static_cast<int>(hi + 0.5)));
  }
  // A join takes about as long for four pieces as a tile: t tiles in p pieces are done after
  // t / p + p / 4 of them, which p = 2 sqrt(t) makes least.
  double pieces_at_most = 0;
  for (const TreeSeg& r : runs) pieces_at_most += std::ceil(2.0 * std::sqrt(static_cast<double>(r.tile1)));
  if (tile.tensor) prefix_sms = static_cast<int>(std::min<double>(prefix_sms, std::max(1.0, pieces_at_most)));
  cut_runs(runs, tile, prefix_sms, true, &segs, &cta_segs);
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
          int rows = decode ? group - r : std::min(group - r, tile.rows - r % tile.rows);
          SharedJoin j = {};
          j.prefix.rows = j.own.rows = 1;
          if (prefix_run[k] >= 0) {
            rows = std::min(rows, tile.rows - row % tile.rows);
            j.prefix = pieces[prefix_run[k] + kvh * prefix_blocks + row / tile.rows];
            j.prefix.row = row % tile.rows;
          }
          if (decode) {
            if (base[i] > 0 || units.splits[i].n > 1) j.own = units.splits[i];   // (else it is written already)
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
  p->n_joins = static_cast<int>(joins.size());
  if (n_seqs == 0) {
    p->valid = true;
    return KVC_OK;
  }
  cudaError_t e;
  if ((e = p->d_part_o.ensure(sizeof(float) * std::max<size_t>(1, part_rows) * g.head_dim)) ||
      (e = p->d_part_ml.ensure(sizeof(float2) * std::max<size_t>(1, part_rows))))
    return cuda_error(e, "plan buffers");
  const size_t split_rows = std::max<size_t>(1, units.n_splits) * num_heads;
  if (decode && ((e = p->d_own_o.ensure(sizeof(float) * split_rows * g.head_dim)) ||
                 (e = p->d_own_ml.ensure(sizeof(float2) * split_rows))))
    return cuda_error(e, "plan buffers");
  const unsigned int zero = 0;
  const PlanPart parts[] = {{segs.data(), sizeof(TreeSeg) * segs.size()},
                            {cta_segs.data(), sizeof(int) * cta_segs.size()},
                            {joins.data(), sizeof(SharedJoin) * joins.size()},
                            {units.recs.data(), sizeof(int4) * units.recs.size()},
                            {&zero, sizeof(zero)}};
  const uint8_t* d[5];
  if (const int rc = upload_plan(p, parts, 5, d, s)) return rc;
  p->dev_units = reinterpret_cast<const int4*>(d[3]);
  p->dev_queue = reinterpret_cast<unsigned int*>(const_cast<uint8_t*>(d[4]));
  p->n_units = static_cast<int>(units.recs.size() / 3);
  p->n_unit_ctas = std::min(sms * kPersistCtasPerSm, (p->n_units + kPersistWarps - 1) / kPersistWarps);
  p->dev_segs = reinterpret_cast<const TreeSeg*>(d[0]);
  p->dev_cta_segs = reinterpret_cast<const int*>(d[1]);
  p->dev_joins = reinterpret_cast<const SharedJoin*>(d[2]);
  p->valid = true;
  return KVC_OK;
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_append_norm_rope(kvc_pool_t* pool, const kvc_norm_rope_args_t* args, void* stream) {
  if (!pool || !args) return set_error(KVC_ERR_INVALID_ARG, "pool and arguments must not be null.");
  return guarded("kvc_append_norm_rope", [&]() -> int {
    DeviceScope dev(pool->device);
    if (dev.rc()) return dev.rc();
    NormRopeArgs a = {};
    if (int rc = norm_rope_args(pool, *args, &a)) return rc;
    if (args->n == 0) return KVC_OK;
    const cudaError_t e = launch_norm_rope(a, pool->g.dtype, args->neox != 0, sms_of(pool->device),
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
    plan->t.release();
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
      plan->t.release();
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
    a.joins = p.dev_joins;
    a.n_joins = p.n_joins;
    cudaError_t e = launch_tree(a, p.tile, static_cast<cudaStream_t>(stream));
    if (e == cudaSuccess && p.n_units > 0) {
      const DecodeArgs own = unit_args(&p, a, p.n_ctas > 0);
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
    if (pool->g.layer_bytes >= (size_t{1} << 36))   // (places are 32-bit counts of 16 bytes)
      return set_error(KVC_ERR_INVALID_ARG, "a layer's K of 64 GB or more cannot be cut back.");
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
