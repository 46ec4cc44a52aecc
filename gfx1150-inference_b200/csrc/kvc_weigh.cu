// Attention weights summed per cached slot (kvc_decode_tree_weights), behind the attention
// of kvc_tree.cu, which leaves every row's final max and sum (and, of short row lists, the
// scores):
//
//   weights[row, kvh, p] += sum over the rows (token, q-head of kvh) of
//                           2^(s scale log2(e) - max) / sum
//
//   finish_kernel        from kept scores, and the joins of split rows
//   recount_mma_kernel   computes the scores again on the tensor cores
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kvc_device.cuh"
#include "kvc_spec.h"
#include "kvc_tcgen05.cuh"
#include "kvc_tree.cuh"

namespace kvc {
namespace {

// =====================================================================================
// From kept scores, in one launch with the joins of the split rows.  A thread owns four slots
// and adds the rows in order, so the sums do not depend on the schedule; slots of the call's
// own tokens start from zero.  A row's final max and sum are joined here again from its
// pieces (a few numbers a row), so that this does not wait for the rows' joins.  Bound by latency:
// four rows' scores, the sums so far and the pieces' statistics are on their way together, and
// the plan's records, no kernel's output, are read while the attention still runs.
// =====================================================================================
constexpr int kFinishThreads = kWeighSlots / 4, kWeighAtOnce = 4;
static_assert(kFinishThreads == kMergeThreads, "a join's CTA has as many threads");

// The pieces of row `row` (a record of the plan).
__device__ __forceinline__ JoinPieces row_chain(const TreeArgs& a, const TreeWeigh& w, int row) {
  return row < w.nodes * a.group ? a.chains[w.chain + (a.own_o ? 0 : row / a.chain_rows)] : JoinPieces{};
}

__device__ __forceinline__ float2 row_statistics(const TreeArgs& a, const TreeWeigh& w,
                                                 const JoinPieces& c, int row) {
  const int node = row / a.group, head = w.kvh * a.group + row - node * a.group;
  if (c.n == 0 || (a.own_o && c.n == 1))
    return a.row_ml[static_cast<size_t>(w.tok0 + node) * a.num_heads + head];
  const float2* ml = a.own_o ? a.own_ml + static_cast<size_t>(c.part) * a.num_heads + head
                             : a.part_ml + c.part + row % a.chain_rows;
  const size_t step = a.own_o ? a.num_heads : c.rows;
  float2 all = make_float2(kNegBig, 0.f);
  for (int k0 = 0; k0 < c.n; k0 += 8) {
    float2 e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = k0 + k < c.n ? ml[(k0 + k) * step] : make_float2(kNegBig, 0.f);
    float m = all.x;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, e[k].x);
    float sum = all.y * fast_exp2(all.x - m);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += e[k].y * fast_exp2(e[k].x - m);
    all = make_float2(m, sum);
  }
  return all;
}

// Where a wait of the attention gave up, in this call or an earlier one of the plan, what rows and
// scores hold is an older call's: the sums stay as they are.  (The mark is read with the first
// loads and looked at in front of the stores.)
__device__ __forceinline__ bool attention_gave_up(const TreeArgs& a, unsigned int mark) {
  if (mark == 0u) return false;
  if (threadIdx.x == 0) report_error_at(a.p.err, KVC_DEVERR_WAIT_LIMIT, blockIdx.x);
  return true;
}

// chain: that of row threadIdx.x.
__device__ __forceinline__ void weigh(const TreeArgs& a, const TreeWeigh& w, JoinPieces chain,
                                      float2* s_ml) {
  const int end = w.ctx + w.nodes, rows = w.nodes * a.group, pitch = (end + 15) & ~15;
  const int p = w.slot0 + 4 * threadIdx.x;
  const bool mine = p < end;
  const unsigned int mark = __ldcg(a.gave_up);
  const float* s = a.scores + static_cast<size_t>(w.scores) * 16 + p;
  float* out = a.weights + (static_cast<size_t>(w.bt_row) * a.p.num_kv_heads + w.kvh) * a.weight_slots + p;
  float old[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
  float4 x[kWeighAtOnce];
  auto load = [&](int r0) {
#pragma unroll
    for (int r = 0; r < kWeighAtOnce; ++r)
      x[r] = mine && r0 + r < rows ? __ldcs(reinterpret_cast<const float4*>(s + static_cast<size_t>(r0 + r) * pitch))
                                   : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  };
  load(0);
#pragma unroll
  for (int i = 0; i < 4; ++i) old[i] = p + i < w.ctx ? out[i] : 0.f;
  for (int b = 0; b < rows; b += kFinishThreads) {
    if (b > 0) __syncthreads();
    if (b + threadIdx.x < rows) {
      if (b > 0) chain = row_chain(a, w, b + threadIdx.x);
      const float2 e = row_statistics(a, w, chain, b + threadIdx.x);
      s_ml[threadIdx.x] = make_float2(e.x, e.y > 0.f ? 1.0f / e.y : e.y);   // (0: no weight)
    }
    __syncthreads();
    const int n = min(kFinishThreads, rows - b);
    for (int r0 = 0; r0 < n; r0 += kWeighAtOnce) {
      if (b + r0 > 0) load(b + r0);
#pragma unroll
      for (int r = 0; r < kWeighAtOnce; ++r) {
        if (r0 + r >= n) break;
        const float2 e = s_ml[r0 + r];
        const float v[4] = {x[r].x, x[r].y, x[r].z, x[r].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (v[i] != -INFINITY) sum[i] += fast_exp2(fmaf(v[i], a.score_scale, -e.x)) * e.y;
      }
    }
  }
  if (attention_gave_up(a, mark)) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (p + i < end) out[i] = old[i] + sum[i];
}

// CTAs of the grid: n_weighs, then those of the merges or the joins (one at least).
template <typename T>
__global__ void __launch_bounds__(kFinishThreads, 4) finish_kernel(const TreeArgs a, const int per_merge) {
  __shared__ float2 s_ml[kFinishThreads];
  const int b = blockIdx.x - a.n_weighs;
  TreeWeigh w = {};
  JoinPieces chain = {};
  if (b < 0) {
    w = a.weighs[blockIdx.x];
    chain = row_chain(a, w, threadIdx.x);
  }
  wait_prerequisites();
  if (b == 0) rearm_queue(a);
  launch_dependents();
  if (b < 0) {
    weigh(a, w, chain, s_ml);
  } else if (a.own_o) {
    if (b < a.n_joins) join_rows<T>(a, a.joins[b], kFinishThreads);
  } else if (b < a.n_merges * per_merge) {
    merge_rows<T>(a, a.merges[b / per_merge], b % per_merge * kFinishThreads + threadIdx.x);
  }
}

template <typename T>
cudaError_t run_finish(const TreeArgs& a, cudaStream_t s) {
  const int per_merge = merge_ctas(a, sizeof(T));
  const int joins = a.own_o ? std::max(1, a.n_joins) : a.n_merges * per_merge;
  if (a.n_weighs + joins == 0) return cudaSuccess;
  const cudaError_t e = prefer_shared<finish_kernel<T>>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.n_weighs + joins));
  cfg.blockDim = dim3(kFinishThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, finish_kernel<T>, a, per_merge);
}

// =====================================================================================
// Recount.  With many rows, writing the scores out and reading them back (8 bytes a score)
// costs more than computing them again from K (2 D bytes a position and KV head, once).
// The product is turned round, S^T = K Q^T: a tensor memory lane is a position, so a thread
// owns one and adds its row of 128 columns up in registers, without a sum across threads.
// 1 / sum goes into the exponent: the weight is 2^(s scale log2(e) - (max + log2(sum))).
//
// A CTA takes one tile of 128 positions and goes through the (token, q-head) rows in blocks
// of 128, two warpgroups taking every other one by themselves: each copies its block of Q,
// has it multiplied into its half of tensor memory and adds it up while the next block of Q
// is on its way.  So an SM's two CTAs have four products and sums in different phases.
//
// 4 prompts of 29-82 tokens at 1.6K-3.9K, 32 q-heads on 8 x 128 dims, bf16: 28.5 us (48 with one
// warpgroup and two blocks of Q, 37 with Q in the pool's layout); the whole call 63, and 218
// with all scores kept.  23.4 million exponentials are 6 us of it at 16 a cycle and SM; the rest is
// the chain of a CTA: K and Q from memory, product, sums, and the next of its two or three blocks.
// Where a sequence has few rows, keeping is less: 8 tokens x 4 q-heads 61.5 against 76.5 us, 16 x 4
// 84.4 against 81.5 (8 sequences at 1K-8K), hence kKeepRows.
// =====================================================================================
constexpr int kRecountThreads = 256, kRecountRows = 128, kRecountCols = 256;

template <int D>
struct RecountShape {
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kHeadBytes = 6144;    // barriers, shifts, visibility
  static constexpr int kSmem = kHeadBytes + 3 * kTileBytes;
};

template <typename T, int D>
__global__ void __launch_bounds__(kRecountThreads, D <= 128 ? 2 : 1)
    recount_mma_kernel(const TreeArgs a) {
  using S = RecountShape<D>;
  constexpr int U = D / 8;
  constexpr uint32_t kSlabBytes = kSlab * D * 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);          // K, the two warpgroups' products
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + 64);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wg = warp >> 2, wt = tid & 127, ww = warp & 3;     // warpgroup; thread and warp in it
  float* s_shift = reinterpret_cast<float*>(smem + 1024) + wg * kRecountRows;
  uint4* s_vis = reinterpret_cast<uint4*>(smem + 2048) + wg * kRecountRows;   // of the 128 positions
  uint8_t* k_mem = smem + S::kHeadBytes;
  uint8_t* q_mem = k_mem + (1 + wg) * S::kTileBytes;
  const uint32_t bar0 = smem_u32(bars), done = bar0 + 8 * (1 + wg);
  const TreeWeigh w = a.weighs[a.n_weighs + blockIdx.x];
  const int end = w.ctx + w.nodes, rows = w.nodes * a.group, p0 = w.slot0;
  const int blocks = (rows + kRecountRows - 1) / kRecountRows;
  const bool edge = p0 + kRecountSlots > w.ctx;
  if (tid == 0) {
    for (int i = 0; i < 3; ++i) mbar_init(bar0 + 8 * i, 1);
    fence_mbar_init();
  }
  wait_prerequisites();
  launch_dependents();
  // (tensor memory only here: see tree_mma_kernel)
  if (warp == 0) tmem_alloc(smem_u32(s_tmem), kRecountCols);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = *s_tmem + wg * kRecountRows;

  if (warp == 0) {
    const int slabs = min(kRecountSlots / kSlab, (end - p0 + kSlab - 1) / kSlab);
    if (lane == 0) mbar_arrive_expect_tx(bar0, slabs * kSlabBytes);
    __syncwarp();
    if (lane < slabs) {
      const int pos = p0 + lane * kSlab;
      const uint8_t* src = a.p.k + (static_cast<size_t>(tree_page(a.p, w.bt_row, pos)) * a.p.num_kv_heads + w.kvh) *
                                       a.p.page_head_bytes +
                           pos % a.p.page_size / kSlab * kSlabBytes;
      bulk_g2s(smem_u32(k_mem) + lane * kSlabBytes, src, kSlabBytes, bar0, l2_policy_evict_first());
    }
  }
  // Block b's rows of Q, and the first one again behind the last (its scores are taken back by
  // the shift; with zeros there, an infinite key would leave what is not a number).
  using R = RowBlocks<D>;
  auto copy_q = [&](int b) {
    copy_rows<T, D, true>(smem_u32(q_mem), 0u, false,
                    reinterpret_cast<const T*>(a.q) +
                        (static_cast<size_t>(w.tok0) * a.num_heads + w.kvh * a.group) * D,
                    b * kRecountRows, rows - b * kRecountRows, kRecountRows, a.group, a.num_heads * D, ww, 4,
                    lane);
  };
  // Thread r: row r's max and sum.
  auto statistics = [&](int b) {
    const int row = b * kRecountRows + wt, node = row / a.group;
    return row < rows ? a.row_ml[static_cast<size_t>(w.tok0 + node) * a.num_heads + w.kvh * a.group + row -
                                 node * a.group]
                      : make_float2(0.f, 0.f);
  };
  // Thread r: what row r's scores are shifted by, and which positions of an edge tile it sees.
  auto constants = [&](int b, float2 e) {
    const int row = b * kRecountRows + wt;
    uint32_t vis[4] = {0, 0, 0, 0};
    if (edge && row < rows) {
      const int node = row / a.group;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j0 = p0 + 32 * k - w.ctx, m = j0 >> 5;
        vis[k] = __funnelshift_r(mask_word(a, w.tok0, w.nodes, node, m),
                                 mask_word(a, w.tok0, w.nodes, node, m + 1), j0 & 31);
      }
    }
    s_shift[wt] = e.y == 0.f ? INFINITY : e.x + log2f(e.y);     // (infinity: no weight)
    if (edge) s_vis[wt] = make_uint4(vis[0], vis[1], vis[2], vis[3]);
  };
  bool failed = false;
  const unsigned int mark = __ldcg(a.gave_up);
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (!mbar_wait_bounded(bar, parity)) {
      report_error_at(a.p.err, KVC_DEVERR_WAIT_LIMIT, blockIdx.x);
      failed = true;
    }
  };
  // A barrier of the warpgroup; true if a wait of any of its threads gave up (all get the same
  // answer, so all leave the loop at the same barrier).
  auto group_failed = [&]() {
    uint32_t any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, %2, 128, p;\n"
        " selp.b32 %0, 1, 0, q;\n}"
        : "=r"(any)
        : "r"(static_cast<uint32_t>(failed)), "r"(1 + wg)
        : "memory");
    return any != 0;
  };
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  const float2 sc = make_float2(a.scale_log2, a.scale_log2);   // (q as it is, whatever the sign)
  int issued = 0;
  float2 next = make_float2(0.f, 0.f);
  if (wg < blocks) {
    copy_q(wg);
    next = statistics(wg);
    wait(bar0, 0);                     // K is here
  }
  for (int b = wg, n = 0; b < blocks; b += 2, ++n) {
    constants(b, next);
    copy_async_wait();
    fence_proxy_async();
    tmem_fence_before();
    const bool stop = group_failed();  // the block is here, and the last one's sums are made
    tmem_fence_after();
    if (stop) break;
    if (ww == 0 && elect_one()) {
      constexpr uint32_t kDesc = mma_desc<T>(128, kRecountRows, false);
      const uint64_t kd = operand_desc(smem_u32(k_mem), 128, U * 128);
      const uint64_t qd = R::desc(smem_u32(q_mem));
#pragma unroll
      for (int k = 0; k < D / 16; ++k) mma_ss(tmem, kd + 16 * k, qd + R::step(k), kDesc, k > 0);
      mma_commit(done);
    }
    __syncwarp();
    ++issued;
    if (b + 2 < blocks) next = statistics(b + 2);
    wait(done, n & 1);
    tmem_fence_after();
    if (b + 2 < blocks) copy_q(b + 2);   // (the product has read the last block)
    const uint32_t* vis = reinterpret_cast<const uint32_t*>(s_vis) + ww;
    const uint32_t t_s = tmem + (static_cast<uint32_t>(ww * 32) << 16);
    const int cols = min(kRecountRows, (rows - b * kRecountRows + 31) & ~31);
    // 32 columns at a time, the next ones on their way
    auto add = [&](int c, const uint32_t* s) {
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 m = *reinterpret_cast<const float4*>(s_shift + c + i);
        float2 e0 = fma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), sc, make_float2(-m.x, -m.y));
        float2 e1 = fma2(make_float2(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), sc, make_float2(-m.z, -m.w));
        e0.x = fast_exp2(e0.x);
        e0.y = fast_exp2(e0.y);
        e1.x = fast_exp2(e1.x);
        e1.y = fast_exp2(e1.y);
        if (edge) {
          if (!((vis[4 * (c + i)] >> lane) & 1u)) e0.x = 0.f;
          if (!((vis[4 * (c + i + 1)] >> lane) & 1u)) e0.y = 0.f;
          if (!((vis[4 * (c + i + 2)] >> lane) & 1u)) e1.x = 0.f;
          if (!((vis[4 * (c + i + 3)] >> lane) & 1u)) e1.y = 0.f;
        }
        sum[0] = add2(sum[0], e0);
        sum[1] = add2(sum[1], e1);
      }
    };
    uint32_t sa[32], sb[32];
    tmem_ld32(t_s, sa);
#pragma unroll 1
    for (int c = 0; c < cols; c += 64) {
      tmem_wait_ld();
      tmem_loaded<32>(sa);
      if (c + 32 < cols) tmem_ld32(t_s + c + 32, sb);
      add(c, sa);
      if (c + 32 < cols) {
        tmem_wait_ld();
        tmem_loaded<32>(sb);
        if (c + 64 < cols) tmem_ld32(t_s + c + 64, sa);
        add(c + 32, sb);
      }
    }
    tmem_fence_before();
    if (group_failed()) break;         // the shifts have been read by all
  }
  copy_async_wait();
  float* s_sum = reinterpret_cast<float*>(smem + 1024) + kRecountRows;   // (the second group's shifts)
  const float add = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
  if (wg == 1) s_sum[wt] = add;
  tmem_fence_before();
  const bool stopped = __syncthreads_or(failed);
  const int p = p0 + wt;
  if (wg == 0 && !stopped && !attention_gave_up(a, mark) && p < end) {
    float* out = a.weights + (static_cast<size_t>(w.bt_row) * a.p.num_kv_heads + w.kvh) * a.weight_slots + p;
    const float total = add + s_sum[wt];
    *out = p < w.ctx ? *out + total : total;
  }
  if (stopped && wt == 0) {            // what is in flight lands before the memory goes
    mbar_wait_bounded(bar0, 0);
    if (issued > 0) mbar_wait_bounded(done, (issued - 1) & 1);
  }
  __syncthreads();
  tmem_fence_after();
  if (warp == 0) tmem_dealloc(*s_tmem, kRecountCols);
}

template <typename T, int D>
cudaError_t run_recount(const TreeArgs& a, cudaStream_t s) {
  using S = RecountShape<D>;
  const cudaError_t e = allow_smem<recount_mma_kernel<T, D>>(S::kSmem);
  if (e != cudaSuccess) return e;
  return launch_early(recount_mma_kernel<T, D>, dim3(a.n_recounts), kRecountThreads, S::kSmem, s, a);
}

template <typename T>
cudaError_t run_recount_any(const TreeArgs& a, cudaStream_t s) {
  switch (a.head_dim) {
    case 32: return run_recount<T, 32>(a, s);
    case 64: return run_recount<T, 64>(a, s);
    case 96: return run_recount<T, 96>(a, s);
    case 128: return run_recount<T, 128>(a, s);
    case 160: return run_recount<T, 160>(a, s);
    case 192: return run_recount<T, 192>(a, s);
    case 256: return run_recount<T, 256>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t launch_weigh(const TreeArgs& a, const TreeTile& t, cudaStream_t s) {
  const cudaError_t e = a.dtype == KVC_DTYPE_F16    ? run_finish<__half>(a, s)
                        : a.dtype == KVC_DTYPE_BF16 ? run_finish<__nv_bfloat16>(a, s)
                                                    : run_finish<float>(a, s);
  if (e != cudaSuccess || a.n_recounts == 0) return e;
  if (!t.tensor) return cudaErrorInvalidValue;
  return a.dtype == KVC_DTYPE_F16 ? run_recount_any<__half>(a, s) : run_recount_any<__nv_bfloat16>(a, s);
}

}  // namespace kvc
