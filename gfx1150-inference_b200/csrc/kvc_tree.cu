// Attention of drafted tokens over the paged cache (kvc_decode_tree).
//
//   out[t, h] = sum_j softmax_j((q[t, h] . k_j) * scale) v_j
//
// over the cached positions of the token's sequence and those drafted tokens that
// its mask row names.  The (node, q-head) pairs of one KV head are the rows of one
// tile, so a K/V byte is read once for all drafted tokens and the whole head group.
//
//   tree_mma_kernel     tcgen05 tensor cores: 16-bit pools, head dims 32 ... 256
//   tree_f32_kernel     CUDA cores: fp32 pools
//   tree_simt_kernel    CUDA cores: 16-bit pools with head dims without a tensor tile
//   tree_merge_kernel   joins the pieces of rows whose positions were split over CTAs
//   shared_join_kernel  the same for rows of a shared prefix and their own positions
//                       (kvc_decode_shared)
// With row_ml they also leave what kvc_weigh.cu makes the weights per slot of
// (kvc_decode_tree_weights): every row's final max and sum, and the kScores variants the scores
// of short row lists.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kvc_device.cuh"
#include "kvc_spec.h"
#include "kvc_tcgen05.cuh"
#include "kvc_tree.cuh"
#include "kvcache.h"

namespace kvc {
namespace {

// Whether node `node` of a sequence sees its drafted token j.
__device__ __forceinline__ bool sees(const TreeArgs& a, int tok0, int node, int j) {
  if (!a.mask) return j <= node;
  const int w = j >> 5;
  return w < a.mask_words &&
         ((a.mask[static_cast<size_t>(tok0 + node) * a.mask_words + w] >> (j & 31)) & 1u);
}

// =====================================================================================
// Tensor-core kernel.  One CTA per SM; each takes its share of the plan's position tiles.
//
// A tile of 128 positions (64 above head_dim 128) of K and of V arrives by bulk copies, slab
// by slab, in the pool's own layout: 8-position x 16-byte core matrices, which is the
// unswizzled operand layout of tcgen05.mma, k-major for K (S = Q K^T) and mn-major for V (O = P V),
// so nothing is rearranged.  S, P and O live in tensor memory; P takes the place of its S.
//
// Two streams share the tensor cores, each with a softmax warpgroup whose thread r owns
// row r (tensor memory lane r), so that one stream's softmax runs under the other's
// products.  With more than 128 rows the streams are the two halves of the rows and each
// tile serves both; with fewer they are the even and the odd tiles of the same rows,
// joined when the piece ends.  (Head dims above 128 fill tensor memory with one stream.)
//
// O is rescaled only when a row's max has grown by more than 2^8 since the last time: the
// probabilities then stay below 2^8 and a tile normally touches O with the MMA alone.
// fp16 probabilities are 2^7 times that, at most 2^15: fp16 keeps 11 bits of those down to
// 2^-21 of the row's largest, and of smaller ones all but 2^-32 of it, so a flat tail of
// 10^5 positions far below one peak loses less than the output's rounding.  As 2^-14 and
// 2^-25 (without the factor) it lost a hundredth of the output and more.
//
// Warps: 0 and 2 bring K/V tiles into a ring of stages, 1 issues the MMAs, 3 loads each
// piece's Q and looks through V tiles with drafted tokens, 4 ... 11 are the two softmax
// warpgroups.  Every wait is bounded; a wait that gives up raises the CTA's abort flag, all
// roles then run through their loops without waiting, copying or issuing, and the kernel
// returns.
//
// Measured on B200 (replayed passes; in parentheses the time of the bytes at the copy rate of
// 6.46 TB/s): 32 sequences of 5-16 nodes at 1K-8K, fp16, 114 us (111); 8 x 12 at 32K,
// 172 us (167); 16 x 63 at 3K-9K, bf16, 118 us (67).  The first two are bound by memory, the
// last by the chain scores -> softmax -> sums of one stream: 3300 cycles for 256 rows x 128
// positions, of which the tensor cores work 2050 and the exponentials of a stream alone
// take 1024.  In seconds of calls without a pause the 1000 W limit holds the clock
// at 1.55-1.7 GHz and the three take 128, 204 and 137 us.  Tiles of 128 positions fill the
// 128 columns that two S and two O tiles leave each other; two streams because one alone
// leaves the tensor cores idle through its softmax.
// =====================================================================================
constexpr int kTmemCols = 512;
constexpr float kRescaleAt = 8.0f;   // log2
// log2 of the factor on the probabilities of a storage type (bf16 has fp32's exponents).
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
// What a row's largest scaled score (log2 units) is taken for.  Past 2^22, where the
// rounding of the score itself comes on top and counts, the factor would take probabilities
// out of fp16's range.
template <typename T>
__device__ __forceinline__ float row_max(float score, float scale) {
  if (score == -INFINITY) return kNegBig;
  const float x = score * scale;
  return fabsf(x) < 4194304.0f ? x - kLift<T> : x;
}
constexpr int kPieceCost = 4;        // a piece's start and end, in tiles

template <int D>
struct TreeShape {
  static constexpr int kStreams = D <= 128 ? 2 : 1;
  static constexpr int kPos = D <= 128 ? 128 : 64;               // positions of a tile
  static constexpr int kThreads = 128 + 128 * kStreams;
  static constexpr int kStageBytes = kPos * D * 2;
  static constexpr int kQBytes = 128 * D * 2;
  static constexpr int kHeadBytes = 3072;                        // barriers, exchange
  static constexpr int kFit = (232448 - kHeadBytes - kStreams * kQBytes) / kStageBytes;
  static constexpr int kStages = kFit > 12 ? 12 : kFit;
  static constexpr int kSmem = kHeadBytes + kStreams * kQBytes + kStages * kStageBytes;
};

template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t h) {
  constexpr uint32_t e = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return (h & e) == e;
}

// Whether one of two packed values may not be finite (never false when one is not).
template <typename T>
__device__ __forceinline__ bool maybe_odd(uint32_t two) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u;
  const uint32_t t = (two & e) ^ e;   // a half is zero where its exponent is all ones
  return ((t - 0x00010001u) & ~t & 0x80008000u) != 0u;
}

template <typename T, int D, bool kScores>
__global__ void __launch_bounds__(TreeShape<D>::kThreads, 1) tree_mma_kernel(const TreeArgs a) {
  using S = TreeShape<D>;
  constexpr int U = D / 8, KP = S::kPos;
  constexpr uint32_t kSlabBytes = kSlab * D * 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  static_assert(S::kHeadBytes % 1024 == 0 && S::kQBytes % 1024 == 0, "swizzled rows start a pattern");
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(smem + 512);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + 516);
  volatile int* s_dirty = reinterpret_cast<volatile int*>(smem + 520);   // [4]
  float2* s_ml = reinterpret_cast<float2*>(smem + 1024);                 // [2][128]
  uint8_t* q_mem = smem + S::kHeadBytes;
  uint8_t* stage_mem = q_mem + S::kStreams * S::kQBytes;
  const uint32_t bar0 = smem_u32(bars);
  auto full = [&](int st) { return bar0 + 8u * st; };
  auto empty = [&](int st) { return bar0 + 8u * (12 + st); };
  auto s_ready = [&](int x) { return bar0 + 8u * (24 + x); };
  auto p_ready = [&](int x) { return bar0 + 8u * (26 + x); };
  auto o_ready = [&](int x) { return bar0 + 8u * (28 + x); };
  const uint32_t q_ready = bar0 + 8u * 30, q_free = bar0 + 8u * 31;
  // (two of each: K may run two edge tiles ahead of the helpers, and they of the sums)
  auto edge_go = [&](uint32_t i) { return bar0 + 8u * (32 + (i & 1)); };
  auto edge_done = [&](uint32_t i) { return bar0 + 8u * (34 + (i & 1)); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int st = 0; st < S::kStages; ++st) {
      mbar_init(full(st), 1);
      mbar_init(empty(st), 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_ready(x), 1);
      mbar_init(p_ready(x), 128);
      mbar_init(o_ready(x), 1);
    }
    mbar_init(q_ready, 32);
    mbar_init(q_free, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(edge_go(i), 1);
      mbar_init(edge_done(i), 32);
    }
    fence_mbar_init();
    *s_abort = 0;
    for (int i = 0; i < 4; ++i) s_dirty[i] = -1;
  }
  // Rows without a token are zeros: whatever else Q's memory holds reaches no result, but it
  // costs power in every MMA (32 ragged trees: 143 us for 132).
  for (int i = threadIdx.x; i < S::kStreams * S::kQBytes / 16; i += S::kThreads)
    reinterpret_cast<uint4*>(q_mem)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  // (the plan's records are no kernel's output: they may be read before the wait)
  const int seg0 = a.cta_segs[blockIdx.x], seg1 = a.cta_segs[blockIdx.x + 1];
  wait_prerequisites();
  launch_dependents();
  // Tensor memory is taken only here: a CTA that held it while it waits could keep a launch
  // ahead of it from ever getting its own.
  if (warp == 1) tmem_alloc(smem_u32(s_tmem), kTmemCols);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = *s_tmem;

  // false: some wait of this CTA gave up
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
#pragma unroll 1
      for (int i = 0; i < 64; ++i)
        if (mbar_try_wait(bar, parity)) return true;
      if (*s_abort) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        report_error_at(a.p.err, KVC_DEVERR_WAIT_LIMIT, blockIdx.x);
        *s_abort = 1;
        return false;
      }
    }
  };

  // Registers move from the other warps to the softmax warpgroups: 128 x 104 + 256 x 200
  // is what 384 threads were launched with (168 each).
  if (warp < 4) {
    if constexpr (S::kStreams == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 0 || warp == 2) {
      // ---- K/V tiles into the ring, in the order the MMAs take them: one warp issues the
      // even entries, the other the odd ones (a tile of 16-position pages is eight copies,
      // and issuing them takes a warp a quarter of the time that memory needs for them).
      // A lane keeps the place of one slab: 32 slabs of page-table entries at a time, the
      // next 32 on their way.
      constexpr int kTileSlabs = KP / kSlab, kWinTiles = 32 / kTileSlabs;
      const uint64_t policy = l2_policy_evict_first();
      const int spp = a.p.page_size / kSlab;             // slabs of a page: neighbours are copied
      const int run = spp % 8 == 0 ? 8 : spp % 4 == 0 ? 4 : spp % 2 == 0 ? 2 : 1;   // together
      const uint32_t parity = warp >> 1;
      uint32_t n = 0;  // ring entries so far
      bool ok = true;
      for (int si = seg0; si < seg1 && ok; ++si) {
        const TreeSeg sg = a.segs[si];
        const int tiles = sg.tile1 - sg.tile0, end = sg.ctx + sg.nodes;
        const int last_slab = (end - 1) / kSlab, slab0 = sg.base / kSlab + sg.tile0 * kTileSlabs;
        const int32_t* table = a.p.block_tables + static_cast<size_t>(sg.bt_row) * a.p.bt_stride;
        auto entry_of = [&](int win) -> int {            // page-table entry of a window's slab
          const int slab = slab0 + win * kWinTiles * kTileSlabs + lane;
          const int col = slab / spp;
          return slab <= last_slab && col < a.p.bt_stride ? table[col] : -1;
        };
        int win = 0, now = entry_of(0), next = entry_of(1);
        const int ahead = S::kStreams == 2 && sg.rows <= 128 ? 2 : 1;  // K runs this far ahead
        for (int step = 0; step < tiles + ahead && ok; ++step) {
          // step: V of tile step - ahead, then K of tile step
          for (int kv = 1; kv >= 0 && ok; --kv) {
            const int t = kv ? step - ahead : step;
            if (t < 0 || t >= tiles) continue;
            if ((n & 1) == parity) {
              const int w = t / kWinTiles;
              if (w != win) {
                now = w == win + 1 ? next : entry_of(w);
                next = entry_of(w + 1);
                win = w;
              }
              const int slabs = min(kTileSlabs, last_slab + 1 - slab0 - t * kTileSlabs);
              int page = __shfl_sync(0xffffffffu, now, t % kWinTiles * kTileSlabs + (lane & (kTileSlabs - 1)));
              const bool mine = lane < slabs && lane % run == 0;
              const uint8_t* src = nullptr;
              if (mine) {
                if (page < 0 || page >= a.p.num_pages) {   // reported, and page 0 read instead
                  report_error_at(a.p.err, KVC_DEVERR_BAD_PAGE, static_cast<uint32_t>(page));
                  page = 0;
                }
                const int slab = slab0 + t * kTileSlabs + lane;
                src = (kv ? a.p.v : a.p.k) +
                      (static_cast<size_t>(page) * a.p.num_kv_heads + sg.kvh) * a.p.page_head_bytes +
                      slab % spp * kSlabBytes;
              }
              const int st = n % S::kStages;
              if (n >= S::kStages) ok = wait(empty(st), (n / S::kStages - 1) & 1);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              if (lane == 0) mbar_arrive_expect_tx(full(st), slabs * kSlabBytes);
              __syncwarp();
              if (mine)
                bulk_g2s(smem_u32(stage_mem) + st * S::kStageBytes + lane * kSlabBytes, src,
                         min(run, slabs - lane) * kSlabBytes, full(st), policy);
            }
            ++n;
          }
        }
      }
      if (!ok) {  // copies in flight land before the CTA's memory goes
        for (uint32_t i = n > 2 * S::kStages ? n - 2 * S::kStages : 0; i < n; ++i)
          if ((i & 1) == parity) mbar_wait_bounded(full(i % S::kStages), (i / S::kStages) & 1);
      }
    } else if (warp == 1) {
      // ---- MMAs: the warp waits together, one lane issues.  Everything an MMA takes is
      // the same in all lanes (broadcast where the compiler could not tell), so it sits in
      // uniform registers: with operands in ordinary ones an issue took over 100 cycles,
      // twice as long as the MMA itself.
      constexpr uint32_t kDescS = mma_desc<T>(128, KP, false);
      constexpr uint32_t kDescO = mma_desc<T>(128, D, true);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t q_desc = RowBlocks<D>::desc(smem_u32(q_mem));
      const uint64_t k_desc = operand_desc(smem_u32(stage_mem), 128, U * 128);
      const uint64_t v_desc = operand_desc(smem_u32(stage_mem), U * 128, 128);
      const bool leader = elect_one();
      uint32_t n = 0;                       // ring tiles consumed
      uint32_t np[2] = {0, 0}, nq = 0, ng = 0, ne = 0;
      bool ok = true;
      auto wait_all = [&](uint32_t bar, uint32_t parity) {
        ok = __all_sync(0xffffffffu, ok && wait(bar, parity));
      };
      auto take = [&]() -> int {            // the next tile of the ring
        const int st = n % S::kStages;
        wait_all(full(st), (n / S::kStages) & 1);
        ++n;
        return st;
      };
      auto commit = [&](uint32_t bar) {
        if (leader) mma_commit(bar);
      };
      auto scores = [&](int x, int st) {    // S_x = Q_x K^T
        const uint64_t qd = q_desc + x * (S::kQBytes / 16), kd = k_desc + st * (S::kStageBytes / 16);
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)  // 16 dims: two core matrices of K on
            mma_ss(tm + x * 128, qd + RowBlocks<D>::step(k), kd + 16 * k, kDescS, k > 0);
          mma_commit(s_ready(x));
        }
      };
      auto sums = [&](int x, int st, int slabs, bool accumulate) {   // O_x += P_x V
        const uint64_t vd = v_desc + st * (S::kStageBytes / 16);
        if (leader) {
          if (slabs == KP / kSlab) {
#pragma unroll
            for (int k = 0; k < KP / kSlab; ++k)
              mma_ts(tm + 256 + x * 128, tm + x * 128 + 8 * k, vd + (kSlabBytes / 16) * k, kDescO,
                     accumulate || k > 0);
          } else {
#pragma unroll 1
            for (int k = 0; k < slabs; ++k)
              mma_ts(tm + 256 + x * 128, tm + x * 128 + 8 * k, vd + (kSlabBytes / 16) * k, kDescO,
                     accumulate || k > 0);
          }
        }
      };
      for (int si = seg0; si < seg1 && ok; ++si) {
        const TreeSeg sg = a.segs[si];
        const int tiles = __shfl_sync(0xffffffffu, sg.tile1 - sg.tile0, 0);
        const int left = __shfl_sync(0xffffffffu, sg.ctx + sg.nodes - sg.base - sg.tile0 * KP, 0);
        const bool two = __shfl_sync(0xffffffffu, sg.rows, 0) > 128;
        const int ahead = S::kStreams == 2 && !two ? 2 : 1;
        const int edge0 = __shfl_sync(0xffffffffu, sg.ctx - sg.base - sg.tile0 * KP, 0);
        auto slabs_of = [&](int t) { return min(KP / kSlab, (left - t * KP + kSlab - 1) / kSlab); };
        auto is_edge = [&](int t) { return (t + 1) * KP > edge0; };
        // K of tile t is here: when the tile holds drafted positions the helper warps may
        // take its V on, which the sums then wait for
        auto take_k = [&](int t) {
          const int st = take();
          if (is_edge(t)) {
            if (ok && leader) mbar_arrive(edge_go(ng));
            ++ng;
          }
          return st;
        };
        auto edge_wait = [&](int t) {
          if (is_edge(t)) {
            wait_all(edge_done(ne), (ne >> 1) & 1);
            ++ne;
          }
        };
        wait_all(q_ready, nq++ & 1);
        if (two) {
          int kst = take_k(0);
          if (!ok) break;
          scores(0, kst);
          scores(1, kst);
          commit(empty(kst));
          if (tiles == 1) commit(q_free);
          for (int t = 0; t < tiles && ok; ++t) {
            const int vst = take();
            edge_wait(t);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              wait_all(p_ready(x), np[x]++ & 1);
              if (!ok) break;
              tmem_fence_after();
              sums(x, vst, slabs_of(t), t > 0);
              if (x == 1) commit(empty(vst));
              if (t + 1 == tiles) commit(o_ready(x));
              if (t + 1 < tiles) {
                if (x == 0) kst = take_k(t + 1);
                if (!ok) break;
                scores(x, kst);
                if (x == 1) commit(empty(kst));
                if (x == 1 && t + 2 == tiles) commit(q_free);
              }
            }
          }
        } else {
          for (int x = 0; x < ahead && x < tiles && ok; ++x) {
            const int kst = take_k(x);
            if (!ok) break;
            scores(x, kst);
            commit(empty(kst));
            if (x + 1 == tiles) commit(q_free);
          }
          for (int t = 0; t < tiles && ok; ++t) {
            const int x = ahead == 2 ? t & 1 : 0;
            const int vst = take();
            edge_wait(t);
            wait_all(p_ready(x), np[x]++ & 1);
            if (!ok) break;
            tmem_fence_after();
            sums(x, vst, slabs_of(t), t >= ahead);
            commit(empty(vst));
            if (t + ahead < tiles) {
              const int kst = take_k(t + ahead);
              if (!ok) break;
              scores(x, kst);
              commit(empty(kst));
              if (t + ahead + 1 == tiles) commit(q_free);
            } else {
              commit(o_ready(x));
            }
          }
        }
      }
      if (!ok && leader) {  // MMAs in flight end before tensor memory is freed
        mbar_init(bar0 + 8u * 40, 1);
        fence_mbar_init();
        mma_commit(bar0 + 8u * 40);
        mbar_wait_bounded(bar0 + 8u * 40, 0);
      }
      __syncwarp();
    } else {
      // ---- helper: each piece's Q, and the V tiles that hold drafted positions --------------
      const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
      int high0 = 0, high1 = 0;   // rows of the streams' copies that may not be zero
      uint32_t ring = 0, nf = 0, ng = 0;
      bool ok = true;
      for (int si = seg0; si < seg1; ++si) {
        const TreeSeg sg = a.segs[si];
        const int tiles = sg.tile1 - sg.tile0, end = sg.ctx + sg.nodes;
        const bool two = sg.rows > 128;
        const int ahead = S::kStreams == 2 && !two ? 2 : 1;
        // Q, all its copies in flight together, and zeros as far as an earlier piece had rows.
        // Streams that share their rows get a copy each.
        if (si > seg0) ok = ok && wait(q_free, nf++ & 1);   // the last piece's scores are done
        if (ok) {
          using R = RowBlocks<D>;
          int n_rows = (sg.rows + 7) & ~7;
          const int now0 = two ? 128 : n_rows, now1 = two ? n_rows - 128 : n_rows;
          n_rows = two ? 128 + max(now1, high1) : max(n_rows, max(high0, high1));
          high0 = now0;
          high1 = now1;
          copy_rows<T, D>(smem_u32(q_mem), S::kQBytes, S::kStreams == 2 && !two,
                          reinterpret_cast<const T*>(a.q) +
                              (static_cast<size_t>(sg.tok0) * a.num_heads + sg.kvh * a.group) * D,
                          sg.row0, sg.rows, n_rows, a.group, a.num_heads * D, 0, 1, lane);
          copy_async_wait();
          if (flip) {   // a negative scale turns q: what other lanes have copied, too
            __syncwarp();
            for (int x = 0; x < S::kStreams * (D / R::kChunk); ++x) {
              const int st = x / (D / R::kChunk), i = x - st * (D / R::kChunk);
              const int n = !two ? n_rows : st == 0 ? 128 : n_rows - 128;
              uint32_t* words = reinterpret_cast<uint32_t*>(q_mem + st * S::kQBytes + i * R::kBytes);
              for (int k = lane; k < n * R::kChunk / 2; k += 32) words[k] ^= flip;
            }
          }
        }
        fence_proxy_async();
        mbar_arrive(q_ready);
        // V of drafted tokens: what is not finite would spread through zero weights to rows
        // that do not see it, so it leaves the tile here (and comes back at the end, to the
        // rows that do); positions past the end hold anything, and go to zero.
        for (int t = max(0, (sg.ctx - sg.base) / KP - sg.tile0); t < tiles; ++t) {
          const int p0 = sg.base + (sg.tile0 + t) * KP;
          ok = ok && wait(edge_go(ng), (ng >> 1) & 1);
          // ring order of the piece: `ahead` K tiles, then V t, K t + ahead, ...
          const uint32_t vi = ring + t + min(ahead + t, tiles);
          const int st = vi % S::kStages;
          ok = ok && wait(full(st), (vi / S::kStages) & 1);
          if (ok) {
            uint8_t* vt = stage_mem + st * S::kStageBytes;
            const int from = max(0, sg.ctx - p0), to = min(KP, (end - p0 + kSlab - 1) / kSlab * kSlab);
            bool dirty = false;
            auto cell = [&](int i) {
              const int pt = i / U, u = i - pt * U;
              return reinterpret_cast<uint4*>(vt + (pt >> 3) * U * 128 + u * 128 + (pt & 7) * 16);
            };
            const int live = min(to, end - p0) * U;      // units of drafted positions
            for (int i0 = from * U + lane; i0 < live; i0 += 4 * 32) {
              uint4 v[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                v[k] = i0 + 32 * k < live ? *cell(i0 + 32 * k) : make_uint4(0, 0, 0, 0);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (!(maybe_odd<T>(v[k].x) || maybe_odd<T>(v[k].y) || maybe_odd<T>(v[k].z) ||
                      maybe_odd<T>(v[k].w)))
                  continue;
                uint32_t e[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                  if (not_finite<T>(e[w] & 0xffffu)) e[w] &= 0xffff0000u, dirty = true;
                  if (not_finite<T>(e[w] >> 16)) e[w] &= 0x0000ffffu, dirty = true;
                }
                *cell(i0 + 32 * k) = make_uint4(e[0], e[1], e[2], e[3]);
              }
            }
            for (int i = live + lane; i < to * U; i += 32) *cell(i) = make_uint4(0, 0, 0, 0);
            // The helper is in piece p once the MMAs are, when softmax group 0 is past piece
            // p - 2.  Group 1 is too, or still at the end of p - 2 (if p - 1 is one tile, all of
            // it group 0's).  So three places suffice for a piece's flag to be read before it
            // is written again; two do not.
            if (dirty) s_dirty[si & 3] = si;
          }
          __threadfence_block();
          fence_proxy_async();
          mbar_arrive(edge_done(ng));
          ++ng;
        }
        ring += 2 * tiles;
      }
    }
  } else {
    if constexpr (S::kStreams == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---- softmax: thread r of stream x owns row r ---------------------------------------------
    const int x = (warp - 4) >> 2, w4 = warp & 3, r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(w4 * 32) << 16;
    const uint32_t t_s = tmem + lanes + x * 128, t_o = tmem + lanes + 256 + x * 128;
    const float sc = fabsf(a.scale_log2);
    uint32_t ns = 0, no[2] = {0, 0};
    bool ok = true;
    for (int si = seg0; si < seg1; ++si) {
      const TreeSeg* seg = a.segs + si;   // (read again where it is needed again: no spills)
      const int tiles = seg->tile1 - seg->tile0, p00 = seg->base + seg->tile0 * KP, ctx = seg->ctx;
      const bool two = seg->rows > 128;
      const int ahead = S::kStreams == 2 && !two ? 2 : 1;
      const bool joint = ahead == 2;
      const int row = (two ? x * 128 : 0) + r;
      const bool live = (two ? x * 128 : 0) + w4 * 32 < seg->rows;   // some row of the warp
      const bool mine = row < seg->rows; 
      // where the row's scores go, 16 positions to 64 bytes (its pitch is a multiple of that)
      float* keep = nullptr;
      int keep_end = 0;
      if constexpr (kScores) {
        const TreeSeg sg = *seg;
        keep_end = sg.ctx + sg.nodes;
        if (mine && sg.scores >= 0) keep = a.scores + score_row(sg, sg.row0 + row);
      }
      float m = kNegBig, l = 0.f;     // max in log2 units, less kLift
      // One tile of the stream: scores to probabilities, in place, and the running max and
      // sum.  Edge tiles hold positions that some rows do not see.
      auto softmax = [&](auto edge_tag, int t, const uint32_t* vis) {
        constexpr bool kEdge = decltype(edge_tag)::value;
        // One pass with the max as it was: the probabilities wait in registers, and only
        // when a row's max turns out to have grown too far is the pass made again.  The
        // first tile has no such max: it looks for one.
        uint32_t pk[KP / 2];
        float mt;
        float2 l2[2];
        auto pass = [&]() {
          uint32_t s[2][16];
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          const float2 sc2 = make_float2(sc, sc), m2 = make_float2(-m, -m);
          l2[0] = l2[1] = make_float2(0.f, 0.f);
          tmem_ld16(t_s, s[0]);
#pragma unroll
          for (int w = 0; w < KP / 16; ++w) {
            const uint32_t* now = s[w & 1];
            tmem_wait_ld();
            tmem_loaded<16>(s[w & 1]);
            if (w + 1 < KP / 16) tmem_ld16(t_s + 16 * (w + 1), s[(w + 1) & 1]);
            if constexpr (kScores) {
              if (keep && (!kEdge || p00 + t * KP + 16 * w < keep_end)) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                  uint4 v = make_uint4(now[i], now[i + 1], now[i + 2], now[i + 3]);
                  if constexpr (kEdge) {
                    const uint32_t bits = vis[w >> 1] >> ((w & 1) * 16 + i);
                    if (!(bits & 1u)) v.x = kUnseen;
                    if (!(bits & 2u)) v.y = kUnseen;
                    if (!(bits & 4u)) v.z = kUnseen;
                    if (!(bits & 8u)) v.w = kUnseen;
                  }
                  *reinterpret_cast<uint4*>(keep + p00 + t * KP + 16 * w + i) = v;
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float a0 = __uint_as_float(now[i]), a1 = __uint_as_float(now[i + 1]);
              float2 e = fma2(make_float2(a0, a1), sc2, m2);
              e.x = fast_exp2(e.x);
              e.y = fast_exp2(e.y);
              if constexpr (kEdge) {
                const uint32_t bits = vis[w >> 1] >> ((w & 1) * 16 + i);
                if (bits & 1u)
                  m4[i & 3] = fmaxf(m4[i & 3], a0);
                else
                  e.x = 0.f;
                if (bits & 2u)
                  m4[(i & 3) + 1] = fmaxf(m4[(i & 3) + 1], a1);
                else
                  e.y = 0.f;
              } else {
                m4[i & 3] = fmaxf(m4[i & 3], a0);
                m4[(i & 3) + 1] = fmaxf(m4[(i & 3) + 1], a1);
              }
              l2[(i >> 1) & 1] = add2(l2[(i >> 1) & 1], e);
              pk[w * 8 + i / 2] = Mma<T>::pack(e.x, e.y);
            }
          }
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          mt = row_max<T>(mx, sc);
        };
        if (t < ahead) {
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int w = 0; w < KP / 32; ++w) {
            uint32_t s[32];
            tmem_ld32(t_s + 32 * w, s);
            tmem_wait_ld();
            tmem_loaded<32>(s);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!kEdge || ((vis[w] >> i) & 1u)) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(s[i]));
          }
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          m = row_max<T>(mx, sc);
        }
        for (;;) {
          pass();
          const bool grew = mine && mt > m + kRescaleAt;
          if (!__any_sync(0xffffffffu, grew)) break;
          const float m2 = grew ? mt : m;
          const float f = fast_exp2(m - m2);
          m = m2;
          l *= f;
          // the sums of earlier tiles are complete: the scores came after them
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(t_o + c, o);
            tmem_wait_ld();
            tmem_loaded<16>(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(t_o + c, o);
          }
        }
#pragma unroll
        for (int w = 0; w < KP / 32; ++w) tmem_st16(t_s + 16 * w, pk + 16 * w);
        l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
        tmem_wait_st();
      };
      for (int t = joint ? x : 0; t < tiles; t += ahead) {
        const int p0 = p00 + t * KP;
        const bool edge = p0 + KP > ctx;
        uint32_t vis[KP / 32];   // of an edge tile: the positions that the row sees
        if (edge && live) {
          const TreeSeg sg = *seg;
          const int node = (sg.row0 + min(row, sg.rows - 1)) / a.group;
#pragma unroll
          for (int w = 0; w < KP / 32; ++w) {
            const int j0 = p0 + 32 * w - ctx;
            const int k = j0 >> 5;
            vis[w] = __funnelshift_r(mask_word(a, sg, node, k), mask_word(a, sg, node, k + 1), j0 & 31);
          }
        }
        ok = ok && wait(s_ready(x), ns & 1);
        ++ns;
        tmem_fence_after();
        if (live) {
          if (edge)
            softmax(std::true_type(), t, vis);
          else
            softmax(std::false_type(), t, vis);
        }
        tmem_fence_before();
        mbar_arrive(p_ready(x));
      }
      // ---- the piece's rows leave tensor memory -----------------------------------------------
      if (joint) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
          if (y < tiles) {
            ok = ok && wait(o_ready(y), no[y] & 1);
            ++no[y];
          }
        s_ml[x * 128 + r] = make_float2(m, l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
      } else {
        ok = ok && wait(o_ready(x), no[x] & 1);
        ++no[0];
        if (two) ++no[1];
      }
      ok = __all_sync(0xffffffffu, ok);
      tmem_fence_after();
      if (live && ok) {
        const TreeSeg sg = *seg;
        const bool live_row = row < sg.rows;
        const int grow = sg.row0 + min(row, sg.rows - 1);
        const int node = grow / a.group, head = sg.kvh * a.group + grow - node * a.group;
        const size_t io_row = (static_cast<size_t>(sg.tok0 + node) * a.num_heads + head) * D;
        float w0 = 1.f, w1 = 0.f, mm = m, ll = l;
        if (joint) {
          const float2 e0 = s_ml[r], e1 = s_ml[128 + r];
          mm = fmaxf(e0.x, e1.x);
          w0 = fast_exp2(e0.x - mm);
          w1 = fast_exp2(e1.x - mm);
          ll = e0.y * w0 + e1.y * w1;
        }
        const bool dirty = s_dirty[si & 3] == si;
        // rare: what was taken out of V comes back, for the nodes that this row sees
        auto restore = [&](int c, float* f) {
          const int t0 = max(sg.base + sg.tile0 * KP, sg.ctx), t1 = min(sg.base + sg.tile1 * KP, sg.ctx + sg.nodes);
          for (int pos = t0; pos < t1; ++pos) {
            const int j = pos - sg.ctx;
            if (!((mask_word(a, sg, node, j >> 5) >> (j & 31)) & 1u)) continue;
            const int page = tree_page(a.p, sg.bt_row, pos);
            const uint8_t* vrow = a.p.v + (static_cast<size_t>(page) * a.p.num_kv_heads + sg.kvh) *
                                              a.p.page_head_bytes;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const T e = reinterpret_cast<const T*>(
                  vrow + unit_offset(kLayoutCore, pos % a.p.page_size, (c + i) / 8, U) * 16)[(c + i) % 8];
              const float v = to_f32<T>(e);
              if (!isfinite(v)) f[i] += v;
            }
          }
        };
        const int c0 = joint ? x * (D / 2) : 0, c1 = joint ? c0 + D / 2 : D;
        const uint32_t o0 = tmem + lanes + 256 + (joint ? 0 : x * 128);
        const float inv = ll > 0.f ? 1.0f / ll : (ll == 0.f ? 0.f : ll);
        if (live_row && sg.part >= 0 && (!joint || x == 0))
          a.part_ml[sg.part + row] = make_float2(mm, ll);
        if (a.row_ml && live_row && sg.part < 0 && (!joint || x == 0)) a.row_ml[io_row / D] = make_float2(mm, ll);
        const bool add = joint && tiles > 1;
        auto load = [&](int c, uint32_t* o, uint32_t* q) {
          tmem_ld16(o0 + c, o);
          if (add) tmem_ld16(o0 + 128 + c, q);
        };
        auto store = [&](int c, const uint32_t* o, const uint32_t* q) {
          float f[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            f[i] = add ? __uint_as_float(o[i]) * w0 + __uint_as_float(q[i]) * w1 : __uint_as_float(o[i]);
          if (live_row) {
            if (dirty) restore(c, f);
            if (sg.part >= 0) {
              float4* po = reinterpret_cast<float4*>(a.part_o + static_cast<size_t>(sg.part) * D) +
                           (c / 4) * sg.rows + row;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                po[i * sg.rows] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
            } else {
              uint32_t pk[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) pk[i] = Mma<T>::pack(f[2 * i] * inv, f[2 * i + 1] * inv);
              uint4* po = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + io_row + c);
              po[0] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
              po[1] = make_uint4(pk[4], pk[5], pk[6], pk[7]);
            }
          }
          __syncwarp();
        };
        // 16 columns at a time, the next ones on their way
        uint32_t oa[16], qa[16], ob[16], qb[16];
        load(c0, oa, qa);
#pragma unroll 1
        for (int c = c0; c < c1; c += 32) {
          tmem_wait_ld();
          tmem_loaded<16>(oa);
          tmem_loaded<16>(qa);
          if (c + 16 < c1) load(c + 16, ob, qb);
          store(c, oa, qa);
          if (c + 16 < c1) {
            tmem_wait_ld();
            tmem_loaded<16>(ob);
            tmem_loaded<16>(qb);
            if (c + 32 < c1) load(c + 32, oa, qa);
            store(c + 16, ob, qb);
          }
        }
      }
      tmem_fence_before();
      if (joint) asm volatile("bar.sync 1, 256;" ::: "memory");  // both streams' sums are read
      tmem_fence_after();
    }
  }
  __syncthreads();
  // (here, not in the wait, where it costs the loops 4 %)
  if (warp == 1) {
    if (*s_abort && a.gave_up) atomicExch(a.gave_up, 1u);
    tmem_dealloc(tmem, kTmemCols);
  }
}

// =====================================================================================
// fp32 kernel: 64 rows x 64 positions per step in fp32 throughout.  Thread (ty, tx) of
// 16 x 16 takes rows 4 ty ... 4 ty + 3: their scores with positions tx, tx + 16, ..., then
// 16-byte pieces tx, tx + 16, ... of their sums, so that 64 FMAs share 8 shared-memory
// reads of 16 bytes.  A row's scores live in the 16 lanes of a half warp.  The next
// tile's K and V are copied while this one is worked on, where two fit (head_dim <= 128).
// =====================================================================================
constexpr int kF32Rows = 64, kF32Pos = 64, kF32Threads = 256;

template <int NJ>
struct F32Shape {
  static constexpr int kBuffers = NJ <= 2 ? 2 : 1;
};

template <int NJ, bool kScores>
__global__ void __launch_bounds__(kF32Threads, 1) tree_f32_kernel(const TreeArgs a) {
  constexpr int kBuf = F32Shape<NJ>::kBuffers, kPld = kF32Pos + 4;
  extern __shared__ float4 smem4[];
  const int D = a.head_dim, ld = D + 4, U = a.p.row_units;
  float* sq = reinterpret_cast<float*>(smem4);      // [64][D + 4]
  float* sp = sq + kF32Rows * ld;                   // [64][68]
  float* sk = sp + kF32Rows * kPld;                 // [kBuf][64][D + 4]
  float* sv = sk + kBuf * kF32Pos * ld;             // [kBuf][64][D]
  __shared__ size_t s_off[2][kF32Pos];              // byte offset of a position's row, ~0: none
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const uint32_t half = 0xffffu << (threadIdx.x & 16);
  // (the plan's records are no kernel's output: they may be read before the wait)
  const int seg0 = a.cta_segs[blockIdx.x], seg1 = a.cta_segs[blockIdx.x + 1];
  TreeSeg next = a.segs[seg0];
  wait_prerequisites();
  launch_dependents();

  for (int si = seg0; si < seg1; ++si) {
    const TreeSeg sg = next;
    next = a.segs[min(si + 1, seg1 - 1)];
    const int end = sg.ctx + sg.nodes, tiles = sg.tile1 - sg.tile0;
    auto places = [&](int i) {   // threads 0 ... 63: where tile i's rows are
      if (threadIdx.x >= kF32Pos || i >= tiles) return;
      const int pos = sg.base + (sg.tile0 + i) * kF32Pos + threadIdx.x;
      size_t off = ~static_cast<size_t>(0);
      if (pos < end)
        off = (static_cast<size_t>(tree_page(a.p, sg.bt_row, pos)) * a.p.num_kv_heads + sg.kvh) *
                  a.p.page_head_bytes +
              static_cast<size_t>(pos % a.p.page_size) * U * 16;
      s_off[i & 1][threadIdx.x] = off;
    };
    // positions behind the sequence's last are zero, whatever their page holds
    auto fetch = [&](int i) {
      float* k = sk + (i % kBuf) * kF32Pos * ld;
      float* v = sv + (i % kBuf) * kF32Pos * D;
      for (int x = threadIdx.x; x < kF32Pos * U; x += kF32Threads) {
        const int t = x / U, u = x - t * U;
        const size_t off = s_off[i & 1][t];
        const bool there = off != ~static_cast<size_t>(0);
        const size_t at = there ? off + u * 16 : 0;
        copy16_async(smem_u32(k + t * ld + u * 4), a.p.k + at, there ? 16 : 0);
        copy16_async(smem_u32(v + t * D + u * 4), a.p.v + at, there ? 16 : 0);
      }
    };
    __syncthreads();
    places(0);
    for (int x = threadIdx.x; x < kF32Rows * U; x += kF32Threads) {
      const int r = x / U, u = x - r * U;
      const int row = sg.row0 + min(r, sg.rows - 1), node = row / a.group;
      const float* src = reinterpret_cast<const float*>(a.q) +
                         (static_cast<size_t>(sg.tok0 + node) * a.num_heads + sg.kvh * a.group + row -
                          node * a.group) * D;
      copy16_async(smem_u32(sq + r * ld + u * 4), src + u * 4, r < sg.rows ? 16 : 0);
    }
    __syncthreads();
    fetch(0);
    places(1);
    const bool works = 4 * ty < sg.rows;
    float m[4], l[4];
    float4 acc[4][NJ];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = kNegBig;
      l[i] = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int it = 0; it < tiles; ++it) {
      copy_async_wait();
      __syncthreads();
      if (kBuf == 2) {
        if (it + 1 < tiles) fetch(it + 1);
        places(it + 2);
      }
      const float* k = sk + (it % kBuf) * kF32Pos * ld;
      const float* v = sv + (it % kBuf) * kF32Pos * D;
      if (works) {
        float s[4][4] = {};
        for (int d = 0; d < D; d += 4) {
          float4 q4[4], k4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) q4[i] = *reinterpret_cast<const float4*>(sq + (4 * ty + i) * ld + d);
#pragma unroll
          for (int j = 0; j < 4; ++j) k4[j] = *reinterpret_cast<const float4*>(k + (tx + 16 * j) * ld + d);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              s[i][j] = fmaf(q4[i].x, k4[j].x, s[i][j]);
              s[i][j] = fmaf(q4[i].y, k4[j].y, s[i][j]);
              s[i][j] = fmaf(q4[i].z, k4[j].z, s[i][j]);
              s[i][j] = fmaf(q4[i].w, k4[j].w, s[i][j]);
            }
        }
        const int p0 = sg.base + (sg.tile0 + it) * kF32Pos;
        const bool edge = p0 + kF32Pos > sg.ctx;
        const float sc = a.scale_log2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int node = (sg.row0 + min(4 * ty + i, sg.rows - 1)) / a.group;
          float mx = m[i];
          bool see[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int pos = p0 + tx + 16 * j;
            see[j] = !edge || pos < sg.ctx || (pos < end && sees(a, sg.tok0, node, pos - sg.ctx));
            if constexpr (kScores) {
              if (4 * ty + i < sg.rows && pos < end)
                a.scores[score_row(sg, sg.row0 + 4 * ty + i) + pos] = see[j] ? s[i][j] : -INFINITY;
            }
            s[i][j] *= sc;
            if (see[j]) mx = fmaxf(mx, s[i][j]);
          }
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(half, mx, o));
          const float corr = fast_exp2(m[i] - mx);
          m[i] = mx;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = see[j] ? fast_exp2(s[i][j] - mx) : 0.f;
            sum += e;
            sp[(4 * ty + i) * kPld + tx + 16 * j] = e;
          }
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(half, sum, o);
          l[i] = l[i] * corr + sum;
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            acc[i][j].x *= corr;
            acc[i][j].y *= corr;
            acc[i][j].z *= corr;
            acc[i][j].w *= corr;
          }
        }
        __syncwarp(half);
#pragma unroll 2
        for (int t = 0; t < kF32Pos; t += 4) {
          float4 p4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) p4[i] = *reinterpret_cast<const float4*>(sp + (4 * ty + i) * kPld + t);
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) {
            float4 v4[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
              v4[j] = 4 * (tx + 16 * j) < D
                          ? *reinterpret_cast<const float4*>(v + (t + tt) * D + 4 * (tx + 16 * j))
                          : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = (&p4[i].x)[tt];
              // (a position without weight adds nothing, not even where its V is not finite)
              if (edge && p == 0.f) continue;
#pragma unroll
              for (int j = 0; j < NJ; ++j) {
                acc[i][j].x = fmaf(p, v4[j].x, acc[i][j].x);
                acc[i][j].y = fmaf(p, v4[j].y, acc[i][j].y);
                acc[i][j].z = fmaf(p, v4[j].z, acc[i][j].z);
                acc[i][j].w = fmaf(p, v4[j].w, acc[i][j].w);
              }
            }
          }
        }
      }
      if (kBuf == 1 && it + 1 < tiles) {
        __syncthreads();
        fetch(it + 1);
        places(it + 2);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * ty + i;
      if (r >= sg.rows) continue;
      const int row = sg.row0 + r, node = row / a.group;
      const int head = sg.kvh * a.group + row - node * a.group;
      const float inv = l[i] > 0.f ? 1.0f / l[i] : (l[i] == 0.f ? 0.f : l[i]);
      float4* po = sg.part >= 0
                       ? reinterpret_cast<float4*>(a.part_o + static_cast<size_t>(sg.part) * D) + r
                       : reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) +
                                                   (static_cast<size_t>(sg.tok0 + node) * a.num_heads + head) * D);
      const int step = sg.part >= 0 ? sg.rows : 1;
      const float f = sg.part >= 0 ? 1.0f : inv;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = tx + 16 * j;
        if (4 * c < D)
          po[c * step] = make_float4(acc[i][j].x * f, acc[i][j].y * f, acc[i][j].z * f, acc[i][j].w * f);
      }
      if (sg.part >= 0 && tx == 0) a.part_ml[sg.part + r] = make_float2(m[i], l[i]);
      if (a.row_ml) {
        if (sg.part < 0 && tx == 0)
          a.row_ml[static_cast<size_t>(sg.tok0 + node) * a.num_heads + head] = make_float2(m[i], l[i]);
      }
    }
  }
}

// =====================================================================================
// CUDA-core kernel: 32 rows x 32 positions per step, eight warps of four rows.  A lane
// owns one position for the scores and every 32nd dim for the sums; the running max
// and sum of a row are the same in all lanes of its warp.  Bound by latency in small
// batches (4 nodes of one sequence at 511, fp32: 13.5 us with the join), by shared-memory
// reads in large ones (10 TFLOP/s).
// =====================================================================================
constexpr int kSimtRows = kTreeSmall, kSimtPos = kTreeSmall, kSimtThreads = 256;

template <typename T, int DPL, bool kScores>
__global__ void __launch_bounds__(kSimtThreads) tree_simt_kernel(const TreeArgs a) {
  extern __shared__ float4 smem4[];
  const int D = a.head_dim, ld = D + 4;
  float* sq = reinterpret_cast<float*>(smem4);   // [32][D + 4]
  float* sk = sq + kSimtRows * ld;               // [32][D + 4]
  float* sv = sk + kSimtPos * ld;                // [32][D]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int N = 16 / sizeof(T);
  const int U = a.p.row_units;
  // (the plan's records are no kernel's output: they may be read before the wait)
  const int seg0 = a.cta_segs[blockIdx.x], seg1 = a.cta_segs[blockIdx.x + 1];
  TreeSeg next = a.segs[seg0];
  wait_prerequisites();
  launch_dependents();

  for (int si = seg0; si < seg1; ++si) {
    const TreeSeg sg = next;
    next = a.segs[min(si + 1, seg1 - 1)];
    const int end = sg.ctx + sg.nodes;
    __syncthreads();
    for (int x = threadIdx.x; x < kSimtRows * U; x += kSimtThreads) {
      const int r = x / U, u = x - r * U;
      float f[N];
      if (r < sg.rows) {
        const int row = sg.row0 + r, node = row / a.group;
        const int head = sg.kvh * a.group + row - node * a.group;
        const T* src = reinterpret_cast<const T*>(a.q) +
                       (static_cast<size_t>(sg.tok0 + node) * a.num_heads + head) * D + u * N;
        T v[N];
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(src);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = to_f32<T>(v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) sq[r * ld + u * N + e] = f[e];
    }
    float m[4], l[4], acc[4][DPL];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = kNegBig;
      l[i] = 0.f;
#pragma unroll
      for (int d = 0; d < DPL; ++d) acc[i][d] = 0.f;
    }
    for (int tile = sg.tile0; tile < sg.tile1; ++tile) {
      const int p0 = sg.base + tile * kSimtPos;
      __syncthreads();
      // rows behind the sequence's last position are zero, whatever their page holds
      for (int x = threadIdx.x; x < kSimtPos * U; x += kSimtThreads) {
        const int t = x / U, u = x - t * U, pos = p0 + t;
        T kv[N], vv[N];
        uint4 z = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(kv) = z;
        *reinterpret_cast<uint4*>(vv) = z;
        if (pos < end) {
          const int page = tree_page(a.p, sg.bt_row, pos);
          const size_t at = (static_cast<size_t>(page) * a.p.num_kv_heads + sg.kvh) *
                                a.p.page_head_bytes +
                            unit_offset(a.p.layout, pos % a.p.page_size, u, U) * 16;
          *reinterpret_cast<uint4*>(kv) = *reinterpret_cast<const uint4*>(a.p.k + at);
          *reinterpret_cast<uint4*>(vv) = *reinterpret_cast<const uint4*>(a.p.v + at);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          sk[t * ld + u * N + e] = to_f32<T>(kv[e]);
          sv[t * D + u * N + e] = to_f32<T>(vv[e]);
        }
      }
      __syncthreads();
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      const float* kr = sk + lane * ld;
      for (int d = 0; d < D; d += 4) {
        const float4 k4 = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 q4 = *reinterpret_cast<const float4*>(sq + (warp * 4 + i) * ld + d);
          s[i] += q4.x * k4.x + q4.y * k4.y + q4.z * k4.z + q4.w * k4.w;
        }
      }
      const int pos = p0 + lane, j = pos - sg.ctx;
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int node = (sg.row0 + min(warp * 4 + i, sg.rows - 1)) / a.group;
        const bool vis = j < 0 || (pos < end && sees(a, sg.tok0, node, j));
        if constexpr (kScores) {
          if (warp * 4 + i < sg.rows && pos < end)
            a.scores[score_row(sg, sg.row0 + warp * 4 + i) + pos] = vis ? s[i] : -INFINITY;
        }
        const float sc = vis ? s[i] * a.scale_log2 : kNegBig;
        float mx = fmaxf(sc, m[i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float corr = fast_exp2(m[i] - mx);
        p[i] = vis ? fast_exp2(sc - mx) : 0.f;
        float sum = p[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[i] = l[i] * corr + sum;
        m[i] = mx;
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[i][d] *= corr;
      }
#pragma unroll 4
      for (int t = 0; t < kSimtPos; ++t) {
        float v[DPL];
#pragma unroll
        for (int d = 0; d < DPL; ++d) v[d] = lane + 32 * d < D ? sv[t * D + lane + 32 * d] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float pt = __shfl_sync(0xffffffffu, p[i], t);
          // a position without weight adds nothing, not even where its V is not finite
#pragma unroll
          for (int d = 0; d < DPL; ++d) acc[i][d] = fmaf(pt, pt != 0.f ? v[d] : 0.f, acc[i][d]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = warp * 4 + i;
      if (r >= sg.rows) continue;
      if (sg.part >= 0) {
        float* po = a.part_o + static_cast<size_t>(sg.part) * D;
#pragma unroll
        for (int d = 0; d < DPL; ++d) {
          const int c = lane + 32 * d;
          if (c < D) po[(c / 4 * sg.rows + r) * 4 + c % 4] = acc[i][d];
        }
        if (lane == 0) a.part_ml[sg.part + r] = make_float2(m[i], l[i]);
      } else {
        const int row = sg.row0 + r, node = row / a.group;
        const int head = sg.kvh * a.group + row - node * a.group;
        T* po = reinterpret_cast<T*>(a.out) +
                (static_cast<size_t>(sg.tok0 + node) * a.num_heads + head) * D;
        const float inv = l[i] > 0.f ? 1.0f / l[i] : (l[i] == 0.f ? 0.f : l[i]);
        if (a.row_ml) {
          if (lane == 0)
            a.row_ml[static_cast<size_t>(sg.tok0 + node) * a.num_heads + head] = make_float2(m[i], l[i]);
        }
#pragma unroll
        for (int d = 0; d < DPL; ++d)
          if (lane + 32 * d < D) po[lane + 32 * d] = from_f32<T>(acc[i][d] * inv);
      }
    }
  }
}

// =====================================================================================
// Joins: see Join and the functions behind it.
// =====================================================================================
template <typename T>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(const TreeArgs a) {
  const TreeMerge mg = a.merges[blockIdx.x];
  wait_prerequisites();
  launch_dependents();
  merge_rows<T>(a, mg, blockIdx.y * kMergeThreads + threadIdx.x);
}

constexpr int kSharedJoinThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kSharedJoinThreads) shared_join_kernel(const TreeArgs a) {
  const bool mine = blockIdx.x < a.n_joins;
  SharedJoin j = {};
  if (mine) j = a.joins[blockIdx.x];
  wait_prerequisites();
  if (blockIdx.x == 0) rearm_queue(a);
  launch_dependents();
  if (mine) join_rows<T>(a, j, kSharedJoinThreads);
}

// Every kernel here lets its successor begin right behind its own wait, so that nothing
// written ahead of it is still on its way then.  The joins ask for the attention kernels'
// shared-memory split, so that an SM passes from one to the other without a change of it.
template <typename T, int DPL, bool kScores>
cudaError_t run_simt(const TreeArgs& a, cudaStream_t s) {
  const size_t smem = sizeof(float) * (static_cast<size_t>(kSimtRows + kSimtPos) * (a.head_dim + 4) +
                                       static_cast<size_t>(kSimtPos) * a.head_dim);
  const cudaError_t e = allow_smem<tree_simt_kernel<T, DPL, kScores>>(smem);
  if (e != cudaSuccess) return e;
  return launch_early(tree_simt_kernel<T, DPL, kScores>, dim3(a.n_ctas), kSimtThreads, smem, s, a);
}

template <int NJ, bool kScores>
cudaError_t run_f32(const TreeArgs& a, cudaStream_t s) {
  const size_t ld = a.head_dim + 4, buf = F32Shape<NJ>::kBuffers;
  const size_t smem = sizeof(float) * (kF32Rows * ld + kF32Rows * (kF32Pos + 4) +
                                       buf * kF32Pos * (ld + a.head_dim));
  const cudaError_t e = allow_smem<tree_f32_kernel<NJ, kScores>>(smem);
  if (e != cudaSuccess) return e;
  return launch_early(tree_f32_kernel<NJ, kScores>, dim3(a.n_ctas), kF32Threads, smem, s, a);
}

template <typename T, int D, bool kScores>
cudaError_t run_mma(const TreeArgs& a, cudaStream_t s) {
  using S = TreeShape<D>;
  const cudaError_t e = allow_smem<tree_mma_kernel<T, D, kScores>>(S::kSmem);
  if (e != cudaSuccess) return e;
  return launch_early(tree_mma_kernel<T, D, kScores>, dim3(a.n_ctas), S::kThreads, S::kSmem, s, a);
}

template <typename T, bool kScores>
cudaError_t run_mma_any(const TreeArgs& a, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    switch (a.head_dim) {
      case 32: return run_mma<T, 32, kScores>(a, s);
      case 64: return run_mma<T, 64, kScores>(a, s);
      case 96: return run_mma<T, 96, kScores>(a, s);
      case 128: return run_mma<T, 128, kScores>(a, s);
      case 160: return run_mma<T, 160, kScores>(a, s);
      case 192: return run_mma<T, 192, kScores>(a, s);
      case 256: return run_mma<T, 256, kScores>(a, s);
      default: break;
    }
  }
  return cudaErrorInvalidValue;
}

template <typename T, bool kScores>
cudaError_t run_cuda_cores(const TreeArgs& a, const TreeTile& t, cudaStream_t s) {
  if constexpr (sizeof(T) == 4) {
    if (t.rows != kSimtRows) {
      if (a.head_dim <= 64) return run_f32<1, kScores>(a, s);
      if (a.head_dim <= 128) return run_f32<2, kScores>(a, s);
      return run_f32<4, kScores>(a, s);
    }
  }
  if (a.head_dim <= 64) return run_simt<T, 2, kScores>(a, s);
  if (a.head_dim <= 128) return run_simt<T, 4, kScores>(a, s);
  return run_simt<T, 8, kScores>(a, s);
}

template <typename T>
cudaError_t run_tree(const TreeArgs& a, const TreeTile& t, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (a.n_ctas > 0) {
    if (a.weights && a.n_weighs > 0)   // (scores are kept)
      e = t.tensor ? run_mma_any<T, true>(a, s) : run_cuda_cores<T, true>(a, t, s);
    else
      e = t.tensor ? run_mma_any<T, false>(a, s) : run_cuda_cores<T, false>(a, t, s);
  }
  if (e == cudaSuccess && a.weights) return launch_weigh(a, t, s);   // (joins the pieces, too)
  if (e == cudaSuccess && a.n_merges > 0) {
    if ((e = prefer_shared<tree_merge_kernel<T>>()) != cudaSuccess) return e;
    e = launch_early(tree_merge_kernel<T>, dim3(a.n_merges, merge_ctas(a, sizeof(T))), kMergeThreads, 0, s, a);
  }
  return e;
}

}  // namespace

// fp32: the larger tiles do 64 FMAs for 8 shared-memory reads (27 TFLOP/s where the small
// ones reach 10, 32 drafted tokens of 4 sequences at 4000), the small ones start sooner and
// spread further (14.8 against 17.3 us, 4 tokens of one sequence at 511, both with the join
// as it was then, 1.3 us slower): they are taken while all of their tiles find a place on
// the GPU at once.
TreeTile tree_tile(const PoolGeom& g, int64_t small_tiles, int sms) {
  if (decode_uses_mma(g.dtype, g.head_dim, g.page_size) && g.layout == kLayoutCore)
    return g.head_dim <= 128 ? TreeTile{128, 256, 1, kPieceCost, true}
                             : TreeTile{64, 128, 1, kPieceCost, true};
  if (g.elem_size == 4 && small_tiles > 2 * sms) return TreeTile{kF32Pos, kF32Rows, 1, 1, false};
  return TreeTile{kSimtPos, kSimtRows, 2, 0, false};
}

namespace {
template <typename T>
cudaError_t run_shared_join(const TreeArgs& a, cudaStream_t s) {
  const cudaError_t e = prefer_shared<shared_join_kernel<T>>();
  if (e != cudaSuccess) return e;
  return launch_early(shared_join_kernel<T>, dim3(std::max(1, a.n_joins)), kSharedJoinThreads, 0, s, a);
}
}  // namespace

cudaError_t launch_shared_join(const TreeArgs& a, cudaStream_t s) {
  if (a.n_joins == 0 && !a.own_queue) return cudaSuccess;
  switch (a.dtype) {
    case KVC_DTYPE_F16: return run_shared_join<__half>(a, s);
    case KVC_DTYPE_BF16: return run_shared_join<__nv_bfloat16>(a, s);
    case KVC_DTYPE_F32: return run_shared_join<float>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_tree(const TreeArgs& a, const TreeTile& t, cudaStream_t s) {
  switch (a.dtype) {
    case KVC_DTYPE_F16: return run_tree<__half>(a, t, s);
    case KVC_DTYPE_BF16: return run_tree<__nv_bfloat16>(a, t, s);
    case KVC_DTYPE_F32: return run_tree<float>(a, t, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace kvc
