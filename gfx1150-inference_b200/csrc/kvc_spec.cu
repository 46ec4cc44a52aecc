// Kernels that move cached rows for drafted tokens and beams:
//   append_rope_kernel    rotation of q and the new K rows fused with the scatter of
//                         the K/V rows into the paged pool
//   commit_kernel         an accepted path's rows moved together, all layers
//   reorder_kernel        beams' open pages and page tables following their parents
// All three are bound by memory traffic: each byte is read once and written once,
// in 16-byte units, and the address arithmetic of a row is shared by its units.
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <algorithm>

#include "kvc_device.cuh"
#include "kvc_paged.cuh"
#include "kvc_spec.h"
#include "kvcache.h"

namespace kvc {
namespace {

// (x0, x1) rotated by the pair's (cos, sin), in 32 bits, rounded once.
template <typename T>
__device__ __forceinline__ void rotate(T& x0, T& x1, float2 cs) {
  const float a = to_f32<T>(x0), b = to_f32<T>(x1);
  x0 = from_f32<T>(a * cs.x - b * cs.y);
  x1 = from_f32<T>(a * cs.y + b * cs.x);
}

// =====================================================================================
// Rotate + append.  kPer threads take a token: its head_dim / 2 angles are computed once and
// serve all its heads.  The angle p * inv_freq is taken in turns, p * (inv_freq / 2 pi) in
// 64 bits with the whole turns removed, so a far position loses nothing; the rest goes
// through sincospif in 32 bits.  A thread owns two 16-byte units that hold each other's
// pairs (units 2i, 2i + 1, or i and i + half the row for NeoX), keeps their angles in
// registers and goes through the heads of q, K and V, kAppendBatch of them on their way;
// the first are asked for before the angles are computed.  Bound by memory traffic: 8,895
// tokens of 32 + 8 + 8 heads of 128 dims, bf16, 45 us for 219 MB (a plain copy of as many
// bytes takes 37); the pool's layout puts a row's pieces 128 bytes apart, which costs 4 us
// of it.  64 threads per token measured best of 32, 64, 128 and 256, and four CTAs of two
// pairs a thread better than three of three (47 us).
// =====================================================================================
constexpr int kAppendThreads = 256;
constexpr int kAppendBatch = 2;

template <typename T, bool kNeox, int kPer>
__global__ void __launch_bounds__(kAppendThreads, 4) append_rope_kernel(const AppendRopeArgs a) {
  constexpr int kTok = kAppendThreads / kPer;
  __shared__ float2 cs[kTok * kMaxRopePairs];
  __shared__ int s_page[kTok], s_slot[kTok];
  const int tok0 = blockIdx.x * kTok, half = a.head_dim / 2;
  const int toks = min(kTok, a.n - tok0);
  const int U = a.p.row_units, Hkv = a.p.num_kv_heads;
  constexpr int N = Unit<T>::N;
  const int pairs = U / 2;                     // unit pairs of a head
  const int heads = a.num_heads + 2 * Hkv;     // q, K and V heads
  const bool whole = U % 2 == 0;               // units pair up
  const int tok = threadIdx.x / kPer, me = threadIdx.x % kPer;
  const int at_once = whole ? kPer / pairs : 1;
  const int row0 = whole ? me / pairs : 0, i = whole ? me - row0 * pairs : 0;
  const int u0 = kNeox ? i : 2 * i, du = kNeox ? pairs : 1;
  const bool works = whole && tok < toks && row0 < at_once;
  const size_t t = tok0 + tok;
  const size_t row_bytes = static_cast<size_t>(U) * 16;
  wait_prerequisites();

  struct Item {
    Unit<T> x0, x1;
  };
  const uint8_t* q_src = a.q + t * a.q_stride + u0 * 16;
  const uint8_t* k_src = a.k_new + t * a.k_stride + u0 * 16;
  const uint8_t* v_src = a.v_new + t * a.v_stride + u0 * 16;
  auto load = [&](int head, Item& it) {
    const uint8_t* src = head < a.num_heads         ? q_src + head * row_bytes
                         : head < a.num_heads + Hkv ? k_src + (head - a.num_heads) * row_bytes
                                                    : v_src + (head - a.num_heads - Hkv) * row_bytes;
    it.x0.raw = *reinterpret_cast<const uint4*>(src);
    it.x1.raw = *reinterpret_cast<const uint4*>(src + du * 16);
  };
  Item items[kAppendBatch];
#pragma unroll
  for (int k = 0; k < kAppendBatch; ++k)
    if (works && row0 + k * at_once < heads) load(row0 + k * at_once, items[k]);

  for (int x = threadIdx.x; x < toks * half; x += kAppendThreads) {
    const int tk = kTok == 1 ? 0 : x / half, j = x - tk * half;
    double turn = static_cast<double>(a.rope_positions[tok0 + tk]) * a.turns[j];
    turn -= rint(turn);
    // (by pair of a unit pair, then unit pair: neighbouring threads read neighbouring angles)
    float2& out = cs[tk * half + (whole ? j % N * pairs + j / N : j)];
    sincospif(2.0f * static_cast<float>(turn), &out.y, &out.x);
  }
  if (threadIdx.x < toks) {
    const int pos = a.positions[tok0 + threadIdx.x];
    s_page[threadIdx.x] = pos < 0 ? -1 : page_of(a.p, a.rows ? a.rows[tok0 + threadIdx.x] : 0, pos);
    s_slot[threadIdx.x] = pos < 0 ? 0 : pos % a.p.page_size;
  }
  __syncthreads();
  if (works) {
    const int page = s_page[tok];
    if (page < 0) return;                      // padding, or reported
    float2 c[N];
#pragma unroll
    for (int k = 0; k < N; ++k) c[k] = cs[tok * half + k * pairs + i];
    uint8_t* q_dst = a.q_out + t * a.num_heads * row_bytes + u0 * 16;
    const size_t place = unit_at(a.p, page, 0, s_slot[tok], u0);
    const int dp = du * (a.p.layout == kLayoutCore ? 128 : 16);
    for (int h0 = row0; h0 < heads; h0 += kAppendBatch * at_once) {
#pragma unroll
      for (int k = 0; k < kAppendBatch; ++k) {
        const int head = h0 + k * at_once;
        if (head >= heads) break;
        Item& it = items[k];
        if (head < a.num_heads + Hkv) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            if (kNeox)
              rotate(it.x0.v[e], it.x1.v[e], c[e]);
            else if (e < N / 2)
              rotate(it.x0.v[2 * e], it.x0.v[2 * e + 1], c[e]);
            else
              rotate(it.x1.v[2 * e - N], it.x1.v[2 * e - N + 1], c[e]);
          }
        }
        if (head < a.num_heads) {
          uint8_t* d = q_dst + head * row_bytes;
          *reinterpret_cast<uint4*>(d) = it.x0.raw;
          *reinterpret_cast<uint4*>(d + du * 16) = it.x1.raw;
        } else {
          const bool is_k = head < a.num_heads + Hkv;
          uint8_t* d = (is_k ? a.p.k : a.p.v) + place +
                       (head - a.num_heads - (is_k ? 0 : Hkv)) * a.p.page_head_bytes;
          *reinterpret_cast<uint4*>(d) = it.x0.raw;
          *reinterpret_cast<uint4*>(d + dp) = it.x1.raw;
        }
      }
      const int next = h0 + kAppendBatch * at_once;
#pragma unroll
      for (int k = 0; k < kAppendBatch; ++k)
        if (next + k * at_once < heads) load(next + k * at_once, items[k]);
    }
    return;
  }
  if (whole) return;
  // An odd number of units per row (head_dim 8, 24, 40 ... of 16-bit types): element pairs.
  for (int x = threadIdx.x; x < toks * heads * half; x += kAppendThreads) {
    const int tk = x / (heads * half), r = x - tk * heads * half;
    const int head = r / half, j = r - head * half;
    const int page = s_page[tk];
    if (page < 0) continue;
    const size_t row = tok0 + tk;
    const int i0 = kNeox ? j : 2 * j, i1 = kNeox ? j + half : 2 * j + 1;
    const bool is_q = head < a.num_heads, is_k = !is_q && head < a.num_heads + Hkv;
    const int h = head - (is_q ? 0 : is_k ? a.num_heads : a.num_heads + Hkv);
    const T* src = reinterpret_cast<const T*>(is_q   ? a.q + row * a.q_stride
                                              : is_k ? a.k_new + row * a.k_stride
                                                     : a.v_new + row * a.v_stride) +
                   static_cast<size_t>(h) * a.head_dim;
    T x0 = src[i0], x1 = src[i1];
    if (is_q || is_k) rotate(x0, x1, cs[tk * half + j]);
    if (is_q) {
      T* dst = reinterpret_cast<T*>(a.q_out) + (row * a.num_heads + h) * a.head_dim;
      dst[i0] = x0;
      dst[i1] = x1;
    } else {
      uint8_t* dst = is_k ? a.p.k : a.p.v;
      reinterpret_cast<T*>(dst + unit_at(a.p, page, h, s_slot[tk], i0 / N))[i0 % N] = x0;
      reinterpret_cast<T*>(dst + unit_at(a.p, page, h, s_slot[tk], i1 / N))[i1 % N] = x1;
    }
  }
}

// =====================================================================================
// Commit of an accepted path.  A CTA moves one layer's K and V of one sequence.  Eight threads
// take eight steps of the path in one 16-byte column (a unit of one head), whose new places
// lie side by side in the pool's 8-position blocks; longer paths go eight steps at a time.
// All of a batch is read before any of it is written, and ascending paths keep the batches
// apart: a later source lies behind every slot written before it.
// The rows come in 16-byte pieces 128 bytes apart, and memory is read 64 bytes at a time:
// the sources alone cost four times their bytes, which is what bounds this (32 paths of up
// to 8 nodes, 32 layers: 18 MB moved, 107 MB read; 27 us over states in turn that do not stay
// in L2, 22 on one that does).
// =====================================================================================
constexpr int kCommitThreads = 128;
constexpr int kCommitSteps = 8;     // of a path at a time
constexpr int kCommitCols = 8;      // columns of a thread in flight

__global__ void __launch_bounds__(kCommitThreads) commit_kernel(const CommitArgs a) {
  __shared__ int s_page[2][kMaxTreeNodes], s_t[2][kMaxTreeNodes];   // [source, target]
  __shared__ int s_bad;
  if (threadIdx.x == 0) s_bad = 0;
  wait_prerequisites();
  const int seq = blockIdx.y;
  const int len = a.path_lens[seq], ctx = a.ctx[seq];
  const int row = a.rows ? a.rows[seq] : seq;
  const int32_t* path = a.paths + static_cast<size_t>(seq) * a.path_stride;
  if (len <= 0) return;
  __syncthreads();
  for (int j = threadIdx.x; j < min(len, a.path_stride); j += kCommitThreads) {
    const int node = path[j];
    // (a context near 2^31 would overflow the sums below, and with them page_of's checks)
    const bool ok = node >= j && node < kMaxTreeNodes && (j == 0 || path[j - 1] < node) && ctx >= 0 &&
                    ctx <= INT_MAX - kMaxTreeNodes && len <= a.path_stride;
    const int sp = ok ? page_of(a.p, row, ctx + node) : -1, dp = ok ? page_of(a.p, row, ctx + j) : -1;
    if (sp < 0 || dp < 0) {
      report_error_at(a.p.err, KVC_DEVERR_BAD_POSITION, static_cast<uint32_t>(node));
      s_bad = 1;
    }
    s_page[0][j] = sp;
    s_page[1][j] = node == j ? -1 : dp;   // a row that stays is not touched
    s_t[0][j] = ok ? (ctx + node) % a.p.page_size : 0;
    s_t[1][j] = ok ? (ctx + j) % a.p.page_size : 0;
  }
  if (len > a.path_stride && threadIdx.x == 0) {
    report_error_at(a.p.err, KVC_DEVERR_BAD_POSITION, static_cast<uint32_t>(len));
    s_bad = 1;
  }
  __syncthreads();
  if (s_bad) return;
  const int U = a.p.row_units, half = a.p.num_kv_heads * U, cols = 2 * half;
  const size_t layer = blockIdx.x * a.layer_bytes;
  auto cell = [&](int c, int page, int t) {
    const int d = c < half ? c : c - half;
    return reinterpret_cast<uint4*>((c < half ? a.p.k : a.p.v) + layer + unit_at(a.p, page, d / U, t, d % U));
  };
  const int step = threadIdx.x % kCommitSteps, col0 = threadIdx.x / kCommitSteps;
  constexpr int kColsAtOnce = kCommitThreads / kCommitSteps;
  for (int j0 = 0; j0 < len; j0 += kCommitSteps) {
    const int j = j0 + step;
    const bool moves = j < len && s_page[1][j] >= 0;
    const int rounds = (cols + kColsAtOnce - 1) / kColsAtOnce;
    for (int c0 = 0; c0 < rounds; c0 += kCommitCols) {
      uint4 v[kCommitCols];
#pragma unroll
      for (int k = 0; k < kCommitCols; ++k) {
        const int c = col0 + (c0 + k) * kColsAtOnce;
        if (moves && c < cols)
          v[k] = *cell(c, s_page[0][j], s_t[0][j]);
      }
      __syncwarp();   // a column's steps are threads of one warp: all read, then all write
#pragma unroll
      for (int k = 0; k < kCommitCols; ++k) {
        const int c = col0 + (c0 + k) * kColsAtOnce;
        if (moves && c < cols) *cell(c, s_page[1][j], s_t[1][j]) = v[k];
      }
    }
  }
}

// =====================================================================================
// Beam reorder.  blockIdx.x 0 permutes the sequence's page-table columns, every other CTA one
// head of one layer's K or V in the open pages.  A thread owns one 16-byte unit of a page
// for all beams: it reads every moved beam's new value, then writes, so the permutation
// happens in place without a second buffer.  The units in front of `tail` positions are
// taken in the order of memory; of the last 8-position block only some rows are.  8 x 8
// beams, 32 layers, 149 MB: 32.4 us over states in turn (23 at the copy rate), where each of
// the 4,104 short CTAs makes its sequence's checks before its first byte moves; replayed on
// one state, part of which stays in L2, 27 (28.4 with 128 threads, 44 with 256).
// =====================================================================================
constexpr int kReorderThreads = 64;

template <int kBeams>
__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const ReorderArgs a) {
  __shared__ int s_parent[kMaxBeams], s_page[kMaxBeams], s_bad;
  if (threadIdx.x == 0) s_bad = 0;
  wait_prerequisites();
  const int seq = blockIdx.y, B = a.beams, ps = a.p.page_size;
  const int ctx = a.ctx[seq];
  const int full = ctx / ps, tail = ctx - full * ps;
  int32_t* table = a.tables + static_cast<size_t>(seq) * B * a.p.bt_stride;
  __syncthreads();
  if (threadIdx.x < B) {
    const int b = threadIdx.x;
    const int par = a.parents[static_cast<size_t>(seq) * B + b];
    const bool fits = ctx >= 0 && static_cast<int64_t>(ctx) <= static_cast<int64_t>(a.p.bt_stride) * ps;
    if (par < 0 || par >= B || !fits) {
      report_error_at(a.p.err, KVC_DEVERR_BAD_POSITION, static_cast<uint32_t>(fits ? par : ctx));
      s_bad = 1;
    }
    int page = -1 - b;
    if (fits && tail > 0) {
      page = table[static_cast<size_t>(b) * a.p.bt_stride + full];
      if (page < 0 || page >= a.p.num_pages) {
        report_error_at(a.p.err, KVC_DEVERR_BAD_PAGE, static_cast<uint32_t>(page));
        s_bad = 1;
      }
    }
    s_parent[b] = par;
    s_page[b] = page;
  }
  __syncthreads();
  if (threadIdx.x < B && tail > 0) {
    for (int b = 0; b < threadIdx.x; ++b)
      if (s_page[b] == s_page[threadIdx.x]) {  // an open page of two beams
        report_error_at(a.p.err, KVC_DEVERR_BAD_PAGE, static_cast<uint32_t>(s_page[b]));
        s_bad = 1;
      }
  }
  __syncthreads();
  if (s_bad) return;
  if (blockIdx.x == 0) {
    for (int c = threadIdx.x; c < full; c += kReorderThreads) {
      int32_t v[kBeams];
#pragma unroll
      for (int b = 0; b < kBeams; ++b)
        if (b < B && s_parent[b] != b) v[b] = table[static_cast<size_t>(s_parent[b]) * a.p.bt_stride + c];
#pragma unroll
      for (int b = 0; b < kBeams; ++b)
        if (b < B && s_parent[b] != b) table[static_cast<size_t>(b) * a.p.bt_stride + c] = v[b];
    }
    return;
  }
  const int r = blockIdx.x - 1, h = r % a.p.num_kv_heads, lk = r / a.p.num_kv_heads;
  uint8_t* base = ((lk & 1) ? a.p.v : a.p.k) + static_cast<size_t>(lk >> 1) * a.layer_bytes +
                  static_cast<size_t>(h) * a.p.page_head_bytes;
  const size_t page_bytes = a.p.page_head_bytes * a.p.num_kv_heads;
  const int U = a.p.row_units;
  const bool core = a.p.layout == kLayoutCore;
  const int whole = core ? tail / 8 * 8 * U : tail * U;        // units of whole blocks
  const int units = core ? (tail + 7) / 8 * 8 * U : whole, rows = tail & 7;
  for (int x = threadIdx.x; x < units; x += kReorderThreads) {
    if (x >= whole && (x & 7) >= rows) continue;
    uint4 v[kBeams];
#pragma unroll
    for (int b = 0; b < kBeams; ++b)
      if (b < B && s_parent[b] != b)
        v[b] = *reinterpret_cast<const uint4*>(base + s_page[s_parent[b]] * page_bytes + x * 16);
#pragma unroll
    for (int b = 0; b < kBeams; ++b)
      if (b < B && s_parent[b] != b) *reinterpret_cast<uint4*>(base + s_page[b] * page_bytes + x * 16) = v[b];
  }
}

// No kernel here lets its successor begin early: they write K/V rows, and a decode two
// launches on may stream those as soon as the launch between them has begun.

// Many tokens: 64 threads each, four in a CTA; few tokens: a CTA each.
template <typename T, bool kNeox>
cudaError_t run_append_rope(const AppendRopeArgs& a, cudaStream_t s) {
  if (a.n >= 4 * a.sms)
    return launch_early(append_rope_kernel<T, kNeox, 64>, dim3((a.n + 3) / 4), kAppendThreads, 0, s, a);
  return launch_early(append_rope_kernel<T, kNeox, kAppendThreads>, dim3(a.n), kAppendThreads, 0, s, a);
}

}  // namespace

cudaError_t launch_append_rope(const AppendRopeArgs& a, cudaStream_t s) {
  if (a.n <= 0) return cudaSuccess;
  switch (a.dtype) {
    case KVC_DTYPE_F16: return a.neox ? run_append_rope<__half, true>(a, s) : run_append_rope<__half, false>(a, s);
    case KVC_DTYPE_BF16: 
      return a.neox ? run_append_rope<__nv_bfloat16, true>(a, s) : run_append_rope<__nv_bfloat16, false>(a, s);
    case KVC_DTYPE_F32: return a.neox ? run_append_rope<float, true>(a, s) : run_append_rope<float, false>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_commit(const CommitArgs& a, cudaStream_t s) {
  return launch_early(commit_kernel, dim3(static_cast<unsigned>(a.n_layers), static_cast<unsigned>(a.n)),
                      kCommitThreads, 0, s, a);
}

cudaError_t launch_reorder(const ReorderArgs& a, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(2 * a.n_layers * a.p.num_kv_heads + 1), static_cast<unsigned>(a.n));
  if (a.beams <= 4) return launch_early(reorder_kernel<4>, grid, kReorderThreads, 0, s, a);
  if (a.beams <= 8) return launch_early(reorder_kernel<8>, grid, kReorderThreads, 0, s, a);
  return launch_early(reorder_kernel<16>, grid, kReorderThreads, 0, s, a);
}

}  // namespace kvc
