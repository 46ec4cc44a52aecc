// Kernels that move cached rows for drafted tokens and beams:
//   append_rope_kernel    rotation of q and the new K rows fused with the scatter of
//                         the K/V rows into the paged pool
//   commit_kernel         an accepted path's rows moved together, all layers
//   reorder_kernel        beams' open pages and page tables following their parents
// All three are bound by memory traffic: each byte is read once and written once,
// in 16-byte units, and the address arithmetic of a row is shared by its units.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kvc_device.cuh"
#include "kvc_spec.h"
#include "kvcache.h"

namespace kvc {
namespace {

// Byte offset of unit u of position t of a page's KV head h.
__device__ __forceinline__ size_t unit_at(const PagedView& p, int page, int h, int t, int u) {
  return (static_cast<size_t>(page) * p.num_kv_heads + h) * p.page_head_bytes +
         unit_offset(p.layout, t, u, p.row_units) * 16;
}

// The page of `pos` in block-table row `row`, or -1 with the error reported.
__device__ __forceinline__ int page_of(const PagedView& p, int row, int pos) {
  const int col = pos / p.page_size;
  if (row < 0 || row >= p.bt_rows || pos < 0 || col >= p.bt_stride) {
    report_error_at(p.err, KVC_DEVERR_BAD_POSITION, static_cast<uint32_t>(pos));
    return -1;
  }
  const int page = p.block_tables[static_cast<size_t>(row) * p.bt_stride + col];
  if (page < 0 || page >= p.num_pages) {
    report_error_at(p.err, KVC_DEVERR_BAD_PAGE, static_cast<uint32_t>(page));
    return -1;
  }
  return page;
}

template <typename T>
struct Unit {
  static constexpr int N = 16 / sizeof(T);
  union {
    uint4 raw;
    T v[N];
  };
  __device__ Unit() {}
};

// (x0, x1) rotated by the pair's (cos, sin), in 32 bits, rounded once.
template <typename T>
__device__ __forceinline__ void rotate(T& x0, T& x1, float2 cs) {
  const float a = to_f32<T>(x0), b = to_f32<T>(x1);
  x0 = from_f32<T>(a * cs.x - b * cs.y);
  x1 = from_f32<T>(a * cs.y + b * cs.x);
}

// =====================================================================================
// Rotate + append.  One CTA per token: its head_dim / 2 angles are computed once and
// serve all its heads.  The angle p * inv_freq is taken in turns, p * (inv_freq / 2 pi)
// in 64 bits with the whole turns removed, so a far position loses nothing; the rest
// goes through sincospif in 32 bits.  A thread then rotates two 16-byte units whose
// pairs they hold (units 2i, 2i + 1, or i and i + half the row for NeoX) of one head.
// =====================================================================================
constexpr int kAppendThreads = 256;

template <typename T, bool kNeox>
__global__ void __launch_bounds__(kAppendThreads) append_rope_kernel(const AppendRopeArgs a) {
  __shared__ float2 cs[kMaxRopePairs];
  __shared__ int s_page;
  const int tok = blockIdx.x;
  const int pos = a.positions[tok];
  if (pos < 0) return;  // padding
  const int half = a.head_dim / 2;
  for (int i = threadIdx.x; i < half; i += kAppendThreads) {
    double turn = static_cast<double>(a.rope_positions[tok]) * a.turns[i];
    turn -= rint(turn);
    sincospif(2.0f * static_cast<float>(turn), &cs[i].y, &cs[i].x);
  }
  if (threadIdx.x == 0) s_page = page_of(a.p, a.rows ? a.rows[tok] : 0, pos);
  __syncthreads();
  const int page = s_page;
  if (page < 0) return;
  const int t = pos % a.p.page_size;
  const int U = a.p.row_units, Hkv = a.p.num_kv_heads;
  constexpr int N = Unit<T>::N;

  if (U % 2 == 0) {
    const int pairs = U / 2;  // unit pairs of a head
    const int total = (a.num_heads + 2 * Hkv) * pairs;
    for (int x = threadIdx.x; x < total; x += kAppendThreads) {
      const int head = x / pairs, i = x - head * pairs;
      const int u0 = kNeox ? i : 2 * i, u1 = kNeox ? i + pairs : 2 * i + 1;
      const uint8_t* src;
      if (head < a.num_heads)
        src = a.q + tok * a.q_stride + static_cast<size_t>(head) * U * 16;
      else if (head < a.num_heads + Hkv)
        src = a.k_new + tok * a.k_stride + static_cast<size_t>(head - a.num_heads) * U * 16;
      else
        src = a.v_new + tok * a.v_stride + static_cast<size_t>(head - a.num_heads - Hkv) * U * 16;
      Unit<T> x0, x1;
      x0.raw = *reinterpret_cast<const uint4*>(src + u0 * 16);
      x1.raw = *reinterpret_cast<const uint4*>(src + u1 * 16);
      if (head < a.num_heads + Hkv) {
        if (kNeox) {
#pragma unroll
          for (int e = 0; e < N; ++e) rotate(x0.v[e], x1.v[e], cs[u0 * N + e]);
        } else {
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            rotate(x0.v[e], x0.v[e + 1], cs[(u0 * N + e) / 2]);
            rotate(x1.v[e], x1.v[e + 1], cs[(u1 * N + e) / 2]);
          }
        }
      }
      if (head < a.num_heads) {
        uint8_t* dst = a.q_out + (static_cast<size_t>(tok) * a.num_heads + head) * U * 16;
        *reinterpret_cast<uint4*>(dst + u0 * 16) = x0.raw;
        *reinterpret_cast<uint4*>(dst + u1 * 16) = x1.raw;
      } else {
        const bool is_k = head < a.num_heads + Hkv;
        const int h = head - a.num_heads - (is_k ? 0 : Hkv);
        uint8_t* dst = is_k ? a.p.k : a.p.v;
        *reinterpret_cast<uint4*>(dst + unit_at(a.p, page, h, t, u0)) = x0.raw;
        *reinterpret_cast<uint4*>(dst + unit_at(a.p, page, h, t, u1)) = x1.raw;
      }
    }
    return;
  }
  // An odd number of units per row (head_dim 8, 24, 40 ... of 16-bit types): element pairs.
  const int total = (a.num_heads + 2 * Hkv) * half;
  for (int x = threadIdx.x; x < total; x += kAppendThreads) {
    const int head = x / half, i = x - head * half;
    const int i0 = kNeox ? i : 2 * i, i1 = kNeox ? i + half : 2 * i + 1;
    const bool is_q = head < a.num_heads, is_k = !is_q && head < a.num_heads + Hkv;
    const int h = head - (is_q ? 0 : is_k ? a.num_heads : a.num_heads + Hkv);
    const T* src = reinterpret_cast<const T*>(is_q   ? a.q + tok * a.q_stride
                                              : is_k ? a.k_new + tok * a.k_stride
                                                     : a.v_new + tok * a.v_stride) +
                   static_cast<size_t>(h) * a.head_dim;
    T x0 = src[i0], x1 = src[i1];
    if (is_q || is_k) rotate(x0, x1, cs[i]);
    if (is_q) {
      T* dst = reinterpret_cast<T*>(a.q_out) +
               (static_cast<size_t>(tok) * a.num_heads + h) * a.head_dim;
      dst[i0] = x0;
      dst[i1] = x1;
    } else {
      uint8_t* dst = is_k ? a.p.k : a.p.v;
      reinterpret_cast<T*>(dst + unit_at(a.p, page, h, t, i0 / N))[i0 % N] = x0;
      reinterpret_cast<T*>(dst + unit_at(a.p, page, h, t, i1 / N))[i1 % N] = x1;
    }
  }
}

// =====================================================================================
// Commit of an accepted path.  A thread owns one 16-byte unit column of one (layer, K
// or V, head) and moves it for the whole path: it reads up to kCommitBatch sources,
// then writes them, so no thread reads what another writes.  Ascending paths keep the
// batches apart: a later source lies behind every slot written before it.
// =====================================================================================
constexpr int kCommitThreads = 256;
constexpr int kCommitBatch = 8;

__global__ void __launch_bounds__(kCommitThreads) commit_kernel(const CommitArgs a) {
  __shared__ int s_src[kMaxTreeNodes], s_dst[kMaxTreeNodes];   // pages
  __shared__ int s_bad;
  const int seq = blockIdx.y;
  const int len = a.path_lens[seq];
  if (len <= 0) return;
  if (threadIdx.x == 0) s_bad = len > a.path_stride;
  __syncthreads();
  const int ctx = a.ctx[seq];
  const int row = a.rows ? a.rows[seq] : seq;
  const int32_t* path = a.paths + static_cast<size_t>(seq) * a.path_stride;
  for (int j = threadIdx.x; j < min(len, a.path_stride); j += kCommitThreads) {
    const int node = path[j];
    bool ok = node >= j && node < kMaxTreeNodes && (j == 0 || path[j - 1] < node) && ctx >= 0;
    if (!ok) report_error_at(a.p.err, KVC_DEVERR_BAD_POSITION, static_cast<uint32_t>(node));
    int sp = -1, dp = -1;
    if (ok) {
      sp = page_of(a.p, row, ctx + node);
      dp = page_of(a.p, row, ctx + j);
      ok = sp >= 0 && dp >= 0;
    }
    if (!ok) {
      s_bad = 1;
    } else {
      s_src[j] = sp;
      s_dst[j] = dp;
    }
  }
  __syncthreads();
  if (s_bad) {
    if (threadIdx.x == 0) report_error_at(a.p.err, KVC_DEVERR_BAD_POSITION, static_cast<uint32_t>(len));
    return;
  }
  const int U = a.p.row_units, Hkv = a.p.num_kv_heads, ps = a.p.page_size;
  const int total = a.n_layers * 2 * Hkv * U;
  const int x = blockIdx.x * kCommitThreads + threadIdx.x;
  if (x >= total) return;
  const int u = x % U;
  int r = x / U;
  const int h = r % Hkv;
  r /= Hkv;
  uint8_t* base = ((r & 1) ? a.p.v : a.p.k) + static_cast<size_t>(r >> 1) * a.layer_bytes;
  for (int j0 = 0; j0 < len; j0 += kCommitBatch) {
    uint4 v[kCommitBatch];
#pragma unroll
    for (int b = 0; b < kCommitBatch; ++b) {
      const int j = j0 + b;
      if (j < len && path[j] != j)
        v[b] = *reinterpret_cast<const uint4*>(base + unit_at(a.p, s_src[j], h, (ctx + path[j]) % ps, u));
    }
#pragma unroll
    for (int b = 0; b < kCommitBatch; ++b) {
      const int j = j0 + b;
      if (j < len && path[j] != j)
        *reinterpret_cast<uint4*>(base + unit_at(a.p, s_dst[j], h, (ctx + j) % ps, u)) = v[b];
    }
  }
}

// =====================================================================================
// Beam reorder.  blockIdx.x 0 permutes the sequence's page-table columns, the other
// CTAs the rows of its open pages.  A thread owns one column (one 16-byte unit of one
// position, head, layer and K or V) for all beams: it reads every moved beam's new
// value, then writes, so the permutation happens in place without a second buffer.
// =====================================================================================
constexpr int kReorderThreads = 128;

__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const ReorderArgs a) {
  __shared__ int s_parent[kMaxBeams], s_page[kMaxBeams], s_bad;
  const int seq = blockIdx.y, B = a.beams, ps = a.p.page_size;
  const int ctx = a.ctx[seq];
  const int full = ctx / ps, tail = ctx - full * ps;
  int32_t* table = a.tables + static_cast<size_t>(seq) * B * a.p.bt_stride;
  if (threadIdx.x == 0) s_bad = 0;
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
      int32_t v[kMaxBeams];
#pragma unroll
      for (int b = 0; b < kMaxBeams; ++b)
        if (b < B && s_parent[b] != b) v[b] = table[static_cast<size_t>(s_parent[b]) * a.p.bt_stride + c];
#pragma unroll
      for (int b = 0; b < kMaxBeams; ++b)
        if (b < B && s_parent[b] != b) table[static_cast<size_t>(b) * a.p.bt_stride + c] = v[b];
    }
    return;
  }
  const int U = a.p.row_units, Hkv = a.p.num_kv_heads;
  const int per = tail * U;                     // units of one head's open rows
  const size_t total = static_cast<size_t>(a.n_layers) * 2 * Hkv * per;
  const size_t step = static_cast<size_t>(gridDim.x - 1) * kReorderThreads;
  for (size_t x = static_cast<size_t>(blockIdx.x - 1) * kReorderThreads + threadIdx.x; x < total;
       x += step) {
    size_t r = x / per;
    const int tu = static_cast<int>(x - r * per);
    const int h = static_cast<int>(r % Hkv);
    r /= Hkv;
    uint8_t* base = ((r & 1) ? a.p.v : a.p.k) + (r >> 1) * a.layer_bytes;
    // neighbouring threads take neighbouring 16-byte units of the page's layout
    int t, u;
    if (a.p.layout == kLayoutCore) {
      const int blk = tu / (8 * U), in = tu - blk * 8 * U;
      const int rows = min(8, tail - blk * 8);  // rows of the last block may be fewer
      u = in / rows;
      t = blk * 8 + in - u * rows;
    } else {
      t = tu / U;
      u = tu - t * U;
    }
    uint4 v[kMaxBeams];
#pragma unroll
    for (int b = 0; b < kMaxBeams; ++b)
      if (b < B && s_parent[b] != b)
        v[b] = *reinterpret_cast<const uint4*>(base + unit_at(a.p, s_page[s_parent[b]], h, t, u));
#pragma unroll
    for (int b = 0; b < kMaxBeams; ++b)
      if (b < B && s_parent[b] != b)
        *reinterpret_cast<uint4*>(base + unit_at(a.p, s_page[b], h, t, u)) = v[b];
  }
}

template <typename T>
cudaError_t run_append_rope(const AppendRopeArgs& a, cudaStream_t s) {
  if (a.neox)
    append_rope_kernel<T, true><<<a.n, kAppendThreads, 0, s>>>(a);
  else
    append_rope_kernel<T, false><<<a.n, kAppendThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append_rope(const AppendRopeArgs& a, cudaStream_t s) {
  if (a.n <= 0) return cudaSuccess;
  switch (a.dtype) {
    case KVC_DTYPE_F16: return run_append_rope<__half>(a, s);
    case KVC_DTYPE_BF16: return run_append_rope<__nv_bfloat16>(a, s);
    case KVC_DTYPE_F32: return run_append_rope<float>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_commit(const CommitArgs& a, cudaStream_t s) {
  const int64_t total = static_cast<int64_t>(a.n_layers) * 2 * a.p.num_kv_heads * a.p.row_units;
  if (total > (1ll << 30) || a.n > 65535) return cudaErrorInvalidValue;
  const unsigned gx = static_cast<unsigned>((total + kCommitThreads - 1) / kCommitThreads);
  commit_kernel<<<dim3(gx, static_cast<unsigned>(a.n)), kCommitThreads, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_reorder(const ReorderArgs& a, cudaStream_t s) {
  if (a.n > 65535) return cudaErrorInvalidValue;
  const size_t most = static_cast<size_t>(a.n_layers) * 2 * a.p.num_kv_heads * a.p.page_size *
                      a.p.row_units;
  const size_t gx = std::min<size_t>((most + kReorderThreads - 1) / kReorderThreads, 4096);
  reorder_kernel<<<dim3(static_cast<unsigned>(gx) + 1, static_cast<unsigned>(a.n)),
                   kReorderThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace kvc
