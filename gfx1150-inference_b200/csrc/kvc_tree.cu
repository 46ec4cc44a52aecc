// Attention of drafted tokens over the paged cache (kvc_decode_tree).
//
//   out[t, h] = sum_j softmax_j((q[t, h] . k_j) * scale) v_j
//
// over the cached positions of the token's sequence and those drafted tokens that
// its mask row names.  The (node, q-head) pairs of one KV head are the rows of one
// tile, so a K/V byte is read once for all drafted tokens and the whole head group.
//
//   tree_simt_kernel    CUDA cores: fp32 pools and head dims without a tensor tile
//   tree_merge_kernel   joins the pieces of rows whose positions were split over CTAs
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "kvc_device.cuh"
#include "kvc_spec.h"
#include "kvcache.h"

namespace kvc {
namespace {

// Page of `pos` of a sequence; a bad entry is reported and reads page 0.
__device__ __forceinline__ int tree_page(const PagedView& p, int bt_row, int pos) {
  const int col = pos / p.page_size;
  const int page = col < p.bt_stride
                       ? p.block_tables[static_cast<size_t>(bt_row) * p.bt_stride + col]
                       : -1;
  if (page < 0 || page >= p.num_pages) {
    report_error_at(p.err, KVC_DEVERR_BAD_PAGE, static_cast<uint32_t>(page));
    return 0;
  }
  return page;
}

// Whether node `node` of a sequence sees its drafted token j.
__device__ __forceinline__ bool sees(const TreeArgs& a, int tok0, int node, int j) {
  if (!a.mask) return j <= node;
  const int w = j >> 5;
  return w < a.mask_words &&
         ((a.mask[static_cast<size_t>(tok0 + node) * a.mask_words + w] >> (j & 31)) & 1u);
}

// =====================================================================================
// CUDA-core kernel: 32 rows x 32 positions per step, eight warps of four rows.  A lane
// owns one position for the scores and every 32nd dim for the sums; the running max
// and sum of a row are the same in all lanes of its warp.
// =====================================================================================
constexpr int kSimtRows = 32, kSimtPos = 32, kSimtThreads = 256;

template <typename T, int DPL>
__global__ void __launch_bounds__(kSimtThreads) tree_simt_kernel(const TreeArgs a) {
  extern __shared__ float4 smem4[];
  const int D = a.head_dim, ld = D + 4;
  float* sq = reinterpret_cast<float*>(smem4);   // [32][D + 4]
  float* sk = sq + kSimtRows * ld;               // [32][D + 4]
  float* sv = sk + kSimtPos * ld;                // [32][D]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int N = 16 / sizeof(T);
  const int U = a.p.row_units;

  for (int si = a.cta_segs[blockIdx.x]; si < a.cta_segs[blockIdx.x + 1]; ++si) {
    const TreeSeg sg = a.segs[si];
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
      const int p0 = tile * kSimtPos;
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
        float* po = a.part_o + static_cast<size_t>(sg.part + r) * D;
#pragma unroll
        for (int d = 0; d < DPL; ++d)
          if (lane + 32 * d < D) po[lane + 32 * d] = acc[i][d];
        if (lane == 0) a.part_ml[sg.part + r] = make_float2(m[i], l[i]);
      } else {
        const int row = sg.row0 + r, node = row / a.group;
        const int head = sg.kvh * a.group + row - node * a.group;
        T* po = reinterpret_cast<T*>(a.out) +
                (static_cast<size_t>(sg.tok0 + node) * a.num_heads + head) * D;
        const float inv = l[i] > 0.f ? 1.0f / l[i] : (l[i] == 0.f ? 0.f : l[i]);
#pragma unroll
        for (int d = 0; d < DPL; ++d)
          if (lane + 32 * d < D) po[lane + 32 * d] = from_f32<T>(acc[i][d] * inv);
      }
    }
  }
}

// =====================================================================================
// Join of split rows: out = sum_k O_k 2^(m_k - m*) / sum_k l_k 2^(m_k - m*).  A thread
// owns four dims of one row; the pieces of a row are added in position order, so the
// result does not depend on which CTA finished first.
// =====================================================================================
constexpr int kMergeThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(const TreeArgs a) {
  const TreeMerge mg = a.merges[blockIdx.x];
  const int D = a.head_dim, C = D / 4;
  const int x = blockIdx.y * kMergeThreads + threadIdx.x;
  const int r = x / C, c = x - r * C;
  if (r >= mg.rows) return;
  const float2* ml = a.part_ml + mg.part + r;
  float mx = kNegBig;
  for (int k = 0; k < mg.n_parts; ++k) mx = fmaxf(mx, ml[static_cast<size_t>(k) * mg.rows].x);
  float sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < mg.n_parts; ++k) {
    const size_t at = static_cast<size_t>(k) * mg.rows;
    const float2 e = ml[at];
    const float w = fast_exp2(e.x - mx);
    const float4 p = *reinterpret_cast<const float4*>(
        a.part_o + (static_cast<size_t>(mg.part + r) + at) * D + 4 * c);
    sum += e.y * w;
    o.x += p.x * w;
    o.y += p.y * w;
    o.z += p.z * w;
    o.w += p.w * w;
  }
  const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
  const int row = mg.row0 + r, node = row / a.group;
  const int head = mg.kvh * a.group + row - node * a.group;
  T* out = reinterpret_cast<T*>(a.out) +
           (static_cast<size_t>(mg.tok0 + node) * a.num_heads + head) * D + 4 * c;
  out[0] = from_f32<T>(o.x * inv);
  out[1] = from_f32<T>(o.y * inv);
  out[2] = from_f32<T>(o.z * inv);
  out[3] = from_f32<T>(o.w * inv);
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

template <typename T, int DPL>
cudaError_t run_simt(const TreeArgs& a, cudaStream_t s) {
  const size_t smem = sizeof(float) * (static_cast<size_t>(kSimtRows + kSimtPos) * (a.head_dim + 4) +
                                       static_cast<size_t>(kSimtPos) * a.head_dim);
  const cudaError_t e = allow_smem<tree_simt_kernel<T, DPL>>(smem);
  if (e != cudaSuccess) return e;
  tree_simt_kernel<T, DPL><<<a.n_ctas, kSimtThreads, smem, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_tree(const TreeArgs& a, const TreeTile&, cudaStream_t s) {
  cudaError_t e;
  if (a.head_dim <= 64)
    e = run_simt<T, 2>(a, s);
  else if (a.head_dim <= 128)
    e = run_simt<T, 4>(a, s);
  else
    e = run_simt<T, 8>(a, s);
  if (e != cudaSuccess || a.n_merges == 0) return e;
  const int per = a.max_merge_rows * (a.head_dim / 4);
  tree_merge_kernel<T><<<dim3(a.n_merges, (per + kMergeThreads - 1) / kMergeThreads), kMergeThreads,
                         0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

TreeTile tree_tile(const PoolGeom&) { return TreeTile{kSimtPos, kSimtRows, 2, false}; }

cudaError_t launch_tree(const TreeArgs& a, const TreeTile& t, cudaStream_t s) {
  if (a.n_ctas <= 0) return cudaSuccess;
  switch (a.dtype) {
    case KVC_DTYPE_F16: return run_tree<__half>(a, t, s);
    case KVC_DTYPE_BF16: return run_tree<__nv_bfloat16>(a, t, s);
    case KVC_DTYPE_F32: return run_tree<float>(a, t, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace kvc
