// What the attention of drafted tokens and the sums of its weights share on the device.
#pragma once

#include "kvc_device.cuh"
#include "kvc_spec.h"
#include "kvc_tcgen05.cuh"
#include "kvcache.h"

namespace kvc {

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

// A score that the row does not see, as it is kept (-inf).
constexpr uint32_t kUnseen = 0xff800000u;
// Where row r of a (sequence, KV head) keeps its scores: rows of whole 16s, in a row.
__device__ __forceinline__ size_t score_row(const TreeSeg& sg, int r) {
  const int pitch = (sg.ctx + sg.nodes + 15) & ~15;
  return static_cast<size_t>(sg.scores) * 16 + static_cast<size_t>(r) * pitch;
}

// Mask word k (drafted tokens 32 k ... 32 k + 31) of a row; below 0: cached positions.
__device__ __forceinline__ uint32_t mask_word(const TreeArgs& a, int tok0, int nodes, int node, int k) {
  if (k < 0) return 0xffffffffu;
  const int left = nodes - 32 * k;
  if (left <= 0) return 0u;
  uint32_t w;
  if (a.mask) {
    w = k < a.mask_words ? a.mask[static_cast<size_t>(tok0 + node) * a.mask_words + k] : 0u;
  } else {
    const int upto = node - 32 * k;  // a chain
    w = upto < 0 ? 0u : (upto >= 31 ? 0xffffffffu : (2u << upto) - 1u);
  }
  return left < 32 ? w & ((1u << left) - 1u) : w;
}

__device__ __forceinline__ uint32_t mask_word(const TreeArgs& a, const TreeSeg& sg, int node, int k) {
  return mask_word(a, sg.tok0, sg.nodes, node, k);
}

// Copies (token, q-head) rows of one KV head into RowBlocks: rows row0 ... row0 + live - 1 of
// the list to places 0 ..., then zeros (kRepeat: the list's first row) up to place n (a
// multiple of 8).  Places from 128 on go `second` bytes further; with `twin` every row goes
// there, too.  Warp w of `warps` takes its eighths of rows; q is that of the list's first token
// and the KV head's first q-head.  What a row needs is carried along: with a division, or a
// handful of instructions more, one warp's copies of 256 rows take 3 us.
template <typename T, int D, bool kRepeat = false>
__device__ __forceinline__ void copy_rows(uint32_t dst, uint32_t second, bool twin, const T* q, int row0,
                                          int live, int n, int group, int row_step, int w, int warps,
                                          int lane) {
  using R = RowBlocks<D>;
  constexpr int kSteps = 8 / R::kRowsPer;       // of eight rows
  const int rr = lane / R::kPieces, piece = lane % R::kPieces;
  const int dn = 8 * warps / group, dr = 8 * warps - dn * group;
  const T* src[kSteps];
  int rem[kSteps];
  uint32_t off[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int r = 8 * w + s * R::kRowsPer + rr, node = (row0 + r) / group;
    rem[s] = row0 + r - node * group;
    src[s] = q + static_cast<size_t>(node) * row_step + rem[s] * D + piece * 8;
    off[s] = dst + R::place((s * R::kRowsPer + rr) & 7, piece);
  }
  const int step = dn * row_step + dr * D, wrap = row_step - group * D;
#pragma unroll 2
  for (int g0 = 8 * w; g0 < n; g0 += 8 * warps) {
    const uint32_t at = (g0 & 127) * (R::kChunk * 2) + (g0 >= 128 ? second : 0u);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const bool here = g0 + s * R::kRowsPer + rr < live;
      const uint32_t bytes = here || kRepeat ? 16 : 0;
      const T* from = here ? src[s] : kRepeat ? q + piece * 8 : q;
#pragma unroll
      for (int i = 0; i < D / R::kChunk; ++i) {
        copy16_async(off[s] + at + i * R::kBytes, from + i * R::kChunk, bytes);
        if (twin) copy16_async(off[s] + at + second + i * R::kBytes, from + i * R::kChunk, bytes);
      }
      src[s] += step;
      rem[s] += dr;
      if (rem[s] >= group) {
        rem[s] -= group;
        src[s] += wrap;
      }
    }
  }
}

// =====================================================================================
// Join of split rows: out = sum_k O_k 2^(m_k - m*) / sum_k l_k 2^(m_k - m*).  A piece's
// partials are stored four dims of all its rows after one another, so that the threads
// of a warp, which own a row each, write and read them side by side.  A thread joins 16
// bytes of output of one row; the pieces are added in position order, so the result does
// not depend on which CTA finished first.
// =====================================================================================
// 16 bytes of output of one row, gathered from pieces.
template <typename T>
struct Join {
  static constexpr int N = 16 / sizeof(T), F = N / 4;
  static constexpr int kAtOnce = 4;   // pieces on their way together
  float mx = kNegBig, sum = 0.f;
  float4 o[F];

  __device__ __forceinline__ Join() {
#pragma unroll
    for (int i = 0; i < F; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // n pieces from partial row `part` on, of `rows` rows each; 16 bytes c of their row r.
  __device__ __forceinline__ void add(const TreeArgs& a, int part, int n, int rows, int r, int c) {
    const float2* ml = a.part_ml + part + r;
    const float4* po = reinterpret_cast<const float4*>(a.part_o + static_cast<size_t>(part) * a.head_dim) +
                       c * F * rows + r;
    const size_t po_step = static_cast<size_t>(rows) * a.head_dim / 4;
    for (int k0 = 0; k0 < n; k0 += kAtOnce) {
      float2 e[kAtOnce];
      float4 v[kAtOnce][F];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const bool there = k0 + k < n;
        e[k] = there ? ml[static_cast<size_t>(k0 + k) * rows] : make_float2(kNegBig, 0.f);
#pragma unroll
        for (int i = 0; i < F; ++i)
          v[k][i] = there ? po[(k0 + k) * po_step + i * rows] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      take(e, v);
    }
  }
  __device__ __forceinline__ void take(const float2 (&e)[kAtOnce], const float4 (&v)[kAtOnce][F]) {
    float m2 = mx;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) m2 = fmaxf(m2, e[k].x);
    const float f = fast_exp2(mx - m2);
    mx = m2;
    sum *= f;
#pragma unroll
    for (int i = 0; i < F; ++i) {
      o[i].x *= f;
      o[i].y *= f;
      o[i].z *= f;
      o[i].w *= f;
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const float w = fast_exp2(e[k].x - mx);
      sum += e[k].y * w;
#pragma unroll
      for (int i = 0; i < F; ++i) {
        o[i].x += v[k][i].x * w;
        o[i].y += v[k][i].y * w;
        o[i].z += v[k][i].z * w;
        o[i].w += v[k][i].w * w;
      }
    }
  }
  // n splits from `split` on of the decode kernel, whose rows are plain; head `head`.
  __device__ __forceinline__ void add_splits(const TreeArgs& a, int split, int n, int head, int c) {
    for (int k0 = 0; k0 < n; k0 += kAtOnce) {
      float2 e[kAtOnce];
      float4 v[kAtOnce][F];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const bool there = k0 + k < n;
        const size_t row = static_cast<size_t>(split + k0 + k) * a.num_heads + head;
        e[k] = there ? a.own_ml[row] : make_float2(kNegBig, 0.f);
#pragma unroll
        for (int i = 0; i < F; ++i)
          v[k][i] = there ? reinterpret_cast<const float4*>(a.own_o + row * a.head_dim)[c * F + i]
                          : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      take(e, v);
    }
  }
  // into 16 bytes c of row `row` of the output, (tokens * heads) rows
  __device__ __forceinline__ void store(const TreeArgs& a, size_t row, int c) const {
    const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
    T v[N];
#pragma unroll
    for (int i = 0; i < F; ++i) {
      v[4 * i] = from_f32<T>(o[i].x * inv);
      v[4 * i + 1] = from_f32<T>(o[i].y * inv);
      v[4 * i + 2] = from_f32<T>(o[i].z * inv);
      v[4 * i + 3] = from_f32<T>(o[i].w * inv);
    }
    T* out = reinterpret_cast<T*>(a.out) + row * a.head_dim + c * N;
    *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(v);
  }
};

// 16 bytes of a merge's output, the x-th along its rows first.
template <typename T>
__device__ __forceinline__ void merge_rows(const TreeArgs& a, const TreeMerge& mg, int x) {
  const int c = x / mg.rows, r = x - c * mg.rows;   // 16 bytes c of row r
  if (c * Join<T>::N >= a.head_dim) return;
  Join<T> join;
  join.add(a, mg.part, mg.n_parts, mg.rows, r, c);
  const int row = mg.row0 + r, node = row / a.group;
  const int head = mg.kvh * a.group + row - node * a.group;
  const size_t out_row = static_cast<size_t>(mg.tok0 + node) * a.num_heads + head;
  join.store(a, out_row, c);
  if (a.row_ml && c == 0) a.row_ml[out_row] = make_float2(join.mx, join.sum);
}

// A run of rows (a sequence's q-heads of one KV head) whose pieces are those of its group's
// prefix, then those of its own positions; by a CTA, 16 bytes of one row a thread.
template <typename T>
__device__ __forceinline__ void join_rows(const TreeArgs& a, const SharedJoin& j, int threads) {
  const int n = j.rows * (a.head_dim / Join<T>::N);
  for (int x = threadIdx.x; x < n; x += threads) {
    const int c = x / j.rows, r = x - c * j.rows;
    Join<T> join;
    join.add(a, j.prefix.part, j.prefix.n, j.prefix.rows, j.prefix.row + r, c);
    if (a.own_o)
      join.add_splits(a, j.own.part, j.own.n, j.head + r, c);
    else
      join.add(a, j.own.part, j.own.n, j.own.rows, j.own.row + r, c);
    const size_t row = static_cast<size_t>(j.token) * a.num_heads + j.head + r;
    join.store(a, row, c);
    if (a.row_ml && c == 0) a.row_ml[row] = make_float2(join.mx, join.sum);
  }
}

// The decode is done: its work list for the next call.  By one CTA, behind its wait and in
// front of the launch of what may use it.
__device__ __forceinline__ void rearm_queue(const TreeArgs& a) {
  if (!a.own_queue) return;
  if (threadIdx.x == 0) {
    *a.own_queue = 0u;
    __threadfence();
  }
  __syncthreads();
}

}  // namespace kvc
