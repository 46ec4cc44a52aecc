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
// the list to places 0 ..., then zeros up to place n (a multiple of 8).  Places from 128 on go
// `second` bytes further; with `twin` every row goes there, too.  Warp w of `warps` takes its
// eighths of rows; q is that of the list's first token and the KV head's first q-head.  What a
// row needs is carried along: with a division, or a handful of instructions more, one warp's
// copies of 256 rows take 3 us.
template <typename T, int D>
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
      const uint32_t bytes = g0 + s * R::kRowsPer + rr < live ? 16 : 0;
      const T* from = bytes ? src[s] : q;
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

}  // namespace kvc
