// What the attention of drafted tokens and the sums of its weights share on the device.
#pragma once

#include "kvc_device.cuh"
#include "kvc_spec.h"
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

}  // namespace kvc
