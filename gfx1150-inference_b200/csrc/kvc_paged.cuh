// Addresses of the paged pool, and 16-byte units of rows, for the kernels that move them.
#pragma once

#include "kvc_device.cuh"
#include "kvc_spec.h"

namespace kvc {

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

// (x0, x1) turned by a pair's (cos, sin), in 32 bits.
__device__ __forceinline__ void turn_pair(float& x0, float& x1, float2 cs) {
  const float a = x0, b = x1;
  x0 = a * cs.x - b * cs.y;
  x1 = a * cs.y + b * cs.x;
}

}  // namespace kvc
