// Paged key/value cache in e4m3 with one scale per page and KV head: what the append and the attention kernel share.
//   codes  [pages][Hkv][page][D] e4m3,  scales [pages][Hkv] fp32,  value = code * scale
//   page_table [B][max_pages] int32: page_table[b][i] holds tokens [i * page, (i+1) * page) of sequence b
#pragma once
#include "emk_common.cuh"

namespace emk {

constexpr int KV8_MIN_PAGE = 16, KV8_MAX_PAGE = 256;  // powers of two: a 16-token tile lies inside one page

__host__ __device__ __forceinline__ bool kv8_page_ok(int64_t page) {
  return page >= KV8_MIN_PAGE && page <= KV8_MAX_PAGE && (page & (page - 1)) == 0;
}

// A page id from the table, made safe: ids outside the pool are clamped into it (recorded in the bounds-check build).
__device__ __forceinline__ int kv8_page_id(const int* table_row, int64_t slot, int num_pages, int* status) {
  const int p = table_row[slot];
  if (p < 0 || p >= num_pages) emk_record_bounds(status, EMK_DEV_BOUNDS_PAGE);
  return min(max(p, 0), num_pages - 1);
}

}  // namespace emk
