// The KV cache in 4 bits and in pages, as the kernels see one layer of it (include/malkin_hip.h has the layout).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mk {

struct Kv4 {
  uint8_t *k, *v;
  uint16_t *ks, *vs;
  const int32_t* table;
  int n_layer, layer, n_page, KV, n_seq, max_pages;
  int shift;  // log2 of a page's rows

  // Page of row `row` of sequence `seq`, or -1.
  __device__ __forceinline__ int page_of(int seq, int row) const {
    if (seq < 0 || seq >= n_seq || row < 0 || (row >> shift) >= max_pages) return -1;
    const int p = table[(int64_t)seq * max_pages + (row >> shift)];
    return p >= 0 && p < n_page ? p : -1;
  }
  // Number of the first row of KV head g in page p, among all rows of the pool.
  __device__ __forceinline__ int64_t first_row(int p, int g) const {
    return (((int64_t)p * n_layer + layer) * KV + g) << shift;
  }
};

constexpr int kKv4Group = 32;  // elements that share a scale

}  // namespace mk
