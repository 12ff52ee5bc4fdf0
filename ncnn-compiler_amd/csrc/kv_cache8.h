// The 8-bit cache as its kernels see it.
#pragma once

#include "nhip_internal.h"

namespace nhip {

constexpr float kScaleLeast = 1.17549435e-38f;  // 2^-126: the reciprocal stays finite

struct Kv8 {
  int8_t* k;  // [pages][kv_heads][1 << shift][head_dim]
  int8_t* v;
  float* k_scale;  // [pages][kv_heads]
  float* v_scale;
  const int32_t* table;  // [batch][table_pages]
  int64_t pages, table_pages;
  int32_t kv_heads, head_dim, shift;
};

// Checks the cache and its table; fills *c.
int kv8_args(const nhip_kv8_cache* cache, const int32_t* table, int64_t table_pages, Kv8* c);

// Page `page` of sequence b, -1 where there is none.
__device__ __forceinline__ int64_t kv8_page(const Kv8& c, int b, int64_t page) {
  if (page >= c.table_pages) return -1;
  const int64_t id = c.table[b * c.table_pages + page];
  return id >= 0 && id < c.pages ? id : -1;
}

}  // namespace nhip
