// A paged key-value cache of one attention layer, and the attention of one new
// token per sequence over it (uqm_kv_cache.hip, uqm_paged_attention.hip).
//
// Keys and values each lie in pages [pages, kv_heads, page_size, head_dim]: the
// tokens of a page and head next to each other, so that what one head reads of a
// page is one piece. Sequence b's position p is in page table[b, p / page_size],
// place p % page_size. A table entry outside [0, pages) is no page: nothing is
// written there, and nothing of it is read or attended to.
//
// Elements are BF16, or e4m3 codes with one FP32 scale for a token's head
// ([pages, kv_heads, page_size]; definitions of scales and codes in uqm_fp8.h, a
// group being the head's head_dim values).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace uqm {

constexpr int kMaxHeadDim = 256;   // head_dim: a multiple of 16
constexpr int kMinPage = 16, kMaxPage = 256;  // page_size: a power of two

struct KvPages {
  void* key;
  void* value;
  float* key_scales;    // NULL: BF16
  float* value_scales;
  int64_t pages;
  int kv_heads, page_log2, dim;
};

// Pages of each sequence: entry i of sequence b is table[b * stride + i], i < width.
struct PageTable {
  const int32_t* table;
  int64_t stride;
  int32_t width;
};

// One of the two tensors of new rows: row (b, h, j) starts at
// data + b * batch + h * head + j * token (elements; all multiples of 8).
struct KvRows {
  const uint16_t* data;
  int64_t batch, head, token;
};

struct KvAppendArgs {
  KvPages cache;
  PageTable pages;
  KvRows key, value;
  int64_t batch;
  int32_t tokens;
  const int32_t* starts;  // [batch]
  const int32_t* counts;  // [batch] or NULL: tokens
};
hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t stream);

struct KvReadArgs {
  KvPages cache;
  PageTable pages;
  int64_t batch;
  int32_t length;          // positions of an output row
  const int32_t* lengths;  // [batch]
  uint16_t* key;           // [batch, kv_heads, length, dim]
  uint16_t* value;
};
hipError_t launch_kv_read(const KvReadArgs& a, hipStream_t stream);

struct PagedAttentionArgs {
  KvPages cache;
  PageTable pages;
  const uint16_t* query;   // [batch, heads, dim]
  int64_t batch;
  int heads;
  const int32_t* lengths;  // [batch]
  int32_t window;          // positions seen, from the last one back
  float scale;
  uint16_t* out;           // [batch, heads, dim]
  float* workspace;
};
// Whether the work can be numbered (below 2^30 tiles of 128 positions and 16 query heads).
bool paged_attention_fits(const PagedAttentionArgs& a);
size_t paged_attention_workspace(const PagedAttentionArgs& a, int cus);
hipError_t launch_paged_attention(const PagedAttentionArgs& a, int cus, hipStream_t stream);

}  // namespace uqm
