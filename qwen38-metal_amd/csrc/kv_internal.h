// The paged KV cache object and its bookkeeping, shared by runtime_kv.cpp
// (caches, attention) and runtime_kv_append.cpp (appends and reads of rows).
#pragma once
#include <stdint.h>

#include <vector>

#include "attention.h"
#include "runtime_internal.h"

struct qm_kv {
  qm_runtime* rt = nullptr;
  uint32_t kv_heads = 0;
  uint32_t head_dim = 0;  // the caller's head dimension
  uint32_t dp = 0;        // storage width of a page row (attn_padded_dim)
  uint32_t bits = 8;      // 8 (below) or 4: `k` holds q4kv_block_bytes(dp) a (page, KV head), the others nothing
  uint32_t page_tokens = 16;
  uint32_t max_tokens = 0;  // hard limit (LogicalPageTable capacity); 0 = grow without limit
  uint32_t cap_pages = 0;   // physical pages allocated
  uint32_t length = 0;
  std::vector<int32_t> pages;  // logical page -> physical id, -1 if not materialised [cap_pages]
  int32_t next_page_id = 0;
  int32_t* d_pt = nullptr;  // device page table [cap_pages]
  int8_t* k = nullptr;      // [cap_pages][kv_heads][16][dp]
  int8_t* v = nullptr;      // [cap_pages][kv_heads][dp][16]
  float* ks = nullptr;      // [cap_pages][kv_heads][16]
  float* vs = nullptr;
};

namespace qm {

// Physical capacity for `tokens` tokens: the next power of two (at least 16
// tokens), clamped to the hard limit, copying the materialised pages.
// Synchronous when it grows; a no-op otherwise.
qm_status kv_grow(qm_kv* kv, uint64_t tokens);
// The pages an append of [start, end) would materialise, without changing
// the table: the first new logical page, how many, and the first new id
// (ids are sequential, LogicalPageTable::append).
void plan_pages(const qm_kv* kv, uint32_t start, uint32_t end, int32_t* first_new, int32_t* count, int32_t* first_id);
// Records a planned append in the host table, and takes it back.
void commit_pages(qm_kv* kv, int32_t first_new, int32_t count);
void rollback_pages(qm_kv* kv, int32_t first_new, int32_t count);
// Fills in a prefill's waves, splits and split_tiles (q4: over a 4-bit cache), and takes
// the splits back where there is no room for their partials.
void plan_prefill(const qm_runtime* rt, bool q4, AttnArgs* at);
void unsplit_prefill(AttnArgs* at);

}  // namespace qm
