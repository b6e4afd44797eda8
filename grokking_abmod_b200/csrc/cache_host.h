// Host-side checks shared by the cache operators' entry points.
#pragma once

#include <climits>

#include "cache.cuh"
#include "host.h"

namespace mb {
namespace cache {

inline View view_of(const mb_kv_cache& given, uint32_t head_dim) {
  const mb_kv_cache* c = &given;
  need(c->k, "cache k");
  need(c->v, "cache v");
  need(c->k_scale, "cache k_scale");
  need(c->v_scale, "cache v_scale");
  require(c->page_tokens == 16 || c->page_tokens == 32 || c->page_tokens == 64 || c->page_tokens == 128,
          "page_tokens must be 16, 32, 64 or 128");
  require(c->pages >= 1 && c->pages <= (uint32_t)INT_MAX, "pages must be in 1..2^31-1");
  require(c->heads >= 1 && c->heads <= 1024, "cache heads must be in 1..1024");
  require(head_dim >= 1, "head_dim must be positive");
  require(head_dim <= (uint32_t)kMaxHeadDim, "head_dim above 128", MB_ERR_UNSUPPORTED);
  require(c->width == (head_dim + 31) / 32 * 32, "cache width must be head_dim rounded up to 32");
  for (const void* p : {(const void*)c->k, (const void*)c->v})
    require((reinterpret_cast<uintptr_t>(p) & 15) == 0, "cache codes must be 16-byte aligned");
  for (const void* p : {(const void*)c->k_scale, (const void*)c->v_scale})
    require((reinterpret_cast<uintptr_t>(p) & 3) == 0, "cache scales must be aligned");
  int shift = 4;
  while ((1u << shift) < c->page_tokens) ++shift;
  return View{c->k, c->v, c->k_scale, c->v_scale, (int)c->pages, (int)c->heads, (int)c->page_tokens, shift,
              (int)c->width};
}

inline Batch batch_of(const mb_cache_rows& given, uint32_t max_new) {
  const mb_cache_rows* r = &given;
  require(r->batch <= (1u << 24), "batch must be at most 2^24");
  require(r->rows <= (size_t)INT_MAX, "rows must be below 2^31");
  require(max_new <= (uint32_t)INT_MAX, "max_new must be below 2^31");
  if (r->batch > 0) {
    need(r->table, "table");
    need(r->lengths, "lengths");
    require(r->table_pages >= 1 && r->table_pages <= (1u << 26) && r->table_stride >= r->table_pages,
            "the table must hold 1..2^26 pages a sequence, its stride at least as many");
    require(r->offsets != nullptr || max_new == 0 || r->rows == r->batch,
            "without offsets every sequence brings one row");
  }
  return Batch{r->table, r->table_stride, (int)r->table_pages, r->lengths, r->offsets, (int)r->batch, r->rows};
}

}  // namespace cache
}  // namespace mb
