// What the paged entry points check of their cache and batch.
#pragma once

#include <stdint.h>

#include "dnx_kernels.h"

namespace dnx {

inline bool cache_ok(const dnx_paged_cache* c) {
  return c != nullptr && c->keys != nullptr && c->values != nullptr &&
         (((uintptr_t)c->keys | (uintptr_t)c->values) & 15) == 0 && c->pages > 0 &&
         c->page >= 16 && c->page <= 4096 && (c->page & (c->page - 1)) == 0 &&
         c->pages <= 0x7fffffff / c->page && (c->hd == 64 || c->hd == 128) && c->kv_heads > 0 &&
         c->kv_heads <= 1024 &&
         (c->type == DNX_F32 || c->type == DNX_BF16 ||
          (c->type == DNX_I8 && c->key_scales != nullptr && c->value_scales != nullptr &&
           (((uintptr_t)c->key_scales | (uintptr_t)c->value_scales) & 15) == 0));
}

// An int8 cache's scales; the fields are not touched for other types, whose callers
// may hold the struct as it was without them.
struct CacheScales {
  float *keys, *values;
};
inline CacheScales cache_scales(const dnx_paged_cache* c) {
  if (c->type != DNX_I8) return {nullptr, nullptr};
  return {c->key_scales, c->value_scales};
}

inline bool batch_ok(const dnx_paged_batch* b) {
  return b != nullptr && b->seqs > 0 && b->seqs <= (1 << 20) && b->tokens >= 0 &&
         b->tokens <= (1 << 22) && b->max_tokens > 0 && b->max_tokens <= (1 << 22) &&
         b->max_len >= 0 && b->max_len <= (1 << 30) && b->prefix_len >= 0 &&
         b->prefix_len <= (1 << 30) && b->prefix_len + b->max_len <= 0x7fffffff && b->table_stride >= 0 && b->table_stride <= (1 << 26) &&
         b->starts != nullptr && b->lens != nullptr &&
         (((uintptr_t)b->starts | (uintptr_t)b->lens | (uintptr_t)b->tables |
           (uintptr_t)b->prefix_pages) & 3) == 0 &&
         (b->tables != nullptr || b->max_len == 0 || b->table_stride == 0) &&
         (b->prefix_pages != nullptr || b->prefix_len == 0);
}

}  // namespace dnx
