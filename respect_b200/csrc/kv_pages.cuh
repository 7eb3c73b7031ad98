// Paged KV cache: device view of the caller's rb_kv_pages.
#pragma once

#include <stdint.h>

#include "../../include/respect_b200.h"

namespace rb {

struct PagesDev {
  uint8_t* store;            // [layers, 2, pages, kv_heads, page_size, row_bytes]
  int layers, pages, kv_heads, page_size, row_bytes;
  int max_seqs, max_pages;
  int32_t *table, *lengths, *held, *refs, *status;
};

}  // namespace rb
