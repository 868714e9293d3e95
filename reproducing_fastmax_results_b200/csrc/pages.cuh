// Pages of moment states: what the serving entry points (decode.cu, tree.cu, cache.cu) check about them.
#pragma once
#include "../../include/fastmax_b200.h"
#include "common.cuh"

namespace fm {

// pb: batch, heads, d and order have been checked before
inline int check_pages(const fastmax_problem* pb, const fastmax_pages& c) {
  if (!c.state || c.pages <= 0) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (c.table == nullptr && c.pages < pb->batch) return FASTMAX_ERR_INVALID_ARGUMENT;
  const long long page = (long long)pb->heads * state_rows(pb->d, pb->order) * state_ld(pb->d);
  if (c.pages > 1 && c.page_stride < page) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(c.state) % 16 != 0 || c.page_stride % 4 != 0) return FASTMAX_ERR_MISALIGNED;
  return FASTMAX_OK;
}

}  // namespace fm
