// paged.cuh — what kernels over a paged cache share: pages of a table, lengths, bf16 pairs.
#pragma once
#include "common.cuh"

namespace ssdk {

// the page that a table names, -1 where it is none of the cache's
SSDK_DEVINL int page_at(const int32_t* entry, int64_t num_blocks) {
  const int page = *entry;
  return page >= 0 && page < num_blocks ? page : -1;
}
// tokens of a sequence, held to what its table has room for
SSDK_DEVINL int tokens_of(const int32_t* lens, int b, int max_blocks, int block_size) {
  const long long cap = (long long)max_blocks * block_size, len = lens[b];
  return (int)(len < 0 ? 0 : len < cap ? len : cap);
}

// two channels at once, NaN if one is
#ifndef SSDK_HOST_EMU
SSDK_DEVINL uint32_t min_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
SSDK_DEVINL uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
#endif

}  // namespace ssdk
