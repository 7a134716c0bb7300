// paged.cuh — what kernels over a paged cache share: pages of a table, lengths, pairs of values, bounded waits.
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
SSDK_DEVINL uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// A bounded wait (about two seconds; then the word is set and false comes back): the clock is read only where the first look fails.
SSDK_DEVINL bool tile_wait(uint64_t* bar, uint32_t parity, unsigned* timeout) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity))
    if (clock64() - t0 > 4000000000LL) {
      if (timeout) *(volatile unsigned*)timeout = 1u;
      return false;
    }
  return true;
}
SSDK_DEVINL bool tile_wait_warp(uint64_t* bar, uint32_t parity, unsigned* timeout) { return __all_sync(0xffffffffu, tile_wait(bar, parity, timeout)); }
#endif

// eight bf16 values as four pairs of fp32, and back
SSDK_DEVINL void pairs_of(const uint4& v, uint64_t* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = (uint64_t)(w[i] & 0xffff0000u) << 32 | w[i] << 16;
}
SSDK_DEVINL uint4 bf16_of(const uint64_t* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x, y;
    unpack2(f[i], &x, &y);
    w[i] = pack_bf16x2(x, y);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kNoPosition = 0x7fffff00;   // of a key that is not there: behind every context

}  // namespace ssdk
