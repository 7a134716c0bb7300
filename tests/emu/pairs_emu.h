// Host stand-ins for the instructions on two values at once (include behind cuda_emu.h, with SSDK_HOST_EMU defined).  TEST INFRASTRUCTURE.
#pragma once
#include "cuda_emu.h"
namespace ssdk {
template <bool MAX>
uint32_t pick_bf16x2(uint32_t a, uint32_t b) {
  uint32_t out = 0;
  for (int i = 0; i < 32; i += 16) {
    const __nv_bfloat16 u{(uint16_t)(a >> i)}, v{(uint16_t)(b >> i)};
    const float x = __bfloat162float(u), y = __bfloat162float(v);
    const uint16_t w = x != x || y != y ? 0x7fff : (MAX ? (x > y ? u.v : v.v) : (x < y ? u.v : v.v));
    out |= (uint32_t)w << i;
  }
  return out;
}
inline void unpack2(uint64_t v, float* x, float* y) {
  const uint32_t a = (uint32_t)v, b = (uint32_t)(v >> 32);
  std::memcpy(x, &a, 4);
  std::memcpy(y, &b, 4);
}
inline uint64_t pack2(float x, float y) {
  uint32_t a, b;
  std::memcpy(&a, &x, 4);
  std::memcpy(&b, &y, 4);
  return (uint64_t)b << 32 | a;
}
inline uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  float x[2], y[2], z[2];
  unpack2(a, x, x + 1);
  unpack2(b, y, y + 1);
  unpack2(c, z, z + 1);
  return pack2(std::fma(x[0], y[0], z[0]), std::fma(x[1], y[1], z[1]));
}
inline uint64_t mul2(uint64_t a, uint64_t b) {
  float x[2], y[2];
  unpack2(a, x, x + 1);
  unpack2(b, y, y + 1);
  return pack2(x[0] * y[0], x[1] * y[1]);
}
inline uint32_t min_bf16x2(uint32_t a, uint32_t b) { return pick_bf16x2<false>(a, b); }
inline uint32_t max_bf16x2(uint32_t a, uint32_t b) { return pick_bf16x2<true>(a, b); }
}  // namespace ssdk
