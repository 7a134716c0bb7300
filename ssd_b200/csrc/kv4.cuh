// kv4.cuh — a paged cache whose keys and values are held in 4 bits: rows quantised as they are written (behind a norm and a rotation, or as they are), and read back.
//
// A cache is uint8 [num_blocks, KV, block_size * (hd / 2 + 4)]: of a page and head first the codes of its tokens, hd / 2 bytes each (byte i: channel 2 i in its low half,
// 2 i + 1 in its high one), then their pairs (scale, minimum) in bf16.  A page's keys of a head are one piece, 17408 bytes for 256 tokens of 128.
// Of a row x of hd bf16 values: minimum m = min x, scale s = (max x - m) / 15 rounded to bf16 (0 where below 2^-126), code = floor((x - m) / s + 1/2), 0 where s = 0;
// the value that stands there is s code + m, rounded once to bf16.  m is one of the values, so it is exact; s rounded down by at most 2^-8 leaves (x - m) / s below 15.06,
// so no code passes 15.  A row that holds something that is not finite, or whose spread passes fp32, is NaN as a whole (both of its pair are).
#pragma once
#include "paged.cuh"

namespace ssdk {

constexpr int kv4_row_bytes(int HD) { return HD / 2 + 4; }   // of a token and head: codes and pair
constexpr uint32_t kKv4Nan = 0x7fc07fc0u;

#ifndef SSDK_HOST_EMU
// (x & a) | b in one operation (two constants would be two)
SSDK_DEVINL uint32_t and_or(uint32_t x, uint32_t a, uint32_t b) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(a), "r"(b));
  return d;
}
// 1 where a >= b, else 0
SSDK_DEVINL float one_if_ge(float a, float b) {
  float d;
  asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// two differences a - b, rounded toward zero
SSDK_DEVINL uint64_t less2_rz(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("sub.rz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// a - b and a b + c of two bf16 values, each rounded once
SSDK_DEVINL uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
SSDK_DEVINL uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
#else   // the same on the host
inline float less_rz(float x, float y) {
  const double a = x, b = y, d = a - b, t = d - a, rest = (a - (d - t)) - (b + t);   // d + rest is the difference
  const float f = (float)d;
  return std::fabs((double)f) > std::fabs(d) || ((double)f == d && rest * d < 0) ? std::nextafter(f, 0.f) : f;
}
inline uint64_t less2_rz(uint64_t a, uint64_t b) {
  float x[2], y[2];
  unpack2(a, x, x + 1);
  unpack2(b, y, y + 1);
  return pack2(less_rz(x[0], y[0]), less_rz(x[1], y[1]));
}
inline uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t out[2];
  for (int i = 0; i < 2; ++i) {
    const double p = (double)__uint_as_float(a >> (16 * i) << 16) * __uint_as_float(b >> (16 * i) << 16), q = __uint_as_float(c >> (16 * i) << 16), d = p + q, t = d - p, rest = (p - (d - t)) + (q - t);
    float f = (float)d;   // toward zero, the last bit set where that is not the sum: such a number is rounded once more as the sum would be
    if (std::isfinite(d) && ((double)f != d || rest != 0)) {
      if (std::fabs((double)f) > std::fabs(d) || ((double)f == d && rest * d < 0)) f = std::nextafter(f, 0.f);
      f = __uint_as_float(__float_as_uint(f) | 1u);
    }
    out[i] = pack_bf16x2(f, 0.f);
  }
  return out[1] << 16 | out[0];
}
inline uint32_t sub_bf16x2(uint32_t a, uint32_t b) { return fma_bf16x2(0x3f803f80u, a, b ^ 0x80008000u); }
#endif

// nibbles P and P + 4 of a word as 16 + c in bf16, and as scale c + low, both of which are there twice
template <int P>
SSDK_DEVINL uint32_t kv4_pair16(uint32_t w) {
  return and_or(P == 0 ? w << 3 : w >> (4 * P - 3), 0x00780078u, 0x41804180u);
}
template <int P>
SSDK_DEVINL uint32_t kv4_value(uint32_t w, uint32_t scale, uint32_t low) {
  return fma_bf16x2(sub_bf16x2(kv4_pair16<P>(w), 0x41804180u), scale, low);
}
// a pair's scale and minimum, twice each
SSDK_DEVINL uint32_t kv4_scales(uint32_t pair) { return __byte_perm(pair, 0, 0x1010); }
SSDK_DEVINL uint32_t kv4_lows(uint32_t pair) { return __byte_perm(pair, 0, 0x3232); }

// Codes of a row whose 16 x LPH values lie with LPH neighbouring lanes, 16 a lane in two pieces of eight.  code: a word of eight channels for each piece; pair: scale | minimum;
// VALUES: the pieces become what the codes stand for.
// A quotient is often a code and a half exactly (x - m has some sixteen bits, s has eight), where a product with 1 / s goes either way.  So the product is made with something below
// 1 / s, which gives the code or the one in front of it, and what it leaves, x - m - code s, is exact in fp32 and decides.  (x - m itself is not, where one of them lies far below the other: it is rounded down,
// which never brings a value to a border that it lies under, and borders are fp32 numbers.)  The nearest whole number stands in the low bits of
// (x - m) r + 1.5 2^23; these words are put together as they are, and their constant parts taken off at the end.  Two values at once: seven instructions a value (32003 rows of 16 heads of 128
// 105 us with one at a time, twice as many; see kv4_store_kernel).
template <int LPH, bool VALUES>
SSDK_DEVINL void kv4_codes(uint4& x, uint4& y, uint32_t (&code)[2], uint32_t& pair) {
  uint32_t w[2][4] = {{x.x, x.y, x.z, x.w}, {y.x, y.y, y.z, y.w}};
  uint32_t lo = w[0][0], hi = w[0][0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_bf16x2(lo, w[i >> 2][i & 3]);
    hi = max_bf16x2(hi, w[i >> 2][i & 3]);
  }
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) {
    lo = min_bf16x2(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_bf16x2(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  lo = min_bf16x2(lo, __byte_perm(lo, lo, 0x1032));
  hi = max_bf16x2(hi, __byte_perm(hi, hi, 0x1032));
  float m = __uint_as_float(lo << 16) + 0.f;   // (a minimum of zero has no sign)
  const float spread = __uint_as_float(hi << 16) - m;
  const bool fine = spread < INFINITY;   // (no NaN, no infinity)
  float s = bf16_round(spread / 15.f);
  if (s < 1.17549435e-38f) s = 0.f;
  pair = fine ? __float_as_uint(s) >> 16 | (__float_as_uint(m) & 0xffff0000u) : kKv4Nan;
  if (!fine) s = m = __uint_as_float(kKv4Nan);
  const float r = s > 0.f ? 1.f / s * (1.f - 0x1p-20f) : 0.f, half = s > 0.f ? 0.5f * s : INFINITY;
  constexpr float kWhole = 12582912.f;   // 1.5 2^23, the word 0x4b400000
  constexpr uint32_t kOff = 0x4b400000u * 0x11111111u;
  const uint64_t one2 = pack2(1.f, 1.f), r2 = pack2(r, r), whole2 = pack2(kWhole, kWhole), less2 = pack2(-kWhole, -kWhole), m2 = pack2(m, m), minus_s2 = pack2(-s, -s);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t acc = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      const uint64_t d = less2_rz((uint64_t)(w[h][i] & 0xffff0000u) << 32 | w[h][i] << 16, m2), c = fma2(fma2(d, r2, whole2), one2, less2);
      float e0, e1;
      unpack2(fma2(c, minus_s2, d), &e0, &e1);
      const uint64_t up = fma2(c, one2, pack2(one_if_ge(e0, half), one_if_ge(e1, half)));   // the codes
      float u0, u1;
      unpack2(fma2(up, one2, whole2), &u0, &u1);
      acc = acc * 256u + (__float_as_uint(u1) * 16u + __float_as_uint(u0));
      if (VALUES) {   // (by way of fp32 a value would be rounded twice)
        float c0, c1;
        unpack2(up, &c0, &c1);
        w[h][i] = fma_bf16x2(pack_bf16x2(c0, c1), kv4_scales(pair), kv4_lows(pair));
      }
    }
    code[h] = fine ? acc - kOff : 0u;
  }
  if (VALUES) {
    x = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
    y = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
  }
}

// ----------------------------------------------------------------------------------
// kv4_store_kernel.  ROPE: queries and keys turn (rope_axes_kernel with one axis), optional norms in front, queries go to q_out; without it rows of keys and values are quantised
// as they are.  Queries are fp32 with one rounding.  A key is rounded to bf16 (what an unquantised cache would hold) and then quantised, and that rounding decides its code next to a
// border: keys' norm and rotation are in 64 bits, so that codes are those of the definition whatever the order of sums.  (Keys are an eighth to a third of the heads.)
// 2 bytes read a channel, 2 written for queries and values that are asked for, 0.53 for codes.  Issue slots 60 % busy with rotation, 69 % without, beside memory: 16000 rows of 32 heads over
// 8 of 128 91 us (71 % of the copy rate; 103 with norms), 32003 rows of 8 heads as they are 60 (76 %), both with the values written back; without them 85 (64 %) and 49 (53 %); 7 rows 2.8.
// Of the 91 and 103 keys in 64 bits make 5 and 11, the remainder that settles a code 1 (none of the 60).  HD / 16 lanes own a head, a warp takes groups of
// 32 / (HD / 16) heads of a row (queries, keys, values behind one another), one or two groups' loads in flight; the rows' groups lie one behind the other and each warp has a stretch of them.
// A row with a position outside the table has NaN queries (and values) and stores nothing; slots outside the cache store nothing.
// ----------------------------------------------------------------------------------
struct Kv4StoreParams {
  const __nv_bfloat16 *q, *k, *v;   // rows of heads; ROPE: of one array, q | k | v
  int64_t q_row, k_row, v_row;      // elements from row to row
  const int64_t* positions;         // [M]
  const int32_t* slots;             // [M]
  const float* table;               // [top, rot] cos | sin
  const __nv_bfloat16 *q_norm_w, *k_norm_w;   // [hd] or null
  __nv_bfloat16 *q_out, *k_values, *v_values;   // [M, H, hd], [M, KV, hd] each or null
  uint8_t *k_cache, *v_cache;
  int64_t top, num_slots;
  float eps;
  int M, heads, kv_heads, rot, block_size;
  int groups;                       // of heads that a warp takes at once, in a row
  int warps, each, longer;          // the rows' groups one behind the other: a warp has a stretch of `each`, the first `longer` one more
};
constexpr int kKv4StoreThreads = 128;
constexpr int kv4_store_blocks(bool rope) { return rope ? 4 : 6; }   // resident on an SM
constexpr int kv4_store_ahead(bool rope) { return rope ? 2 : 1; }    // groups whose loads are in flight beside the one that is worked on
constexpr int kv4_store_heads(int HD) { return 32 / (HD / 16); }   // of a group

SSDK_DEVINL double shfl_xor_f64(double v, int o) {
  union { double d; uint32_t w[2]; } u;
  u.d = v;
  u.w[0] = __shfl_xor_sync(0xffffffffu, u.w[0], o);
  u.w[1] = __shfl_xor_sync(0xffffffffu, u.w[1], o);
  return u.d;
}

// norm (weights w0, w1 of the two pieces, or none) and rotation of a lane's two pieces: in 64 bits, rounded to bf16 by way of fp32
template <int LPH>
SSDK_DEVINL void kv4_turn_f64(uint4& x, uint4& y, const __nv_bfloat16* w0, const __nv_bfloat16* w1, float eps, bool turns, const uint64_t (&co)[4], const uint64_t (&si)[4]) {
  float a[8], b[8];
  unpack_bf16x8(x, a);
  unpack_bf16x8(y, b);
  double scale = 1;
  float wa[8], wb[8];
  if (w0) {   // (the whole warp)
    double sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += (double)a[i] * (double)a[i] + (double)b[i] * (double)b[i];
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) sum += shfl_xor_f64(sum, o);
    scale = 1.0 / sqrt(sum / (16.0 * LPH) + (double)eps);
    unpack_bf16x8(*reinterpret_cast<const uint4*>(w0), wa);
    unpack_bf16x8(*reinterpret_cast<const uint4*>(w1), wb);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    double u = a[i], v = b[i];
    if (w0) {
      u = u * scale * (double)wa[i];
      v = v * scale * (double)wb[i];
    }
    float c[2], s[2];
    unpack2(co[i >> 1], &c[0], &c[1]);
    unpack2(si[i >> 1], &s[0], &s[1]);
    a[i] = (float)(turns ? u * (double)c[i & 1] - v * (double)s[i & 1] : u);
    b[i] = (float)(turns ? v * (double)c[i & 1] + u * (double)s[i & 1] : v);
  }
  x = pack_bf16x8(a);
  y = pack_bf16x8(b);
}
// the same in fp32, two values at once
template <int LPH>
SSDK_DEVINL void kv4_turn_f32(uint4& x, uint4& y, const __nv_bfloat16* w0, const __nv_bfloat16* w1, float eps, bool turns, const uint64_t (&co)[4], const uint64_t (&si)[4]) {
  uint64_t a[4], b[4];
  pairs_of(x, a);
  pairs_of(y, b);
  if (w0) {
    uint64_t sum2 = mul2(a[0], a[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) sum2 = fma2(a[i], a[i], sum2);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum2 = fma2(b[i], b[i], sum2);
    float s0, s1;
    unpack2(sum2, &s0, &s1);
    s0 += s1;
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
    const float scale = rsqrtf(s0 / (16.f * LPH) + eps);
    const uint64_t scale2 = pack2(scale, scale);
    uint64_t w[4];
    pairs_of(*reinterpret_cast<const uint4*>(w0), w);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = mul2(mul2(a[i], scale2), w[i]);
    pairs_of(*reinterpret_cast<const uint4*>(w1), w);
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = mul2(mul2(b[i], scale2), w[i]);
  }
  if (turns) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t t = fma2(a[i], co[i], mul2(b[i], si[i] ^ 0x8000000080000000ull));
      b[i] = fma2(b[i], co[i], mul2(a[i], si[i]));
      a[i] = t;
    }
  }
  x = bf16_of(a);
  y = bf16_of(b);
}

template <int HD, bool ROPE, bool VALUES>
__global__ void __launch_bounds__(kKv4StoreThreads, kv4_store_blocks(ROPE)) kv4_store_kernel(const __grid_constant__ Kv4StoreParams p) {
  constexpr int LPH = HD / 16, SIDE = 32 / LPH, AHEAD = kv4_store_ahead(ROPE);   // lanes of a head, heads side by side
  pdl_wait();
  pdl_launch_dependents();
  const int warp = (int)blockIdx.x * (kKv4StoreThreads / 32) + (int)(threadIdx.x >> 5);
  if (warp >= p.warps) return;
  int unit = warp * p.each + min(warp, p.longer);   // (below 2^31: the host sees to it)
  const int last = unit + p.each + (warp < p.longer);
  const int piece = threadIdx.x % LPH, side = threadIdx.x % 32 / LPH, half = p.rot / 2;
  const int first_k = ROPE ? p.heads : 0, first_v = first_k + p.kv_heads, end = first_v + p.kv_heads;   // of a row's heads
  const bool turns = ROPE && piece < p.rot / 16;
  // channels of a lane's pieces: of heads that turn, and of others
  const int t0 = turns ? piece * 8 : p.rot + (piece - p.rot / 16) * 16, t1 = turns ? half + piece * 8 : t0 + 8;
  const int record = p.block_size * kv4_row_bytes(HD);   // bytes of a page and head

  uint4 a[AHEAD], b[AHEAD];
  int at_m = unit / p.groups, at_head = (unit - at_m * p.groups) * SIDE + side;   // row and head that are asked for next
  auto load = [&](uint4& x, uint4& y) {
    x = y = make_uint4(0, 0, 0, 0);
    if (at_head < end) {
      const bool value = at_head >= first_v;
      const __nv_bfloat16* src;
      if (ROPE) src = p.q + at_m * p.q_row + at_head * HD;
      else src = value ? p.v + at_m * p.v_row + (at_head - first_v) * HD : p.k + at_m * p.k_row + at_head * HD;
      const bool turned = ROPE && !value;
      x = ld_nc_v4(src + (turned ? t0 : piece * 16));
      y = ld_nc_v4(src + (turned ? t1 : piece * 16 + 8));
    }
    at_head += SIDE;
    if (at_head - side >= p.groups * SIDE) {
      at_head = side;
      ++at_m;
    }
  };
  int m = at_m, head0 = at_head - side, row = -1, next_slot = -1;
  int64_t next_at = -1;
  if (unit < last) {
    next_slot = p.slots[m];
    if (ROPE) next_at = p.positions[m];
  }
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (unit + i < last) load(a[i], b[i]);
  bool known = true, stores = false;
  uint64_t co[4] = {}, si[4] = {};
  uint8_t *k_page = p.k_cache, *v_page = p.v_cache;   // of the row's slot: its codes in the page of the first head
  int off = 0;
  auto work = [&](uint4& next_x, uint4& next_y) {
    if (m != row) {
      row = m;
      const int slot = next_slot;
      const int64_t at = next_at;
      if (m + 1 < p.M) {   // (the next row's, which may be another warp's)
        next_slot = p.slots[m + 1];
        if (ROPE) next_at = p.positions[m + 1];
      }
      known = true;
      if (ROPE) {
        known = at >= 0 && at < p.top;
        if (turns && known) {
          const float* angles = p.table + (size_t)at * p.rot + piece * 8;
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float4 c = *reinterpret_cast<const float4*>(angles + 2 * i), s = *reinterpret_cast<const float4*>(angles + half + 2 * i);
            co[i] = pack2(c.x, c.y); co[i + 1] = pack2(c.z, c.w);
            si[i] = pack2(s.x, s.y); si[i + 1] = pack2(s.z, s.w);
          }
        }
      }
      stores = known && slot >= 0 && slot < p.num_slots;
      if (stores) {
        const int page = slot / p.block_size;
        off = slot - page * p.block_size;
        const int64_t at = (int64_t)page * p.kv_heads * record;
        k_page = p.k_cache + at;
        v_page = p.v_cache + at;
      }
    }
    uint4 x = next_x, y = next_y;
    const int head = head0 + side;
    const bool key = head >= first_k && head < first_v, value = head >= first_v, there = head < end;
    const bool some_q = ROPE && head0 < first_k, some_k = head0 < first_v && head0 + SIDE > first_k, some_kv = head0 + SIDE > first_k;   // (of the warp's heads)
    head0 += SIDE;
    if (head0 >= p.groups * SIDE) {
      head0 = 0;
      ++m;
    }
    if (unit + AHEAD < last) load(next_x, next_y);
    const bool turned = ROPE && !value;
    const int c0 = turned ? t0 : piece * 16, c1 = turned ? t1 : piece * 16 + 8;
    if (some_q) {
      uint4 u = x, v = y;
      kv4_turn_f32<LPH>(u, v, p.q_norm_w ? p.q_norm_w + t0 : nullptr, p.q_norm_w ? p.q_norm_w + t1 : nullptr, p.eps, turns, co, si);
      if (head < first_k) {
        x = u;
        y = v;
      }
    }
    if (ROPE && some_k) {
      uint4 u = x, v = y;
      kv4_turn_f64<LPH>(u, v, p.k_norm_w ? p.k_norm_w + t0 : nullptr, p.k_norm_w ? p.k_norm_w + t1 : nullptr, p.eps, turns, co, si);
      if (key) {
        x = u;
        y = v;
      }
    }
    uint32_t code[2], pair;
    if (some_kv) {
      uint4 u = x, v = y;
      kv4_codes<LPH, VALUES>(u, v, code, pair);
      if (VALUES && (key || value)) {
        x = u;
        y = v;
      }
    }
    if (ROPE && !known) x = y = make_uint4(kKv4Nan, kKv4Nan, kKv4Nan, kKv4Nan);
    if (!there) return;
    const int kv_head = head - (value ? first_v : first_k);
    if (!(key || value) || VALUES) {
      __nv_bfloat16* dst = key ? p.k_values + ((size_t)row * p.kv_heads + kv_head) * HD : value ? p.v_values + ((size_t)row * p.kv_heads + kv_head) * HD : p.q_out + ((size_t)row * p.heads + head) * HD;
      __stcs(reinterpret_cast<uint4*>(dst + c0), x);   // (evicted first: 16000 rows rotated 114 -> 110 us)
      __stcs(reinterpret_cast<uint4*>(dst + c1), y);
    }
    if ((key || value) && stores) {
      uint8_t* at = (value ? v_page : k_page) + (int64_t)kv_head * record;
      uint8_t* codes = at + off * (HD / 2);
      if (turned) {
        *reinterpret_cast<uint32_t*>(codes + c0 / 2) = code[0];
        *reinterpret_cast<uint32_t*>(codes + c1 / 2) = code[1];
      } else {
        *reinterpret_cast<uint2*>(codes + c0 / 2) = make_uint2(code[0], code[1]);
      }
      if (piece == 0) *reinterpret_cast<uint32_t*>(at + p.block_size * (HD / 2) + off * 4) = pair;
    }
  };
  while (unit < last) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (unit < last) {
        work(a[i], b[i]);
        ++unit;
      }
  }
}

// ----------------------------------------------------------------------------------
// kv4_load_kernel: value = s code + m of the rows in `slots`, rounded once; rows with a slot outside the cache are zero.
// Bound by memory, mostly by what is written, 2 bytes a channel of 2.53: 64004 rows of 8 heads of 128 56 us, 92 % of the copy rate (codes to floats without conversions, two channels at once; with conversions and places in 64 bits 60).  HD / 8 lanes own a row of a head, eight channels each; a warp takes kKv4LoadRows times as many rows
// as it has room for, all loads in front of the first use.
// ----------------------------------------------------------------------------------
struct Kv4LoadParams {
  const uint8_t *k_cache, *v_cache;
  const int32_t* slots;             // [M]
  __nv_bfloat16 *k, *v;             // [M, KV, hd]
  int64_t num_slots;
  int M, kv_heads, block_size;
};
constexpr int kKv4LoadThreads = 256, kKv4LoadRows = 4;
constexpr int kv4_load_tile(int HD) { return 32 / (HD / 8) * kKv4LoadRows; }   // rows of a warp's tile, of one head

SSDK_DEVINL uint4 kv4_values(uint32_t codes, uint32_t pair) {
  const uint32_t s = kv4_scales(pair), m = kv4_lows(pair);
  const uint32_t v[4] = {kv4_value<0>(codes, s, m), kv4_value<1>(codes, s, m), kv4_value<2>(codes, s, m), kv4_value<3>(codes, s, m)};   // channels P and P + 4
  return make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632));
}

template <int HD>
__global__ void __launch_bounds__(kKv4LoadThreads) kv4_load_kernel(Kv4LoadParams p) {
  constexpr int LPR = HD / 8, SIDE = 32 / LPR, ROWS = kKv4LoadRows;
  pdl_wait();
  pdl_launch_dependents();
  const int piece = threadIdx.x % LPR, side = threadIdx.x % 32 / LPR;
  const uint32_t kv_heads = p.kv_heads, block_size = p.block_size, tiles = (uint32_t)((p.M + SIDE * ROWS - 1) / (SIDE * ROWS)) * kv_heads, step = gridDim.x * (kKv4LoadThreads / 32);   // (below 2^31: the host sees to it)
  const size_t record = (size_t)p.block_size * kv4_row_bytes(HD), pairs = (size_t)p.block_size * (HD / 2);
  for (uint32_t tile = blockIdx.x * (kKv4LoadThreads / 32) + (threadIdx.x >> 5); tile < tiles; tile += step) {
    const uint32_t group = tile / kv_heads, head = tile - group * kv_heads;
    const int m0 = (int)group * (SIDE * ROWS) + side;
    int slot[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int m = m0 + i * SIDE;
      slot[i] = m < p.M ? p.slots[m] : -1;
    }
    uint32_t c[2][ROWS], w[2][ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      c[0][i] = c[1][i] = w[0][i] = w[1][i] = 0;
      if (slot[i] >= 0 && slot[i] < p.num_slots) {
        const uint32_t page = (uint32_t)slot[i] / block_size, off = slot[i] - page * block_size;
        const size_t at = ((size_t)page * kv_heads + head) * record, code = at + (size_t)off * (HD / 2) + piece * 4, pair = at + pairs + (size_t)off * 4;
        c[0][i] = *reinterpret_cast<const uint32_t*>(p.k_cache + code);
        c[1][i] = *reinterpret_cast<const uint32_t*>(p.v_cache + code);
        w[0][i] = *reinterpret_cast<const uint32_t*>(p.k_cache + pair);
        w[1][i] = *reinterpret_cast<const uint32_t*>(p.v_cache + pair);
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int m = m0 + i * SIDE;
      if (m >= p.M) continue;
      const size_t to = ((size_t)m * p.kv_heads + head) * HD + piece * 8;
      __stcs(reinterpret_cast<uint4*>(p.k + to), kv4_values(c[0][i], w[0][i]));
      __stcs(reinterpret_cast<uint4*>(p.v + to), kv4_values(c[1][i], w[1][i]));
    }
  }
}

}  // namespace ssdk
