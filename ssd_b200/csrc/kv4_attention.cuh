// kv4_attention.cuh — attention over a paged cache held in 4 bits (kv4.cuh), on mma.sync: a step's tokens of a sequence, up to sixteen query rows of a key head at a time.
#pragma once
#include <cooperative_groups.h>

#include <type_traits>

#include "async_copy.cuh"
#include "kv4.cuh"

namespace ssdk {

// ----------------------------------------------------------------------------------
// kv4_attn_kernel: softmax(scale q k^T) v, causal to the end of the context as in paged attention (query j of a sequence sees positions <= len - Q + j), grouped heads.
// With k = s c + m and v = s' c' + m' of a token (c codes)
//   q k = s (q c) + m sum(q)          O = sum_j (P_j s'_j) (c'_j - 8) + sum_j P_j (m'_j + 8 s'_j)
// so that what meets in the products are codes, which are exact: keys and values are not rounded at all.  What is rounded is P s' (bf16, 2^-8 of a term at most, the codes
// around their middle so that it is of the value's size); sums, references and the second term are fp32.
// Bound by the instructions that make codes into fragments, then by the bytes of the cache: 48 contexts of 16000 (64 heads over 8 of 128) 129 us, 76 % of the copy rate, integer pipe 56 % (in
// loops of seconds the power limit makes that 144, 68 %); one of 32000 (32 heads) 20, where it is latency.  The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that
// keys (sixteen) and channels (sixteen) are the m of mma and the eight query rows of a usual group its n.
//   Scores are whole numbers: a mask (and a shift) makes four codes of a word bytes, and a query row, scaled by a power of two so that its largest lies in 2^14 .. 2^15 and rounded, is 256 h + l with a
// byte each, so that its values are off by at most 2^-15 of its largest (those above 2^-7 of it by nothing).  (bf16 codes take 64 instructions for sixteen keys where these take 24; mma on e4m3 is
// made of conversions and f16 here: four times as slow.)  Which channels a product's k stands for is free: a quad's lanes read a key's row, 16 bytes each, and the query's fragments follow.
//   Values: P has no such range, it is bf16 and so are the codes: 16 + c has c in the top of bf16's mantissa, 128 + c in its end (no shift for the first of four codes).  ldmatrix turns the rows of
// codes so that a register's halves are four channels each of two keys, which is what the fragments of four products need.  A product of P s' with ones beside them sums what the constants too many
// amount to, of the rounded weights, and is taken off every 256 keys, while the sums that cancel are small.
// Chunks of 32 keys go round a block's warps, each with a ring of its own (cp.async, no barrier between warps) and a softmax of its own; at the end warps meet, then blocks.
// Which blocks work on which keys: few keys are shared by the blocks of a cluster, one to a sequence and key head, whose parts meet in shared memory (one launch).  Many keys (SHARED) are one
// long row of turns, W chunks each, of which every block has an equal stretch, whatever the lengths: where a stretch begins or ends inside a head's keys it leaves a part in global memory, and
// kv4_join_kernel puts the parts together.
// A page outside the cache is passed over, a row that sees no key is zero; a NaN row of keys or values makes NaN of the rows that see it and of no other.
// ----------------------------------------------------------------------------------
struct Kv4AttnParams {
  const __nv_bfloat16* q;        // [B * Q, H, hd]
  const uint8_t *k_cache, *v_cache;
  const int32_t* tables;         // [B, max_blocks]
  const int32_t* lens;           // [B]
  __nv_bfloat16* out;            // [B * Q, H, hd]
  int64_t num_blocks;
  int B, Q, heads, kv_heads, block_size, max_blocks;
  float scale_log2;              // scale * log2(e)
  float* parts;                  // SHARED: [blocks][2][rows of a key head][HD + 4]: O, reference, sum of a block's first stretch where it began in front of it, and of its last
};
// Weights are exp2(score - reference), the reference the largest score that it was raised for, raised again when a score passes that by 2^8.  Keys whose values have a scale or minimum of 2^65 or more find it
// 2^32 above their scores: of them and the sum of weights all sums are 2^-32 of what they would be, and values up to bf16's largest number (here times codes less 8 that come with 128 more) pass fp32's in none.
// What that costs is weights below 2^-94 of the largest (else 2^-126); in front of small values it would cost their own bits, since P s' is subnormal in bf16 then (for scales below 2^-94; zero from 2^-102 on).
constexpr float kKv4Slack = 8.f, kKv4Above = 32.f;
SSDK_DEVINL bool kv4_large(uint32_t pair) { return (pair & pair << 1 & 0x40004000u) != 0; }   // (an exponent's two top bits)
constexpr int kKv4Most = 16, kKv4Stages = 3, kKv4Keys = 32;   // blocks of a cluster, a warp's ring, keys of a chunk
constexpr int kv4_stage_bytes(int HD) { return 2 * kKv4Keys * (HD / 2 + 4); }   // keys' codes | values' codes | keys' pairs | values' pairs
constexpr int kv4_attn_smem(int HD, int NT, int W) {
  const int ring = W * kKv4Stages * kv4_stage_bytes(HD), join = (W + 1) * 8 * NT * (HD + 8) * 4;
  return ring > join ? ring : join;
}

SSDK_DEVINL uint32_t transpose_8x8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// 16 x 8 (+)= codes (bytes) x 32 bytes of a query, signed or not; the first product of a sum takes zeros that need no registers
template <bool SIGNED, bool FIRST>
SSDK_DEVINL void mma_u8_16832(int (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
#define SSDK_U8(TYPE)                                                                                                                                                             \
  if (FIRST)                                                                                                                                                                      \
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8." TYPE ".s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"                                           \
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));                                       \
  else                                                                                                                                                                            \
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8." TYPE ".s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                                             \
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  if constexpr (SIGNED) { SSDK_U8("s8") } else { SSDK_U8("u8") }
#undef SSDK_U8
}
// where the 16-byte piece c of the codes of value r lies in its stage: pieces c of eight rows, which ldmatrix reads together, are in banks of their own
template <int HD>
SSDK_DEVINL int kv4_v_place(int r, int c) {
  return HD == 128 ? r * 64 + ((c ^ (r >> 1 & 3)) << 4) : r * 32 + ((c ^ (r >> 2 & 1)) << 4);
}
// nibble P of both halves of a word as 16 + c (128 + c for the first) in bf16
template <int P>
SSDK_DEVINL uint32_t kv4_nibble(uint32_t w) {
  return P == 0 ? and_or(w, 0x000f000fu, 0x43004300u) : and_or(w >> (4 * P - 3), 0x00780078u, 0x41804180u);
}

// ---- shares of all turns: turn x of the row of them is one of the key heads of sequence b, kv_heads * (turns of a head of those in front) + head * turns(b) + ..; fewer than 2^31 in all (the host sees
// to it) ----
// turns of a key head's keys, one at least (whose block writes the zeros of rows that see nothing)
template <int KEYS>
SSDK_DEVINL int kv4_turns(const Kv4AttnParams& p, int b) { return max(1, (tokens_of(p.lens, b, p.max_blocks, p.block_size) + KEYS - 1) / KEYS); }
// turns of a head of all sequences, and of those in front of sequence b (every lane of a warp asks, and gets them)
template <int KEYS>
SSDK_DEVINL int2 kv4_turns_of_all(const Kv4AttnParams& p, int b) {
  int all = 0, before = 0;
  for (int x = threadIdx.x & 31; x < p.B; x += 32) {
    const int turns = kv4_turns<KEYS>(p, x);
    all += turns;
    before += x < b ? turns : 0;
  }
  return make_int2((int)__reduce_add_sync(0xffffffffu, (unsigned)all), (int)__reduce_add_sync(0xffffffffu, (unsigned)before));
}
// the sequence that turn `at` of the whole row belongs to, and the turns of a head in front of it
template <int KEYS>
SSDK_DEVINL int kv4_sequence_of(const Kv4AttnParams& p, int at, int* before) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  for (int base = 0; base < p.B; base += 32) {
    const int mine = base + lane < p.B ? kv4_turns<KEYS>(p, base + lane) : 0;
    int sum = mine;
#pragma unroll
    for (int w = 1; w < 32; w *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, sum, w);
      if (lane >= w) sum += x;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, base + lane < p.B && at < (run + sum) * p.kv_heads);
    if (past) {
      const int x = __ffs(past) - 1;
      *before = run + __shfl_sync(0xffffffffu, sum - mine, x);
      return base + x;
    }
    run += __shfl_sync(0xffffffffu, sum, 31);
  }
  *before = run;
  return p.B;   // (behind the end)
}
// stretches of `all` turns for so many blocks: the first ones have one more; where block x begins, and which block has turn t
struct Kv4Stretch {
  int each, longer;
  SSDK_DEVINL Kv4Stretch(int all, int blocks) : each(all / blocks), longer(all - all / blocks * blocks) {}
  SSDK_DEVINL int first(int x) const { return x * each + min(x, longer); }
  SSDK_DEVINL int block(int t) const {
    const int split = longer * (each + 1);
    return t < split ? t / (each + 1) : longer + (t - split) / each;   // (each > 0 where t >= split)
  }
};

// NT tiles of eight rows, W warps; sixteen (eight with two tiles) warps are resident on an SM
template <int HD, int NT, int W, bool SHARED>
__global__ void __launch_bounds__(W * 32, 16 / NT / W) kv4_attn_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int KW = HD / 32, VW = HD / 64, CODES = HD / 2, K = kKv4Keys, STAGE = kv4_stage_bytes(HD);
  extern __shared__ __align__(16) uint8_t kv4_smem[];
  pdl_wait();
  pdl_launch_dependents();
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = SHARED ? 1 : (int)cluster.num_blocks(), rank = SHARED ? 0 : (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.heads / p.kv_heads, R = G * p.Q;   // at most 8 NT rows
  int kvh = blockIdx.x / C, b = blockIdx.y;
  // SHARED: this block's turns at .. end, the first of them turn `turn` of its head
  int at = 0, end = 1, turn = 0, turns = 0;
  if constexpr (SHARED) {
    const Kv4Stretch stretch(kv4_turns_of_all<W * K>(p, 0).x * p.kv_heads, gridDim.x);
    at = stretch.first(blockIdx.x);
    end = stretch.first(blockIdx.x + 1);
    if (at >= end) return;
    int before;
    b = kv4_sequence_of<W * K>(p, at, &before);
    if (b >= p.B) return;   // (only where lengths change meanwhile)
    turns = kv4_turns<W * K>(p, b);
    const int from = at - before * p.kv_heads;
    kvh = from / turns;
    turn = from - kvh * turns;
  }
#pragma unroll 1
  for (bool again = false;; again = true) {
  if constexpr (SHARED) {
    if (again) {
      if (at >= end) break;
      turn = 0;
      if (++kvh == p.kv_heads) {
        kvh = 0;
        if (++b >= p.B) break;   // (only where lengths change meanwhile)
        turns = kv4_turns<W * K>(p, b);
      }
    }
  }
  const int len = tokens_of(p.lens, b, p.max_blocks, p.block_size), ctx = len - p.Q;
  const int seen_by_all = ctx + 1;   // positions that all rows see

  // ---- a warp's chunks of 32 keys: own, own + stride, ... ----
  const int tiles = (len + 15) >> 4, last_turn = SHARED ? min(turns, turn + (end - at)) : 0;
  const int chunks = SHARED ? min((tiles + 1) >> 1, last_turn * W) : (tiles + 1) >> 1, stride = C * W, own = (SHARED ? turn * W : rank * W) + warp;
  const int n = own < chunks ? (chunks - own + stride - 1) / stride : 0;
  const int record = p.block_size * kv4_row_bytes(HD);   // bytes of a page and head
  uint8_t* ring = kv4_smem + warp * kKv4Stages * STAGE;
  // Where a chunk lies is looked up by a lane: pages of whole chunks 32 chunks at a time, others sixteen, two lanes (of sixteen keys each) a chunk; the next ones' on their way.
  const bool one_page = p.block_size % K == 0;
  const int per = one_page ? 1 : 2, ahead = 32 / per;
  const int64_t page_step = (int64_t)p.kv_heads * record;
  struct Where { int64_t codes; int pairs; };   // bytes from the head's first code of the cache (-1: no page), and from there to the pairs
  auto look_up = [&](int first) {
    Where w = {-1, 0};
    const long long chunk = own + (long long)(first + lane / per) * stride, tile = one_page ? 2 * chunk : 2 * chunk + (lane & 1);
    if (tile < tiles) {
      const int pos = (int)tile * 16, x = pos / p.block_size, off = pos - x * p.block_size;
      const int page = page_at(p.tables + (size_t)b * p.max_blocks + x, p.num_blocks);
      if (page >= 0) w.codes = page * page_step + off * CODES;
      w.pairs = (p.block_size - off) * CODES + off * 4;
    }
    return w;
  };
  Where here = {-1, 0}, next = look_up(0);
  const uint8_t *k_from = p.k_cache + (int64_t)kvh * record + lane * 16, *v_from = p.v_cache + (int64_t)kvh * record + lane * 16;
  const uint8_t* pair_from = ((one_page ? lane & 8 : lane & 4) ? p.v_cache : p.k_cache) + (int64_t)kvh * record + (one_page ? lane & 7 : lane & 3) * 16;
  const int v_to = K * CODES + kv4_v_place<HD>(lane / (CODES / 16), lane % (CODES / 16));
  const int pair_to = 2 * K * CODES + (one_page ? lane * 16 : (lane >> 2) * K * 4 + (lane & 3) * 16);
  uint32_t missing = 0;   // two bits a stage: sixteen keys without a page
  auto load = [&](int i, int stage) {
    if (i >= n) return;
    if ((i & (ahead - 1)) == 0) {
      here = next;
      next = look_up(i + ahead);
    }
    uint8_t* to = ring + stage * STAGE;
    missing &= ~(3u << (2 * stage));
    auto from_lane = [&](int src) {
      Where w;
      w.codes = (int64_t)((uint64_t)(uint32_t)__shfl_sync(0xffffffffu, (int)(here.codes >> 32), src) << 32 | (uint32_t)__shfl_sync(0xffffffffu, (int)here.codes, src));
      w.pairs = __shfl_sync(0xffffffffu, here.pairs, src);
      return w;
    };
    if (one_page) {
      const Where w = from_lane(i & 31);
      if (w.codes < 0) {
        missing |= 3u << (2 * stage);
        return;
      }
      const uint8_t *kc = k_from + w.codes, *vc = v_from + w.codes;
#pragma unroll
      for (int u = 0; u < K * CODES; u += 512) {   // (32 rows of a values' place are 512 bytes on, too)
        cp_async16(to + u + lane * 16, kc + u, true);
        cp_async16(to + u + v_to, vc + u, true);
      }
      if (lane < 16) cp_async16(to + pair_to, pair_from + w.codes + w.pairs, true);
      return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Where w = from_lane((2 * i + h) & 31);
      if (w.codes < 0) {
        missing |= 1u << (2 * stage + h);
        continue;
      }
      const uint8_t *kc = k_from + w.codes, *vc = v_from + w.codes;
#pragma unroll
      for (int u = 0; u < 16 * CODES; u += 512) {
        cp_async16(to + h * 16 * CODES + u + lane * 16, kc + u, true);
        cp_async16(to + h * 16 * CODES + u + v_to, vc + u, true);
      }
      if (lane < 8) cp_async16(to + h * 64 + pair_to, pair_from + w.codes + w.pairs, true);
    }
  };
#pragma unroll
  for (int s = 0; s < kKv4Stages - 1; ++s) {
    load(s, s);
    cp_async_commit();
  }

  // ---- queries: fragments in the order of the keys' words (channels 0, 2, 4, 6 and 1, 3, 5, 7 of a word), sums ----
  uint32_t qb[NT][KW][2][2];   // [.., byte, half of k]
  float qs[NT][2], qf[NT][2];  // of rows 2 t, 2 t + 1: sum and unit, times scale * log2(e)
  int lim[NT][2];              // first position that they do not see
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + g;
    const __nv_bfloat16* q = p.q + ((size_t)(b * p.Q + r / G) * p.heads + kvh * G + r % G) * HD + t * (HD / 4);
    float f[KW][8], sum = 0.f, top = 0.f;
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      unpack_bf16x8(nt * 8 + g < R ? *reinterpret_cast<const uint4*>(q + j * 8) : make_uint4(0, 0, 0, 0), f[j]);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        sum += f[j][c];
        top = fmaxf(top, fabsf(f[j][c]));
      }
    }
#pragma unroll
    for (int w = 1; w < 4; w *= 2) {
      sum += __shfl_xor_sync(0xffffffffu, sum, w);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    }
    const int e = max((int)(__float_as_uint(top) >> 23), 14);   // (biased exponent)
    const float up = __uint_as_float((uint32_t)(268 - e) << 23);   // 2^(14 - (e - 127))
#pragma unroll
    for (int j = 0; j < KW; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        qb[nt][j][0][h] = qb[nt][j][1][h] = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t w = (uint32_t)__float2int_rn(f[j][2 * c + h] * up);   // 256 h + l
          qb[nt][j][0][h] |= (w >> 8 & 0xffu) << (8 * c);
          qb[nt][j][1][h] |= (w & 0xffu) << (8 * c);
        }
      }
    // a score is 1 / up = 2^(e - 127) 2^-14 times what the products give; a query that is not finite makes NaN (its sum alone might not)
    float unit = __uint_as_float((uint32_t)min(e, 254) << 23) * p.scale_log2 * 0x1p-14f;
    if (!(fabsf(sum) < INFINITY) || e == 255) unit = __uint_as_float(kKv4Nan);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = nt * 8 + 2 * t + i;
      qs[nt][i] = __shfl_sync(0xffffffffu, sum, (2 * t + i) * 4) * p.scale_log2;
      qf[nt][i] = __shfl_sync(0xffffffffu, unit, (2 * t + i) * 4);
      lim[nt][i] = row < R ? ctx + row / G + 1 : 0;
    }
  }

  float o[NT][HD / 16][4], one[NT][4], ref[NT][2], l[NT][2], low[NT][2];   // O^T, sum of P s', reference, sum, sum of P (m' + 8 s')
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    one[nt][0] = one[nt][1] = one[nt][2] = one[nt][3] = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      ref[nt][e] = -INFINITY;
      l[nt][e] = low[nt][e] = 0.f;
    }
  }

  // scores of a chunk's keys g, g + 8, .. and rows 2 t, 2 t + 1 to weights, and their product with the values.  MASK: some row does not see some key, or a page is missing
  const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  auto work = [&](const uint8_t* in, int x, int pos, uint32_t none, bool large, auto mask) {   // (x: which sixteen of the chunk; large: some value of it is, kKv4Above)
    constexpr bool MASK = decltype(mask)::value;
    const uint32_t* pairs = reinterpret_cast<const uint32_t*>(in + 2 * K * CODES) + g;
    float s[NT][4];
    uint32_t hidden = 0;   // bits of the scores
    {
      uint32_t k[2][KW];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* row = in + (x * 16 + h * 8 + g) * CODES + t * (CODES / 4);
        if constexpr (HD == 128) {
          const uint4 w = *reinterpret_cast<const uint4*>(row);
          k[h][0] = w.x; k[h][1] = w.y; k[h][2] = w.z; k[h][3] = w.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(row);
          k[h][0] = w.x; k[h][1] = w.y;
        }
      }
      int whole[NT][2][4];
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        const uint32_t a[4] = {k[0][j] & 0x0f0f0f0fu, k[1][j] & 0x0f0f0f0fu, k[0][j] >> 4 & 0x0f0f0f0fu, k[1][j] >> 4 & 0x0f0f0f0fu};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (j == 0) {
            mma_u8_16832<true, true>(whole[nt][0], a, qb[nt][j][0][0], qb[nt][j][0][1]);
            mma_u8_16832<false, true>(whole[nt][1], a, qb[nt][j][1][0], qb[nt][j][1][1]);
          } else {
            mma_u8_16832<true, false>(whole[nt][0], a, qb[nt][j][0][0], qb[nt][j][0][1]);
            mma_u8_16832<false, false>(whole[nt][1], a, qb[nt][j][1][0], qb[nt][j][1][1]);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w = pairs[x * 16 + h * 8];
        const float sk = __uint_as_float(w << 16), mk = __uint_as_float(w & 0xffff0000u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& v = s[nt][2 * h + e];
            v = (float)(whole[nt][0][2 * h + e] * 256 + whole[nt][1][2 * h + e]);   // (below 2^27)
            v = fmaf(v, sk * qf[nt][e], mk * qs[nt][e]);
            if (MASK && ((none >> x & 1u) || pos + x * 16 + h * 8 + g >= lim[nt][e])) {
              v = -INFINITY;
              hidden |= 1u << (nt * 4 + 2 * h + e);
            }
          }
      }
    }
    // a row's reference is raised, and its sums rescaled, only when a score passes it by kKv4Slack (base 2)
    float most[NT][2];
    bool grow = large;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        most[nt][e] = fmaxf(s[nt][e], s[nt][2 + e]);
        grow = grow || most[nt][e] > ref[nt][e] + kKv4Slack;
      }
    if (__any_sync(0xffffffffu, grow)) {
      const float above = __any_sync(0xffffffffu, large) ? kKv4Above : 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = most[nt][e];
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) + above, ref[nt][e]);
          const float f = top == ref[nt][e] ? 1.f : ex2_ftz(ref[nt][e] - top);   // (from -inf: 0)
          ref[nt][e] = top;
          l[nt][e] *= f;
          low[nt][e] *= f;
          one[nt][e] *= f;
          one[nt][2 + e] *= f;
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            o[nt][i][e] *= f;
            o[nt][i][2 + e] *= f;
          }
        }
    }
    {
      uint32_t pb[NT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t pair = pairs[K + x * 16 + h * 8];
        const float sv = __uint_as_float(pair << 16), mv = fmaf(8.f, sv, __uint_as_float(pair & 0xffff0000u));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float y = ex2_ftz(s[nt][2 * h + e] - (MASK && ref[nt][e] == -INFINITY ? 0.f : ref[nt][e]));
            l[nt][e] += y;
            if (MASK && (hidden >> (nt * 4 + 2 * h + e) & 1u)) {   // (its pair may be anything: 0 x NaN is NaN)
              w[e] = 0.f;
            } else {
              low[nt][e] = fmaf(y, mv, low[nt][e]);
              w[e] = y * sv;
            }
          }
          pb[nt][h] = transpose_8x8(pack_bf16x2(w[0], w[1]));
        }
      }
      // [keys 0 .. 7, 8 .. 15][32 channels of 64]: lane 8 i + r names row r of matrix i
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        uint32_t w[4];   // keys 2 t, 2 t + 1 of channels 64 j + 4 g .., of 32 more; the same of keys 8 on
        ldmatrix_x4_trans(w, in + K * CODES + x * 16 * CODES + kv4_v_place<HD>((lane & 7) + 8 * (lane >> 4), 2 * j + (lane >> 3 & 1)));
        const uint32_t a[4][4] = {{kv4_nibble<0>(w[0]), kv4_nibble<0>(w[1]), kv4_nibble<0>(w[2]), kv4_nibble<0>(w[3])}, {kv4_nibble<1>(w[0]), kv4_nibble<1>(w[1]), kv4_nibble<1>(w[2]), kv4_nibble<1>(w[3])},
                                  {kv4_nibble<2>(w[0]), kv4_nibble<2>(w[1]), kv4_nibble<2>(w[2]), kv4_nibble<2>(w[3])}, {kv4_nibble<3>(w[0]), kv4_nibble<3>(w[1]), kv4_nibble<3>(w[2]), kv4_nibble<3>(w[3])}};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(o[nt][4 * j + i], a[i], pb[nt][0], pb[nt][1]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(one[nt], ones, pb[nt][0], pb[nt][1]);
    }
  };

  auto take_off = [&]() {   // (the rows of `one` are alike)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = fmaf(i & 3 ? -24.f : -136.f, one[nt][e], o[nt][i][e]);   // (codes less 8)
      one[nt][0] = one[nt][1] = one[nt][2] = one[nt][3] = 0.f;
    }
  };
  for (int i = 0, stage = 0; i < n; ++i, stage = stage + 1 == kKv4Stages ? 0 : stage + 1) {
    __syncwarp();   // every lane is done with the stage that is filled now
    load(i + kKv4Stages - 1, stage == 0 ? kKv4Stages - 1 : stage - 1);
    cp_async_commit();
    cp_async_wait<kKv4Stages - 1>();
    __syncwarp();   // every lane's copies of this stage have landed
    const int pos = (own + i * stride) * K;
    const uint32_t none = missing >> (2 * stage) & 3u;
    const bool whole = pos + K <= seen_by_all && !none;
    const bool large = kv4_large(reinterpret_cast<const uint32_t*>(ring + stage * STAGE + 2 * K * CODES)[K + lane]);   // a lane looks at one pair of the values
    if (whole) {
      work(ring + stage * STAGE, 0, pos, 0u, large, std::false_type());
      work(ring + stage * STAGE, 1, pos, 0u, large, std::false_type());
    } else {   // (behind the context's end, seen_by_all + Q - 1, or without a page a pair may be anything)
      const bool there = large && pos + lane < seen_by_all + p.Q - 1 && !(none >> (lane >> 4) & 1u);
#pragma unroll 1
      for (int x = 0; x < 2; ++x) work(ring + stage * STAGE, x, pos, none, there, std::true_type());
    }
    if ((i & 7) == 7) take_off();
  }
  take_off();
  cp_async_wait<0>();
  __syncthreads();   // the rings are read: their memory is the parts' now

  // ---- the warps' parts meet: [warp][row][HD + 8] O | reference, sum ----
  constexpr int LDO = HD + 8, ROWS = 8 * NT;
  float* parts = reinterpret_cast<float*>(kv4_smem);
  float* joined = parts + W * ROWS * LDO;   // [row][HD + 8]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int w = 4; w < 32; w *= 2) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], w);
        low[nt][e] += __shfl_xor_sync(0xffffffffu, low[nt][e], w);
      }
      float* row = parts + (warp * ROWS + nt * 8 + 2 * t + e) * LDO;
#pragma unroll
      for (int j = 0; j < VW; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<float4*>(row + 64 * j + 32 * h + 4 * g) =
              make_float4(o[nt][4 * j][2 * h + e] + low[nt][e], o[nt][4 * j + 1][2 * h + e] + low[nt][e], o[nt][4 * j + 2][2 * h + e] + low[nt][e], o[nt][4 * j + 3][2 * h + e] + low[nt][e]);
      if (g == 0) *reinterpret_cast<float2*>(row + HD) = make_float2(ref[nt][e], l[nt][e]);
    }
  __syncthreads();
  // four columns of a row; SHARED: of a head's part, unless the whole of it is here
  const bool whole_head = !SHARED || (turn == 0 && last_turn == turns);
  auto store = [&](int r, int d, float4 acc, float top, float sum) {
    if (!whole_head) {
      float* part = p.parts + ((size_t)(2 * blockIdx.x + (turn == 0)) * R + r) * (HD + 4);
      *reinterpret_cast<float4*>(part + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(part + HD) = make_float2(top, sum);
      return;
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // (a row that sees no key is zero, NaN stays)
    __nv_bfloat16* dst = p.out + ((size_t)(b * p.Q + r / G) * p.heads + kvh * G + r % G) * HD + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  };
  for (int idx = threadIdx.x; idx < R * (HD / 4); idx += W * 32) {
    const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, parts[(w * ROWS + r) * LDO + HD]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* row = parts + (w * ROWS + r) * LDO;
      const float2 ml = *reinterpret_cast<const float2*>(row + HD);
      const float4 v = *reinterpret_cast<const float4*>(row + d);
      const float f = top == -INFINITY ? 1.f : exp2f(ml.x - top);   // (no score, or NaN only: zeros and NaN add up)
      acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
      sum += ml.y * f;
    }
    if (C == 1) {
      store(r, d, acc, top, sum);
    } else {
      *reinterpret_cast<float4*>(joined + r * LDO + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(joined + r * LDO + HD) = make_float2(top, sum);
    }
  }
  if constexpr (SHARED) {
    at += last_turn - turn;
    __syncthreads();   // (the parts are read: their memory is the rings' again)
    continue;
  } else {
  if (C == 1) return;
  // the blocks' parts meet over the cluster's shared memory, each block joins a share of the columns
  cluster.sync();
  for (int idx = rank * W * 32 + threadIdx.x; idx < R * (HD / 4); idx += C * W * 32) {
    const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int c = 0; c < C; ++c) top = fmaxf(top, cluster.map_shared_rank(joined, c)[r * LDO + HD]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < C; ++c) {
      const float* row = cluster.map_shared_rank(joined, c) + r * LDO;
      const float2 ml = *reinterpret_cast<const float2*>(row + HD);
      const float4 v = *reinterpret_cast<const float4*>(row + d);
      const float f = top == -INFINITY ? 1.f : exp2f(ml.x - top);
      acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
      sum += ml.y * f;
    }
    store(r, d, acc, top, sum);
  }
  cluster.sync();   // no block leaves while its part is read
  return;
  }
  }
}

// ----------------------------------------------------------------------------------
// kv4_join_kernel: the parts that the blocks of a shared launch left of a head's keys, put together; heads that one block had whole are in their place already.  KEYS: of a turn; blocks: of the
// launch in front.  A warp puts a row together, a lane asks for a part's reference and sum, and then for the columns that are its own.  SPREAD: few heads in many parts, a block's warps take
// them in turns and meet in shared memory (one context of 32000 in 64 parts a head: 7.5 us with four warps and loads in fours).
// ----------------------------------------------------------------------------------
constexpr int kKv4JoinThreads = 256;
template <int HD, int KEYS, bool SPREAD>
__global__ void __launch_bounds__(kKv4JoinThreads, 2) kv4_join_kernel(const __grid_constant__ Kv4AttnParams p, const int blocks) {
  constexpr int W = kKv4JoinThreads / 32, V = HD / 32;   // channels of a lane
  __shared__ float sums[SPREAD ? W : 1][HD];
  __shared__ float2 totals[W];
  const int G = p.heads / p.kv_heads, R = G * p.Q, kvh = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int2 heads = kv4_turns_of_all<KEYS>(p, b);
  const Kv4Stretch stretch(heads.x * p.kv_heads, blocks);
  const int turns = kv4_turns<KEYS>(p, b), first = heads.y * p.kv_heads + kvh * turns, from = stretch.block(first), to = stretch.block(first + turns - 1);
  pdl_wait();   // (the lengths are there before: the kernel in front, which lets this one begin behind its own wait, has read them)
  pdl_launch_dependents();
  if (from == to) return;   // (the whole block; behind the wait, as whoever waits for this grid waits for the one in front too)
  for (int r = SPREAD ? (int)blockIdx.z : (int)blockIdx.z * W + warp; r < R; r += SPREAD ? (int)gridDim.z : (int)gridDim.z * W) {
    const int step = SPREAD ? W : 1;
    float top = -INFINITY, sum = 0.f, acc[V] = {};
    for (int base = from + (SPREAD ? warp : 0); base <= to; base += 32 * step) {   // 32 parts
      const int n = min(32, (to - base) / step + 1), mine = base + lane * step;
      auto part = [&](int x) { return p.parts + ((size_t)(2 * x + (x == from)) * R + r) * (HD + 4); };
      const float2 ml = lane < n ? *reinterpret_cast<const float2*>(part(mine) + HD) : make_float2(-INFINITY, 0.f);
      const float now = fmaxf(top, warp_max(ml.x)), f = now == -INFINITY ? 1.f : exp2f(top - now);   // (no score, or NaN only: zeros and NaN add up)
      const float w = now == -INFINITY ? 1.f : exp2f(ml.x - now);
      top = now;
      sum = sum * f + warp_sum(ml.y * w);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] *= f;
#pragma unroll 8
      for (int x = 0; x < n; ++x) {
        const float* at = part(base + x * step);
        const float g = __shfl_sync(0xffffffffu, w, x);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(at[lane + 32 * i], g, acc[i]);
      }
    }
    if constexpr (SPREAD) {
      __syncthreads();   // (of the row in front, all is read)
#pragma unroll
      for (int i = 0; i < V; ++i) sums[warp][lane + 32 * i] = acc[i];
      if (lane == 0) totals[warp] = make_float2(top, sum);
      __syncthreads();
      if (warp > 0) continue;
      const float2 ml = lane < W ? totals[lane] : make_float2(-INFINITY, 0.f);
      top = warp_max(ml.x);
      const float w = top == -INFINITY ? 1.f : exp2f(ml.x - top);
      sum = warp_sum(ml.y * w);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const float g = __shfl_sync(0xffffffffu, w, x);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(sums[x][lane + 32 * i], g, acc[i]);
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // (a row that sees no key is zero, NaN stays)
    __nv_bfloat16* dst = p.out + ((size_t)(b * p.Q + r / G) * p.heads + kvh * G + r % G) * HD;
#pragma unroll
    for (int i = 0; i < V; ++i) dst[lane + 32 * i] = f2bf(acc[i] * inv);
  }
}

}  // namespace ssdk
