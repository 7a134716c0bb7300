// kv4_attention.cuh — attention over a paged cache held in 4 bits (kv4.cuh), on mma.sync: a step's tokens of a sequence, up to sixteen query rows of a key head at a time.
#pragma once
#include <cooperative_groups.h>

#include "kv4.cuh"

namespace ssdk {

// ----------------------------------------------------------------------------------
// kv4_attn_kernel: softmax(scale q k^T) v, causal to the end of the context as in paged attention (query j of a sequence sees positions <= len - Q + j), grouped heads.
// With k = s c + m and v = s' c' + m' of a token (c codes)
//   q k = s (q c) + m sum(q)          O = sum_j (P_j s'_j) (c'_j - 8) + sum_j P_j (m'_j + 8 s'_j)
// so that what meets in the products are codes, exact in bf16: keys and values are not rounded at all.  What is rounded is P s' (bf16, 2^-9 of a term at most, the codes
// around their middle so that it is of the value's size); sums, references and the second term are fp32.
// Bound by the bytes of the cache, then by the instructions that make codes into fragments.  The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that
// keys (sixteen) and channels (sixteen) are the m of mma and the eight query rows of a usual group its n.  Nothing goes through shared memory: a quad's lanes read a key's row, 16
// bytes each, as the A fragment of any eight products (which channels a product's k stands for is free, the query's fragments follow), eight lanes a value's row, and a
// word of eight channels is four pairs of bf16 by a shift and a mask each: 16 + c has c in the top of its mantissa.  Of two values' words one byte_perm makes words whose halves
// are the two keys of a fragment's register.
// A cluster of blocks shares the keys of a key head of one sequence: pieces of 16 keys go round the blocks' warps, each with a softmax of its own; at the end warps meet, then blocks.
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
};
constexpr float kKv4Slack = 8.f;
constexpr int kKv4Warps = 8, kKv4Most = 16;   // warps of a block, blocks of a cluster
constexpr int kv4_attn_smem(int HD, int NT) { return (kKv4Warps + 1) * 8 * NT * (HD + 8) * 4; }

SSDK_DEVINL uint32_t ld_nc_u32(const void* p) {
  uint32_t r;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}
SSDK_DEVINL uint2 ld_nc_v2(const void* p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
// nibbles P and P + 4 of a word as 16 + c in bf16
template <int P>
SSDK_DEVINL uint32_t kv4_pair(uint32_t w) {
  const uint32_t x = P == 0 ? w << 3 : w >> (4 * P - 3);
  return (x & 0x00780078u) | 0x41804180u;
}
SSDK_DEVINL uint32_t minus24(uint32_t x) {   // of both halves: codes around their middle (exact)
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x41c041c0u));
  return d;
}
SSDK_DEVINL uint32_t transpose_8x8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

// what a lane holds of sixteen keys: words of the keys' rows g, g + 8 (of S^T) and of the values' rows, their pairs
template <int HD>
struct Kv4Piece {
  uint32_t k[2][HD / 32], v[4][HD / 64], pk[2], pv[2];
  int pos;   // of the first key, -1: no page
};

template <int HD, int NT>
__global__ void __launch_bounds__(kKv4Warps * 32, NT == 1 ? 2 : 1) kv4_attn_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int KS = HD / 16, KW = HD / 32, VW = HD / 64, CODES = HD / 2;
  extern __shared__ __align__(16) uint8_t kv4_smem[];
  pdl_wait();
  pdl_launch_dependents();
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int kvh = blockIdx.x / C, b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.heads / p.kv_heads, r0 = blockIdx.z * 8 * NT, R = min(G * p.Q - r0, 8 * NT);   // rows of this block: r0 ..
  const int len = tokens_of(p.lens, b, p.max_blocks, p.block_size), ctx = len - p.Q;
  const int seen = min(len, ctx + (r0 + R - 1) / G + 1), seen_by_all = ctx + r0 / G + 1;   // positions that some row sees, that all do

  // ---- queries: fragments in the order of the keys' words, sums ----
  uint32_t qb[NT][KS][2];
  float qs[NT][2];
  int lim[NT][2];   // first position that rows 2 t, 2 t + 1 do not see
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + n * 8 + g;
    const __nv_bfloat16* q = p.q + ((size_t)(b * p.Q + r / G) * p.heads + kvh * G + r % G) * HD + t * (HD / 4);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const uint4 x = n * 8 + g < R ? *reinterpret_cast<const uint4*>(q + j * 8) : make_uint4(0, 0, 0, 0);
      qb[n][2 * j][0] = __byte_perm(x.x, x.z, 0x5410);   // channels 0 and 4 of the word, 1 and 5, 2 and 6, 3 and 7
      qb[n][2 * j][1] = __byte_perm(x.x, x.z, 0x7632);
      qb[n][2 * j + 1][0] = __byte_perm(x.y, x.w, 0x5410);
      qb[n][2 * j + 1][1] = __byte_perm(x.y, x.w, 0x7632);
      float f[8];
      unpack_bf16x8(x, f);
      sum += ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      qs[n][e] = __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4) * p.scale_log2;
      const int row = n * 8 + 2 * t + e;
      lim[n][e] = row < R ? ctx + (r0 + row) / G + 1 : 0;
    }
  }

  float o[NT][HD / 16][4], ref[NT][2], l[NT][2], low[NT][2];   // O^T, reference, sum, sum of P (m' + 8 s')
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      ref[n][e] = -INFINITY;
      l[n][e] = low[n][e] = 0.f;
    }
  }

  // ---- pieces of 16 keys: own, own + stride, ...; pages of 32 of them at a time, one a lane ----
  const int pieces = (max(seen, 0) + 15) >> 4, stride = C * kKv4Warps, own = rank * kKv4Warps + warp;
  const size_t record = (size_t)p.block_size * kv4_row_bytes(HD);
  // The keys of a piece as S^T's rows: row 2 t + (i & 1) + 8 (i >> 1) is key 4 i + t, so that a value's load i takes four neighbouring rows and a key's load eight.
  const int key = 4 * (g & 1) + (g >> 1);
  const int k_at = key * CODES + t * (CODES / 4), v_at = t * CODES + g * (CODES / 8), pair_at = p.block_size * CODES + key * 4;
  int page = -1, off = 0;   // of piece own + (base + lane) * stride
  auto look_up = [&](int first) {
    const long long piece = own + (long long)(first + lane) * stride;
    page = -1;
    if (piece < pieces) {
      const int pos = (int)piece * 16, x = pos / p.block_size;
      off = pos - x * p.block_size;
      page = page_at(p.tables + (size_t)b * p.max_blocks + x, p.num_blocks);
    }
  };
  auto load = [&](Kv4Piece<HD>& x, int i) {   // this warp's piece i
    if ((i & 31) == 0) look_up(i);
    const int at_page = __shfl_sync(0xffffffffu, page, i & 31), at = __shfl_sync(0xffffffffu, off, i & 31);
    x.pos = -1;
    if (at_page < 0) return;
    x.pos = (own + i * stride) * 16;
    const size_t base = ((size_t)at_page * p.kv_heads + kvh) * record;
    const uint8_t *kc = p.k_cache + base, *vc = p.v_cache + base;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* row = kc + at * CODES + k_at + h * 8 * CODES;
      if constexpr (HD == 128) {
        const uint4 w = ld_nc_v4(row);
        x.k[h][0] = w.x; x.k[h][1] = w.y; x.k[h][2] = w.z; x.k[h][3] = w.w;
      } else {
        const uint2 w = ld_nc_v2(row);
        x.k[h][0] = w.x; x.k[h][1] = w.y;
      }
      x.pk[h] = ld_nc_u32(kc + pair_at + at * 4 + h * 32);
      x.pv[h] = ld_nc_u32(vc + pair_at + at * 4 + h * 32);
    }
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const uint8_t* row = vc + at * CODES + v_at + i4 * 4 * CODES;
      if constexpr (HD == 128) {
        const uint2 w = ld_nc_v2(row);
        x.v[i4][0] = w.x; x.v[i4][1] = w.y;
      } else {
        x.v[i4][0] = ld_nc_u32(row);
      }
    }
  };

  auto work = [&](const Kv4Piece<HD>& x) {
    if (x.pos < 0) return;
    float s[NT][4] = {};
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const uint32_t a0[4] = {kv4_pair<0>(x.k[0][j]), kv4_pair<0>(x.k[1][j]), kv4_pair<1>(x.k[0][j]), kv4_pair<1>(x.k[1][j])};
      const uint32_t a1[4] = {kv4_pair<2>(x.k[0][j]), kv4_pair<2>(x.k[1][j]), kv4_pair<3>(x.k[0][j]), kv4_pair<3>(x.k[1][j])};
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_bf16_16816(s[n], a0, qb[n][2 * j][0], qb[n][2 * j][1]);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_bf16_16816(s[n], a1, qb[n][2 * j + 1][0], qb[n][2 * j + 1][1]);
    }
    float sv[2], mv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float sk = __uint_as_float(x.pk[h] << 16), mk = fmaf(-16.f, sk, __uint_as_float(x.pk[h] & 0xffff0000u)), f = sk * p.scale_log2;
      sv[h] = __uint_as_float(x.pv[h] << 16);
      mv[h] = fmaf(8.f, sv[h], __uint_as_float(x.pv[h] & 0xffff0000u));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) s[n][2 * h + e] = fmaf(s[n][2 * h + e], f, mk * qs[n][e]);
    }
    const bool whole = x.pos + 16 <= seen_by_all;   // (the same for the warp)
    uint32_t out_of_sight = 0;   // bits of the scores
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (x.pos + key + 8 * (e >> 1) >= lim[n][e & 1]) {
            s[n][e] = -INFINITY;
            out_of_sight |= 1u << (n * 4 + e);
          }
    }
    // a row's reference is raised, and its sums rescaled, only when a score passes it by kKv4Slack (base 2)
    bool grow = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) grow = grow || fmaxf(s[n][e], s[n][2 + e]) > ref[n][e] + kKv4Slack;
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(s[n][e], s[n][2 + e]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)), ref[n][e]);
          const float f = top == ref[n][e] ? 1.f : ex2_ftz(ref[n][e] - top);   // (from -inf: 0)
          ref[n][e] = top;
          l[n][e] *= f;
          low[n][e] *= f;
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            o[n][i][e] *= f;
            o[n][i][2 + e] *= f;
          }
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float y = ex2_ftz(s[n][2 * h + e] - (ref[n][e] == -INFINITY ? 0.f : ref[n][e]));
          l[n][e] += y;
          const bool none = out_of_sight >> (n * 4 + 2 * h + e) & 1u;   // (its pair may be anything: 0 x NaN is NaN)
          low[n][e] = none ? low[n][e] : fmaf(y, mv[h], low[n][e]);
          w[e] = none ? 0.f : y * sv[h];
        }
        pb[n][h] = transpose_8x8(pack_bf16x2(w[0], w[1]));
      }
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      const uint32_t a01 = __byte_perm(x.v[0][j], x.v[1][j], 0x5410), b01 = __byte_perm(x.v[0][j], x.v[1][j], 0x7632);
      const uint32_t a23 = __byte_perm(x.v[2][j], x.v[3][j], 0x5410), b23 = __byte_perm(x.v[2][j], x.v[3][j], 0x7632);
      const uint32_t a[4][4] = {{minus24(kv4_pair<0>(a01)), minus24(kv4_pair<0>(b01)), minus24(kv4_pair<0>(a23)), minus24(kv4_pair<0>(b23))},
                                {minus24(kv4_pair<1>(a01)), minus24(kv4_pair<1>(b01)), minus24(kv4_pair<1>(a23)), minus24(kv4_pair<1>(b23))},
                                {minus24(kv4_pair<2>(a01)), minus24(kv4_pair<2>(b01)), minus24(kv4_pair<2>(a23)), minus24(kv4_pair<2>(b23))},
                                {minus24(kv4_pair<3>(a01)), minus24(kv4_pair<3>(b01)), minus24(kv4_pair<3>(a23)), minus24(kv4_pair<3>(b23))}};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_bf16_16816(o[n][4 * j + i], a[i], pb[n][0], pb[n][1]);
    }
  };

  const int n_own = own < pieces ? (pieces - own + stride - 1) / stride : 0;
  if (n_own > 0) {
    Kv4Piece<HD> x, y;
    load(x, 0);
    for (int i = 0; i < n_own; i += 2) {
      y.pos = -1;
      if (i + 1 < n_own) load(y, i + 1);
      work(x);
      x.pos = -1;
      if (i + 2 < n_own) load(x, i + 2);
      work(y);
    }
  }

  // ---- the warps' parts meet: [warp][row][HD + 8] O | reference, sum ----
  constexpr int LDO = HD + 8, ROWS = 8 * NT;
  float* parts = reinterpret_cast<float*>(kv4_smem);
  float* joined = parts + kKv4Warps * ROWS * LDO;   // [row][HD + 8]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int w = 4; w < 32; w *= 2) {
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], w);
        low[n][e] += __shfl_xor_sync(0xffffffffu, low[n][e], w);
      }
      float* row = parts + (warp * ROWS + n * 8 + 2 * t + e) * LDO;
#pragma unroll
      for (int j = 0; j < VW; ++j)   // channels g HD / 8 + 8 j ..
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<float4*>(row + g * (HD / 8) + 8 * j + 4 * h) =
              make_float4(o[n][4 * j][2 * h + e] + low[n][e], o[n][4 * j + 1][2 * h + e] + low[n][e], o[n][4 * j + 2][2 * h + e] + low[n][e], o[n][4 * j + 3][2 * h + e] + low[n][e]);
      if (g == 0) *reinterpret_cast<float2*>(row + HD) = make_float2(ref[n][e], l[n][e]);
    }
  __syncthreads();
  // four columns of a row
  auto store = [&](int r, int d, float4 acc, float sum) {
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // (a row that sees no key is zero, NaN stays)
    __nv_bfloat16* dst = p.out + ((size_t)(b * p.Q + (r0 + r) / G) * p.heads + kvh * G + (r0 + r) % G) * HD + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  };
  for (int idx = threadIdx.x; idx < R * (HD / 4); idx += kKv4Warps * 32) {
    const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) top = fmaxf(top, parts[(w * ROWS + r) * LDO + HD]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) {
      const float* row = parts + (w * ROWS + r) * LDO;
      const float2 ml = *reinterpret_cast<const float2*>(row + HD);
      const float4 v = *reinterpret_cast<const float4*>(row + d);
      const float f = top == -INFINITY ? 1.f : exp2f(ml.x - top);   // (no score, or NaN only: zeros and NaN add up)
      acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
      sum += ml.y * f;
    }
    if (C == 1) {
      store(r, d, acc, sum);
    } else {
      *reinterpret_cast<float4*>(joined + r * LDO + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(joined + r * LDO + HD) = make_float2(top, sum);
    }
  }
  if (C == 1) return;
  // the blocks' parts meet over the cluster's shared memory, each block joins a share of the columns
  cluster.sync();
  for (int idx = rank * kKv4Warps * 32 + threadIdx.x; idx < R * (HD / 4); idx += C * kKv4Warps * 32) {
    const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
    float2 ml[kKv4Most];
    float4 v[kKv4Most];
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int c = 0; c < kKv4Most; ++c)
      if (c < C) {
        const float* row = cluster.map_shared_rank(joined, c) + r * LDO;
        ml[c] = *reinterpret_cast<const float2*>(row + HD);
        v[c] = *reinterpret_cast<const float4*>(row + d);
        top = fmaxf(top, ml[c].x);
      }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kKv4Most; ++c)
      if (c < C) {
        const float f = top == -INFINITY ? 1.f : exp2f(ml[c].x - top);
        acc.x += v[c].x * f; acc.y += v[c].y * f; acc.z += v[c].z * f; acc.w += v[c].w * f;
        sum += ml[c].y * f;
      }
    store(r, d, acc, sum);
  }
  cluster.sync();   // no block leaves while its part is read
}

}  // namespace ssdk
