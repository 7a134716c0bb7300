// span_ops.cuh — attention over a part of a long paged cache: spans of keys are chosen by a bound on their scores, and attention reads the chosen ones only.
#pragma once
#include "async_copy.cuh"
#include "cache_ops.cuh"
#include "common.cuh"

namespace ssdk {

// ----------------------------------------------------------------------------------
// select_spans: the score of span s for key head g is the largest over the query rows r of (sequence, g) of
//   sum_d max(q[r, d] lo[s, d], q[r, d] hi[s, d])  >=  max over the span's keys of q[r] . k,
// in 64 bits: products of bf16 values are exact, and sums of a head's size are off by less than two scores of different spans are apart.
// ----------------------------------------------------------------------------------
struct SelectParams {
  const __nv_bfloat16* q;        // [B * Q, H, hd]
  const __nv_bfloat16* bounds;   // [num_blocks, block_size / span, KV, 2, hd]
  const int32_t* tables;         // [B, max_blocks]
  const int32_t* lens;           // [B]
  int32_t* out;                  // [B, KV, count]
  int64_t num_blocks;
  int B, Q, heads, kv_heads, block_size, span, max_blocks, count, first, last;
};
constexpr int kPickThreads = 1024;
constexpr int kMaxSpans = 24576;   // of a sequence

// 64-bit values in their order as unsigned words; zeros of both signs are one value, NaN is above all.  0 is no value
SSDK_DEVINL unsigned long long score_key(double s) {
  if (s != s) return ~0ull;
  const long long b = __double_as_longlong(s + 0.0);
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | (1ull << 63);
}

// A block per key head of a sequence: its warps score the spans into shared memory, then the smallest key that is taken is found bit by bit: the
// first and last spans, then by key, the lowest index first among equal ones.
template <int HD>
__global__ void __launch_bounds__(kPickThreads) span_select_kernel(SelectParams p) {
  constexpr int E = HD / 32;   // channels of a lane
  SSDK_DYN_SMEM(unsigned long long, keys);   // [n]
  SSDK_STATIC_SMEM(int, sums, 64);
  const int g = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, subs = p.block_size / p.span;
  const int G = p.heads / p.kv_heads, rows = G * p.Q;
  const int len = tokens_of(p.lens, b, p.max_blocks, p.block_size), n = (len + p.span - 1) / p.span;
  for (int s = warp; s < n; s += kPickThreads / 32) {
    unsigned long long key = 0;
    const int page = page_at(p.tables + (size_t)b * p.max_blocks + s / subs, p.num_blocks);
    if (page >= 0) {
      const __nv_bfloat16* both = p.bounds + (((size_t)page * subs + s % subs) * p.kv_heads + g) * 2 * HD;
      float lo[E], hi[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        lo[e] = bf2f(both[lane * E + e]);
        hi[e] = bf2f(both[HD + lane * E + e]);
      }
      for (int r = 0; r < rows; ++r) {
        const __nv_bfloat16* q = p.q + ((size_t)(b * p.Q + r / G) * p.heads + g * G + r % G) * HD + lane * E;
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const double x = bf2f(q[e]), u = x * lo[e], v = x * hi[e];
          sum += u != u || v != v ? __longlong_as_double(0x7ff8000000000000ll) : (u > v ? u : v);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        key = max(key, score_key(sum));
      }
    }
    if (lane == 0) keys[s] = key;
  }
  __syncthreads();
  auto kept = [&](int s) { return s < p.first || s >= n - p.last; };
  auto total = [&](int v) {   // over the block
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) sums[warp] = v;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, sums[lane]);
  };
  int always = 0, others = 0;
  for (int s = threadIdx.x; s < n; s += kPickThreads)
    if (keys[s]) (kept(s) ? always : others) += 1;
  always = total(always);
  others = total(others);
  const int want = min(p.count - always, others);
  unsigned long long line = 0;   // the want-th largest key
  int above = 0;
  if (want > 0) {
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long tried = line | (1ull << bit);
      int c = 0;
      for (int s = threadIdx.x; s < n; s += kPickThreads) c += !kept(s) && keys[s] >= tried;
      if (total(c) >= want) line = tried;
    }
    for (int s = threadIdx.x; s < n; s += kPickThreads) above += !kept(s) && keys[s] > line;
    above = total(above);
  }
  const int equal = want - above;   // so many of the keys on the line, the first ones
  int32_t* out = p.out + ((size_t)b * p.kv_heads + g) * p.count;
  int taken = 0, ties = 0;
  for (int base = 0; base < n; base += kPickThreads) {
    const int s = base + threadIdx.x;
    const unsigned long long key = s < n ? keys[s] : 0;
    const bool sure = key && (kept(s) || (want > 0 && key > line)), tie = key && !kept(s) && want > 0 && key == line;
    const unsigned m_sure = __ballot_sync(0xffffffffu, sure), m_tie = __ballot_sync(0xffffffffu, tie), under = (1u << lane) - 1;
    __syncthreads();
    if (lane == 0) {
      sums[warp] = __popc(m_sure);
      sums[32 + warp] = __popc(m_tie);
    }
    __syncthreads();
    int sure_before = taken + __popc(m_sure & under), tie_before = ties + __popc(m_tie & under);
    for (int w = 0; w < 32; ++w) {
      if (w < warp) {
        sure_before += sums[w];
        tie_before += sums[32 + w];
      }
      taken += sums[w];
      ties += sums[32 + w];
    }
    if (sure || (tie && tie_before < equal)) out[sure_before + min(tie_before, equal)] = s;
  }
  for (int i = taken + min(ties, equal) + threadIdx.x; i < p.count; i += kPickThreads) out[i] = -1;
}

// ----------------------------------------------------------------------------------
// span_attn_kernel: softmax(scale q k^T) v over the keys of the listed spans, causal to the end of the context as in paged attention (query j of a sequence
// sees positions <= len - Q + j); grouped heads.  A list may name spans in any order; what lies outside the context or on a page outside the cache
// is passed over, a row that sees no key is zero.
// Bound by the bytes of the listed keys and values.  A block owns one key head of one sequence and up to 16 MT of its query rows; its warps take pieces of 16
// keys in turn, each with a ring of its own (cp.async, no barrier between warps) and a softmax of its own, and meet at the end.
// Weights go into the second product as two bf16 pieces, sums are fp32.
// ----------------------------------------------------------------------------------
struct SpanAttnParams {
  const __nv_bfloat16* q;        // [B * Q, H, hd]
  const __nv_bfloat16 *k_cache, *v_cache;   // [num_blocks, block_size, KV, hd]
  const int32_t* tables;         // [B, max_blocks]
  const int32_t* lens;           // [B]
  const int32_t* spans;          // [B, KV, count]
  __nv_bfloat16* out;            // [B * Q, H, hd]
  int64_t num_blocks;
  int B, Q, heads, kv_heads, block_size, span, max_blocks, count;
  int tokens;                    // query tokens of a block
  float scale_log2;              // scale * log2(e)
};
constexpr int kSpanWarps = 4, kSpanStages = 3, kSpanKeys = 16;
constexpr int span_stage_bytes(int HD) { return 2 * kSpanKeys * (HD + 8) * 2; }
constexpr int span_attn_smem(int HD, int count) { return kSpanWarps * kSpanStages * span_stage_bytes(HD) + count * 8; }

template <int HD, int MT>
__global__ void __launch_bounds__(kSpanWarps * 32, 2) span_attn_kernel(SpanAttnParams p) {
  constexpr int LDS = HD + 8, KS = HD / 16, ND = HD / 8, SEG = HD / 8;
  extern __shared__ __align__(16) uint8_t span_smem[];
  const int kvh = blockIdx.x, b = blockIdx.y, tile = gridDim.z - 1 - blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.heads / p.kv_heads, tq = min(p.tokens, p.Q - tile * p.tokens), R = G * tq;
  const int len = tokens_of(p.lens, b, p.max_blocks, p.block_size);
  int2* where = reinterpret_cast<int2*>(span_smem + kSpanWarps * kSpanStages * span_stage_bytes(HD));   // [count] slot (-1: none) and position of a span's first key
  uint8_t* ring = span_smem + warp * kSpanStages * span_stage_bytes(HD);

  int n_list = 0;
  {
    const int32_t* list = p.spans + ((size_t)b * p.kv_heads + kvh) * p.count;
    for (int i = threadIdx.x; i < p.count; i += kSpanWarps * 32) {
      const int s = list[i];
      int2 at = make_int2(-1, 0);
      if (s >= 0 && (long long)s * p.span < len) {
        at.y = s * p.span;
        const int page = page_at(p.tables + (size_t)b * p.max_blocks + at.y / p.block_size, p.num_blocks);
        if (page >= 0) at.x = page * p.block_size + at.y % p.block_size;
      }
      where[i] = at;
      if (at.x >= 0) n_list = i + 1;
    }
  }
  {
    __shared__ int last[kSpanWarps];
    n_list = __reduce_max_sync(0xffffffffu, n_list);   // behind the last entry of any use
    if (lane == 0) last[warp] = n_list;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSpanWarps; ++w) n_list = max(n_list, last[w]);
  }

  uint32_t qa[MT][KS][4];
  int lim[MT][2];   // first position that a row does not see
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r0 = mt * 16 + g, r1 = r0 + 8;
    const __nv_bfloat16* q0 = p.q + ((size_t)(b * p.Q + tile * p.tokens + r0 / G) * p.heads + kvh * G + r0 % G) * HD;
    const __nv_bfloat16* q1 = p.q + ((size_t)(b * p.Q + tile * p.tokens + r1 / G) * p.heads + kvh * G + r1 % G) * HD;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const int c = kk * 16 + 2 * t;
      qa[mt][kk][0] = r0 < R ? *reinterpret_cast<const uint32_t*>(q0 + c) : 0u;
      qa[mt][kk][1] = r1 < R ? *reinterpret_cast<const uint32_t*>(q1 + c) : 0u;
      qa[mt][kk][2] = r0 < R ? *reinterpret_cast<const uint32_t*>(q0 + c + 8) : 0u;
      qa[mt][kk][3] = r1 < R ? *reinterpret_cast<const uint32_t*>(q1 + c + 8) : 0u;
    }
    lim[mt][0] = r0 < R ? len - p.Q + tile * p.tokens + r0 / G + 1 : 0;
    lim[mt][1] = r1 < R ? len - p.Q + tile * p.tokens + r1 / G + 1 : 0;
  }

  float o[MT][ND][4], mrow[MT][2], lrow[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int i = 0; i < ND; ++i) o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.f;
    mrow[mt][0] = mrow[mt][1] = -INFINITY;
    lrow[mt][0] = lrow[mt][1] = 0.f;
  }

  const int per = p.span / kSpanKeys, pieces = n_list * per;
  auto load = [&](int piece, int stage) {
    const int i = piece / per, off = (piece - i * per) * kSpanKeys;
    const int2 at = where[i];
    __nv_bfloat16* dk = reinterpret_cast<__nv_bfloat16*>(ring + stage * span_stage_bytes(HD));
    __nv_bfloat16* dv = dk + kSpanKeys * LDS;
    const size_t base = ((size_t)max(at.x, 0) + off) * p.kv_heads + kvh;
#pragma unroll
    for (int u = 0; u < kSpanKeys * SEG / 32; ++u) {
      const int idx = u * 32 + lane, tok = idx / SEG, seg = idx % SEG;
      const bool valid = at.x >= 0 && at.y + off + tok < len;   // what is not in the context is zero: a stale NaN would pass a weight of 0
      const size_t from = valid ? (base + (size_t)tok * p.kv_heads) * HD + seg * 8 : 0;
      cp_async16(dk + tok * LDS + seg * 8, p.k_cache + from, valid);
      cp_async16(dv + tok * LDS + seg * 8, p.v_cache + from, valid);
    }
  };
  const int step = kSpanWarps;
#pragma unroll
  for (int s = 0; s < kSpanStages - 1; ++s) {
    if (warp + s * step < pieces) load(warp + s * step, s);
    cp_async_commit();
  }
  int stage = 0;
  for (int piece = warp; piece < pieces; piece += step, stage = stage + 1 == kSpanStages ? 0 : stage + 1) {
    __syncwarp();   // every lane is done with the stage that is filled now
    if (piece + (kSpanStages - 1) * step < pieces) load(piece + (kSpanStages - 1) * step, stage == 0 ? kSpanStages - 1 : stage - 1);
    cp_async_commit();
    cp_async_wait<kSpanStages - 1>();
    __syncwarp();   // every lane's copies of this stage have landed
    const int2 at = where[piece / per];
    if (at.x < 0) continue;
    const int pos0 = at.y + (piece % per) * kSpanKeys;
    const __nv_bfloat16* cK = reinterpret_cast<const __nv_bfloat16*>(ring + stage * span_stage_bytes(HD));
    const __nv_bfloat16* cV = cK + kSpanKeys * LDS;
    const int mi = lane >> 3, rr = lane & 7;

    float s[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {   // a 16 x 16 piece of the keys: tokens 0 .. 7 and 8 .. 15, channels 0 .. 7 and 8 .. 15
      uint32_t kb[4];
      ldmatrix_x4(kb, cK + ((mi >> 1) * 8 + rr) * LDS + kk * 16 + (mi & 1) * 8);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mma_bf16_16816(s[mt][0], qa[mt][kk], kb[0], kb[1]);
        mma_bf16_16816(s[mt][1], qa[mt][kk], kb[2], kb[3]);
      }
    }
    uint32_t ph[MT][4], pl[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float top[2] = {mrow[mt][0], mrow[mt][1]};
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1, pos = pos0 + nt * 8 + 2 * t + (e & 1);
          s[mt][nt][e] = pos < lim[mt][h] ? s[mt][nt][e] * p.scale_log2 : -INFINITY;
          top[h] = fmaxf(top[h], s[mt][nt][e]);
        }
      float corr[2], ref[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        ref[h] = top[h] == -INFINITY ? 0.f : top[h];
        corr[h] = exp2f(mrow[mt][h] - ref[h]);
        mrow[mt][h] = top[h];
      }
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[mt][nt][e] = exp2f(s[mt][nt][e] - ref[e >> 1]);
          sum[e >> 1] += s[mt][nt][e];
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) lrow[mt][h] = lrow[mt][h] * corr[h] + sum[h];
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          o[mt][i][0] *= corr[0];
          o[mt][i][1] *= corr[0];
          o[mt][i][2] *= corr[1];
          o[mt][i][3] *= corr[1];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // rows g, g + 8 of keys 0 .. 7, then of keys 8 .. 15
        const float x = s[mt][i >> 1][2 * (i & 1)], y = s[mt][i >> 1][2 * (i & 1) + 1];
        ph[mt][i] = pack_bf16x2(x, y);
        pl[mt][i] = pack_bf16x2(x - bf16_round(x), y - bf16_round(y));
      }
    }
#pragma unroll
    for (int nd = 0; nd < ND; nd += 2) {
      uint32_t vb[4];
      ldmatrix_x4_trans(vb, cV + ((mi & 1) * 8 + rr) * LDS + nd * 8 + (mi >> 1) * 8);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mma_bf16_16816(o[mt][nd], ph[mt], vb[0], vb[1]);
        mma_bf16_16816(o[mt][nd + 1], ph[mt], vb[2], vb[3]);
        mma_bf16_16816(o[mt][nd], pl[mt], vb[0], vb[1]);
        mma_bf16_16816(o[mt][nd + 1], pl[mt], vb[2], vb[3]);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // the warps' parts meet: [warp][row][HD + 8] O | maximum, sum (row stride of 8 banks: fragment stores and row reads are free of conflicts)
  constexpr int LDO = HD + 8;
  float* parts = reinterpret_cast<float*>(span_smem);
  {
    float* w = parts + warp * (16 * MT) * LDO;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        lrow[mt][h] += __shfl_xor_sync(0xffffffffu, lrow[mt][h], 1);
        lrow[mt][h] += __shfl_xor_sync(0xffffffffu, lrow[mt][h], 2);
        float* row = w + (mt * 16 + g + 8 * h) * LDO;
#pragma unroll
        for (int i = 0; i < ND; ++i) *reinterpret_cast<float2*>(row + i * 8 + 2 * t) = make_float2(o[mt][i][2 * h], o[mt][i][2 * h + 1]);
        if (t == 0) *reinterpret_cast<float2*>(row + HD) = make_float2(mrow[mt][h], lrow[mt][h]);
      }
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < R * (HD / 4); idx += kSpanWarps * 32) {
    const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSpanWarps; ++w) top = fmaxf(top, parts[(w * 16 * MT + r) * LDO + HD]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    if (top != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kSpanWarps; ++w) {
        const float* row = parts + (w * 16 * MT + r) * LDO;
        const float2 ml = *reinterpret_cast<const float2*>(row + HD);
        const float4 v = *reinterpret_cast<const float4*>(row + d);
        const float f = exp2f(ml.x - top);
        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
        l += ml.y * f;
      }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    __nv_bfloat16* dst = p.out + ((size_t)(b * p.Q + tile * p.tokens + r / G) * p.heads + kvh * G + r % G) * HD + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  }
}

}  // namespace ssdk
