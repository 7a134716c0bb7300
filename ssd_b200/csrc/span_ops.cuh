// span_ops.cuh — attention over a part of a long paged cache: spans of keys are chosen by a bound on their scores, and attention reads the chosen ones only.
#pragma once
#ifndef SSDK_HOST_EMU
#include <cooperative_groups.h>

#include "async_copy.cuh"
#endif
#include "cache_ops.cuh"
#include "common.cuh"

namespace ssdk {

// ----------------------------------------------------------------------------------
// select_spans: the score of span s for key head g is the largest over the query rows r of (sequence, g) of
//   sum_d max(q[r, d] lo[s, d], q[r, d] hi[s, d])  >=  max over the span's keys of q[r] . k.
// Listed are the first and the last spans, then the best by score, the lowest index first among equal ones.  Scores count in 64 bits: 32 would let spans
// change places whose scores differ in the last bits.
// Bound by the bytes of the bounds.  The sum is a product, [lo | hi] . [min(q, 0) | max(q, 0)], so span_estimate_kernel makes an estimate of every score on the
// tensor cores: a warp takes sixteen spans, whose 16-byte loads are the m16 fragments of mma.m16n8k16 (channels permuted alike on both sides), eight rows
// are its n.  The estimate is off by at most eps = 2^-14 max_r sum_d |q[r, d]| max |lo, hi|: lower and upper bounds are a chain of hd / 16 steps each,
// a step adds 17 numbers with 2^-22 of its chain's terms' size lost, and 17 hd / 16 2^-22 is below 2^-14.9 for hd = 128.  With t the want-th largest estimate, a span above t + 2 eps is taken, one under t - 2 eps is not, and span_pick_kernel scores only the few
// in between in 64 bits (products of bf16 values are exact, sums of 128 of them off by 2^-46).  Where values are not finite, or so large that 32 bits
// overflow, it scores all.
// Two kernels, the second's start under the first's end: the estimates fill all SMs in even shares whatever the number of heads, and what picks is one block
// of a head (short tables, few rows and few heads: the block that picks makes its estimates itself, kOwnSpans).  24 contexts of 64000 tokens (150 MB of bounds): 37 us, of it 8 the
// second's.  The first has its loads in flight one turn at a time (registers hold one);
// a ring of cp.async stages, each lane its own pieces or a span's bounds by whole lines, was slower: 49 and 41 us.
// ----------------------------------------------------------------------------------
struct SelectParams {
  const __nv_bfloat16* q;        // [B * Q, H, hd]
  const __nv_bfloat16* bounds;   // [num_blocks, block_size / span, KV, 2, hd]
  const int32_t* tables;         // [B, max_blocks]
  const int32_t* lens;           // [B]
  int32_t* out;                  // [B, KV, count]
  uint32_t* estimates;           // [B, KV, max_spans] bits of fp32, kNoSpan where there is no page
  uint32_t* wide;                // [B, KV, warps] bits of the largest |lo|, |hi| that a warp saw
  int64_t num_blocks;
  unsigned long long sub_magic;  // ceil(2^32 / spans of a page)
  int B, Q, heads, kv_heads, block_size, span, max_blocks, max_spans, count, first, last;
  int warps;                     // to a key head of a sequence: warp w takes groups w, w + warps, ... of sixteen spans
};
constexpr int kEstimateThreads = 256;
constexpr int kPickThreads = 512, kPickWarps = kPickThreads / 32;
constexpr int kMaxSpans = 24576;   // of a sequence
constexpr int kPickBins = 1024;    // a multiple of kPickThreads
constexpr int kPickRanked = 256;   // spans between, up to which each is compared with each
// rows of the query | scores (64 bits; before them the estimates) | taken | between (a bit per span) | bins, then the spans between
constexpr int64_t pick_smem(int spans, int64_t rows, int HD) { return (rows + 7) / 8 * 8 * HD * 2 + spans * 8 + 2 * ((spans + 31) / 32) * 4 + kPickBins * 4; }
constexpr int64_t estimate_smem(int64_t rows, int HD) { return rows > 8 ? (rows + 7) / 8 * 16 * HD : 0; }
constexpr uint32_t kNoSpan = 0xffffffffu;   // estimate of a span that has no page

// 64-bit values in their order as unsigned words; zeros of both signs are one value, NaN is above all.  0 is no value
SSDK_DEVINL unsigned long long score_key(double s) {
  if (s != s) return ~0ull;
  const long long b = __double_as_longlong(s + 0.0);
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | (1ull << 63);
}

// the sum of v over the block's threads up to this one, and over all.  words: not those of the call before
SSDK_DEVINL int pick_running_sum(int v, int* words, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) words[warp] = v;
  __syncthreads();
  const int x = lane < kPickWarps ? words[lane] : 0;
  *total = __reduce_add_sync(0xffffffffu, x);
  return v + __reduce_add_sync(0xffffffffu, lane < warp ? x : 0);
}

// the spans of a bit map, ascending, then -1
SSDK_DEVINL void pick_write(const uint32_t* bits, int words, int32_t* out, int count, int* sums) {
  int done = 0, turn = 0;
  for (int base = 0; base < words; base += kPickThreads, turn ^= 1) {
    const int w = base + threadIdx.x;
    uint32_t m = w < words ? bits[w] : 0;
    int all, at = pick_running_sum(__popc(m), sums + turn * kPickWarps, &all);
    at += done - __popc(m);
    for (; m && at < count; m &= m - 1) out[at++] = w * 32 + __ffs(m) - 1;
    done += all;
  }
  for (int i = done + threadIdx.x; i < count; i += kPickThreads) out[i] = -1;
}
// floats in their order as unsigned words, and back
SSDK_DEVINL uint32_t order_of(uint32_t f) { return f >> 31 ? ~f : f | 0x80000000u; }
SSDK_DEVINL float of_order(uint32_t o) { return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o); }

// a warp: the score of one span in 64 bits.  q: the rows [tiles * 8][HD], those behind the last one zero.  A lane has HD / 32 channels of eight rows at a time;
// their sums halve their number with every exchange.  FINITE: lo <= hi and no product is NaN, so that the sign of q says which bound counts.
template <int HD, bool FINITE>
SSDK_DEVINL unsigned long long exact_score(const __nv_bfloat16* both, const __nv_bfloat16* q, int rows) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  double lo[E], hi[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    lo[e] = bf2f(both[lane * E + e]);
    hi[e] = bf2f(both[HD + lane * E + e]);
  }
  unsigned long long key = 0;
  for (int r0 = 0; r0 < rows; r0 += 8) {
    double sum[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      sum[r] = 0.0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float f = bf2f(q[(r0 + r) * HD + lane * E + e]);
        const double x = f;
        if (FINITE) {
          sum[r] += x * (f >= 0.f ? hi[e] : lo[e]);
        } else {
          const double u = x * lo[e], v = x * hi[e];
          sum[r] += u != u || v != v ? __longlong_as_double(0x7ff8000000000000ll) : (u > v ? u : v);
        }
      }
    }
    int row = 0;   // of the eight, the one that this lane ends with
#pragma unroll
    for (int o = 16, m = 4; o >= 4; o >>= 1, m >>= 1) {
      const bool up = (lane & o) != 0;
      row += up ? m : 0;
#pragma unroll
      for (int r = 0; r < m; ++r) {
        const double give = up ? sum[r] : sum[r + m], keep = up ? sum[r + m] : sum[r];
        sum[r] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    }
    sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 2);
    sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 1);
    if (r0 + row < rows) key = max(key, score_key(sum[0]));
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  return key;
}

SSDK_DEVINL int sub_page(const SelectParams& p, int s) { return (int)((unsigned)s * p.sub_magic >> 32); }   // s / spans of a page: below 2^15 and 2^16
SSDK_DEVINL const __nv_bfloat16* bounds_at(const SelectParams& p, int page, int s, int head, int HD) {
  const int subs = p.block_size / p.span;
  return p.bounds + (((size_t)page * subs + (s - sub_page(p, s) * subs)) * p.kv_heads + head) * 2 * HD;
}

// A warp: the estimates of the groups `group`, `group` + step, ... of sixteen spans of a key head, put(s, bits) by one lane; returns the largest |lo|, |hi| seen (bits
// of bf16).  MANY: more than eight rows, whose fragments the block's warps put into shared memory (all of them are here).
template <int HD, bool MANY, typename Put>
SSDK_DEVINL uint32_t estimate_groups(const SelectParams& p, int b, int head, int n, int group, int step, uint2* frags, Put put) {   // frags [tiles][2 CH][32]
  constexpr int CH = HD / 32;   // 16-byte pieces of a lane per bound
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, groups = (n + 15) / 16;
  const int G = p.heads / p.kv_heads, rows = G * p.Q, tiles = (rows + 7) / 8, subs = p.block_size / p.span;
  const int32_t* table = p.tables + (size_t)b * p.max_blocks;
  // where the bounds of span s start (in channels; negative: no such span, or on no page)
  auto place_of = [&](int s) {
    const int entry = sub_page(p, s), page = s < n ? page_at(table + entry, p.num_blocks) : -1;
    return page < 0 ? -1ll : (((long long)page * subs + (s - entry * subs)) * p.kv_heads + head) * (2 * HD);
  };
  // the query's side: row g of a tile, step k of 16 channels: the lane's channels 8 (t + 4 (k / 2)) + 4 (k % 2) .. + 3.  Lower bounds meet the negative parts,
  // upper bounds the positive ones
  auto load_q = [&](int tile, uint2* f) {
    const int r = tile * 8 + g;
    const __nv_bfloat16* q = p.q + ((size_t)(b * p.Q + r / G) * p.heads + head * G + r % G) * HD + 8 * t;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const uint4 x = r < rows ? *reinterpret_cast<const uint4*>(q + 32 * i) : make_uint4(0, 0, 0, 0);
      f[2 * i] = make_uint2(x.x, x.y);
      f[2 * i + 1] = make_uint2(x.z, x.w);
    }
  };
  auto negative = [](const uint2& f) { return make_uint2(min_bf16x2(f.x, 0u), min_bf16x2(f.y, 0u)); };
  auto positive = [](const uint2& f) { return make_uint2(max_bf16x2(f.x, 0u), max_bf16x2(f.y, 0u)); };
  long long at0 = place_of(group * 16 + g), at1 = place_of(group * 16 + 8 + g);
  uint2 qf[2 * CH];
  if (MANY) {   // every tile's fragments into shared memory, a tile per warp
    for (int tile = threadIdx.x >> 5; tile < tiles; tile += (int)(blockDim.x >> 5)) {
      load_q(tile, qf);
#pragma unroll
      for (int k = 0; k < 2 * CH; ++k) frags[(tile * 2 * CH + k) * 32 + lane] = qf[k];
    }
    __syncthreads();
  } else if (group < groups) {
    load_q(0, qf);
  }
  uint32_t bottom = 0, top = 0;   // two channels: smallest lower, largest upper bound
  for (; group < groups; group += step) {
    const int s0 = group * 16 + g, s1 = s0 + 8;
    const bool there0 = at0 >= 0, there1 = at1 >= 0;
    const __nv_bfloat16 *both0 = p.bounds + at0 + 8 * t, *both1 = p.bounds + at1 + 8 * t;
    uint4 u[2 * CH], v[2 * CH];
#pragma unroll
    for (int i = 0; i < 2 * CH; ++i) {
      u[i] = there0 ? ld_nc_v4(both0 + 32 * i) : make_uint4(0, 0, 0, 0);
      v[i] = there1 ? ld_nc_v4(both1 + 32 * i) : make_uint4(0, 0, 0, 0);
    }
    at0 = place_of(s0 + 16 * step);
    at1 = place_of(s1 + 16 * step);
    float best[2] = {-INFINITY, -INFINITY};   // spans g, g + 8
    for (int tile = 0; tile < (MANY ? tiles : 1); ++tile) {
      float c[2][4] = {};
#pragma unroll
      for (int k = 0; k < 2 * CH; ++k) {
        const uint2 f = MANY ? frags[(tile * 2 * CH + k) * 32 + lane] : qf[k], lo = negative(f), hi = positive(f);
        const uint4 &ul = u[k / 2], &vl = v[k / 2], &uh = u[CH + k / 2], &vh = v[CH + k / 2];
        const uint32_t al[4] = {k & 1 ? ul.z : ul.x, k & 1 ? vl.z : vl.x, k & 1 ? ul.w : ul.y, k & 1 ? vl.w : vl.y};
        const uint32_t ah[4] = {k & 1 ? uh.z : uh.x, k & 1 ? vh.z : vh.x, k & 1 ? uh.w : uh.y, k & 1 ? vh.w : vh.y};
        mma_bf16_16816(c[0], al, lo.x, lo.y);
        mma_bf16_16816(c[1], ah, hi.x, hi.y);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (tile * 8 + 2 * t + e < rows) {
          best[0] = fmaxf(best[0], c[0][e] + c[1][e]);
          best[1] = fmaxf(best[1], c[0][2 + e] + c[1][2 + e]);
        }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      bottom = min_bf16x2(bottom, min_bf16x2(min_bf16x2(u[i].x, u[i].y), min_bf16x2(u[i].z, u[i].w)));
      bottom = min_bf16x2(bottom, min_bf16x2(min_bf16x2(v[i].x, v[i].y), min_bf16x2(v[i].z, v[i].w)));
      top = max_bf16x2(top, max_bf16x2(max_bf16x2(u[i + CH].x, u[i + CH].y), max_bf16x2(u[i + CH].z, u[i + CH].w)));
      top = max_bf16x2(top, max_bf16x2(max_bf16x2(v[i + CH].x, v[i + CH].y), max_bf16x2(v[i + CH].z, v[i + CH].w)));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      best[0] = fmaxf(best[0], __shfl_xor_sync(0xffffffffu, best[0], o));
      best[1] = fmaxf(best[1], __shfl_xor_sync(0xffffffffu, best[1], o));
    }
    if (t < 2) {
      const int s = t ? s1 : s0;
      if (s < n) put(s, (t ? there1 : there0) ? __float_as_uint(t ? best[1] : best[0]) : kNoSpan);
    }
  }
  const uint32_t both = max_bf16x2(bottom & 0x7fff7fffu, top);   // (top is not negative; NaN is above infinity above all)
  return __reduce_max_sync(0xffffffffu, max(both & 0xffffu, both >> 16));
}

template <int HD, bool MANY>
__global__ void __launch_bounds__(kEstimateThreads, 2) span_estimate_kernel(SelectParams p) {
  SSDK_DYN_SMEM(uint2, frags);
  constexpr int W = kEstimateThreads / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z;
  // neighbouring warps take neighbouring heads, whose bounds of a span lie together (MANY: a block's warps share the fragments of their head)
  const int unit = blockIdx.x * W + (int)(threadIdx.x >> 5), head = MANY ? (int)blockIdx.y : unit % p.kv_heads, slot = MANY ? unit : unit / p.kv_heads;
  if (slot >= p.warps) return;   // (MANY: none)
  const int n = (tokens_of(p.lens, b, p.max_blocks, p.block_size) + p.span - 1) / p.span;
  if (n <= p.count) return;   // all are listed
  uint32_t* estimates = p.estimates + ((size_t)b * p.kv_heads + head) * p.max_spans;
  const uint32_t most = estimate_groups<HD, MANY>(p, b, head, n, slot, p.warps, frags, [&](int s, uint32_t e) { estimates[s] = e; });
  if ((threadIdx.x & 31) == 0) p.wide[((size_t)b * p.kv_heads + head) * p.warps + slot] = most << 16;
}

// OWN: the block makes the estimates itself, where a head's are few and heads fewer than SMs: one launch
template <int HD, bool OWN>
__global__ void __launch_bounds__(kPickThreads, OWN ? 1 : 2) span_pick_kernel(SelectParams p) {
  SSDK_DYN_SMEM(uint8_t, pick_smem_bytes);
  SSDK_STATIC_SMEM(int, sums, 4 * kPickWarps);
  SSDK_SHARED_VAR(int, pick_bin);
  SSDK_SHARED_VAR(int, n_sure);
  SSDK_SHARED_VAR(int, n_open);
  SSDK_STATIC_SMEM(int4, stats, kPickWarps);
  SSDK_STATIC_SMEM(uint32_t, wides, kPickWarps);   // bits of the largest |lo|, |hi| of a warp's share
  SSDK_SHARED_VAR(uint32_t, q_most);               // and of the largest sum of |q| over a row
  const int G = p.heads / p.kv_heads, rows = G * p.Q, padded = (rows + 7) / 8 * 8;
  const int words = (p.max_spans + 31) / 32;
  __nv_bfloat16* q_rows = reinterpret_cast<__nv_bfloat16*>(pick_smem_bytes);   // [padded][HD]
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(q_rows + padded * HD);
  uint32_t* estimate = reinterpret_cast<uint32_t*>(keys);
  uint32_t* taken = reinterpret_cast<uint32_t*>(keys + p.max_spans);
  uint32_t* between = taken + words;
  int* bins = reinterpret_cast<int*>(between + words);
  const int head = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (OWN) {
    pdl_wait();
    pdl_launch_dependents();
  }
  const int n = (tokens_of(p.lens, b, p.max_blocks, p.block_size) + p.span - 1) / p.span;
  const int32_t* table = p.tables + (size_t)b * p.max_blocks;
  int32_t* out = p.out + ((size_t)b * p.kv_heads + head) * p.count;

  if (n <= p.count) {   // all of them
    if (!OWN) {
      pdl_wait();
      pdl_launch_dependents();
    }
    for (int base = warp * 32; base < n; base += kPickThreads) {
      const int s = base + lane;
      const uint32_t m = __ballot_sync(0xffffffffu, s < n && page_at(table + sub_page(p, s), p.num_blocks) >= 0);
      if (lane == 0) taken[base / 32] = m;
    }
    __syncthreads();
    pick_write(taken, (n + 31) / 32, out, p.count, sums);
    return;
  }
  if (threadIdx.x == 0) q_most = n_sure = n_open = pick_bin = 0;
  for (int i = threadIdx.x; i < kPickBins; i += kPickThreads) bins[i] = 0;
  __syncthreads();
  for (int base = warp * 32; base < padded * (HD / 8); base += kPickThreads) {   // (whole warps) the query's rows: 8 channels a thread
    const int r = (base + lane) / (HD / 8), c = (base + lane) % (HD / 8) * 8;
    const uint4 v = r < rows ? ld_nc_v4(p.q + ((size_t)(b * p.Q + r / G) * p.heads + head * G + r % G) * HD + c) : make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(q_rows + r * HD + c) = v;
    float x[8], size = 0.f;
    unpack_bf16x8(v, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) size += fabsf(x[j]);
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) size += __shfl_xor_sync(0xffffffffu, size, o);
    const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(size));   // (NaN above infinity above all)
    if (lane == 0) atomicMax(&q_most, most);
  }
  uint32_t wide = 0;
  if (OWN) {
    wide = estimate_groups<HD, false>(p, b, head, n, warp, kPickWarps, nullptr, [&](int s, uint32_t e) { estimate[s] = e; }) << 16;
    __syncthreads();
  } else {
    pdl_wait();   // the estimates are there (what is read above was there before they began: see launcher())
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < p.warps; i += kPickThreads) wide = max(wide, __ldcg(p.wide + ((size_t)b * p.kv_heads + head) * p.warps + i));
  }

  auto kept = [&](int s) { return s < p.first || s >= n - p.last; };
  int always = 0, others = 0;
  uint32_t lowest = ~0u, highest = 0;
  const uint32_t* estimates = p.estimates + ((size_t)b * p.kv_heads + head) * p.max_spans;
  for (int base = threadIdx.x; base < n; base += 4 * kPickThreads) {   // four at a time
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = base + i * kPickThreads >= n ? kNoSpan : OWN ? estimate[base + i * kPickThreads] : __ldcg(estimates + base + i * kPickThreads);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = base + i * kPickThreads;
      if (!OWN && s < n) estimate[s] = e[i];
      const bool there = e[i] != kNoSpan, keep = kept(s);
      always += there && keep;
      others += there && !keep;
      if (there && !keep) {
        lowest = min(lowest, order_of(e[i]));
        highest = max(highest, order_of(e[i]));
      }
    }
  }
  always = __reduce_add_sync(0xffffffffu, always);
  others = __reduce_add_sync(0xffffffffu, others);
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  highest = __reduce_max_sync(0xffffffffu, highest);
  wide = __reduce_max_sync(0xffffffffu, wide);
  if (lane == 0) {
    stats[warp] = make_int4(always, others, (int)lowest, (int)highest);
    wides[warp] = wide;
  }
  __syncthreads();
  {
    const int4 x = stats[lane % kPickWarps];
    always = __reduce_add_sync(0xffffffffu, lane < kPickWarps ? x.x : 0);
    others = __reduce_add_sync(0xffffffffu, lane < kPickWarps ? x.y : 0);
    lowest = __reduce_min_sync(0xffffffffu, (uint32_t)x.z);
    highest = __reduce_max_sync(0xffffffffu, (uint32_t)x.w);
    wide = __reduce_max_sync(0xffffffffu, wides[lane % kPickWarps]);
  }
  const float lo = of_order(lowest), hi = of_order(highest), size = __uint_as_float(q_most) * __uint_as_float(wide);
  const int want = min(p.count - always, others);   // beside those that are kept
  const bool all = want == others, none = want == 0;
  const bool finite = size < 1e38f;
  const float eps2 = size * 0x1p-13f + 0x1p-100f, scale = hi - lo > 1e-30f ? (float)(kPickBins - 1) / (hi - lo) : 0.f;
  auto bin_of = [&](float x) { return (int)fminf(fmaxf((x - lo) * scale, -1.f), (float)(kPickBins - 1)); };   // (rises with x; NaN: -1)
  int line = 0;   // the bin of the want-th largest
  if (!all && !none && finite) {
#pragma unroll 4
    for (int s = threadIdx.x; s < n; s += kPickThreads) {
      const uint32_t e = estimate[s];
      if (e != kNoSpan && !kept(s)) atomicAdd(&bins[max(bin_of(__uint_as_float(e)), 0)], 1);
    }
    __syncthreads();
    constexpr int PER = kPickBins / kPickThreads;   // from the top, each thread some bins
    int mine = 0, total;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += bins[kPickBins - 1 - (int)threadIdx.x * PER - i];
    int upto = pick_running_sum(mine, sums, &total) - mine;
    if (upto < want && upto + mine >= want) {
      int i = kPickBins - 1 - (int)threadIdx.x * PER;
      for (;; --i) {
        upto += bins[i];
        if (upto >= want) break;
      }
      pick_bin = i;
    }
    __syncthreads();
    line = pick_bin;
  }
  int* list = bins;   // (the bins have been read) the spans between, in any order, as far as they are compared with one another
  for (int base = warp * 32; base < n; base += kPickThreads) {
    const int s = base + lane;
    const uint32_t e = s < n ? estimate[s] : kNoSpan;
    const bool there = e != kNoSpan, keep = kept(s);
    bool in = there && (keep || all), maybe = there && !keep && !all && !none;
    if (maybe && finite) {
      const float x = __uint_as_float(e);
      in = bin_of(x - eps2) > line;
      maybe = !in && bin_of(x + eps2) >= line;
    }
    const uint32_t m_in = __ballot_sync(0xffffffffu, in), m_open = __ballot_sync(0xffffffffu, maybe), m_sure = __ballot_sync(0xffffffffu, in && !keep);
    int at = 0;
    if (lane == 0) {
      taken[base / 32] = m_in;
      between[base / 32] = m_open;
      if (m_sure) atomicAdd(&n_sure, __popc(m_sure));
      if (m_open) at = atomicAdd(&n_open, __popc(m_open));
    }
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(m_open & ((1u << lane) - 1));
    if (maybe && at < kPickRanked) list[at] = s;
  }
  __syncthreads();
  const int open = n_open, left = want - n_sure, n_words = (n + 31) / 32;   // so many of the `open` ones are wanted (0 where all or none are)

  if (left > 0 && left == open) {
    for (int w = threadIdx.x; w < n_words; w += kPickThreads) taken[w] |= between[w];
  } else if (left > 0) {
    // ---- scores in 64 bits, over the estimates ----
    const bool listed = open <= kPickRanked;
    const int m = listed ? open : n;
    auto span_of = [&](int i) { return listed ? list[i] : ((between[i >> 5] >> (i & 31)) & 1 ? i : -1); };
    for (int i = warp; i < m; i += kPickWarps) {
      const int s = span_of(i);
      if (s < 0) continue;
      unsigned long long key = 0;
      const int page = page_at(table + sub_page(p, s), p.num_blocks);
      if (page >= 0) {   // (it was when the estimate was made, unless the table has changed since)
        const __nv_bfloat16* both = bounds_at(p, page, s, head, HD);
        key = finite ? exact_score<HD, true>(both, q_rows, rows) : exact_score<HD, false>(both, q_rows, rows);
      }
      if (lane == 0) keys[i] = key;
    }
    __syncthreads();
    if (listed) {
      for (int i = threadIdx.x; i < m; i += kPickThreads) {
        const unsigned long long key = keys[i];
        const int s = list[i];
        int before = 0;
        for (int j = 0; j < m; ++j) before += keys[j] > key || (keys[j] == key && list[j] < s);
        if (before < left) atomicOr(&taken[s >> 5], 1u << (s & 31));
      }
    } else {   // the left-th largest score bit by bit, then as many of those on it as there is room for, in their order
      auto total = [&](int v) {
        v = __reduce_add_sync(0xffffffffu, v);
        __syncthreads();
        if (lane == 0) sums[warp] = v;
        __syncthreads();
        return __reduce_add_sync(0xffffffffu, lane < kPickWarps ? sums[lane] : 0);
      };
      unsigned long long score = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long tried = score | (1ull << bit);
        int c = 0;
        for (int i = threadIdx.x; i < m; i += kPickThreads) c += span_of(i) >= 0 && keys[i] >= tried;
        if (total(c) >= left) score = tried;
      }
      int above = 0;
      for (int i = threadIdx.x; i < m; i += kPickThreads) above += span_of(i) >= 0 && keys[i] > score;
      int room = left - total(above);
      for (int base = 0, turn = 1; base < m; base += kPickThreads, turn ^= 1) {
        const int i = base + threadIdx.x, s = i < m ? span_of(i) : -1;
        const bool over = s >= 0 && keys[i] > score, on = s >= 0 && keys[i] == score;
        int equal;
        const int at = pick_running_sum(on, sums + turn * kPickWarps, &equal) - on;
        if (over || (on && at < room)) atomicOr(&taken[s >> 5], 1u << (s & 31));
        room -= equal;
      }
    }
  }
  __syncthreads();
  pick_write(taken, n_words, out, p.count, sums + 2 * kPickWarps);
}

#ifndef SSDK_HOST_EMU
// ----------------------------------------------------------------------------------
// span_attn_kernel: softmax(scale q k^T) v over the keys of the listed spans, causal to the end of the context as in paged attention (query j of a sequence
// sees positions <= len - Q + j); grouped heads.  A list may name spans in any order; what lies outside the context or on a page outside the cache
// is passed over, a row that sees no key is zero.
// Bound by the bytes of the listed keys and values.  A cluster of blocks owns one key head of one sequence and up to sixteen of its query rows (more:
// span_tiles.cuh).  Pieces of 16 keys go round the blocks' warps, each with a ring of its own (cp.async, no barrier between warps) and a softmax of its own;
// at the end warps meet, then blocks.  Sums are fp32.  Weights go into the second product as two bf16 pieces, 16 bits of them: with 4096 keys an output is off by 2.4e-6 of
// itself before its own rounding to 8 bits (1e-7 with fp32 weights), 0.24 % of the outputs round to the neighbouring value, and their error against 64 bits stays what their
// rounding makes it, 0.00165 either way.  A third piece would be half as many products again for nothing that the output's type can hold.
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
  int tokens;                    // query tokens of a tile
  uint32_t q_sign;               // the sign of the scale, for two bf16 values
  bool zero_scale;
  float scale_log2;              // |scale| * log2(e), or 1 where the scale is 0
};
// Values that are not finite.  A product with the weight 0 of a query that does not see their token is NaN, so from the first token on that some query does not see
// they go into the product as 0 (take_out), and a row adds those that it sees where it is stored (add_taken_out), read from the cache again.  Where every query sees them the
// two pieces of a weight can make NaN of an infinity: columns that are NaN in a row whose weights are not are the sum of what is not finite in them.
SSDK_DEVINL bool not_finite(uint32_t half) { return (half & 0x7f80u) == 0x7f80u; }
SSDK_DEVINL bool take_out(uint4* at) {
  uint32_t w[4] = {at->x, at->y, at->z, at->w};
  bool some = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = not_finite(w[i]), hi = not_finite(w[i] >> 16);
    some = some || lo || hi;
    w[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
  }
  if (some) *at = make_uint4(w[0], w[1], w[2], w[3]);
  return some;
}
// 0 times two bf16 values: NaN where one is not finite, so that its row's scores are
SSDK_DEVINL uint32_t zero_times(uint32_t w) { return (not_finite(w) ? 0x7fffu : 0u) | (not_finite(w >> 16) ? 0x7fff0000u : 0u); }
// four columns of a row that sees the tokens below lim; all queries see those below `from`.  odd: values were taken out; l: the row's sum
__device__ __noinline__ float4 with_taken_out(const SpanAttnParams& p, int head_dim, int b, int kvh, int from, int lim, int d, float4 acc) {
  float out[4] = {acc.x, acc.y, acc.z, acc.w}, sum[4] = {};
  const bool nan = out[0] != out[0] || out[1] != out[1] || out[2] != out[2] || out[3] != out[3];
#pragma unroll 1
  for (int i = 0; i < p.count; ++i) {
    const int s = p.spans[((size_t)b * p.kv_heads + kvh) * p.count + i];
    if (s < 0 || (long long)s * p.span >= lim) continue;
    const int first = s * p.span, page = page_at(p.tables + (size_t)b * p.max_blocks + first / p.block_size, p.num_blocks);
    if (page < 0) continue;
#pragma unroll 1
    for (int pos = nan ? first : max(first, from); pos < lim && pos - first < p.span; ++pos) {
      const uint2 v = *reinterpret_cast<const uint2*>(p.v_cache + (((size_t)page * p.block_size + pos % p.block_size) * p.kv_heads + kvh) * head_dim + d);
      const uint32_t x[4] = {v.x & 0xffffu, v.x >> 16, v.y & 0xffffu, v.y >> 16};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (not_finite(x[j])) sum[j] += __uint_as_float(x[j] << 16);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = out[j] == out[j] ? out[j] + sum[j] : sum[j] != 0.f ? sum[j] : out[j];
  return make_float4(out[0], out[1], out[2], out[3]);
}
SSDK_DEVINL void add_taken_out(const SpanAttnParams& p, int head_dim, int b, int kvh, int from, int lim, int d, bool odd, float l, float4* acc) {
  const float any = (acc->x + acc->y) + (acc->z + acc->w);   // (NaN if one is, or of infinities of both signs, which come from values that are not finite too)
  if ((odd || any != any) && l == l) *acc = with_taken_out(p, head_dim, b, kvh, from, lim, d, *acc);
}

constexpr float kSpanSlack = 8.f;
constexpr int kSpanWarps = 4, kSpanStages = 3, kSpanKeys = 16;
constexpr int kSpanMost = 16;   // blocks of a cluster
constexpr int span_stage_bytes(int HD) { return 2 * kSpanKeys * (HD + 8) * 2; }
constexpr int span_attn_smem(int HD, int count) { return kSpanWarps * kSpanStages * span_stage_bytes(HD) + count * 8; }

template <int HD>
__global__ void __launch_bounds__(kSpanWarps * 32, 2) span_attn_kernel(const __grid_constant__ SpanAttnParams p) {
  constexpr int LDS = HD + 8, KS = HD / 16, ND = HD / 8, SEG = HD / 8;
  extern __shared__ __align__(16) uint8_t span_smem[];
  pdl_wait();
  pdl_launch_dependents();
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int kvh = blockIdx.x / C, b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.heads / p.kv_heads, R = G * p.Q;
  const int len = tokens_of(p.lens, b, p.max_blocks, p.block_size);
  int2* where = reinterpret_cast<int2*>(span_smem + kSpanWarps * kSpanStages * span_stage_bytes(HD));   // [count] slot (-1: none) and position of a span's first key
  uint8_t* ring = span_smem + warp * kSpanStages * span_stage_bytes(HD);

  __shared__ int s_odd;   // values were taken out
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
    if (threadIdx.x == 0) s_odd = 0;
    n_list = __reduce_max_sync(0xffffffffu, n_list);   // behind the last entry of any use
    if (lane == 0) last[warp] = n_list;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSpanWarps; ++w) n_list = max(n_list, last[w]);
  }

  uint32_t qa[KS][4];
  int lim[2];   // first position that a row does not see
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    const __nv_bfloat16* q = p.q + ((size_t)(b * p.Q + r / G) * p.heads + kvh * G + r % G) * HD + 2 * t;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      qa[kk][h] = r < R ? *reinterpret_cast<const uint32_t*>(q + kk * 16) ^ p.q_sign : 0u;
      qa[kk][2 + h] = r < R ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + 8) ^ p.q_sign : 0u;
    }
    if (p.zero_scale) {   // (scale_log2 is 1: 0 times the mask's minus infinity would be NaN)
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        qa[kk][h] = zero_times(qa[kk][h]);
        qa[kk][2 + h] = zero_times(qa[kk][2 + h]);
      }
    }
    lim[h] = r < R ? len - p.Q + r / G + 1 : 0;
  }
  const int seen_by_all = len - p.Q + 1;   // positions below it are seen by every row

  float o[ND][4], mrow[2] = {-INFINITY, -INFINITY}, lrow[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < ND; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  const int per = p.span / kSpanKeys;   // pieces of a span
  constexpr int TOK = 32 / SEG;   // keys that a warp copies at a time
  const int tok0 = lane / SEG, seg = lane % SEG;
  const size_t row_step = (size_t)TOK * p.kv_heads * HD;
  // places in the list advance by a warp's stride without a division
  const int step = kSpanWarps * C, step_i = step / per, step_r = step - step_i * per;
  struct Place { int i, r; };   // span of the list, piece of the span
  auto advance = [&](Place& at) {
    at.i += step_i;
    at.r += step_r;
    if (at.r >= per) {
      at.r -= per;
      ++at.i;
    }
  };
  const int own = rank * kSpanWarps + warp;
  Place ahead = {own / per, own % per}, now = ahead;
  auto load = [&](int stage) {   // the piece that is next to be asked for
    if (ahead.i >= n_list) return;
    const int off = ahead.r * kSpanKeys;
    const int2 at = where[ahead.i];
    const bool there = at.x >= 0;
    __nv_bfloat16* dk = reinterpret_cast<__nv_bfloat16*>(ring + stage * span_stage_bytes(HD)) + tok0 * LDS + seg * 8;
    __nv_bfloat16* dv = dk + kSpanKeys * LDS;
    size_t from = there ? (((size_t)at.x + off + tok0) * p.kv_heads + kvh) * HD + seg * 8 : 0;
    if (there && at.y + off + kSpanKeys <= len) {
#pragma unroll
      for (int u = 0; u < kSpanKeys / TOK; ++u, from += row_step) {
        cp_async16(dk + u * TOK * LDS, p.k_cache + from, true);
        cp_async16(dv + u * TOK * LDS, p.v_cache + from, true);
      }
    } else {
#pragma unroll 1
      for (int u = 0; u < kSpanKeys / TOK; ++u, from += row_step) {   // what is not in the context is zero: a stale NaN would pass a weight of 0
        const bool valid = there && at.y + off + u * TOK + tok0 < len;
        cp_async16(dk + u * TOK * LDS, p.k_cache + (valid ? from : 0), valid);
        cp_async16(dv + u * TOK * LDS, p.v_cache + (valid ? from : 0), valid);
      }
    }
  };
#pragma unroll
  for (int s = 0; s < kSpanStages - 1; ++s) {
    load(s);
    advance(ahead);
    cp_async_commit();
  }
  for (int stage = 0; now.i < n_list; stage = stage + 1 == kSpanStages ? 0 : stage + 1) {
    __syncwarp();   // every lane is done with the stage that is filled now
    load(stage == 0 ? kSpanStages - 1 : stage - 1);
    advance(ahead);
    cp_async_commit();
    cp_async_wait<kSpanStages - 1>();
    __syncwarp();   // every lane's copies of this stage have landed
    const int2 at = where[now.i];
    const int pos0 = at.y + now.r * kSpanKeys;
    advance(now);
    if (at.x < 0) continue;
    const __nv_bfloat16* cK = reinterpret_cast<const __nv_bfloat16*>(ring + stage * span_stage_bytes(HD));
    const __nv_bfloat16* cV = cK + kSpanKeys * LDS;
    const int mi = lane >> 3, rr = lane & 7;

    float s[2][4] = {};
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {   // a 16 x 16 piece of the keys: tokens 0 .. 7 and 8 .. 15, channels 0 .. 7 and 8 .. 15
      uint32_t kb[4];
      ldmatrix_x4(kb, cK + ((mi >> 1) * 8 + rr) * LDS + kk * 16 + (mi & 1) * 8);
      mma_bf16_16816(s[0], qa[kk], kb[0], kb[1]);
      mma_bf16_16816(s[1], qa[kk], kb[2], kb[3]);
    }
    if (pos0 + kSpanKeys > seen_by_all) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (pos0 + nt * 8 + 2 * t + (e & 1) >= lim[e >> 1]) s[nt][e] = -INFINITY;
      if (seen_by_all < len) {   // the sequence's own new tokens
        bool odd = false;
        for (int i = lane; i < kSpanKeys * SEG; i += 32)
          if (pos0 + i / SEG >= seen_by_all) odd |= take_out(const_cast<uint4*>(reinterpret_cast<const uint4*>(cV + i / SEG * LDS + i % SEG * 8)));
        if (odd) s_odd = 1;
        __syncwarp();
      }
    }
    // A row's reference is raised, and its sums rescaled, only when a score passes it by kSpanSlack (base 2): weights stay below 2^kSpanSlack, where fp32
    // and the two bf16 pieces are as fine relative to a value as below 1.
    float most[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) most[h] = fmaxf(max3(s[0][2 * h], s[0][2 * h + 1], s[1][2 * h]), s[1][2 * h + 1]) * p.scale_log2;
    if (__any_sync(0xffffffffu, most[0] > mrow[0] + kSpanSlack || most[1] > mrow[1] + kSpanSlack)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 1));
        top = fmaxf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)), mrow[h]);
        const float f = top == mrow[h] ? 1.f : ex2_ftz(mrow[h] - top);   // (from -inf: 0)
        mrow[h] = top;
        lrow[h] *= f;
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          o[i][2 * h] *= f;
          o[i][2 * h + 1] *= f;
        }
      }
    }
    uint32_t ph[4], pl[4];
    const float ref[2] = {mrow[0] == -INFINITY ? 0.f : mrow[0], mrow[1] == -INFINITY ? 0.f : mrow[1]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // rows g, g + 8 of keys 0 .. 7, then of keys 8 .. 15
      const int h = i & 1;
      const float x = ex2_ftz(fmaf(s[i >> 1][2 * h], p.scale_log2, -ref[h])), y = ex2_ftz(fmaf(s[i >> 1][2 * h + 1], p.scale_log2, -ref[h]));
      lrow[h] += x + y;
      ph[i] = pack_bf16x2(x, y);
      pl[i] = pack_bf16x2(x - __uint_as_float(ph[i] << 16), y - __uint_as_float(ph[i] & 0xffff0000u));   // (exact differences)
    }
#pragma unroll
    for (int nd = 0; nd < ND; nd += 2) {
      uint32_t vb[4];
      ldmatrix_x4_trans(vb, cV + ((mi & 1) * 8 + rr) * LDS + nd * 8 + (mi >> 1) * 8);
      mma_bf16_16816(o[nd], ph, vb[0], vb[1]);
      mma_bf16_16816(o[nd + 1], ph, vb[2], vb[3]);
      mma_bf16_16816(o[nd], pl, vb[0], vb[1]);
      mma_bf16_16816(o[nd + 1], pl, vb[2], vb[3]);
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // The warps' parts meet: [warp][row][HD + 8] O | reference, sum (row stride of 8 banks: fragment stores and row reads are free of conflicts).
  constexpr int LDO = HD + 8;
  float* parts = reinterpret_cast<float*>(span_smem);
  float* joined = parts + kSpanWarps * 16 * LDO;   // [row][HD + 8]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    lrow[h] += __shfl_xor_sync(0xffffffffu, lrow[h], 1);
    lrow[h] += __shfl_xor_sync(0xffffffffu, lrow[h], 2);
    float* row = parts + (warp * 16 + g + 8 * h) * LDO;
#pragma unroll
    for (int i = 0; i < ND; ++i) *reinterpret_cast<float2*>(row + i * 8 + 2 * t) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
    if (t == 0) *reinterpret_cast<float2*>(row + HD) = make_float2(mrow[h], lrow[h]);
  }
  __syncthreads();
  // four columns of a row
  auto store = [&](int r, int d, float4 acc, float l, bool odd) {
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;   // (a row that sees no key is zero, NaN stays)
    acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    add_taken_out(p, HD, b, kvh, seen_by_all, len - p.Q + r / G + 1, d, odd, l, &acc);
    __nv_bfloat16* dst = p.out + ((size_t)(b * p.Q + r / G) * p.heads + kvh * G + r % G) * HD + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
  };
  for (int idx = threadIdx.x; idx < R * (HD / 4); idx += kSpanWarps * 32) {
    const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSpanWarps; ++w) top = fmaxf(top, parts[(w * 16 + r) * LDO + HD]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    if (top != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kSpanWarps; ++w) {
        const float* row = parts + (w * 16 + r) * LDO;
        const float2 ml = *reinterpret_cast<const float2*>(row + HD);
        const float4 v = *reinterpret_cast<const float4*>(row + d);
        const float f = exp2f(ml.x - top);
        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
        l += ml.y * f;
      }
    } else {   // no score, or NaN only
      for (int w = 0; w < kSpanWarps; ++w) l += parts[(w * 16 + r) * LDO + HD + 1];
    }
    if (C == 1) {
      store(r, d, acc, l, s_odd);
    } else {
      *reinterpret_cast<float4*>(joined + r * LDO + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(joined + r * LDO + HD) = make_float2(top, s_odd ? -l : l);   // (a sum's sign is that word)
    }
  }
  if (C == 1) return;
  // The blocks' parts meet over the cluster's shared memory, each block joins a share of the columns.
  cluster.sync();
  for (int idx = rank * kSpanWarps * 32 + threadIdx.x; idx < R * (HD / 4); idx += C * kSpanWarps * 32) {
    const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
    float2 ml[kSpanMost];
    float4 v[kSpanMost];
    float top = -INFINITY;
#pragma unroll
    for (int c = 0; c < kSpanMost; ++c) {
      if (c < C) {
        const float* row = cluster.map_shared_rank(joined, c) + r * LDO;
        ml[c] = *reinterpret_cast<const float2*>(row + HD);
        v[c] = *reinterpret_cast<const float4*>(row + d);
        top = fmaxf(top, ml[c].x);
      }
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    bool odd = false;
    if (top != -INFINITY) {
#pragma unroll
      for (int c = 0; c < kSpanMost; ++c) {
        if (c < C) {
          const float f = exp2f(ml[c].x - top);
          acc.x += v[c].x * f; acc.y += v[c].y * f; acc.z += v[c].z * f; acc.w += v[c].w * f;
          l += fabsf(ml[c].y) * f;
          odd |= __float_as_int(ml[c].y) < 0;
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < kSpanMost; ++c)
        if (c < C) l += ml[c].y;
    }
    store(r, d, acc, l, odd);
  }
  cluster.sync();   // no block leaves while its part is read
}
#endif  // SSDK_HOST_EMU

}  // namespace ssdk
