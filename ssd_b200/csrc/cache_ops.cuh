// cache_ops.cuh — what surrounds attention over a part of a long paged cache: pages, positions and slots of a step's tokens from the lengths of its
// requests, rotary positions with several axes beside the cache write, and per span of keys the smallest and largest value of every channel.
#pragma once
#include "paged.cuh"

namespace ssdk {

// ----------------------------------------------------------------------------------
// place_tokens_kernel.  Sequence b has ctx[b] tokens in ceil(ctx / S) pages of S tokens and gets new[b] more; need[b] = ceil((ctx + new) / S) - ceil(ctx / S)
// pages come from the list of free ones, in the order of the sequences.  With P[b] the sum of need up to b and R[b] the sum of the new tokens of those that
// have their pages, b is placed where used + P[b] <= free pages (or it needs none) and R[b] <= rows (or it brings none).  Both sums only grow, so that what
// is placed takes a prefix of the list and of the rows.
// A row finds its sequence by bisection over the running sums; the row at a page's first token writes the page into the table (a new page's first
// token is always a new one).  Every block makes the sums of all sequences for itself, so that blocks need not meet and one launch is all: 8 bytes a
// sequence read again by each of at most 148 blocks, out of L2.
// ----------------------------------------------------------------------------------
struct PlaceParams {
  const int32_t* ctx;            // [B]
  const int32_t* fresh;          // [B] new tokens
  int32_t* tables;               // [B, max_blocks]
  const int32_t* free_blocks;    // [n_free]
  const int32_t* free_used;      // [1]
  int64_t* positions;            // [rows]
  int32_t *slots, *seqs;         // [rows]
  int32_t *cu, *lens, *used;     // [B + 1], [B], [1]
  int B, max_blocks, n_free, rows, block_size, num_blocks;
};
constexpr int kPlaceThreads = 512;
constexpr int kPlaceMaxSeqs = 16384;
constexpr int place_smem(int B) { return (2 * B + 1) * 4; }

// sum of v over the threads up to this one, and over the block (64 bits: lengths and their sums are the caller's).  part: a word per warp
SSDK_DEVINL long long block_running_sum(long long v, long long* part, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int src = lane >= o ? lane - o : lane;
    const unsigned lo = __shfl_sync(0xffffffffu, (unsigned)(unsigned long long)v, src), hi = __shfl_sync(0xffffffffu, (unsigned)((unsigned long long)v >> 32), src);
    if (lane >= o) v += (long long)(((unsigned long long)hi << 32) | lo);
  }
  __syncthreads();   // the words of the sum before have been read
  if (lane == 31) part[warp] = v;
  __syncthreads();
  long long before = 0, all = 0;
  for (int i = 0; i < kPlaceThreads / 32; ++i) {
    const long long x = part[i];
    before += i < warp ? x : 0;
    all += x;
  }
  *total = all;
  return before + v;
}

__global__ void __launch_bounds__(kPlaceThreads) place_tokens_kernel(PlaceParams p) {
  SSDK_DYN_SMEM(int32_t, place_words);
  pdl_wait();
  pdl_launch_dependents();
  SSDK_STATIC_SMEM(long long, part, kPlaceThreads / 32);
  SSDK_STATIC_SMEM(int, most, 2);   // pages and rows of all that is placed
  int32_t* cu = place_words;                // [B + 1] first row of a sequence
  int32_t* first = place_words + p.B + 1;   // [B] entry of the free list that would be page 0: page x is free_blocks[first + x] from the first new one on
  const int S = p.block_size, used = max(p.free_used[0], 0);
  const long long cap = (long long)p.max_blocks * S;
  const bool writer = blockIdx.x == 0;
  if (threadIdx.x < 2) most[threadIdx.x] = 0;
  if (threadIdx.x == 0) cu[0] = 0;
  __syncthreads();

  long long pages = 0, rows = 0;   // sums over the sequences in front of this stretch
  for (int base = 0; base < p.B; base += kPlaceThreads) {
    const int b = base + threadIdx.x;
    const int c = b < p.B ? p.ctx[b] : 0, n = b < p.B ? p.fresh[b] : 0;
    bool ok = b < p.B && c >= 0 && n >= 0 && (long long)c + n <= cap;
    const int have = ok ? (int)(((long long)c + S - 1) / S) : 0;
    const int need = ok ? (int)(((long long)c + n + S - 1) / S) - have : 0;
    long long total;
    const long long P = pages + block_running_sum(need, part, &total);
    pages += total;
    ok = ok && (need == 0 || used + P <= p.n_free);
    const long long R = rows + block_running_sum(ok ? n : 0, part, &total);
    rows += total;
    const bool fits = R <= p.rows;
    ok = ok && (n == 0 || fits);
    if (b < p.B) {
      cu[b + 1] = fits ? (int)R : -1;
      first[b] = ok && need > 0 ? (int)(used + P) - need - have : 0;
      if (ok && need > 0) atomicMax(&most[0], (int)P);
      if (fits) atomicMax(&most[1], (int)R);
      if (writer) p.lens[b] = ok ? c + n : c;
    }
  }
  __syncthreads();
  const int n_rows = most[1];
  if (rows > p.rows) {   // sequences behind the first that found no room own no rows
    for (int b = threadIdx.x; b < p.B; b += kPlaceThreads)
      if (cu[b + 1] < 0) cu[b + 1] = n_rows;
    __syncthreads();
  }
  if (writer) {
    for (int b = threadIdx.x; b <= p.B; b += kPlaceThreads) p.cu[b] = cu[b];
    if (threadIdx.x == 0) p.used[0] = used + most[0];
  }

  for (int r = blockIdx.x * kPlaceThreads + threadIdx.x; r < p.rows; r += gridDim.x * kPlaceThreads) {
    int64_t pos = 0;
    int slot = -1, seq = -1;
    if (r < n_rows) {
      int lo = 0, hi = p.B - 1;   // the sequence whose rows end behind r first
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid + 1] > r) hi = mid;
        else lo = mid + 1;
      }
      seq = lo;
      const int c = p.ctx[seq], at = c + (r - cu[seq]);
      const int x = at / S, off = at - x * S, have = (int)(((long long)c + S - 1) / S);
      int32_t* entry = p.tables + (size_t)seq * p.max_blocks + x;
      const int page = x < have ? *entry : p.free_blocks[first[seq] + x];
      if (x >= have && off == 0) *entry = page;
      if (page >= 0 && page < p.num_blocks) slot = page * S + off;
      pos = at;
    }
    p.positions[r] = pos;
    p.slots[r] = slot;
    p.seqs[r] = seq;
  }
}

// ----------------------------------------------------------------------------------
// rope_axes_kernel: frequency i turns the channels (i, i + rot/2) of every query and key head by the angle of the row's position on axis
// axis_of[i] (time, height, width, ...); channels from rot on pass.  Optional RMS norm per head in front.  Norm, rotation and the table's cosines and
// sines are fp32, and a value is rounded once, where it is stored.  Queries go to q, keys and values to their slot of the cache.
// Bound by memory: 2 bytes read and 2 written per channel.  HD / 16 lanes own a head, 16 channels each in two 16-byte pieces, and a warp asks for a batch of
// 2 * 32 / (HD / 16) heads at once, a batch ahead.  The rows' batches lie one behind the other and each warp has a stretch of them: the angles stay in registers for a row,
// the next row's heads are on their way when it begins, and few rows still make as many warps as batches.  Products and sums two at a time.  16000 rows of 32 heads of 128
// with norms 49.4 us (a warp per row 52; four warps a row that gathered the angles through shared memory 58, issue slots 70 % busy; norm weights of the queries kept in
// registers 51), 4003 rows of 48 heads 20.9.
// A row with a position outside the table has NaN queries and stores nothing.
// ----------------------------------------------------------------------------------
struct RopeAxesParams {
  const __nv_bfloat16* qkv;      // [M, (H + 2 KV) hd]
  const int64_t* positions;      // [axes, M]
  const int32_t* slots;          // [M]
  const float* table;            // [top, rot] cos | sin
  const __nv_bfloat16 *q_norm_w, *k_norm_w;   // [hd] or null
  __nv_bfloat16 *q, *k_cache, *v_cache;
  int64_t top, num_slots;
  float eps;
  int M, heads, kv_heads, rot, axes;
  int batches;                   // of heads that a warp asks for at once, in a row
  int warps, each, longer;       // the rows' batches one behind the other: a warp has a stretch of `each`, the first `longer` one more
  uint32_t axis_of[8];           // two bits per frequency
};
constexpr int kRopeAxesThreads = 128, kRopeAxesAhead = 2;
constexpr int rope_axes_heads(int HD) { return 32 / (HD / 16) * kRopeAxesAhead; }   // that a warp asks for at once

template <int HD, bool NORM>
__global__ void __launch_bounds__(kRopeAxesThreads, 4) rope_axes_kernel(RopeAxesParams p) {
  constexpr int LPH = HD / 16, SIDE = 32 / LPH;   // lanes of a head, heads side by side
  pdl_wait();
  pdl_launch_dependents();
  const int warp = (int)blockIdx.x * (kRopeAxesThreads / 32) + (int)(threadIdx.x >> 5);
  if (warp >= p.warps) return;
  int unit = warp * p.each + min(warp, p.longer);   // (below 2^31: the host sees to it)
  const int last = unit + p.each + (warp < p.longer);
  const int piece = threadIdx.x % LPH, side = threadIdx.x % 32 / LPH, half = p.rot / 2;
  const int n_heads = p.heads + 2 * p.kv_heads;
  const bool turns = piece < p.rot / 16;
  const int c0 = turns ? piece * 8 : p.rot + (piece - p.rot / 16) * 16, c1 = turns ? half + piece * 8 : c0 + 8;

  uint4 a[kRopeAxesAhead], b[kRopeAxesAhead];
  auto load = [&](int m, int batch) {
    const __nv_bfloat16* src = p.qkv + (size_t)m * n_heads * HD;
#pragma unroll
    for (int i = 0; i < kRopeAxesAhead; ++i) {
      const int head = (batch * kRopeAxesAhead + i) * SIDE + side;
      a[i] = b[i] = make_uint4(0, 0, 0, 0);
      if (head < n_heads) {
        a[i] = ld_nc_v4(src + head * HD + c0);
        b[i] = ld_nc_v4(src + head * HD + c1);
      }
    }
  };
  int m = unit / p.batches, batch = unit - m * p.batches, row = -1;
  load(m, batch);
  bool known = true, stores = false;
  uint64_t co[4] = {}, si[4] = {}, minus[4] = {};   // cos, sin, -sin of this lane's eight frequencies
  __nv_bfloat16* q_row = p.q;
  size_t in_cache = 0;

  for (; unit < last; ++unit) {
    if (m != row) {
      row = m;
      const int slot = p.slots[m];
      known = true;
      for (int x = 0; x < p.axes; ++x) {
        const int64_t at = p.positions[(size_t)x * p.M + m];
        known = known && at >= 0 && at < p.top;
      }
      if (turns && known) {
        const uint32_t axes = (p.axis_of[piece >> 1] >> (16 * (piece & 1))) & 0xffffu;
        if (axes == (axes & 3) * 0x5555u) {
          const float* angles = p.table + (size_t)p.positions[(size_t)(axes & 3) * p.M + m] * p.rot + piece * 8;
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float4 c = *reinterpret_cast<const float4*>(angles + 2 * i), s = *reinterpret_cast<const float4*>(angles + half + 2 * i);
            co[i] = pack2(c.x, c.y); co[i + 1] = pack2(c.z, c.w);
            si[i] = pack2(s.x, s.y); si[i + 1] = pack2(s.z, s.w);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* r0 = p.table + (size_t)p.positions[(size_t)(axes >> (4 * i) & 3) * p.M + m] * p.rot + piece * 8 + 2 * i;
            const float* r1 = p.table + (size_t)p.positions[(size_t)(axes >> (4 * i + 2) & 3) * p.M + m] * p.rot + piece * 8 + 2 * i + 1;
            co[i] = pack2(r0[0], r1[0]);
            si[i] = pack2(r0[half], r1[half]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) minus[i] = si[i] ^ 0x8000000080000000ull;
      }
      stores = known && slot >= 0 && slot < p.num_slots;
      q_row = p.q + (size_t)m * p.heads * HD;
      in_cache = (size_t)max(slot, 0) * p.kv_heads * HD;
    }
    const int head0 = batch * kRopeAxesAhead * SIDE;
    uint4 now_a[kRopeAxesAhead], now_b[kRopeAxesAhead];
#pragma unroll
    for (int i = 0; i < kRopeAxesAhead; ++i) {
      now_a[i] = a[i];
      now_b[i] = b[i];
    }
    if (++batch == p.batches) {
      batch = 0;
      ++m;
    }
    if (unit + 1 < last) load(m, batch);
#pragma unroll
    for (int i = 0; i < kRopeAxesAhead; ++i) {
      const int head = head0 + i * SIDE + side, kind = head < p.heads ? 0 : (head < p.heads + p.kv_heads ? 1 : 2);   // q, k, v
      uint4 x = now_a[i], y = now_b[i];
      if (head0 + i * SIDE < p.heads + p.kv_heads) {   // (the whole warp: some of its heads are no values)
        uint64_t u[4], v[4];
        pairs_of(x, u);
        pairs_of(y, v);
        if (NORM) {
          uint64_t ss2 = mul2(u[0], u[0]);
#pragma unroll
          for (int j = 1; j < 4; ++j) ss2 = fma2(u[j], u[j], ss2);
#pragma unroll
          for (int j = 0; j < 4; ++j) ss2 = fma2(v[j], v[j], ss2);
          float s0, s1;
          unpack2(ss2, &s0, &s1);
          s0 += s1;
#pragma unroll
          for (int o = LPH / 2; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
          const __nv_bfloat16* weight = kind == 0 ? p.q_norm_w : p.k_norm_w;
          if (weight) {
            const float r = rsqrtf(s0 / (float)HD + p.eps);
            const uint64_t rr = pack2(r, r);
            uint64_t w[4];
            pairs_of(*reinterpret_cast<const uint4*>(weight + c0), w);
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = mul2(mul2(u[j], rr), w[j]);
            pairs_of(*reinterpret_cast<const uint4*>(weight + c1), w);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = mul2(mul2(v[j], rr), w[j]);
          }
        }
        if (turns) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint64_t t = fma2(u[j], co[j], mul2(v[j], minus[j]));
            v[j] = fma2(v[j], co[j], mul2(u[j], si[j]));
            u[j] = t;
          }
        }
        if (kind != 2) {
          x = bf16_of(u);
          y = bf16_of(v);
          if (!known) x = y = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
        }
      }
      if (head < n_heads && (kind == 0 || stores)) {
        __nv_bfloat16* dst = kind == 0 ? q_row + head * HD : (kind == 1 ? p.k_cache + in_cache + (head - p.heads) * HD : p.v_cache + in_cache + (head - p.heads - p.kv_heads) * HD);
        *reinterpret_cast<uint4*>(dst + c0) = x;
        *reinterpret_cast<uint4*>(dst + c1) = y;
      }
    }
  }
}

// ----------------------------------------------------------------------------------
// span_bounds_kernel: lo[d] = min, hi[d] = max of channel d over the keys of a span that are in the context, for every span that holds one of the last
// `fresh` tokens of its sequence.  Read anew from the cache rather than kept up: a rejected draft token leaves no trace, a page that changes hands needs no
// reset, and a span named by two tables gets the same values twice.  min and max are exact in any order; a NaN key makes its channel NaN.
// Bound by memory: a span's keys once.  A thread owns a column of 8 channels (16 bytes).  Few spans: a block takes 32 columns of one, its warps beside one
// another token after token, and they meet in shared memory, so that all loads are in flight together (64 x 7 new rows 4.5 us; 8.2 with a span's tokens in
// two lanes).  Many: a warp takes 32 columns of a span alone, eight tokens at a time (four prompts of 16001 24 us; 35 the other way, bound by its instructions).
// ----------------------------------------------------------------------------------
struct SpanBoundsParams {
  const __nv_bfloat16* k_cache;  // [num_blocks, block_size, KV, hd]
  const int32_t* tables;         // [B, max_blocks]
  const int32_t* lens;           // [B]
  __nv_bfloat16* bounds;         // [num_blocks, block_size / span, KV, 2, hd]: lo, hi
  int64_t num_blocks;
  int B, max_blocks, block_size, span, kv_heads, head_dim, fresh;
  int width;                     // columns of 8 channels of a block: 8, 16 or 32
};
constexpr int kBoundsThreads = 256;

SSDK_DEVINL uint4 min_bf16x8(const uint4& a, const uint4& b) { return make_uint4(min_bf16x2(a.x, b.x), min_bf16x2(a.y, b.y), min_bf16x2(a.z, b.z), min_bf16x2(a.w, b.w)); }
SSDK_DEVINL uint4 max_bf16x8(const uint4& a, const uint4& b) { return make_uint4(max_bf16x2(a.x, b.x), max_bf16x2(a.y, b.y), max_bf16x2(a.z, b.z), max_bf16x2(a.w, b.w)); }

SSDK_DEVINL uint4 shfl_xor_16(const uint4& v, int o) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o), __shfl_xor_sync(0xffffffffu, v.z, o), __shfl_xor_sync(0xffffffffu, v.w, o));
}

template <bool SPLIT>
__global__ void __launch_bounds__(kBoundsThreads, 4) span_bounds_kernel(SpanBoundsParams p) {
  constexpr int WARPS = kBoundsThreads / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.y;
  const int len = tokens_of(p.lens, b, p.max_blocks, p.block_size);
  const int row = p.kv_heads * p.head_dim, slices = (row / 8 + p.width - 1) / p.width;   // columns of a warp: p.width
  const int nth = SPLIT ? (int)blockIdx.x : (int)blockIdx.x * WARPS + (int)(threadIdx.x >> 5), span = nth / slices;
  const long long from = (max(len - p.fresh, 0) / p.span + (long long)span) * p.span;   // (the grid's last warps may be some long spans behind the end)
  if (from >= len) return;
  const int pos0 = (int)from;
  const int page = page_at(p.tables + (size_t)b * p.max_blocks + pos0 / p.block_size, p.num_blocks);
  if (page < 0) return;
  const int off = pos0 % p.block_size, tokens = min(p.span, len - pos0);
  const int who = SPLIT ? (int)threadIdx.x : (int)threadIdx.x % 32;
  const int col = (nth - span * slices) * p.width + who % p.width;                       // of 8 channels
  const int lane = who / p.width, lanes = (SPLIT ? kBoundsThreads : 32) / p.width;       // tokens beside one another
  const bool there = col * 8 < row;
  uint4 lo = make_uint4(0x7f807f80u, 0x7f807f80u, 0x7f807f80u, 0x7f807f80u), hi = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);   // +- infinity
  const __nv_bfloat16* keys = p.k_cache + ((size_t)page * p.block_size + off) * row + col * 8;
  constexpr int AHEAD = SPLIT ? 4 : 8;
  for (int t = lane; t < tokens; t += AHEAD * lanes) {
    uint4 v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (there && t + j * lanes < tokens) v[j] = ld_nc_v4(keys + (size_t)(t + j * lanes) * row);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (there && t + j * lanes < tokens) {
        lo = min_bf16x8(lo, v[j]);
        hi = max_bf16x8(hi, v[j]);
      }
  }
  const int head = col * 8 / p.head_dim;
  __nv_bfloat16* out = p.bounds + ((size_t)page * (p.block_size / p.span) + off / p.span) * 2 * row + (size_t)head * 2 * p.head_dim + (col * 8 - head * p.head_dim);
  if (SPLIT) {
    SSDK_STATIC_SMEM(uint4, meet, 2 * kBoundsThreads);
    meet[threadIdx.x] = lo;
    meet[kBoundsThreads + threadIdx.x] = hi;
    __syncthreads();
    if (lane > 1 || !there) return;   // the first lane joins the smallest values, the second the largest
    const uint4* part = meet + lane * kBoundsThreads + threadIdx.x % p.width;
    uint4 v = part[0];
    for (int l = 1; l < lanes; ++l) v = lane ? max_bf16x8(v, part[l * p.width]) : min_bf16x8(v, part[l * p.width]);
    *reinterpret_cast<uint4*>(out + lane * p.head_dim) = v;
  } else {
    for (int o = p.width; o < 32; o <<= 1) {
      lo = min_bf16x8(lo, shfl_xor_16(lo, o));
      hi = max_bf16x8(hi, shfl_xor_16(hi, o));
    }
    if (lane > 0 || !there) return;
    *reinterpret_cast<uint4*>(out) = lo;
    *reinterpret_cast<uint4*>(out + p.head_dim) = hi;
  }
}

}  // namespace ssdk
