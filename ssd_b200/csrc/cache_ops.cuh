// cache_ops.cuh — what surrounds attention over a part of a long paged cache: pages, positions and slots of a step's tokens from the lengths of its
// requests, rotary positions with several axes beside the cache write, and per span of keys the smallest and largest value of every channel.
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
// Bound by memory: 2 bytes read and 2 written per channel.  HD / 16 lanes own a head, 16 channels each in two 16-byte pieces; a thread keeps its
// frequencies over NH heads of its row, all asked for before the angles, which the block gathers from the rows of the axes into shared memory.
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
  uint32_t axis_of[8];           // two bits per frequency
};
constexpr int kRopeAxesThreads = 128;

SSDK_DEVINL void turn(float& x, float& y, float c, float s) {
  const float u = x * c - y * s;
  y = y * c + x * s;
  x = u;
}

template <int HD, int NH>
__global__ void __launch_bounds__(kRopeAxesThreads, NH <= 3 ? 8 : 6) rope_axes_kernel(RopeAxesParams p) {
  constexpr int LPH = HD / 16, GROUPS = kRopeAxesThreads / LPH;
  SSDK_STATIC_SMEM(float4, cs4, 64);
  float* cs = reinterpret_cast<float*>(cs4);
  const int m = blockIdx.x, lane = threadIdx.x % LPH, half = p.rot / 2;
  const int head0 = blockIdx.y * (NH * GROUPS) + threadIdx.x / LPH, n_heads = p.heads + 2 * p.kv_heads;
  const bool turns = lane < p.rot / 16;
  const int c0 = turns ? lane * 8 : p.rot + (lane - p.rot / 16) * 16, c1 = turns ? half + lane * 8 : c0 + 8;

  const __nv_bfloat16* src = p.qkv + (size_t)m * n_heads * HD;
  const int slot = p.slots[m];
  uint4 a[NH], b[NH];
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const int head = head0 + i * GROUPS;
    a[i] = b[i] = make_uint4(0, 0, 0, 0);
    if (head < n_heads) {
      a[i] = ld_nc_v4(src + (size_t)head * HD + c0);
      b[i] = ld_nc_v4(src + (size_t)head * HD + c1);
    }
  }
  bool known = true;
  for (int x = 0; x < p.axes; ++x) {
    const int64_t at = p.positions[(size_t)x * p.M + m];
    known = known && at >= 0 && at < p.top;
  }
  if (known)
    for (int i = threadIdx.x; i < p.rot; i += kRopeAxesThreads) {
      const int f = i < half ? i : i - half, axis = (p.axis_of[f >> 4] >> (2 * (f & 15))) & 3;
      cs[i] = p.table[(size_t)p.positions[(size_t)axis * p.M + m] * p.rot + i];
    }
  __syncthreads();
  const bool stores = known && slot >= 0 && slot < p.num_slots;
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const int head = head0 + i * GROUPS, kind = head < p.heads ? 0 : (head < p.heads + p.kv_heads ? 1 : 2);   // q, k, v
    float x[8], y[8];
    unpack_bf16x8(a[i], x);
    unpack_bf16x8(b[i], y);
    const __nv_bfloat16* w = kind == 0 ? p.q_norm_w : p.k_norm_w;
    if (w) {   // (the same for all lanes of a head; every lane of a warp takes part in the sums)
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += x[j] * x[j] + y[j] * y[j];
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss / (float)HD + p.eps);
      float wx[8], wy[8];
      unpack_bf16x8(ld_nc_v4(w + c0), wx);
      unpack_bf16x8(ld_nc_v4(w + c1), wy);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] *= r * wx[j];
        y[j] *= r * wy[j];
      }
    }
    if (head >= n_heads || (kind != 0 && !stores)) continue;
    __nv_bfloat16* dst = kind == 0 ? p.q + ((size_t)m * p.heads + head) * HD
                                   : (kind == 1 ? p.k_cache + ((size_t)slot * p.kv_heads + (head - p.heads)) * HD
                                                : p.v_cache + ((size_t)slot * p.kv_heads + (head - p.heads - p.kv_heads)) * HD);
    if (kind != 2) {
      if (turns && known) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const float4 co = *reinterpret_cast<const float4*>(cs + c0 + j), si = *reinterpret_cast<const float4*>(cs + c1 + j);
          turn(x[j], y[j], co.x, si.x);
          turn(x[j + 1], y[j + 1], co.y, si.y);
          turn(x[j + 2], y[j + 2], co.z, si.z);
          turn(x[j + 3], y[j + 3], co.w, si.w);
        }
      }
      a[i] = pack_bf16x8(x);
      b[i] = pack_bf16x8(y);
      if (!known) a[i] = b[i] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
    }
    *reinterpret_cast<uint4*>(dst + c0) = a[i];
    *reinterpret_cast<uint4*>(dst + c1) = b[i];
  }
}

// ----------------------------------------------------------------------------------
// span_bounds_kernel: lo[d] = min, hi[d] = max of channel d over the keys of a span that are in the context, for every span that holds one of the last
// `fresh` tokens of its sequence.  Read anew from the cache rather than kept up: a rejected draft token leaves no trace, a page that changes hands needs no
// reset, and a span named by two tables gets the same values twice.  min and max are exact in any order; a NaN key makes its channel NaN.
// Bound by memory: a span's keys once.  A block takes 32 columns of 8 channels (16 bytes) of a span, a warp beside another token after token, and the warps'
// parts meet in shared memory: all loads of a short span are in flight together.  (With all columns in one block a thread walked half of the span's tokens:
// 64 spans of 32 tokens 8.3 us, 64000 tokens 37.)
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
SSDK_DEVINL uint4 min_bf16x8(const uint4& a, const uint4& b) { return make_uint4(min_bf16x2(a.x, b.x), min_bf16x2(a.y, b.y), min_bf16x2(a.z, b.z), min_bf16x2(a.w, b.w)); }
SSDK_DEVINL uint4 max_bf16x8(const uint4& a, const uint4& b) { return make_uint4(max_bf16x2(a.x, b.x), max_bf16x2(a.y, b.y), max_bf16x2(a.z, b.z), max_bf16x2(a.w, b.w)); }

__global__ void __launch_bounds__(kBoundsThreads) span_bounds_kernel(SpanBoundsParams p) {
  SSDK_STATIC_SMEM(uint4, meet, 2 * kBoundsThreads);
  const int b = blockIdx.y;
  const int len = tokens_of(p.lens, b, p.max_blocks, p.block_size);
  const int slices = (p.kv_heads * p.head_dim / 8 + p.width - 1) / p.width, nth = (int)blockIdx.x / slices;
  const int pos0 = (max(len - p.fresh, 0) / p.span + nth) * p.span;   // (below len + span, which the host holds under 2^31)
  if (pos0 >= len) return;
  const int page = page_at(p.tables + (size_t)b * p.max_blocks + pos0 / p.block_size, p.num_blocks);
  if (page < 0) return;
  const int off = pos0 % p.block_size, tokens = min(p.span, len - pos0);
  const int row = p.kv_heads * p.head_dim;
  const int col = ((int)blockIdx.x - nth * slices) * p.width + (int)threadIdx.x % p.width;   // of 8 channels
  const int lane = threadIdx.x / p.width, lanes = kBoundsThreads / p.width;                  // tokens beside one another
  const bool works = col * 8 < row && lane < tokens;
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (works) {
    const __nv_bfloat16* keys = p.k_cache + ((size_t)page * p.block_size + off) * row + col * 8;
    lo = hi = ld_nc_v4(keys + (size_t)lane * row);
#pragma unroll 7
    for (int t = lane + lanes; t < tokens; t += lanes) {
      const uint4 v = ld_nc_v4(keys + (size_t)t * row);
      lo = min_bf16x8(lo, v);
      hi = max_bf16x8(hi, v);
    }
  }
  meet[threadIdx.x] = lo;
  meet[kBoundsThreads + threadIdx.x] = hi;
  __syncthreads();
  if (lane > 1 || col * 8 >= row) return;   // the first lane joins the smallest values, the second the largest
  const uint4* part = meet + lane * kBoundsThreads + threadIdx.x % p.width;
  uint4 v = part[0];
  for (int l = 1; l < min(lanes, tokens); ++l) {
    const uint4 w = part[l * p.width];
    v = lane ? max_bf16x8(v, w) : min_bf16x8(v, w);
  }
  __nv_bfloat16* out = p.bounds + ((size_t)page * (p.block_size / p.span) + off / p.span) * 2 * row + (size_t)(col * 8 / p.head_dim) * 2 * p.head_dim;
  *reinterpret_cast<uint4*>(out + lane * p.head_dim + col * 8 % p.head_dim) = v;
}

}  // namespace ssdk
