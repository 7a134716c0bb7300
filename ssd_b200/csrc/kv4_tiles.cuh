// kv4_tiles.cuh — attention over a paged cache held in 4 bits (kv4.cuh) of more than sixteen query rows to a key head, on tcgen05.
//
// S = Q C^T of up to 128 rows (query tokens x the heads that share a key head) and 64 keys' codes into TMEM, P = exp2(S s + m sum(q) - reference) one row per thread, O += (P s') (C' - 8) with
// P s' out of TMEM; what the minima give is a sum of its own (kv4_attn_kernel has the formulas).
// Scores are products in e4m3: a byte that holds a code c in 0 .. 15 is the number c 2^-9, so codes become bytes with a mask (and a shift) for four.  A query row, scaled by a power of two so that its largest
// lies in 2^7 .. 2^8, is the sum of two e4m3 numbers, exactly where it is above 2^-10 of the largest, else off by at most 2^-17 of that; both meet the same codes.  The sums are fp32.
// Values stay bf16, c - 8, as P has no such range.  A word of eight channels gives them in the order 0, 4, 1, 5, 2, 6, 3, 7 (outputs are put back), and keys' codes as 0, 2, 4, 6, 1, 3, 5, 7 (queries are
// stored in that order).
// Four warps bring codes in (registers, a chunk ahead of the one that they write, its pages two ahead), one issues the products, four have the rows.  Scales and minima of a chunk's keys lie beside its
// values, as pairs of keys, so that a row takes two at a time.  A cluster of blocks shares the chunks of a key head; their sums meet in shared memory.
// A row takes 32 keys at a time (64 scores and as many scales pass the registers of nine warps twice on an SM).  TWIN: up to 64 rows lie in the tile twice, rows 0 .. 63 take a chunk's first 32 keys and
// 64 .. 127 the others, each with zeros for weights of the other half and a reference of its own: all four warps work on half of the scores where two would on all, and the products are no more.
#pragma once
#include <cuda_fp8.h>

#include "kv4_attention.cuh"
#include "prompt_attention.cuh"

namespace ssdk {

constexpr int kKv4TileRows = 128, kKv4TileKeys = 64, kKv4TileThreads = 288, kKv4Producers = 128;   // warps: 4 of rows, 4 of codes, one of products
constexpr int kv4_tile_body(int HD) { return kKv4TileRows * HD * 2 + 2 * kKv4TileKeys * 128 + 2 * kKv4TileKeys * HD * 2; }   // queries | two stages of keys | of values
constexpr int kv4_tile_smem(int HD) {
  const int join = kKv4TileRows * (HD + 4) * 4, body = kv4_tile_body(HD);
  return (body > join ? body : join) + 1024;
}

// nibbles P and P + 4 of a word as c - 8 in bf16
template <int P>
SSDK_DEVINL uint32_t kv4_pair(uint32_t w) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(kv4_pair16<P>(w)), "r"(0x41c041c0u));
  return d;
}
// four values as e4m3, and what that leaves of them as e4m3
SSDK_DEVINL void e4m3_twice(const float (&x)[4], uint32_t* high, uint32_t* low) {
  *high = *low = 0;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const __nv_fp8x2_storage_t h = __nv_cvt_float2_to_fp8x2(make_float2(x[i], x[i + 1]), __NV_SATFINITE, __NV_E4M3);
    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3)));
    const __nv_fp8x2_storage_t l = __nv_cvt_float2_to_fp8x2(make_float2(x[i] - f.x, x[i + 1] - f.y), __NV_SATFINITE, __NV_E4M3);
    *high |= (uint32_t)h << (8 * i);
    *low |= (uint32_t)l << (8 * i);
  }
}
// D[tmem] (+)= A[smem desc] * B[smem desc], e4m3 x e4m3 -> fp32, 32 bytes of k
SSDK_DEVINL void umma_e4m3_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// its descriptor: A = B = e4m3 (K-major), D = fp32
constexpr uint32_t make_umma_idesc_e4m3(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
SSDK_DEVINL uint4 kv4_words(uint32_t w) { return make_uint4(kv4_pair<0>(w), kv4_pair<1>(w), kv4_pair<2>(w), kv4_pair<3>(w)); }
// 16-byte piece c of a row of 128 bytes under the 128-byte swizzle
SSDK_DEVINL int swizzled(int row, int c) { return row * 128 + ((c ^ (row & 7)) << 4); }

struct Kv4TileParams {
  Kv4AttnParams a;
  int tokens;                    // query tokens of a tile
  unsigned* timeout;             // (rows whose waits ran out are NaN)
};

// SHARED: calls of one tile, whose blocks have equal stretches of all sequences' keys (kv4_attn_kernel, kv4_join_kernel; a turn is a chunk), one head's piece after another
template <int HD, bool TWIN, bool SHARED>
__global__ void __launch_bounds__(kKv4TileThreads, 2) kv4_tile_kernel(const __grid_constant__ Kv4TileParams pp) {
  namespace cg = cooperative_groups;
  constexpr int HALVES = HD / 64, CODES = HD / 2, K = kKv4TileKeys;
  constexpr int kQHalf = kKv4TileRows * 128, kKTile = K * 128, kVHalf = K * 128, kVTile = HALVES * kVHalf;
  const Kv4AttnParams& p = pp.a;
  extern __shared__ uint8_t kv4_tile_raw[];
  __shared__ __align__(8) uint64_t k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2];
  __shared__ __align__(16) float key_pairs[2][K * 2], value_pairs[2][K * 2];   // of two keys: scale, scale, what goes with the sum, the same (times scale * log2(e) for keys)
  __shared__ __align__(16) int at_pos[2][4];   // position of a chunk's sixteen keys, behind every context where they have no page
  __shared__ float2 row_units[kKv4TileRows];   // of a row of queries: what a unit of its products is (NaN: it is not finite), and its sum in them
  __shared__ uint32_t tmem_slot;
  uint8_t* smem = kv4_tile_raw + ((1024u - (smem_u32(kv4_tile_raw) & 1023u)) & 1023u);
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + HALVES * kQHalf;
  uint8_t* sV = sK + 2 * kKTile;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = SHARED ? 1 : (int)cluster.num_blocks(), rank = SHARED ? 0 : (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int kvh = blockIdx.x / C, b = blockIdx.y;
  const int tile = SHARED ? 0 : (int)gridDim.z - 1 - (int)blockIdx.z;   // (the tiles that see most keys first)
  const int G = p.heads / p.kv_heads, tok0 = tile * pp.tokens, tq = min(pp.tokens, p.Q - tok0), rows = tq * G;
  const int half = (rows + 31) & ~31;                // rows of the warps that have some
  const int live = TWIN ? 2 * half : half;           // threads that hand P over

  if (warp == 8) {
    if (lane == 0) {
      for (int s = 0; s < 2; ++s) {
        mbar_init(&k_full[s], kKv4Producers);
        mbar_init(&v_full[s], kKv4Producers);
        mbar_init(&s_full[s], 1);
        mbar_init(&p_full[s], live);
        mbar_init(&pv_done[s], 1);
      }
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(&tmem_slot, 256);
    tmem_relinquish();
  }
  pdl_wait();
  // SHARED: this block's turns at .. end, the first of them turn `turn` of its head
  int at = 0, end = 1, turn = 0, turns = 0, done = 0;   // done: chunks of the pieces before (of stages and barriers)
  if constexpr (SHARED) {
    const Kv4Stretch stretch(kv4_turns_of_all<K>(p, 0).x * p.kv_heads, gridDim.x);
    at = stretch.first(blockIdx.x);
    end = stretch.first(blockIdx.x + 1);
    int before = 0;
    if (at < end) b = kv4_sequence_of<K>(p, at, &before);
    if (at >= end || b >= p.B) {   // nothing to do but to give the tensor memory back (no sequence: only where lengths change meanwhile)
      __syncthreads();
      pdl_launch_dependents();
      if (warp == 8) tmem_dealloc(tmem_slot, 256);
      return;
    }
    turns = kv4_turns<K>(p, b);
    const int from = at - before * p.kv_heads;
    kvh = from / turns;
    turn = from - kvh * turns;
  }
#pragma unroll 1
  for (bool again = false; at < end; again = true) {
  if constexpr (SHARED) {
    if (again) {
      turn = 0;
      if (++kvh == p.kv_heads) {
        kvh = 0;
        if (++b >= p.B) break;   // (only where lengths change meanwhile)
        turns = kv4_turns<K>(p, b);
      }
    }
  }
  const int last_turn = SHARED ? min(turns, turn + (end - at)) : 0;
  if (!again) {   // the barriers, and where tensor memory is
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();   // (this block has its tensor memory: what is scheduled now may take the rest of the SM's and wait for this grid)
  }
  const uint32_t tmem = tmem_slot, tmem_o = tmem + 128;   // S / P buffers at columns 0 and 64, O behind them
  const int len = tokens_of(p.lens, b, p.max_blocks, p.block_size), ctx = len - p.Q + tok0;
  const int seen = max(0, min(len, ctx + tq)), seen_by_all = ctx + 1;   // positions that some row sees, that all do
  const int chunks = (seen + K - 1) / K, front = SHARED ? turn : rank;   // chunk i of this piece is front + i C
  const int n = SHARED ? max(0, min(chunks, last_turn) - turn) : front < chunks ? (chunks - front + C - 1) / C : 0;
  // Chunk i is in stage and on barriers use(i), parity(i) is that use's.  A wait by parity is only right while the barrier is in that use or the one behind it:
  //   k_full, v_full: whoever waits for chunk i has to be through with it before its stage is written anew (the keys' behind s_full, the values' behind pv_done, which needs every row's P).
  //   s_full: the producers and the rows ask for chunk i, and chunk i + 2's needs keys of the former and, through p_full, P of the latter.
  //   p_full: chunk i + 2's needs the rows to have seen its scores, which are issued behind the product of chunk i.
  //   pv_done: the scores of chunk i + 1 ask for chunk i - 1; the producers ask for chunk i - 2 before they bring chunk i's values; the rows ask for chunk i - 1, and chunk i + 1's product needs their P.
  auto use = [&](int i) { return (done + i) & 1; };
  auto parity = [&](int i) { return (uint32_t)((done + i) >> 1) & 1u; };
  float l = 0.f, m = -INFINITY, low = 0.f;
  bool ok = true;

  if (warp < 4 || warp == 8) {
    // Queries: HD / 8 lanes a row, eight channels each.  Heads of 128: high and low parts in halves of their own, heads of 64: in a row's 128 bytes behind one another (the keys' codes stand there twice).
    // Rows behind the last one are zero.
    constexpr int LPR = HD / 8, PIECES = (TWIN ? 64 : kKv4TileRows) * LPR, T = kKv4TileThreads - kKv4Producers, LOADS = (PIECES + T - 1) / T, BATCH = SHARED && LOADS > 7 ? 7 : LOADS;
    const int mine = warp < 4 ? threadIdx.x : threadIdx.x - kKv4Producers;
#pragma unroll 1
    for (int x0 = 0; x0 < LOADS; x0 += BATCH) {
      uint4 q_now[BATCH];
#pragma unroll
      for (int x = 0; x < BATCH; ++x) {
        const int i = (x0 + x) * T + mine, r = i / LPR;
        q_now[x] = make_uint4(0, 0, 0, 0);
        if (r < rows) q_now[x] = ld_nc_v4(p.q + ((size_t)(b * p.Q + tok0 + r / G) * p.heads + kvh * G + r % G) * HD + i % LPR * 8);
      }
#pragma unroll
      for (int x = 0; x < BATCH; ++x) {
        const int i = (x0 + x) * T + mine, r = i / LPR, c = i % LPR;
        if (i >= PIECES) break;   // (a warp's lanes stay together: both numbers are multiples of 32)
        float f[8], sum = 0.f, top = 0.f;
        unpack_bf16x8(q_now[x], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sum += f[j];
          top = fmaxf(top, fabsf(f[j]));
        }
#pragma unroll
        for (int w = 1; w < LPR; w *= 2) {
          sum += __shfl_xor_sync(0xffffffffu, sum, w);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        }
        const int e = max((int)(__float_as_uint(top) >> 23), 9);   // (biased exponent; a unit is 2^9 2^(e - 134), of which the keys' scales have 2^2)
        const float up = __uint_as_float((uint32_t)(261 - e) << 23), unit = __uint_as_float((uint32_t)min(e, 254) << 23);   // 2^(7 - (e - 127)), 2^(e - 127)
        const float even[4] = {f[0] * up, f[2] * up, f[4] * up, f[6] * up}, odd[4] = {f[1] * up, f[3] * up, f[5] * up, f[7] * up};
        uint2 high, low;
        e4m3_twice(even, &high.x, &low.x);
        e4m3_twice(odd, &high.y, &low.y);
#pragma unroll
        for (int at_row = r; at_row < kKv4TileRows; at_row += TWIN ? 64 : kKv4TileRows) {
          uint8_t* to = sQ + swizzled(at_row, c >> 1) + (c & 1) * 8;
          *reinterpret_cast<uint2*>(to) = high;
          if (HD == 128) *reinterpret_cast<uint2*>(to + kQHalf) = low;
          else *reinterpret_cast<uint2*>(sQ + swizzled(at_row, 4 + (c >> 1)) + (c & 1) * 8) = low;
          if (c == 0) row_units[at_row] = fabsf(sum) < INFINITY && e < 255 ? make_float2(unit, sum / unit) : make_float2(__uint_as_float(kKv4Nan), 0.f);
        }
      }
    }
    fence_proxy_async_smem();
    asm volatile("bar.sync 1, %0;" ::"r"(T) : "memory");   // (of these warps: codes are on their way meanwhile)
  }
  if (warp >= 4 && warp < 8) {
    // ---- codes: a thread has PER pieces of 32 channels (eight lanes are eight rows) of the keys and of the values, and the pair of one of either ----
    constexpr int NP = HD / 32, PER = K * NP / kKv4Producers;   // (PER = 2: the second piece is 32 rows on)
    const int tid = threadIdx.x - 128, pw = tid >> 5, piece = (lane >> 3) % NP, key = tid & 63;
    const int row = (HD == 128 ? pw : 2 * pw + (lane >> 4)) * 8 + (lane & 7);
    const int record = p.block_size * kv4_row_bytes(HD), pairs = p.block_size * CODES;   // (bytes of a page and head, of its codes)
    const int64_t page_step = (int64_t)p.kv_heads * record;
    const uint8_t *k_from = p.k_cache + (int64_t)kvh * record + piece * 16, *v_from = p.v_cache + (int64_t)kvh * record + piece * 16;
    const uint8_t* pair_from = (tid < 64 ? p.k_cache : p.v_cache) + (int64_t)kvh * record + pairs;
    const int32_t* table = p.tables + (size_t)b * p.max_blocks;
    const int step = C * K, step_x = step / p.block_size, step_off = step - step_x * p.block_size;
    uint4 kc[PER], vc[PER];   // (without a page they stay what they were: no row sees what comes of it)
#pragma unroll
    for (int u = 0; u < PER; ++u) kc[u] = vc[u] = make_uint4(0, 0, 0, 0);
    uint32_t pair = 0;
    int pos = 0;
    // A page of whole chunks is looked up once a chunk by each warp, others by sixteens of keys.  What a page is, is looked at where it is used, a chunk later.
    const bool one_page = p.block_size % K == 0;
    struct Place { int x, off, pos, page, at; };   // the next chunk's entry of the table, offset in its page and position, and the page and offset that were looked up
    auto first = [&](int sixteen) {
      Place w;
      w.pos = front * K + sixteen * 16;
      w.x = w.pos / p.block_size;
      w.off = w.pos - w.x * p.block_size;
      w.page = -1;
      w.at = 0;
      return w;
    };
    auto look_up = [&](Place& w) {   // (positions stay below 2^31: the host sees to it)
      w.page = w.pos < seen ? table[w.x] : -1;
      w.at = w.off;
      w.pos += step;
      w.x += step_x;
      w.off += step_off;
      if (w.off >= p.block_size) {
        w.off -= p.block_size;
        ++w.x;
      }
    };
    Place mine = first(one_page ? 0 : key >> 4), of[PER];
    look_up(mine);
    if (!one_page) {
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        of[u] = first((row + 32 * u) >> 4);
        look_up(of[u]);
      }
    }
    auto there = [&](int page) { return page >= 0 && page < p.num_blocks; };
    auto load = [&]() {   // of the chunk that was looked up; then the next one's pages
      pair = 0;
      if (one_page) {
        const bool is = there(mine.page);
        const int64_t at = mine.page * page_step + (mine.at + row) * CODES;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          if (is) {
            kc[u] = ld_nc_v4(k_from + at + u * 32 * CODES);
            vc[u] = ld_nc_v4(v_from + at + u * 32 * CODES);
          }
        }
        pos = is ? mine.pos - step + (key & 48) : kNoPosition;
        if (is && pos + (key & 15) < len) pair = *reinterpret_cast<const uint32_t*>(pair_from + mine.page * page_step + (mine.at + key) * 4);   // (behind the context it may be anything)
      } else {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          if (there(of[u].page)) {
            const int64_t at = of[u].page * page_step + (of[u].at + (row & 15)) * CODES;
            kc[u] = ld_nc_v4(k_from + at);
            vc[u] = ld_nc_v4(v_from + at);
          }
          look_up(of[u]);
        }
        const bool is = there(mine.page);
        pos = is ? mine.pos - step : kNoPosition;
        if (is && pos + (key & 15) < len) pair = *reinterpret_cast<const uint32_t*>(pair_from + mine.page * page_step + (mine.at + (key & 15)) * 4);
      }
      look_up(mine);
    };
    // where a piece's 32 bytes of a key go in a stage, and its four words (16 bytes of bf16 each) of a value
    uint8_t *k_to[2], *v_to[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) k_to[j] = sK + swizzled(row, piece * 2 + j);
#pragma unroll
    for (int j = 0; j < 4; ++j) v_to[j] = sV + (piece >> 1) * kVHalf + swizzled(row, (piece & 1) * 4 + j);
    if (n > 0) load();
    for (int i = 0; i < n; ++i) {
      uint4 k_now[PER], v_now[PER];
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        k_now[u] = kc[u];
        v_now[u] = vc[u];
      }
      const uint32_t pair_now = pair;
      const int pos_now = pos, s = use(i);
      if (i + 1 < n) load();
      if (done + i >= 2 && !tile_wait_warp(&s_full[s], parity(i - 2), pp.timeout)) break;   // the scores of chunk i - 2 have read their keys
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const uint32_t w[4] = {k_now[u].x, k_now[u].y, k_now[u].z, k_now[u].w};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 x = make_uint4(w[2 * j] & 0x0f0f0f0fu, w[2 * j] >> 4 & 0x0f0f0f0fu, w[2 * j + 1] & 0x0f0f0f0fu, w[2 * j + 1] >> 4 & 0x0f0f0f0fu);
          *reinterpret_cast<uint4*>(k_to[j] + s * kKTile + u * 32 * 128) = x;
          if (HD == 64) *reinterpret_cast<uint4*>(sK + s * kKTile + swizzled(row, 4 + piece * 2 + j)) = x;
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&k_full[s]);
      if (done + i >= 2 && !tile_wait_warp(&pv_done[s], parity(i - 2), pp.timeout)) break;   // its product has read its values, its rows their pairs
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const uint32_t w[4] = {v_now[u].x, v_now[u].y, v_now[u].z, v_now[u].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(v_to[j] + s * kVTile + u * 32 * 128) = kv4_words(w[j]);
      }
      {
        const float scale = __uint_as_float(pair_now << 16), minimum = __uint_as_float(pair_now & 0xffff0000u);
        float* dst = (tid < 64 ? key_pairs[s] : value_pairs[s]) + (key >> 1) * 4 + (key & 1);
        dst[0] = tid < 64 ? scale * p.scale_log2 * 4.f : scale;   // (a row's unit has 2^2 less)
        dst[2] = tid < 64 ? minimum * p.scale_log2 : fmaf(8.f, scale, minimum);
        if (tid < 64 && (key & 15) == 0) at_pos[s][key >> 4] = pos_now;
      }
      fence_proxy_async_smem();
      mbar_arrive(&v_full[s]);
    }
  } else if (warp == 8) {
    // (the whole warp goes through the waits, and one lane issues: what a product takes stays uniform)
    constexpr uint32_t idesc_s = make_umma_idesc_e4m3(kKv4TileRows, K);
    constexpr uint32_t idesc_o = make_umma_idesc_bf16(kKv4TileRows, HD) | (1u << 16);   // V: b_major = MN
    const uint64_t q_desc = make_umma_desc_k128(sQ), k_desc = make_umma_desc_k128(sK), v_desc = make_umma_desc_mn128(sV, kVHalf);
    auto scores = [&](int i) {
      if (!tile_wait_warp(&k_full[use(i)], parity(i), pp.timeout)) return false;
      tc_fence_after();
      const uint64_t kd = k_desc + (uint64_t)(use(i) * (kKTile >> 4));
      const uint32_t to = tmem + (uint32_t)use(i) * 64u;
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_e4m3_ss(to, q_desc + (h * kQHalf >> 4) + 2 * k, kd + 2 * k, idesc_s, (uint32_t)((h | k) != 0));   // (heads of 128: high parts, then low)
        umma_commit(&s_full[use(i)]);
      }
      __syncwarp();
      return true;
    };
    bool go = n > 0 && scores(0);
    for (int i = 0; i < n && go; ++i) {
      // the scores of chunk i + 1 go over the P that the product of chunk i - 1 reads
      if (i > 0 && !(go = tile_wait_warp(&pv_done[use(i - 1)], parity(i - 1), pp.timeout))) break;
      if (i + 1 < n && !(go = scores(i + 1))) break;
      if (!(go = tile_wait_warp(&v_full[use(i)], parity(i), pp.timeout) && tile_wait_warp(&p_full[use(i)], parity(i), pp.timeout))) break;
      tc_fence_after();
      const uint64_t vd = v_desc + (uint64_t)(use(i) * (kVTile >> 4));
      const uint32_t from = tmem + (uint32_t)use(i) * 64u;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < K / 16; ++k)   // 16 keys: 2048 B of V, 8 columns of P
          umma_bf16_ts(tmem_o, from + 8 * k, vd + 128 * k, idesc_o, (uint32_t)((i | k) != 0));
        umma_commit(&pv_done[use(i)]);
      }
      __syncwarp();
    }
  } else if (warp < 4 && (TWIN ? (warp & 1) * 32 : warp * 32) < half) {
    const int at = warp * 32 + lane, r = TWIN ? at & 63 : at;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const int lim = ctx + r / G + 1;   // first position this row does not see (rows behind the tile's: some, dropped)
    const float unit = row_units[at].x;
    const uint64_t sum2 = pack2(row_units[at].y, row_units[at].y);
    for (int i = 0; i < n && ok; ++i) {
      const uint32_t sp = tmem + lanes + (uint32_t)use(i) * 64u;
      if (!(ok = tile_wait_warp(&v_full[use(i)], parity(i), pp.timeout) && tile_wait_warp(&s_full[use(i)], parity(i), pp.timeout))) break;
      tc_fence_after();
#pragma unroll 1
      for (int h = TWIN ? warp >> 1 : 0; h < (TWIN ? (warp >> 1) + 1 : 2); ++h) {   // 32 keys
        const int2 pos2 = *reinterpret_cast<const int2*>(&at_pos[use(i)][2 * h]);
        const int pos[2] = {pos2.x, pos2.y};
        const bool whole = max(pos[0], pos[1]) + 16 <= seen_by_all;
        const ulonglong2 *kp = reinterpret_cast<const ulonglong2*>(key_pairs[use(i)]) + 16 * h, *vp = reinterpret_cast<const ulonglong2*>(value_pairs[use(i)]) + 16 * h;
        uint32_t u[32];
        tmem_ld_32x32b_x16(sp + 32 * h, u);
        tmem_ld_32x32b_x16(sp + 32 * h + 16, u + 16);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const ulonglong2 w = kp[c >> 1];
          float x, y;
          unpack2(fma2(pack2(__uint_as_float(u[c]), __uint_as_float(u[c + 1])), w.x, mul2(sum2, w.y)), &x, &y);
          u[c] = __float_as_uint(x);
          u[c + 1] = __float_as_uint(y);
        }
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (pos[c / 16] + c % 16 >= lim) u[c] = 0xff800000u;   // -inf
        }
        float top[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) top[c] = max3(__uint_as_float(u[c]), __uint_as_float(u[c + 4]), __uint_as_float(u[c + 8]));
#pragma unroll
        for (int c = 12; c < 28; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(u[c + e]), __uint_as_float(u[c + 4 + e]));
        const float mx = fmaxf(max3(max3(top[0], top[1], __uint_as_float(u[28])), max3(top[2], top[3], __uint_as_float(u[29])), __uint_as_float(u[30])), __uint_as_float(u[31])) * unit;
        const bool grow = mx > m + kPromptSlack;
        if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? exp2f(m - mx) : 1.f;   // (m = -inf: 0)
          if (grow) m = mx;
          l *= f;
          low *= f;
          if (i > 0) {
            if (!(ok = tile_wait_warp(&pv_done[use(i - 1)], parity(i - 1), pp.timeout))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(tmem_o + lanes + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st_32x32b_x16(tmem_o + lanes + c, o);
            }
          }
          if (!TWIN && h) {   // the weights of the 32 keys before (rounded twice then)
            uint32_t o[16];
            tmem_st_wait();
            tmem_ld_32x32b_x16(sp, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = pack_bf16x2(__uint_as_float(o[j] << 16) * f, __uint_as_float(o[j] & 0xffff0000u) * f);
            tmem_st_32x32b_x16(sp, o);
          }
        }
        const float ms = m == -INFINITY ? 0.f : m;
        if (whole) {
          const uint64_t off = pack2(-ms, -ms), unit2 = pack2(unit, unit);
          uint64_t sums = 0, lows = 0;
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const ulonglong2 w = vp[c >> 1];
            float x, y;
            unpack2(fma2(pack2(__uint_as_float(u[c]), __uint_as_float(u[c + 1])), unit2, off), &x, &y);
            const uint64_t e = pack2(ex2_ftz(x), ex2_ftz(y));
            sums = add2(sums, e);
            lows = fma2(e, w.y, lows);
            unpack2(mul2(e, w.x), &x, &y);
            u[c >> 1] = pack_bf16x2(x, y);
          }
          float x, y;
          unpack2(sums, &x, &y);
          l += x + y;
          unpack2(lows, &x, &y);
          low += x + y;
        } else {   // (a pair that a row does not see may be NaN: 0 x NaN)
          const float* w = value_pairs[use(i)] + 64 * h;
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float z[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const bool there = pos[c / 16] + c % 16 + e < lim;
              const float y = ex2_ftz(fmaf(__uint_as_float(u[c + e]), unit, -ms));
              l += y;
              if (there) low = fmaf(y, w[2 * c + 2 + e], low);
              z[e] = there ? y * w[2 * c + e] : 0.f;
            }
            u[c >> 1] = pack_bf16x2(z[0], z[1]);
          }
        }
        tmem_st_32x32b_x16(sp + 16 * h, u);
        if (TWIN) {
#pragma unroll
          for (int c = 0; c < 16; ++c) u[c] = 0;
          tmem_st_32x32b_x16(sp + 16 * (1 - h), u);
        }
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[use(i)]);
    }
    if (ok && n > 0) ok = tile_wait_warp(&pv_done[use(n - 1)], parity(n - 1), pp.timeout);
    tc_fence_after();
  }

  // ---- the sums of a row: [row][HD + 4] O | reference, sum over queries, keys and values (every product has read them) ----
  constexpr int LDO = HD + 4;
  float* joined = reinterpret_cast<float*>(smem);
  __syncthreads();
  if (warp < 4 && (TWIN ? (warp & 1) * 32 : warp * 32) < half) {
    const int r = warp * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const bool some = ok && n > 0;
#pragma unroll 1
    for (int c = 0; c < HD; c += 16) {
      uint32_t o[16];
      if (some) {
        tmem_ld_32x32b_x16(tmem_o + lanes + c, o);
        tmem_ld_wait();
      }
      float f[16];   // channels 0, 4, 1, 5, 2, 6, 3, 7 of eight
#pragma unroll
      for (int j = 0; j < 16; ++j) f[(j & 8) + ((j & 7) >> 1) + 4 * (j & 1)] = some ? __uint_as_float(o[j]) + low : 0.f;
#pragma unroll
      for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(joined + r * LDO + c + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
    }
    // a wait ran out: the row is NaN.  Without chunks (or keys) the row has no part in the sum.
    *reinterpret_cast<float2*>(joined + r * LDO + HD) = ok ? make_float2(m, l) : make_float2(0.f, __uint_as_float(kKv4Nan));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if constexpr (!SHARED) {
    if (warp == 8) tmem_dealloc(tmem, 256);   // (before the other blocks are waited for: they may wait for tensor memory)
    cluster.sync();
  }
  const bool whole_head = !SHARED || (turn == 0 && last_turn == turns);   // (else a part of it)
  constexpr int PER = HD / 4, SIDE = 32 / PER, W = kKv4TileThreads / 32;   // lanes of a row, rows side by side in a warp
  const int part_lane = lane % PER, parts = TWIN ? 2 * C : C;
  for (int base = (rank * W + warp) * SIDE; base < rows; base += C * W * SIDE) {
    const int row = min(base + lane / PER, rows - 1);
    // a part: a block's, or one of the two of a block
    auto part = [&](int x) { return (SHARED ? joined : cluster.map_shared_rank(joined, TWIN ? x >> 1 : x)) + (row + (TWIN ? (x & 1) * 64 : 0)) * LDO; };
    float2 ml = make_float2(-INFINITY, 0.f);
    if (part_lane < parts) ml = *reinterpret_cast<const float2*>(part(part_lane) + HD);
    float top = ml.x;
#pragma unroll
    for (int w = PER / 2; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    float f = top == -INFINITY ? 1.f : exp2f(ml.x - top), total = part_lane < parts ? ml.y * f : 0.f;   // (of this lane's part; no score, or NaN only: zeros and NaN add up)
#pragma unroll
    for (int w = PER / 2; w > 0; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
    if (whole_head) f *= total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;   // (a row that sees no key is zero, NaN stays)
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < parts; ++c) {
      const float4 x = *reinterpret_cast<const float4*>(part(c) + part_lane * 4);
      const float w = __shfl_sync(0xffffffffu, f, (lane & ~(PER - 1)) + c);
      acc.x += x.x * w; acc.y += x.y * w; acc.z += x.z * w; acc.w += x.w * w;
    }
    if (base + lane / PER >= rows) continue;
    if (!whole_head) {
      float* to = p.parts + ((size_t)(2 * blockIdx.x + (turn == 0)) * rows + row) * (HD + 4);
      *reinterpret_cast<float4*>(to + part_lane * 4) = acc;
      if (part_lane == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(top, total);
      continue;
    }
    *reinterpret_cast<uint2*>(p.out + ((size_t)(b * p.Q + tok0 + row / G) * p.heads + kvh * G + row % G) * HD + part_lane * 4) = make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
  }
  if constexpr (SHARED) {
    at += last_turn - turn;
    done += n;
    __syncthreads();   // (the sums are read: their memory is the queries' and stages' again)
  } else {
    cluster.sync();   // no block leaves while its part is read
    return;
  }
  }
  if (SHARED && warp == 8) tmem_dealloc(tmem_slot, 256);
}

}  // namespace ssdk
