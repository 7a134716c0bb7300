// span_tiles.cuh — span_attention of more than sixteen query rows to a key head, on tcgen05.
//
// As in prompt_attn_kernel's twin form: S = Q K^T of up to 64 rows and 64 keys into TMEM, P = exp2(S - m) one row per thread, O += P V with P out of TMEM.  The
// queries lie in rows 0 .. 63 and again in 64 .. 127: these make the low bf16 pieces of the weights (two pieces: see span_attn_kernel), add up in lanes of their own and are added at the
// end.  (With a row's keys shared by its two lanes, zeros in P at the other's keys and the two pieces in a product each, the exponentials halve and the
// products double: 37.0 us against 36.5 where this is 36.5, one warp issuing; tensor and shared memory are what two blocks share.)  Scores and products with V are issued
// by a warp each, with one commit a product: one thread that issued both and looked at five barriers a chunk held it at 2500 clocks a chunk (36.5 -> 33.4 us at the time).
// A chunk of 64 keys is gathered from the listed spans by TMA boxes of gcd(span, 64) keys, in list order; what is missing from the last
// chunk is loaded from behind the cache (zeros) and masked.  A cluster of blocks shares the chunks of a key head; their sums meet in shared memory.
// Up to sixteen rows span_attn_kernel is as fast as the memory; with more its mma.sync products bound it: 8 sequences of 7 rows, 64 heads over 8 of 128,
// 4096 listed keys each: 63 us on two m16 tiles a warp, 32.7 here (32 sequences: 99 us, 84 % of the copy rate).  Of these 33 a block takes 5 until its first scores are
// weights, some 22 for its 16 chunks and 6 to join.  Keys and values are asked for by a warp each, the moment that their stage is read: one thread for both, with a division a box,
// asked for a chunk's keys 1200 clocks late (33.5 us; 32 sequences 102; boxes of 16 keys, one sequence of 160 rows, 32 -> 27).  Two stages of both are what fits twice on an SM; heads of
// 64 have four (32 sequences 84.5 -> 82).
#pragma once
#include <cooperative_groups.h>

#include "prompt_attention.cuh"
#include "span_ops.cuh"

namespace ssdk {

constexpr int kTileRows64 = 64, kTileKeys = 64, kTileThreads = 256;   // warps: loads of keys, scores, 4 of softmax, products with V, loads of values
constexpr int kTileMost = 16;   // blocks of a cluster
constexpr int tile_stages(int HD) { return HD == 64 ? 4 : 2; }   // of keys and of values: as many as fit when two blocks share an SM
// query twice | keys and values; behind them the places of the listed spans
constexpr int span_tile_body(int HD) { return 2 * kTileRows64 * HD * 2 + tile_stages(HD) * 2 * kTileKeys * HD * 2; }
constexpr int span_tile_smem(int HD, int count) { return span_tile_body(HD) + 1024 + count * 8; }

template <int HD>
__global__ void __launch_bounds__(kTileThreads, 2)
span_tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ SpanAttnParams p,
                 const int box, const int q_tokens, unsigned* timeout) {
  namespace cg = cooperative_groups;
  constexpr int HALVES = HD / 64;                    // 64-column boxes of a row
  constexpr int STAGES = tile_stages(HD);
  constexpr int kQHalf = 2 * kTileRows64 * 128, kKHalf = kTileKeys * 128, kTile = HALVES * kKHalf;
  extern __shared__ uint8_t span_tile_raw[];
  __shared__ __align__(8) uint64_t q_full, k_full[STAGES], v_full[STAGES], k_free[STAGES], v_free[STAGES], s_full[2], p_full[2], pv_done[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int s_failed, s_odd, found[kTileThreads / 32];   // s_odd: values were taken out
  uint8_t* smem = span_tile_raw + ((1024u - (smem_u32(span_tile_raw) & 1023u)) & 1023u);
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + HALVES * kQHalf;
  uint8_t* sV = sK + STAGES * kTile;
  int2* where = reinterpret_cast<int2*>(smem + span_tile_body(HD));   // [count] slot and position of the first key of a span that is there
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x / C, b = blockIdx.y, tile = (int)gridDim.z - 1 - (int)blockIdx.z;
  const int G = p.heads / p.kv_heads, tok0 = tile * p.tokens, tq = min(p.tokens, p.Q - tok0), rows = tq * G;
  const int half = (rows + 31) & ~31;                // rows of the warps that have some
  const int live = 2 * half;                         // threads that hand P over

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    mbar_init(&q_full, 1);
    for (int s = 0; s < STAGES; ++s) { mbar_init(&k_full[s], 1); mbar_init(&v_full[s], 1); mbar_init(&k_free[s], 1); mbar_init(&v_free[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 1); mbar_init(&p_full[s], live); mbar_init(&pv_done[s], 1); }
    fence_mbar_init();
    s_failed = s_odd = 0;
  }
  if (warp == 1) { tmem_alloc(&tmem_slot, 256); tmem_relinquish(); }
  pdl_wait();
  // the spans that are there, in the list's order
  const int len = tokens_of(p.lens, b, p.max_blocks, p.block_size);
  int spans = 0;
  for (int base = 0; base < p.count; base += kTileThreads) {
    const int i = base + (int)threadIdx.x, s = i < p.count ? p.spans[((size_t)b * p.kv_heads + kvh) * p.count + i] : -1;
    int2 at = make_int2(-1, 0);
    if (s >= 0 && (long long)s * p.span < len) {
      at.y = s * p.span;
      const int page = page_at(p.tables + (size_t)b * p.max_blocks + at.y / p.block_size, p.num_blocks);
      if (page >= 0) at.x = page * p.block_size + at.y % p.block_size;
    }
    const uint32_t there = __ballot_sync(0xffffffffu, at.x >= 0);
    if (lane == 0) found[warp] = __popc(there);
    __syncthreads();
    if (base == 0 && threadIdx.x == 0) {   // the queries need no list
      mbar_arrive_expect_tx(&q_full, HALVES * 2 * 128 * G * q_tokens);
      for (int h = 0; h < HALVES; ++h)
        for (int x = 0; x < 2 * kTileRows64; x += kTileRows64) tma_load_3d(sQ + h * kQHalf + x * 128, &tmQ, &q_full, h * 64, kvh * G, b * p.Q + tok0);
    }
    int before = spans + __popc(there & ((1u << lane) - 1));
#pragma unroll
    for (int w = 0; w < kTileThreads / 32; ++w) {
      before += w < warp ? found[w] : 0;
      spans += found[w];
    }
    if (at.x >= 0) where[before] = at;
    __syncthreads();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot, tmem_o = tmem + 128;   // S / P buffers at columns 0 and 64, O behind them
  pdl_launch_dependents();   // (this block has its tensor memory: what is scheduled now may take the rest of the SM's and wait for this grid)

  const int per = p.span / box, boxes = kTileKeys / box, pieces = spans * per;   // boxes of a span, of a chunk, in all
  const int chunks = (pieces + boxes - 1) / boxes, share = (chunks + C - 1) / C;
  const int first = rank * share, n = max(0, min(share, chunks - first));
  // Chunk i's scores, weights and product on barrier i & 1, parity(i) is that use's; its keys and values in stage i % STAGES, turn(i).  A wait by parity is only right
  // while the barrier is in that use or the one behind it:
  //   k_full, v_full, p_full: whoever waits for chunk i has to be through with it before the stage, or P, is made anew.
  //   k_free, v_free (with two stages s_full and pv_done): the loads ask for chunk i - STAGES before they bring what the next use of that barrier needs.
  //   s_full: the softmax asks for chunk i, and scores of chunk i + 2 need its P (through pv_done of chunk i).
  //   pv_done: the scores of chunk i + 1 ask for chunk i - 1, the softmax of chunk i for chunk i - 1 or nothing, the end for
  //     chunk n - 1.  Chunk i + 1's product, the next on that barrier, needs the P of chunk i + 1, so its scores, so the first of them; and the P of a warp that
  //     has not gone on, so the second.
  auto parity = [](int i) { return (uint32_t)(i >> 1) & 1u; };
  auto turn = [](int i) { return (uint32_t)(i / STAGES) & 1u; };
  float l = 0.f, m = -INFINITY;
  bool ok = true;
  const int q4 = warp & 3, r = (q4 & 1) * 32 + lane;
  const bool softmax = warp >= 2 && warp < 6, second = q4 >= 2, in = softmax && (r & ~31) < half;   // (whole warps) second: the same row as two warps before, its low pieces
  const uint32_t lanes = (uint32_t)(q4 * 32) << 16;

  if (warp == 0 || warp == 7) {
    if (lane == 0) {
      const CUtensorMap* tm = warp ? &tmV : &tmK;
      uint8_t* ring = warp ? sV : sK;
      uint64_t *full = warp ? v_full : k_full, *free = STAGES == 2 ? (warp ? pv_done : s_full) : (warp ? v_free : k_free);
      int i = 0, at_i = first * boxes / per, at_r = first * boxes - at_i * per;
      for (; i < n; ++i) {
        const int s = i % STAGES;
        int slots[4];   // of the chunk's boxes, behind the last one no keys
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          slots[j] = at_i < spans ? where[at_i].x + at_r * box : (int)(p.num_blocks * p.block_size);
          if (j < boxes && ++at_r == per) {
            at_r = 0;
            ++at_i;
          }
        }
        if (i >= STAGES && !tile_wait(&free[s], turn(i - STAGES), timeout)) break;   // chunk i - STAGES has been read
        mbar_arrive_expect_tx(&full[s], kTile);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < boxes)
            for (int h = 0; h < HALVES; ++h) tma_load_3d(ring + s * kTile + h * kKHalf + j * box * 128, tm, &full[s], h * 64, kvh, slots[j]);
      }
      // nothing is in flight into this block's memory when it leaves, also after a wait ran out
      if (warp == 0) tile_wait(&q_full, 0, timeout);
      for (int j = max(0, i - STAGES); j < i; ++j) tile_wait(&full[j % STAGES], turn(j), timeout);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_umma_idesc_bf16(2 * kTileRows64, kTileKeys);
      bool go = n > 0 && tile_wait(&q_full, 0, timeout);
      for (int i = 0; i < n && go; ++i) {
        // the scores of chunk i go over the P that the product of chunk i - 2 reads
        if (i > 1 && !(go = tile_wait(&pv_done[i & 1], parity(i - 2), timeout))) break;
        if (!(go = tile_wait(&k_full[i % STAGES], turn(i), timeout))) break;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const uint64_t qd = make_umma_desc_k128(sQ + h * kQHalf), kd = make_umma_desc_k128(sK + i % STAGES * kTile + h * kKHalf);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16_ss(tmem + (i & 1) * 64, qd + 2 * k, kd + 2 * k, idesc_s, (uint32_t)((h | k) != 0));
        }
        umma_commit(&s_full[i & 1]);
        if (STAGES > 2) umma_commit(&k_free[i % STAGES]);
      }
    }
    __syncwarp();
  } else if (warp == 6) {
    if (lane == 0) {
      constexpr uint32_t idesc_o = make_umma_idesc_bf16(2 * kTileRows64, HD) | (1u << 16);   // V: b_major = MN
      bool go = true;
      for (int i = 0; i < n && go; ++i) {
        if (!(go = tile_wait(&v_full[i % STAGES], turn(i), timeout) && tile_wait(&p_full[i & 1], parity(i), timeout))) break;
        tc_fence_after();
        const uint64_t vd = make_umma_desc_mn128(sV + i % STAGES * kTile, kKHalf);
#pragma unroll
        for (int k = 0; k < kTileKeys / 16; ++k)   // 16 keys: 2048 B of V, 8 columns of P
          umma_bf16_ts(tmem_o, tmem + (i & 1) * 64 + 8 * k, vd + 128 * k, idesc_o, (uint32_t)((i | k) != 0));
        umma_commit(&pv_done[i & 1]);
        if (STAGES > 2) umma_commit(&v_free[i % STAGES]);
      }
    }
    __syncwarp();
  } else {
    const int lim = len - p.Q + tok0 + r / G + 1;        // first position this row does not see (rows behind the tile's: some, dropped)
    const int seen_by_all = len - p.Q + tok0 + 1;        // positions below it are seen by every row
    ok = in;
    // the lane's box of a chunk, of the spans and of the boxes of a span (advancing by a chunk's boxes without a division)
    const int step_i = boxes / per, step_r = boxes - step_i * per;
    int at_i = (first * boxes + lane) / per, at_r = first * boxes + lane - at_i * per;
    for (int i = 0; i < n && in; ++i) {
      const uint32_t sp = tmem + lanes + (uint32_t)(i & 1) * 64u;
      // positions of the chunk's keys: a lane has a box's, sixteen keys' are taken from there where some row does not see all
      const int mine = lane < boxes ? (at_i < spans ? where[at_i].y + at_r * box : kNoPosition) : 0;
      at_i += step_i;
      at_r += step_r;
      if (at_r >= per) {
        at_r -= per;
        ++at_i;
      }
      const bool whole = __all_sync(0xffffffffu, lane >= boxes || mine + box <= seen_by_all);
      if (!(ok = tile_wait_warp(&s_full[i & 1], parity(i), timeout))) break;
      tc_fence_after();
      uint32_t u[64];
#pragma unroll
      for (int c = 0; c < 64; c += 16) tmem_ld_32x32b_x16(sp + c, u + c);
      tmem_ld_wait();
      if (p.zero_scale) {   // (NaN where a score is not finite)
#pragma unroll
        for (int c = 0; c < 64; ++c) u[c] = __float_as_uint(__uint_as_float(u[c]) * 0.f);
      } else if (p.q_sign) {
#pragma unroll
        for (int c = 0; c < 64; ++c) u[c] ^= 0x80000000u;
      }
      int pos[4];   // of sixteen keys each
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int x = 16 * j / box;
          pos[j] = __shfl_sync(0xffffffffu, mine, x) + (16 * j - x * box);
        }
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (pos[c / 16] + c % 16 >= lim) u[c] = 0xff800000u;   // -inf
      }
      const float mx = row_max(u) * p.scale_log2;
      const bool grow = mx > m + kPromptSlack;
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? exp2f(m - mx) : 1.f;   // (m = -inf: 0)
        if (grow) m = mx;
        l *= f;
        if (i > 0) {
          if (!(ok = tile_wait_warp(&pv_done[(i - 1) & 1], parity(i - 1), timeout))) break;
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
      }
      const float ms = m == -INFINITY ? 0.f : m;
      l += second ? row_exp<false, true>(u, p.scale_log2, ms) : row_exp<true, false>(u, p.scale_log2, ms);
      tmem_st_32x32b_x16(sp, u);
      tmem_st_32x32b_x16(sp + 16, u + 16);
      tmem_st_wait();
      if (!whole) {   // slots behind the context hold anything, new tokens values that are not finite: 0 x NaN is NaN
        const int edge = min(seen_by_all, len);
        bool stale = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) stale = stale || (pos[j] < kNoPosition && pos[j] + 16 > edge);
        if (stale) {   // (the same for all warps)
          if (!(ok = tile_wait_warp(&v_full[i % STAGES], turn(i), timeout))) break;
          bool odd = false;
          for (int j = second ? half + r : r; j < kTileKeys * 8; j += live) {
            const int key = j >> 3, x = key >> 4, at = (x == 0 ? pos[0] : x == 1 ? pos[1] : x == 2 ? pos[2] : pos[3]) + (key & 15);
            if (at >= edge)
#pragma unroll
              for (int h = 0; h < HALVES; ++h) {
                uint4* v = reinterpret_cast<uint4*>(sV + i % STAGES * kTile + h * kKHalf + j * 16);
                if (at >= len) *v = make_uint4(0u, 0u, 0u, 0u);
                else odd |= take_out(v);
              }
          }
          if (odd) s_odd = 1;
          fence_proxy_async_smem();
        }
      }
      tc_fence_before();
      mbar_arrive(&p_full[i & 1]);
    }
    if (ok && n > 0) ok = tile_wait_warp(&pv_done[(n - 1) & 1], parity(n - 1), timeout);
    tc_fence_after();
  }

  // ---- the sums of a row: low pieces to the row's warp, then [row][HD + 4] O | reference, sum over queries, keys and values (every product has read them) ----
  constexpr int LDO = HD + 4;
  float* joined = reinterpret_cast<float*>(smem);
  auto sums = [&](int c, uint32_t* o) {   // 32 columns
    tmem_ld_32x32b_x16(tmem_o + lanes + c, o);
    tmem_ld_32x32b_x16(tmem_o + lanes + c + 16, o + 16);
    tmem_ld_wait();
  };
  __syncthreads();   // nothing is on its way into them
  if (softmax && in && second) {
    if (!ok) s_failed = 1;
    if (ok && n > 0)
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        sums(c, o);
#pragma unroll
        for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4*>(joined + r * LDO + c + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
      }
  }
  __syncthreads();
  if (softmax && in && !second) {
    const bool good = ok && !s_failed, some = good && n > 0;
#pragma unroll 1
    for (int c = 0; c < HD; c += 32) {
      uint32_t o[32];
      if (some) sums(c, o);
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        float4* at = reinterpret_cast<float4*>(joined + r * LDO + c + j);
        const float4 x = *at;
        *at = some ? make_float4(__uint_as_float(o[j]) + x.x, __uint_as_float(o[j + 1]) + x.y, __uint_as_float(o[j + 2]) + x.z, __uint_as_float(o[j + 3]) + x.w)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    // a wait ran out: the row is NaN.  Without chunks (or keys) the row has no part in the sum.  The sum's sign: s_odd.
    *reinterpret_cast<float2*>(joined + r * LDO + HD) = good ? make_float2(m, s_odd ? -l : l) : make_float2(0.f, __int_as_float(0x7fffffff));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 256);   // (before the other blocks are waited for: they may wait for tensor memory)
  cluster.sync();
  constexpr int PER = HD / 4, SIDE = 32 / PER;   // lanes of a row, rows side by side in a warp
  const int part_lane = lane % PER;
  for (int base = (rank * (kTileThreads / 32) + warp) * SIDE; base < rows; base += C * (kTileThreads / 32) * SIDE) {
    const int row = min(base + lane / PER, rows - 1);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (part_lane < C) ml = *reinterpret_cast<const float2*>(cluster.map_shared_rank(joined, part_lane) + row * LDO + HD);
    const bool odd = __any_sync(0xffffffffu, __float_as_int(ml.y) < 0);
    ml.y = fabsf(ml.y);
    float top = ml.x;
#pragma unroll
    for (int w = PER / 2; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    float f = top == -INFINITY ? 0.f : exp2f(ml.x - top), sum = part_lane < C ? ml.y * f : 0.f;   // (of this lane's block)
#pragma unroll
    for (int w = PER / 2; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    f *= sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // (NaN stays)
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < C; ++c) {
      const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(joined, c) + row * LDO + part_lane * 4);
      const float g = __shfl_sync(0xffffffffu, f, (lane & ~(PER - 1)) + c);
      acc.x += x.x * g; acc.y += x.y * g; acc.z += x.z * g; acc.w += x.w * g;
    }
    if (base + lane / PER < rows) {
      add_taken_out(p, HD, b, kvh, len - p.Q + tok0 + 1, len - p.Q + tok0 + row / G + 1, part_lane * 4, odd, sum, &acc);
      __nv_bfloat16* dst = p.out + ((size_t)(b * p.Q + tok0 + row / G) * p.heads + kvh * G + row % G) * HD + part_lane * 4;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
    }
  }
  cluster.sync();   // no block leaves while its part is read
}

}  // namespace ssdk
