// kv4_tiles.cuh — attention over a paged cache held in 4 bits (kv4.cuh) of more than sixteen query rows to a key head, on tcgen05.
//
// S = Q K^T of up to 128 rows (query tokens x the heads that share a key head) and 64 keys into TMEM, P = exp2(S scale - reference) one row per thread, O += P V with P out of TMEM: the usual two
// products in bf16, over what the codes stand for, bf16(scale x code + minimum), which load_kv4 gives too.  That rounding (half a step of bf16) is what lets a row take a score as it comes: with codes as
// operands each of them needs its key's scale and minimum, and each weight its value's, which is twice the work of a row and a read of shared memory for every two keys of it (8 x 7 rows over 16000
// 101 us then, 95 so; 512 rows over 8000 119 and 97).
// A query row is scaled by a power of two so that its largest lies in 2^-9 .. 2^-8 (exact but for what is below 2^-133 then): no sum with keys up to the largest number passes it, and scores are scaled back
// in fp32.  A word of eight channels' codes gives them in the
// order 0, 4, 1, 5, 2, 6, 3, 7: queries are stored in that order, outputs are put back.
// A pair that is not finite makes NaN of the rows that see its key and of no others: a NaN value counts as a NaN key, and is zero itself, since weights of zero meet it too.
// Four kinds of warps: one copies codes as the cache has them (bulk copies, up to three chunks on their way, their pages looked up a chunk ahead), four make them bf16, one issues the products, four have the
// rows.  A cluster of blocks shares the chunks of a key head; their sums meet in shared memory.  SHARED: as in kv4_attn_kernel.
// A row takes 32 keys at a time.  TWIN: up to 64 rows lie in the tile twice, rows 0 .. 63 take a chunk's first 32 keys and 64 .. 127 the others, each with zeros for weights of the other half and a reference
// of its own: all four warps work on half of the scores where two would on all, and the products are no more.
// Bound by instructions and by the hand-offs between the warps: 8 x 7 rows over 16000 (64 heads over 8 of 128) 85 us, where the bytes ask for 17, 66 without making bf16 of codes, 79 without the softmax, 64
// without either; 32 x 7 rows 271; 512 rows over 8000 (32 heads over 8 of 64) 97, 89, 71 and 64.  Two blocks to an SM hide each other's hand-offs (one with chunks of 128 keys: 109 where two had 104).  Loads
// by the warps that make bf16 cost more than the copies (95 and 91), one chunk of copies more than three (91 and 85), which fit because keys have one stage: they are written while the values' product runs.
#pragma once
#include <climits>

#include "kv4_attention.cuh"
#include "prompt_attention.cuh"

namespace ssdk {

constexpr int kKv4TileRows = 128, kKv4TileKeys = 64, kKv4TileThreads = 320, kKv4Producers = 128;   // warps: 4 of rows, 4 of values, one of products, one of copies
constexpr int kKv4Copies = 3;   // chunks on their way or there as the cache has them
constexpr int kv4_tile_body(int HD) { return kKv4TileRows * HD * 2 + 3 * kKv4TileKeys * HD * 2 + kKv4Copies * 2 * kKv4TileKeys * kv4_row_bytes(HD); }   // queries | keys | two stages of values | copies
constexpr int kv4_tile_smem(int HD) {
  const int join = kKv4TileRows * (HD + 4) * 4, body = kv4_tile_body(HD);
  return (body > join ? body : join) + 1024;
}

SSDK_DEVINL uint4 kv4_value8(uint32_t w, uint32_t scale, uint32_t low) {
  return make_uint4(kv4_value<0>(w, scale, low), kv4_value<1>(w, scale, low), kv4_value<2>(w, scale, low), kv4_value<3>(w, scale, low));
}
// A scale that rounding has brought so high that code 15 passes the largest number of bf16 goes one step back (values are of finite rows, so that is below their largest then).
SSDK_DEVINL uint32_t kv4_in_range(uint32_t pair) { return fmaf(15.f, __uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u)) >= 0x1.ffp127f ? pair - 1 : pair; }
SSDK_DEVINL bool kv4_finite(uint32_t pair) { return (pair & 0x7f80u) != 0x7f80u && (pair & 0x7f800000u) != 0x7f800000u; }
SSDK_DEVINL void bulk_copy(void* smem_dst, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)), "l"(from), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// of a warp: what its threads did before is there for whoever waits
SSDK_DEVINL void mbar_arrive_warp(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
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
  constexpr int kQHalf = kKv4TileRows * 128, kHalf = K * 128, kTile = HALVES * kHalf, kCopy = 2 * K * kv4_row_bytes(HD);   // 64 channels of the queries, of the keys or values of a chunk; all of them
  const Kv4AttnParams& p = pp.a;
  extern __shared__ uint8_t kv4_tile_raw[];
  __shared__ __align__(8) uint64_t k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2], codes_full[kKv4Copies], codes_free[kKv4Copies];
  __shared__ int codes_pos[kKv4Copies][4];                 // where a chunk's four sixteens of keys that were copied are in their context: behind every one where they have no page
  __shared__ __align__(16) int at_pos[2][4];   // position of a chunk's sixteen keys, behind every context where they have no page
  __shared__ int first_large;                  // the first chunk of this piece with large values (kKv4Above), of those that have been made bf16
  __shared__ float row_units[kKv4TileRows];   // of a row of queries: what a unit of its scores is (NaN: it is not finite)
  __shared__ uint32_t tmem_slot;
  uint8_t* smem = kv4_tile_raw + ((1024u - (smem_u32(kv4_tile_raw) & 1023u)) & 1023u);
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + HALVES * kQHalf;
  uint8_t* sV = sK + kTile;
  uint8_t* sC = sV + 2 * kTile;   // codes of keys, of values, pairs of keys, of values
  cg::cluster_group cluster = cg::this_cluster();
  const int C = SHARED ? 1 : (int)cluster.num_blocks(), rank = SHARED ? 0 : (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int kvh = blockIdx.x / C, b = blockIdx.y;
  const int tile = SHARED ? 0 : (int)gridDim.z - 1 - (int)blockIdx.z;   // (the tiles that see most keys first)
  const int G = p.heads / p.kv_heads, tok0 = tile * pp.tokens, tq = min(pp.tokens, p.Q - tok0), rows = tq * G;
  const int half = (rows + 31) & ~31;                // rows of the warps that have some
  const int live = (TWIN ? 2 * half : half) / 32;    // warps that hand P over

  if (warp == 8) {
    if (lane == 0) {
      for (int s = 0; s < 2; ++s) {
        mbar_init(&k_full[s], kKv4Producers / 32);
        mbar_init(&v_full[s], kKv4Producers / 32);
        mbar_init(&s_full[s], 1);
        mbar_init(&p_full[s], live);
        mbar_init(&pv_done[s], 1);
      }
      for (int s = 0; s < kKv4Copies; ++s) {
        mbar_init(&codes_full[s], 1);
        mbar_init(&codes_free[s], kKv4Producers / 32);
      }
      first_large = INT_MAX;
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(&tmem_slot, 256);
    tmem_relinquish();
  }
  pdl_wait();
  // SHARED: this block's turns at .. end, the first of them turn `turn` of its head
  int at = 0, end = 1, turn = 0, turns = 0, done = 0;   // done: chunks of the pieces before (of stages and barriers)
  bool lost = false;                                    // a wait ran out: all rows from there on are NaN
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
  const int n = SHARED ? lost ? 0 : max(0, min(chunks, last_turn) - turn) : front < chunks ? (chunks - front + C - 1) / C : 0;
  // Chunk i is on barriers use(i), its values and positions in that stage (keys have one), parity(i) is that use's.  A wait by parity is only right while the barrier is in that use or the one behind it:
  //   k_full, v_full: whoever waits for chunk i has to be through with it before the next but one comes: keys are written behind the scores of the chunk in front, values behind the product of the one before that,
  //     which needs every row's P.
  //   s_full: the producers and the rows ask for chunk i; chunk i + 2's needs chunk i + 1's keys, behind the former's wait, and through pv_done P of the latter.
  //   p_full: chunk i + 2's needs the rows to have seen its scores, which are issued behind the product of chunk i.
  //   pv_done: the scores of chunk i + 1 ask for chunk i - 1; the producers ask for chunk i - 2 before they write chunk i's values; the rows ask for chunk i - 1, and chunk i + 1's product needs their P.
  //   codes_full, codes_free (kKv4Copies of either, in turn): the producers ask for chunk i, whose place is filled again only when they have freed it, and each use is freed once.
  auto use = [&](int i) { return (done + i) & 1; };
  auto parity = [&](int i) { return (uint32_t)((done + i) >> 1) & 1u; };
  float l = 0.f, m = -INFINITY;
  bool ok = !lost;

  if (warp < 4 || warp == 8) {
    // Queries: HD / 8 lanes a row, eight channels each; rows behind the last one are zero.
    constexpr int LPR = HD / 8, PIECES = (TWIN ? 64 : kKv4TileRows) * LPR, T = 160, LOADS = (PIECES + T - 1) / T, BATCH = SHARED && LOADS > 7 ? 7 : LOADS;
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
        float f[8], top = 0.f;
        unpack_bf16x8(q_now[x], f);
        bool fine = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          fine = fine && fabsf(f[j]) < INFINITY;
          top = fmaxf(top, fabsf(f[j]));
        }
        const uint32_t all = __ballot_sync(0xffffffffu, fine) >> (lane & ~(LPR - 1)) & ((1u << LPR) - 1);
#pragma unroll
        for (int w = 1; w < LPR; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const int e = min(max((int)(__float_as_uint(top) >> 23), 9), 244);   // (biased exponent)
        const float up = copysignf(__uint_as_float((uint32_t)(245 - e) << 23), p.scale_log2), unit = __uint_as_float((uint32_t)e << 23) * fabsf(p.scale_log2) * 512.f;   // 2^(-9 - (e - 127)) with the scale's sign
        const uint4 to = make_uint4(pack_bf16x2(f[0] * up, f[4] * up), pack_bf16x2(f[1] * up, f[5] * up), pack_bf16x2(f[2] * up, f[6] * up), pack_bf16x2(f[3] * up, f[7] * up));
#pragma unroll
        for (int at_row = r; at_row < kKv4TileRows; at_row += TWIN ? 64 : kKv4TileRows) {
          *reinterpret_cast<uint4*>(sQ + (c >> 3) * kQHalf + swizzled(at_row, c & 7)) = to;
          if (c == 0) row_units[at_row] = all == (1u << LPR) - 1 ? unit : __uint_as_float(kKv4Nan);
        }
      }
    }
    fence_proxy_async_smem();
    asm volatile("bar.sync 1, %0;" ::"r"(T) : "memory");   // (of these warps: codes are on their way meanwhile)
  }
  if (warp >= 4 && warp < 8) {
    // ---- keys and values in bf16: a thread has PER pieces of 32 channels of either ----
    constexpr int NP = HD / 32, PER = K * NP / kKv4Producers;   // (PER = 2: the second piece is 32 rows on)
    const int tid = threadIdx.x - 128, piece = tid % NP, row = tid / NP;   // (neighbours are next to one another in the cache)
    // Where a piece's four words (16 bytes of bf16 each) go in a stage.  Heads of 128: of eight lanes, two rows of four pieces, the upper two begin with their third word, so that all go to banks of their own.
    const bool later = HD == 128 && piece >= 2;
    int to[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) to[j] = (piece >> 1) * kHalf + swizzled(row, (piece & 1) * 4 + (later ? j ^ 2 : j));
    auto write = [&](uint8_t* stage, const uint4& codes, uint32_t pair) {
      const uint32_t scale = kv4_scales(pair), low = kv4_lows(pair);
      const uint32_t w[4] = {later ? codes.z : codes.x, later ? codes.w : codes.y, later ? codes.x : codes.z, later ? codes.y : codes.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stage + to[j]) = kv4_value8(w[j], scale, low);
    };
    for (int i = 0; i < n; ++i) {
      const int s = use(i), c = (done + i) % kKv4Copies;
      if (!tile_wait_warp(&codes_full[c], (uint32_t)((done + i) / kKv4Copies) & 1u, pp.timeout)) break;
      const uint8_t* from = sC + c * kCopy;
      uint4 kc[PER], vc[PER];
      uint32_t k_pair[PER], v_pair[PER];
      int pos[PER];
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int key = row + 32 * u;
        kc[u] = *reinterpret_cast<const uint4*>(from + key * CODES + piece * 16);
        vc[u] = *reinterpret_cast<const uint4*>(from + (K + key) * CODES + piece * 16);
        k_pair[u] = *reinterpret_cast<const uint32_t*>(from + 2 * K * CODES + key * 4);
        v_pair[u] = *reinterpret_cast<const uint32_t*>(from + 2 * K * CODES + (K + key) * 4);
        pos[u] = codes_pos[c][key >> 4];
      }
      mbar_arrive_warp(&codes_free[c]);
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        if (pos[u] + (row & 15) >= len) k_pair[u] = v_pair[u] = 0;   // (behind the context they may be anything; without a page they are left from before)
        k_pair[u] = kv4_in_range(k_pair[u]);
        if (!kv4_finite(v_pair[u])) {
          k_pair[u] = 0x7fc07fc0u;
          v_pair[u] = 0;
        }
        if (kv4_large(v_pair[u])) atomicMin(&first_large, done + i);
      }
      if (done + i >= 1 && !tile_wait_warp(&s_full[use(i - 1)], parity(i - 1), pp.timeout)) break;   // the scores of chunk i - 1 have read their keys
#pragma unroll
      for (int u = 0; u < PER; ++u) write(sK + u * 32 * 128, kc[u], k_pair[u]);
      fence_proxy_async_smem();
      mbar_arrive_warp(&k_full[s]);
      if (done + i >= 2 && !tile_wait_warp(&pv_done[s], parity(i - 2), pp.timeout)) break;   // its product has read its values, its rows their positions
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        write(sV + s * kTile + u * 32 * 128, vc[u], kv4_in_range(v_pair[u]));
        if (piece == 0 && (row & 15) == 0) at_pos[s][(row + 32 * u) >> 4] = pos[u];
      }
      fence_proxy_async_smem();
      mbar_arrive_warp(&v_full[s]);
    }
  } else if (warp == 9) {
    // ---- copies of a chunk, as soon as the one before has been taken to registers: four lanes have sixteen keys each, whose pages they look up a chunk ahead ----
    const int record = p.block_size * kv4_row_bytes(HD), pairs = p.block_size * CODES;   // (bytes of a page and head, of its codes)
    const int64_t page_step = (int64_t)p.kv_heads * record, head = (int64_t)kvh * record;
    const int32_t* table = p.tables + (size_t)b * p.max_blocks;
    const int step = C * K, step_x = step / p.block_size, step_off = step - step_x * p.block_size;
    int pos = front * K + (lane & 3) * 16, x = pos / p.block_size, off = pos - x * p.block_size;   // (positions stay below 2^31: the host sees to it)
    int page = lane < 4 && pos < seen ? table[x] : -1, i = 0;
    for (; i < n; ++i) {
      const int c = (done + i) % kKv4Copies;
      if (done + i >= kKv4Copies && !tile_wait_warp(&codes_free[c], (uint32_t)((done + i) / kKv4Copies - 1) & 1u, pp.timeout)) break;
      const bool is = page >= 0 && page < p.num_blocks;
      const int64_t from = page * page_step + head, codes = from + off * CODES, two = from + pairs + off * 4;
      if (lane < 4) codes_pos[c][lane] = is ? pos : kNoPosition;
      const int count = __popc(__ballot_sync(0xffffffffu, is));
      __syncwarp();   // (all four positions are there before lane 0 arrives for them: a vote orders no memory)
      if (lane == 0) mbar_arrive_expect_tx(&codes_full[c], (uint32_t)(count * 32 * kv4_row_bytes(HD)));
      __syncwarp();
      if (is) {
        uint8_t* to = sC + c * kCopy + lane * 16 * CODES;
        bulk_copy(to, p.k_cache + codes, 16 * CODES, &codes_full[c]);
        bulk_copy(to + K * CODES, p.v_cache + codes, 16 * CODES, &codes_full[c]);
        to = sC + c * kCopy + 2 * K * CODES + lane * 64;
        bulk_copy(to, p.k_cache + two, 64, &codes_full[c]);
        bulk_copy(to + K * 4, p.v_cache + two, 64, &codes_full[c]);
      }
      pos += step;
      x += step_x;
      off += step_off;
      if (off >= p.block_size) {
        off -= p.block_size;
        ++x;
      }
      page = lane < 4 && pos < seen ? table[x] : -1;
    }
    for (int x = max(0, i - kKv4Copies); x < i; ++x) tile_wait_warp(&codes_full[(done + x) % kKv4Copies], (uint32_t)((done + x) / kKv4Copies) & 1u, pp.timeout);   // (no copy is on its way when the block ends)
  } else if (warp == 8) {
    // (the whole warp goes through the waits, and one lane issues: what a product takes stays uniform)
    constexpr uint32_t idesc_s = make_umma_idesc_bf16(kKv4TileRows, K);
    constexpr uint32_t idesc_o = make_umma_idesc_bf16(kKv4TileRows, HD) | (1u << 16);   // V: b_major = MN
    const uint64_t q_desc = make_umma_desc_k128(sQ), k_desc = make_umma_desc_k128(sK), v_desc = make_umma_desc_mn128(sV, kHalf);
    auto scores = [&](int i) {
      if (!tile_wait_warp(&k_full[use(i)], parity(i), pp.timeout)) return false;
      tc_fence_after();
      const uint32_t to = tmem + (uint32_t)use(i) * 64u;
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16_ss(to, q_desc + (h * kQHalf >> 4) + 2 * k, k_desc + (h * kHalf >> 4) + 2 * k, idesc_s, (uint32_t)((h | k) != 0));
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
      const uint64_t vd = v_desc + (uint64_t)(use(i) * (kTile >> 4));
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
    const float unit = row_units[at];
    for (int i = 0; i < n && ok; ++i) {
      const uint32_t sp = tmem + lanes + (uint32_t)use(i) * 64u;
      if (!(ok = tile_wait_warp(&v_full[use(i)], parity(i), pp.timeout))) break;
      const float above = *(volatile int*)&first_large <= done + i ? kKv4Above : 0.f;
      if (!(ok = tile_wait_warp(&s_full[use(i)], parity(i), pp.timeout))) break;
      tc_fence_after();
#pragma unroll 1
      for (int h = TWIN ? warp >> 1 : 0; h < (TWIN ? (warp >> 1) + 1 : 2); ++h) {   // 32 keys
        const int2 pos2 = *reinterpret_cast<const int2*>(&at_pos[use(i)][2 * h]);
        const int pos[2] = {pos2.x, pos2.y};
        const bool whole = max(pos[0], pos[1]) + 16 <= seen_by_all;
        uint32_t u[32];
        tmem_ld_32x32b_x16(sp + 32 * h, u);
        tmem_ld_32x32b_x16(sp + 32 * h + 16, u + 16);
        tmem_ld_wait();
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
        const bool grow = mx > m + (kKv4Slack - above);
        if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? exp2f(m - (mx + above)) : 1.f;   // (m = -inf: 0)
          if (grow) m = mx + above;
          l *= f;
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
          uint64_t sums = 0;
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float x, y;
            unpack2(fma2(pack2(__uint_as_float(u[c]), __uint_as_float(u[c + 1])), unit2, off), &x, &y);
            x = ex2_ftz(x);
            y = ex2_ftz(y);
            sums = add2(sums, pack2(x, y));
            u[c >> 1] = pack_bf16x2(x, y);
          }
          float x, y;
          unpack2(sums, &x, &y);
          l += x + y;
        } else {   // (a score that a row does not see may be NaN, and 0 x -inf is)
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float z[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              z[e] = pos[c / 16] + c % 16 + e < lim ? ex2_ftz(fmaf(__uint_as_float(u[c + e]), unit, -ms)) : 0.f;
              l += z[e];
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
      mbar_arrive_warp(&p_full[use(i)]);
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
      for (int j = 0; j < 16; ++j) f[(j & 8) + ((j & 7) >> 1) + 4 * (j & 1)] = some ? __uint_as_float(o[j]) : 0.f;
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
    if (threadIdx.x == 0) first_large = INT_MAX;
    lost = __syncthreads_or(!ok) != 0;   // (and the sums are read: their memory is the queries' and stages' again)
  } else {
    cluster.sync();   // no block leaves while its part is read
    return;
  }
  }
  if (SHARED && warp == 8) tmem_dealloc(tmem_slot, 256);
}

}  // namespace ssdk
