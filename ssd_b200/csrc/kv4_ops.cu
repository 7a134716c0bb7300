// kv4_ops.cu — entry points (include/ssdk.h) of the paged cache held in 4 bits: kv4.cuh, kv4_attention.cuh, kv4_tiles.cuh.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/ssdk.h"
#include "kv4_attention.cuh"
#include "kv4_tiles.cuh"
#include "op_host.cuh"

using namespace ssdk;
typedef __nv_bfloat16 bf16;

constexpr int kSms = 148;

// a cache of pages whose slots are numbered in 32 bits
static int check_kv4(const char* who, int64_t num_blocks, int block_size, int kv_heads, int head_dim) {
  if (head_dim != 64 && head_dim != 128) return fail("%s: heads of %d (64 or 128)", who, head_dim);
  if (kv_heads < 1 || kv_heads > 65535 || num_blocks < 1 || block_size < 16 || block_size % 16 || block_size > 65536)
    return fail("%s: %lld pages of %d tokens (a multiple of 16, at most 65536), %d key heads", who, (long long)num_blocks, block_size, kv_heads);
  if (num_blocks >= (1ll << 31) / block_size) return fail("%s: a cache of %lld pages of %d tokens passes 32 bits", who, (long long)num_blocks, block_size);
  return 0;
}
static int64_t kv4_bytes(int64_t num_blocks, int block_size, int kv_heads, int head_dim) { return num_blocks * block_size * kv_heads * kv4_row_bytes(head_dim); }

template <int HD, bool ROPE, bool VALUES>
static int launch_store(Launcher& L, Kv4StoreParams p) {
  constexpr int SIDE = kv4_store_heads(HD), W = kKv4StoreThreads / 32;
  p.groups = ((ROPE ? p.heads : 0) + 2 * p.kv_heads + SIDE - 1) / SIDE;
  const int64_t units = (int64_t)p.M * p.groups;
  if (units >= (1ll << 31)) return fail("%s: %d rows of %d heads", ROPE ? "rope_store_kv4" : "store_kv4", p.M, p.heads + 2 * p.kv_heads);
  p.warps = (int)std::min<int64_t>(units, kSms * kv4_store_blocks(ROPE) * W);
  p.each = (int)(units / p.warps);
  p.longer = (int)(units - (int64_t)p.each * p.warps);
  return L.go(kv4_store_kernel<HD, ROPE, VALUES>, dim3((unsigned)((p.warps + W - 1) / W)), dim3(kKv4StoreThreads), 0, p);
}
template <bool ROPE>
static int store(const Kv4StoreParams& p, int head_dim, void* stream) {
  Launcher L = launcher(stream);
  if (head_dim == 64) return p.k_values ? launch_store<64, ROPE, true>(L, p) : launch_store<64, ROPE, false>(L, p);
  return p.k_values ? launch_store<128, ROPE, true>(L, p) : launch_store<128, ROPE, false>(L, p);
}

// How a call's keys are shared.  Costs are in keys of a block: a block's start and end as long as some 512, the join of a cluster grows with its blocks; the longest context that the tables have room for.
struct Kv4Plan {
  int cluster, blocks;   // blocks: of a shared launch, 0 where clusters do
};
static Kv4Plan kv4_plan(int64_t units, int64_t keys, int resident, int most, int turn, int64_t share_from, bool may_share) {
  Kv4Plan plan = {1, 0};
  const int64_t slots = resident * kSms;
  int64_t least = INT64_MAX;
  for (int c = 1; c <= (units > 8 ? std::min(most, 8) : most); c *= 2) {   // (more than eight clusters of sixteen, which wait for one another's places: us with them and without, 4 contexts of 4000 17.1 and 9.8, 2 with 56 rows 32.6 and 20.5)
    const int64_t cost = (units * c + slots - 1) / slots * (512 + 16 * c + keys / c);
    if (cost < least) {
      least = cost;
      plan.cluster = c;
    }
  }
  // Equal stretches cost a second launch, but their time goes by the sum of all lengths, not by the longest, and more than the blocks of a cluster can share a head: they are taken where the clusters' cost
  // passes share_from.  With a head or more to every place on the device blocks are dealt out as others end.  us, clusters and stretches, of the streaming kernel: one context of 8000 (8 heads) 10.5
  // and 11.9, of 16000 14.7 and 15.1, of 32000 22.9 and 19.3, of 64000 40 and 26.8, 8 of 8000 23 and 26, 16 of 8000 37 and 35, 48 of 16000 131 and 128, 148 of 4000 95 and 113; of 56 rows on tiles: one context of 8000 25.9 and
  // 27.5, of 16000 36.5 and 32.8, of 32000 59 and 42, 4 of 16000 56 and 61, 8 of 4000 33 and 38, 8 of 16000 99 and 85, 16 of 4000 53 and 56, 16 of 16000 181 and 146, 32 of 16000 347 and 270.
  // (What counts is the table's room, since lengths are on the device: short contexts in tables made for long ones take the second launch for nothing, one of 500 5.4 and, in a table of 64000, 7.5; 8 x 7 rows of 500 14 and 24.)
  if (may_share && least > share_from && units < slots && units * ((keys + turn - 1) / turn) < (1ll << 31)) plan.blocks = (int)std::min(std::min(slots, units * 64), units * ((keys + turn - 1) / turn));
  return plan;
}
constexpr int kKv4Warps = 4, kMaxShared = 1024;   // warps of a block; sequences of a shared launch (each block goes through their lengths)
static Kv4Plan kv4_few_plan(int batch, int q_len, int heads, int kv_heads, int64_t keys) {
  const int tiles = (heads / kv_heads * q_len + 7) / 8;
  return kv4_plan((int64_t)batch * kv_heads, keys, 16 / tiles / kKv4Warps, kKv4Most, kKv4Warps * kKv4Keys, 2048, batch <= kMaxShared);
}
// of tiles: up to 64 rows lie in one twice
static int kv4_tile_tokens(int q_len, int group, int* tiles) {
  const int most = (group * q_len <= 64 ? kKv4TileRows / 2 : kKv4TileRows) / group;
  *tiles = (q_len + most - 1) / most;
  return (q_len + *tiles - 1) / *tiles;
}
static Kv4Plan kv4_tile_plan(int batch, int q_len, int heads, int kv_heads, int head_dim, int64_t keys) {
  int tiles;
  kv4_tile_tokens(q_len, heads / kv_heads, &tiles);
  const int most = head_dim == 64 && heads / kv_heads * q_len <= 64 ? 8 : kKv4Most;   // (their join has a lane of HD / 4 for each part)
  const int64_t units = (int64_t)batch * kv_heads * tiles;
  return kv4_plan(units, keys, 2, most, kKv4TileKeys, 1100 + (int64_t)((double)units * keys / (2 * kSms)), tiles == 1 && batch <= kMaxShared);   // (a block's start and its two parts; its share)
}
template <int HD, int KEYS>
static int launch_join(Launcher& L, const Kv4AttnParams& p, int blocks) {
  const int rows = p.heads / p.kv_heads * p.Q;
  if (blocks > 8 * p.B * p.kv_heads) return L.go(kv4_join_kernel<HD, KEYS, true>, dim3(p.kv_heads, p.B, rows), dim3(kKv4JoinThreads), 0, p, blocks);
  return L.go(kv4_join_kernel<HD, KEYS, false>, dim3(p.kv_heads, p.B, (rows + kKv4JoinThreads / 32 - 1) / (kKv4JoinThreads / 32)), dim3(kKv4JoinThreads), 0, p, blocks);
}
template <int HD, int NT>
static int launch_attn(Launcher& L, const Kv4AttnParams& p) {
  constexpr int W = kKv4Warps, smem = kv4_attn_smem(HD, NT, W);
  const Kv4Plan plan = kv4_few_plan(p.B, p.Q, p.heads, p.kv_heads, (int64_t)p.max_blocks * p.block_size);
  if (plan.blocks) {
    static std::atomic<bool> done[64];
    CKI(with_smem(kv4_attn_kernel<HD, NT, W, true>, smem, kSmemCarveout, done));
    if (!p.parts) return fail("paged_attn_kv4: null argument (scratch)");
    CKI(L.go(kv4_attn_kernel<HD, NT, W, true>, dim3(plan.blocks), dim3(W * 32), smem, p));
    return launch_join<HD, W * kKv4Keys>(L, p, plan.blocks);
  }
  static std::atomic<bool> done[64];
  CKI(with_smem(kv4_attn_kernel<HD, NT, W, false>, smem, kSmemClusters, done));
  L.cluster = plan.cluster;
  return L.go(kv4_attn_kernel<HD, NT, W, false>, dim3(p.kv_heads * L.cluster, p.B), dim3(W * 32), smem, p);
}
template <int HD, bool TWIN>
static int launch_tiles(Launcher& L, const Kv4AttnParams& a) {
  WaitWord* waits = op_waits();
  if (!waits) return fail("paged_attn_kv4: pinned word for bounded waits not allocated");
  CKI(waits->check("an earlier call of attention without an engine left is not complete (NaN rows)"));
  Kv4TileParams p;
  int tiles;
  p.a = a;
  p.tokens = kv4_tile_tokens(a.Q, a.heads / a.kv_heads, &tiles);
  p.timeout = waits->word;
  if (tiles > 65535) return fail("paged_attn_kv4: q_len=%d", a.Q);
  const Kv4Plan plan = kv4_tile_plan(a.B, a.Q, a.heads, a.kv_heads, HD, (int64_t)a.max_blocks * a.block_size);
  if (plan.blocks) {
    static std::atomic<bool> done[64];
    CKI(with_smem(kv4_tile_kernel<HD, TWIN, true>, kv4_tile_smem(HD), kSmemCarveout, done));
    if (!a.parts) return fail("paged_attn_kv4: null argument (scratch)");
    CKI(L.go(kv4_tile_kernel<HD, TWIN, true>, dim3(plan.blocks), dim3(kKv4TileThreads), kv4_tile_smem(HD), p));
    return launch_join<HD, kKv4TileKeys>(L, a, plan.blocks);
  }
  static std::atomic<bool> done[64];
  CKI(with_smem(kv4_tile_kernel<HD, TWIN, false>, kv4_tile_smem(HD), kSmemClusters, done));
  L.cluster = plan.cluster;
  return L.go(kv4_tile_kernel<HD, TWIN, false>, dim3(a.kv_heads * L.cluster, a.B, tiles), dim3(kKv4TileThreads), kv4_tile_smem(HD), p);
}

extern "C" {

int ssdk_rope_store_kv4(const void* qkv, const int64_t* positions, const int32_t* slot_mapping, const float* rope_table, int64_t max_pos,
                        int rot_dim, const void* q_norm_w, const void* k_norm_w, float norm_eps, void* q_out, void* k_cache, void* v_cache,
                        void* k_values, void* v_values, int64_t num_blocks, int block_size, int M, int heads, int kv_heads, int head_dim,
                        void* stream) {
  CKI(check_kv4("rope_store_kv4", num_blocks, block_size, kv_heads, head_dim));
  if (M < 1 || heads < 1 || heads > 65535) return fail("rope_store_kv4: %d rows of %d heads", M, heads);
  if (rot_dim < 16 || rot_dim % 16 || rot_dim > head_dim || max_pos < 1) return fail("rope_store_kv4: %d rotated channels of %d (a multiple of 16), %lld positions", rot_dim, head_dim, (long long)max_pos);
  if (!qkv || !positions || !slot_mapping || !rope_table || !q_out || !k_cache || !v_cache || !k_values != !v_values) return fail("rope_store_kv4: null argument");
  if (off16(qkv, q_out, k_cache, v_cache) || off16(q_norm_w, k_norm_w, rope_table) || off16(k_values, v_values)) return fail("rope_store_kv4: arrays must start at multiples of 16 bytes");
  const int64_t row = 2ll * M * head_dim, all = heads + 2 * (int64_t)kv_heads, cache = kv4_bytes(num_blocks, block_size, kv_heads, head_dim);
  // (of larger numbers of positions only as much counts as keeps the bytes in 64 bits)
  CKI(check_apart("rope_store_kv4", {{"q_out", q_out, row * heads}, {"k_cache", k_cache, cache}, {"v_cache", v_cache, cache}, {"k_values", k_values, row * kv_heads}, {"v_values", v_values, row * kv_heads}},
                  {{"qkv", qkv, row * all}, {"positions", positions, 8ll * M}, {"slot_mapping", slot_mapping, 4ll * M}, {"rope_table", rope_table, 4 * std::min<int64_t>(max_pos, 1ll << 40) * rot_dim},
                   {"q_norm_w", q_norm_w, 2ll * head_dim}, {"k_norm_w", k_norm_w, 2ll * head_dim}}));
  Kv4StoreParams p;
  memset(&p, 0, sizeof(p));
  p.q = (const bf16*)qkv; p.k = p.q + (int64_t)heads * head_dim; p.v = p.k + (int64_t)kv_heads * head_dim;
  p.q_row = p.k_row = p.v_row = all * head_dim;
  p.positions = positions; p.slots = slot_mapping; p.table = rope_table; p.top = max_pos; p.rot = rot_dim;
  p.q_norm_w = (const bf16*)q_norm_w; p.k_norm_w = (const bf16*)k_norm_w; p.eps = norm_eps;
  p.q_out = (bf16*)q_out; p.k_cache = (uint8_t*)k_cache; p.v_cache = (uint8_t*)v_cache; p.k_values = (bf16*)k_values; p.v_values = (bf16*)v_values;
  p.num_slots = num_blocks * block_size; p.block_size = block_size; p.M = M; p.heads = heads; p.kv_heads = kv_heads;
  return store<true>(p, head_dim, stream);
}

int ssdk_store_kv4(const void* k, const void* v, int64_t k_row, int64_t v_row, const int32_t* slot_mapping, void* k_cache, void* v_cache,
                   void* k_values, void* v_values, int64_t num_blocks, int block_size, int M, int kv_heads, int head_dim, void* stream) {
  CKI(check_kv4("store_kv4", num_blocks, block_size, kv_heads, head_dim));
  const int64_t n = (int64_t)kv_heads * head_dim, most = 1ll << 31;
  if (M < 1 || k_row < 0 || v_row < 0 || k_row % 8 || v_row % 8 || k_row >= most || v_row >= most) return fail("store_kv4: %d rows, %lld and %lld elements apart (multiples of 8)", M, (long long)k_row, (long long)v_row);
  if (!k || !v || !slot_mapping || !k_cache || !v_cache || !k_values != !v_values) return fail("store_kv4: null argument");
  if (off16(k, v, k_cache, v_cache) || off16(k_values, v_values)) return fail("store_kv4: arrays must start at multiples of 16 bytes");
  const int64_t values = 2ll * M * n, cache = kv4_bytes(num_blocks, block_size, kv_heads, head_dim);
  CKI(check_apart("store_kv4", {{"k_cache", k_cache, cache}, {"v_cache", v_cache, cache}, {"k_values", k_values, values}, {"v_values", v_values, values}},
                  {{"k", k, 2 * ((M - 1) * k_row + n)}, {"v", v, 2 * ((M - 1) * v_row + n)}, {"slot_mapping", slot_mapping, 4ll * M}}));
  Kv4StoreParams p;
  memset(&p, 0, sizeof(p));
  p.k = (const bf16*)k; p.v = (const bf16*)v; p.k_row = k_row; p.v_row = v_row; p.slots = slot_mapping;
  p.k_cache = (uint8_t*)k_cache; p.v_cache = (uint8_t*)v_cache; p.k_values = (bf16*)k_values; p.v_values = (bf16*)v_values;
  p.num_slots = num_blocks * block_size; p.block_size = block_size; p.M = M; p.kv_heads = kv_heads;
  return store<false>(p, head_dim, stream);
}

int ssdk_load_kv4(const void* k_cache, const void* v_cache, const int32_t* slot_mapping, void* k, void* v, int64_t num_blocks, int block_size,
                  int M, int kv_heads, int head_dim, void* stream) {
  CKI(check_kv4("load_kv4", num_blocks, block_size, kv_heads, head_dim));
  if (M < 1 || M > (1 << 30)) return fail("load_kv4: %d rows", M);
  if (!k_cache || !v_cache || !slot_mapping || !k || !v) return fail("load_kv4: null argument");
  if (off16(k_cache, v_cache, k, v)) return fail("load_kv4: arrays must start at multiples of 16 bytes");
  const int64_t rows = 2ll * M * kv_heads * head_dim, cache = kv4_bytes(num_blocks, block_size, kv_heads, head_dim);
  CKI(check_apart("load_kv4", {{"k", k, rows}, {"v", v, rows}}, {{"k_cache", k_cache, cache}, {"v_cache", v_cache, cache}, {"slot_mapping", slot_mapping, 4ll * M}}));
  Kv4LoadParams p;
  p.k_cache = (const uint8_t*)k_cache; p.v_cache = (const uint8_t*)v_cache; p.slots = slot_mapping; p.k = (bf16*)k; p.v = (bf16*)v;
  p.num_slots = num_blocks * block_size; p.M = M; p.kv_heads = kv_heads; p.block_size = block_size;
  Launcher L = launcher(stream);
  const int tile = kv4_load_tile(head_dim), W = kKv4LoadThreads / 32;
  const int64_t tiles = (int64_t)((M + tile - 1) / tile) * kv_heads;
  if (tiles >= (1ll << 31)) return fail("load_kv4: %d rows of %d heads", M, kv_heads);
  const dim3 grid((unsigned)std::min<int64_t>((tiles + W - 1) / W, kSms * 32)), block(kKv4LoadThreads);
  return head_dim == 64 ? L.go(kv4_load_kernel<64>, grid, block, 0, p) : L.go(kv4_load_kernel<128>, grid, block, 0, p);
}

int64_t ssdk_paged_attn_kv4_scratch_bytes(int batch, int q_len, int heads, int kv_heads, int head_dim, int block_size, int max_blocks_per_seq) {
  if (batch < 1 || q_len < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || heads / kv_heads > 32 || head_dim < 1 || block_size < 1 || max_blocks_per_seq < 1) return 0;
  const int64_t rows = (int64_t)(heads / kv_heads) * q_len;
  if (rows >= (1ll << 31) - 65536) return 0;
  const int64_t keys = (int64_t)max_blocks_per_seq * block_size;
  const Kv4Plan plan = rows <= 16 ? kv4_few_plan(batch, q_len, heads, kv_heads, keys) : kv4_tile_plan(batch, q_len, heads, kv_heads, head_dim, keys);
  return 8ll * plan.blocks * rows * (head_dim + 4);
}
int ssdk_paged_attn_kv4(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables, const int32_t* context_lens,
                        void* out, void* scratch, int batch, int q_len, int heads, int kv_heads, int head_dim, int block_size, int max_blocks_per_seq,
                        int64_t num_blocks, float scale, void* stream) {
  CKI(check_kv4("paged_attn_kv4", num_blocks, block_size, kv_heads, head_dim));
  CKI(check_pages("paged_attn_kv4", batch, block_size, max_blocks_per_seq, num_blocks));
  const float scale_log2 = scale * 1.4426950408889634f;
  if (q_len < 1 || heads < 1 || heads % kv_heads || heads / kv_heads > 32 || !std::isfinite(scale_log2))
    return fail("paged_attn_kv4: q_len=%d, %d heads over %d (at most 32 to a key head), scale %g (finite, log2(e) times it too)", q_len, heads, kv_heads, (double)scale);
  if ((int64_t)batch * q_len >= (1ll << 31) || (int64_t)q_len * (heads / kv_heads) >= (1ll << 31) - 65536) return fail("paged_attn_kv4: %d rows of %d sequences", q_len, batch);
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out) return fail("paged_attn_kv4: null argument");
  if (off16(q, k_cache, v_cache, out) || off16(scratch)) return fail("paged_attn_kv4: arrays must start at multiples of 16 bytes");
  const int64_t rows = 2ll * batch * q_len * heads * head_dim, cache = kv4_bytes(num_blocks, block_size, kv_heads, head_dim);
  CKI(check_apart("paged_attn_kv4", {{"out", out, rows}, {"scratch", scratch, ssdk_paged_attn_kv4_scratch_bytes(batch, q_len, heads, kv_heads, head_dim, block_size, max_blocks_per_seq)}},
                  {{"q", q, rows}, {"k_cache", k_cache, cache}, {"v_cache", v_cache, cache}, {"block_tables", block_tables, 4ll * batch * max_blocks_per_seq}, {"context_lens", context_lens, 4ll * batch}}));
  Kv4AttnParams p;
  p.q = (const bf16*)q; p.k_cache = (const uint8_t*)k_cache; p.v_cache = (const uint8_t*)v_cache; p.tables = block_tables; p.lens = context_lens; p.out = (bf16*)out;
  p.num_blocks = num_blocks; p.B = batch; p.Q = q_len; p.heads = heads; p.kv_heads = kv_heads; p.block_size = block_size; p.max_blocks = max_blocks_per_seq;
  p.scale_log2 = scale_log2; p.parts = (float*)scratch;
  Launcher L = launcher(stream);
  if ((int64_t)(heads / kv_heads) * q_len <= 8) return head_dim == 64 ? launch_attn<64, 1>(L, p) : launch_attn<128, 1>(L, p);
  if ((int64_t)(heads / kv_heads) * q_len <= 16) return head_dim == 64 ? launch_attn<64, 2>(L, p) : launch_attn<128, 2>(L, p);
  if ((int64_t)(heads / kv_heads) * q_len <= 64) return head_dim == 64 ? launch_tiles<64, true>(L, p) : launch_tiles<128, true>(L, p);
  return head_dim == 64 ? launch_tiles<64, false>(L, p) : launch_tiles<128, false>(L, p);
}

}  // extern "C"
