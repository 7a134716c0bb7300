// cache_ops.cu — entry points (include/ssdk.h) of the operators of cache_ops.cuh and span_ops.cuh.
#include <atomic>
#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <numeric>

#include "../../include/ssdk.h"
#include "cache_ops.cuh"
#include "host.cuh"
#include "span_ops.cuh"
#include "span_tiles.cuh"

using namespace ssdk;
typedef __nv_bfloat16 bf16;

static bool off16(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) != 0;
}
// An array of a call.  What is written lies apart from everything else: other blocks still read the inputs, or write the other outputs, while one writes.
struct Array {
  const char* name;
  const void* at;
  int64_t bytes;
};
static bool overlap(const Array& a, const Array& b) {
  return a.at && b.at && (uintptr_t)a.at < (uintptr_t)b.at + (uintptr_t)b.bytes && (uintptr_t)b.at < (uintptr_t)a.at + (uintptr_t)a.bytes;
}
static int check_apart(const char* who, std::initializer_list<Array> written, std::initializer_list<Array> read) {
  for (const Array* w = written.begin(); w != written.end(); ++w) {
    const Array* other = nullptr;
    for (const Array* x = w + 1; x != written.end(); ++x)
      if (overlap(*w, *x)) other = x;
    for (const Array& x : read)
      if (overlap(*w, x)) other = &x;
    if (other) return fail("%s: %s lies over %s (an output needs memory of its own, inputs keep theirs: arrays of their own)", who, w->name, other->name);
  }
  return 0;
}
// a cache whose slots are numbered in 32 bits, and tables over it
static int check_pages(const char* who, int batch, int block_size, int max_blocks, int64_t num_blocks) {
  if (batch < 1 || batch > 65535 || block_size < 1 || max_blocks < 1 || num_blocks < 1)
    return fail("%s: batch=%d, pages of %d, %d to a sequence, %lld in all", who, batch, block_size, max_blocks, (long long)num_blocks);
  if ((int64_t)max_blocks * block_size >= (1ll << 31) - 65536 || num_blocks * block_size >= (1ll << 31))
    return fail("%s: tables of %d pages or a cache of %lld of %d tokens pass 32 bits", who, max_blocks, (long long)num_blocks, block_size);
  return 0;
}
static int check_spans(const char* who, int heads, int kv_heads, int head_dim, int block_size, int span) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || kv_heads > 65535 || (head_dim != 64 && head_dim != 128))
    return fail("%s: %d heads over %d of %d (64 or 128)", who, heads, kv_heads, head_dim);
  if (span < 16 || span % 16 || block_size % span) return fail("%s: spans of %d tokens (multiples of 16 that divide pages of %d)", who, span, block_size);
  return 0;
}
// The attributes that a kernel needs, once per device.  The large carve-out is for kernels whose blocks are to share an SM: loads into registers wait in the cache
// that it takes (span_estimate_kernel for sixteen rows, 24 contexts of 64000: 67 us with it, 37 without).
enum { kSmemOnly = 0, kSmemCarveout = 1, kSmemClusters = 3 };
template <typename Kernel>
static int with_smem(Kernel* kernel, int bytes, int what, std::atomic<bool>* done) {
  int dev = 0;
  CK(cudaGetDevice(&dev));
  if (dev < 64 && done[dev].load(std::memory_order_acquire)) return 0;
  CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (what & 1) CK(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  if (what & 2) CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (dev < 64) done[dev].store(true, std::memory_order_release);
  return 0;
}

// Every kernel here may be scheduled under the end of the one in front (whatever it is): it touches no global memory before griddepcontrol.wait, and lets its own
// successor be scheduled only behind that wait.  (So span_pick_kernel may read before its wait what span_estimate_kernel, right in front of it, waited for.)  us a call, back to back
// on one stream, without and with: 4003 rows rotated 22.5 -> 20.7, four prompts' bounds 25.6 -> 24.3, 24 selections 44.4 -> 40.0, 8 x 7 rows' attention 38.0 -> 36.8.
static Launcher launcher(void* stream) {
  Launcher L;
  L.st = (cudaStream_t)stream;
  L.pdl = L.prev_kernel = true;
  return L;
}

constexpr int kSms = 148, kMaxSmem = 227 * 1024 - 1024;   // (statics beside it)
constexpr int kMaxListed = 4096;   // spans of a list
// Blocks that share the listed keys of a key head (a cluster).  Two blocks are resident on an SM, so that units x blocks take waves; a block's start and end
// cost as much as some 512 keys, and the join grows with the blocks.  us for one, two, four, eight blocks: 48 sequences of 8 key heads and 4096 keys 143, 131,
// 145, 178; one sequence of 8 key heads and 2048 keys 24.9, 15.9, 10.8, 8.1 (sixteen: 8.6); 8 x 7 rows over 8 key heads and 4096 keys (tiles) 77, 46, 34, 44.
static int span_cluster(int64_t units, int64_t keys, int most) {
  int best = 1;
  int64_t least = INT64_MAX;
  for (int c = 1; c <= most; c *= 2) {
    const int64_t cost = (units * c + 2 * kSms - 1) / (2 * kSms) * (512 + 16 * c + keys / c);
    if (cost < least) {
      least = cost;
      best = c;
    }
  }
  return best;
}
template <int HD>
static int launch_span_attn(Launcher& L, const SpanAttnParams& p) {
  static std::atomic<bool> done[64];
  CKI(with_smem(span_attn_kernel<HD>, span_attn_smem(HD, kMaxListed), kSmemClusters, done));
  L.cluster = span_cluster((int64_t)p.B * p.kv_heads, (int64_t)p.count * p.span, kSpanMost);
  return L.go(span_attn_kernel<HD>, dim3(p.kv_heads * L.cluster, p.B), dim3(kSpanWarps * 32), span_attn_smem(HD, p.count), p);
}
template <int HD>
static int launch_span_tiles(Launcher& L, SpanAttnParams p) {
  static std::atomic<bool> done[64];
  CKI(with_smem(span_tile_kernel<HD>, span_tile_smem(HD, kMaxListed), kSmemClusters, done));
  WaitWord* waits = op_waits();
  if (!waits) return fail("span_attn: pinned word for bounded waits not allocated");
  CKI(waits->check("an earlier call of attention without an engine left is not complete (NaN rows)"));
  const int G = p.heads / p.kv_heads, most = kTileRows64 / G, tiles = (p.Q + most - 1) / most, box = std::gcd(p.span, kTileKeys);
  if (tiles > 65535) return fail("span_attn: q_len=%d", p.Q);
  p.tokens = (p.Q + tiles - 1) / tiles;
  const int64_t slots = p.num_blocks * p.block_size;
  CUtensorMap tmQ, tmK, tmV;
  CKI(make_tmap_heads(&tmQ, p.q, (int64_t)p.B * p.Q, p.heads, HD, G, most));
  CKI(make_tmap_heads(&tmK, p.k_cache, slots, p.kv_heads, HD, 1, box));
  CKI(make_tmap_heads(&tmV, p.v_cache, slots, p.kv_heads, HD, 1, box));
  L.cluster = span_cluster((int64_t)p.B * p.kv_heads * tiles, (int64_t)p.count * p.span, kTileMost);
  return L.go(span_tile_kernel<HD>, dim3(p.kv_heads * L.cluster, p.B, tiles), dim3(kTileThreads), span_tile_smem(HD, p.count), tmQ, tmK, tmV, p, box, most, waits->word);
}

template <int HD>
static int launch_rope_axes(Launcher& L, RopeAxesParams p) {
  const int n = p.heads + 2 * p.kv_heads;
  p.batches = (n + rope_axes_heads(HD) - 1) / rope_axes_heads(HD);
  constexpr int W = kRopeAxesThreads / 32;
  const int64_t units = (int64_t)p.M * p.batches;
  if (units >= (1ll << 31)) return fail("rope_axes: %d rows of %d heads", p.M, n);
  p.warps = (int)std::min<int64_t>(units, kSms * 4 * W);   // four blocks on an SM
  p.each = (int)(units / p.warps);
  p.longer = (int)(units - (int64_t)p.each * p.warps);
  const dim3 grid((unsigned)((p.warps + W - 1) / W)), block(kRopeAxesThreads);
  return p.q_norm_w || p.k_norm_w ? L.go(rope_axes_kernel<HD, true>, grid, block, 0, p) : L.go(rope_axes_kernel<HD, false>, grid, block, 0, p);
}
// One launch while an SM brings in a head's bounds about as fast as a second launch begins.  us on the device, two kernels and one: contexts of 250 spans, 8 heads 8.4 and
// 7.8, 64 heads 9.4 and 8.3; of 500, 144 heads 14.4 and 11.9; of 1000, 64 heads 14.5 and 14.0, but 8 heads 9.0 and 12.6 (2 us less of the host either way).
constexpr int kOwnSpans = 512;
template <int HD>
static int launch_select(Launcher& L, const SelectParams& p) {
  constexpr int W = kEstimateThreads / 32;
  const int64_t rows = (int64_t)p.Q * (p.heads / p.kv_heads);
  const dim3 heads(p.kv_heads, p.B);
  if (rows <= 8 && p.max_spans <= kOwnSpans && (int64_t)p.kv_heads * p.B <= kSms) {
    static std::atomic<bool> own_done[64];
    CKI(with_smem(span_pick_kernel<HD, true>, kMaxSmem, kSmemOnly, own_done));
    return L.go(span_pick_kernel<HD, true>, heads, dim3(kPickThreads), pick_smem(p.max_spans, rows, HD), p);
  }
  static std::atomic<bool> done[64];
  CKI(with_smem(span_pick_kernel<HD, false>, kMaxSmem, kSmemOnly, done));
  const dim3 grid(rows > 8 ? p.warps / W : (p.warps * p.kv_heads + W - 1) / W, rows > 8 ? p.kv_heads : 1, p.B), block(kEstimateThreads);
  if (rows > 8) {
    static std::atomic<bool> many_done[64];
    CKI(with_smem(span_estimate_kernel<HD, true>, kMaxSmem, kSmemOnly, many_done));
    CKI(L.go(span_estimate_kernel<HD, true>, grid, block, estimate_smem(rows, HD), p));
  } else {
    CKI(L.go(span_estimate_kernel<HD, false>, grid, block, 0, p));
  }
  return L.go(span_pick_kernel<HD, false>, heads, dim3(kPickThreads), pick_smem(p.max_spans, rows, HD), p);
}
// Warps to a key head, which go over its groups of sixteen spans in turns: as many as make the fewest turns and waves (two blocks on an SM), a block's start and the
// query's fragments as long as two turns.  us for 1, 2, 4, 6, 8, 11 turns of 24 contexts of 64000 (8 key heads): 49.3, 42.7, 40.4, 39.2, 41.4, 39.2; 8 of them 24.7, 22.9, 21.7,
// 22.8, 25.1, 26.7; one of 32000 9.2, 10.3, 12.6, 14.9.
static int select_warps(int batch, int kv_heads, int64_t max_spans, bool many) {
  constexpr int W = kEstimateThreads / 32;
  const int groups = (int)((max_spans + 15) / 16);
  int best = groups;
  int64_t least = INT64_MAX;
  for (int turns = 1; turns <= std::min(groups, 32); ++turns) {
    int warps = (groups + turns - 1) / turns;
    if (many) warps = (warps + W - 1) / W * W;   // (a block's are of one head)
    const int64_t blocks = (int64_t)((warps * (unsigned)kv_heads + W - 1) / W) * batch, cost = (blocks + 2 * kSms - 1) / (2 * kSms) * (turns + 2);
    if (cost < least) {
      least = cost;
      best = warps;
    }
    if (blocks <= 2 * kSms) break;   // (more turns of one wave only last longer)
  }
  return best;
}

extern "C" {

uint32_t* ssdk_debug_op_wait_word(void) {
  WaitWord* waits = op_waits();
  return waits ? waits->word : nullptr;
}

int ssdk_place_tokens(const int32_t* context_lens, const int32_t* new_lens, int32_t* block_tables, const int32_t* free_blocks,
                      const int32_t* free_used, int64_t* positions, int32_t* slot_mapping, int32_t* row_seqs, int32_t* cu_rows,
                      int32_t* lens, int32_t* used, int batch, int max_blocks_per_seq, int n_free, int rows, int block_size,
                      int64_t num_blocks, void* stream) {
  CKI(check_pages("place_tokens", batch, block_size, max_blocks_per_seq, num_blocks));
  if (batch > kPlaceMaxSeqs || rows < 1 || rows > (1 << 30) || n_free < 0) return fail("place_tokens: %d sequences (at most %d), %d rows, %d free pages", batch, kPlaceMaxSeqs, rows, n_free);
  if (!context_lens || !new_lens || !block_tables || !free_used || (n_free && !free_blocks) || !positions || !slot_mapping || !row_seqs || !cu_rows || !lens || !used)
    return fail("place_tokens: null argument");
  const int64_t n_seq = batch, n_rows = rows;
  CKI(check_apart("place_tokens",
                  {{"block_tables", block_tables, n_seq * max_blocks_per_seq * 4}, {"positions", positions, n_rows * 8}, {"slot_mapping", slot_mapping, n_rows * 4},
                   {"row_seqs", row_seqs, n_rows * 4}, {"cu_rows", cu_rows, (n_seq + 1) * 4}, {"lens", lens, n_seq * 4}, {"used", used, 4}},
                  {{"context_lens", context_lens, n_seq * 4}, {"new_lens", new_lens, n_seq * 4}, {"free_blocks", free_blocks, 4ll * n_free}, {"free_used", free_used, 4}}));
  PlaceParams p;
  p.ctx = context_lens; p.fresh = new_lens; p.tables = block_tables; p.free_blocks = free_blocks; p.free_used = free_used;
  p.positions = positions; p.slots = slot_mapping; p.seqs = row_seqs; p.cu = cu_rows; p.lens = lens; p.used = used;
  p.B = batch; p.max_blocks = max_blocks_per_seq; p.n_free = n_free; p.rows = rows; p.block_size = block_size; p.num_blocks = (int)num_blocks;
  Launcher L = launcher(stream);
  static std::atomic<bool> done[64];
  if (place_smem(batch) > 48000) CKI(with_smem(place_tokens_kernel, place_smem(kPlaceMaxSeqs), kSmemOnly, done));
  return L.go(place_tokens_kernel, dim3(std::min((rows + kPlaceThreads - 1) / kPlaceThreads, 148)), dim3(kPlaceThreads), place_smem(batch), p);
}

int ssdk_rope_axes_store_kv(const void* qkv, const int64_t* positions, int axes, const uint8_t* axis_of, const int32_t* slot_mapping,
                            const float* rope_table, int64_t max_pos, int rot_dim, const void* q_norm_w, const void* k_norm_w,
                            float norm_eps, void* q_out, void* k_cache, void* v_cache, int64_t num_slots, int M, int heads,
                            int kv_heads, int head_dim, void* stream) {
  if (M < 1 || heads < 1 || kv_heads < 1 || (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return fail("rope_axes: %d rows of %d heads over %d of %d (64, 128 or 256)", M, heads, kv_heads, head_dim);
  if (rot_dim < 16 || rot_dim % 16 || rot_dim > head_dim) return fail("rope_axes: %d rotated channels of %d (a multiple of 16)", rot_dim, head_dim);
  if (axes < 1 || axes > 4 || max_pos < 1 || num_slots < 1) return fail("rope_axes: %d axes (1 to 4), %lld positions, %lld slots", axes, (long long)max_pos, (long long)num_slots);
  if (heads + 2 * (int64_t)kv_heads > 65535) return fail("rope_axes: too many heads");
  if (!qkv || !positions || !axis_of || !slot_mapping || !rope_table || !q_out || !k_cache || !v_cache) return fail("rope_axes: null argument");
  if (off16(qkv, q_out, k_cache, v_cache) || off16(q_norm_w, k_norm_w, rope_table)) return fail("rope_axes: arrays must start at multiples of 16 bytes");
  // (a slot has 32 bits; of larger numbers only as much counts as keeps the bytes in 64)
  const int64_t row = 2ll * M * head_dim, cache = 2 * std::min<int64_t>(num_slots, 1ll << 31) * kv_heads * head_dim, angles = 4 * std::min<int64_t>(max_pos, 1ll << 40) * rot_dim;
  CKI(check_apart("rope_axes", {{"q_out", q_out, row * heads}, {"k_cache", k_cache, cache}, {"v_cache", v_cache, cache}},
                  {{"qkv", qkv, row * (heads + 2 * (int64_t)kv_heads)}, {"positions", positions, 8ll * axes * M}, {"slot_mapping", slot_mapping, 4ll * M},
                   {"rope_table", rope_table, angles}, {"q_norm_w", q_norm_w, 2ll * head_dim}, {"k_norm_w", k_norm_w, 2ll * head_dim}}));
  RopeAxesParams p;
  memset(&p, 0, sizeof(p));
  for (int i = 0; i < rot_dim / 2; ++i) {
    if (axis_of[i] >= axes) return fail("rope_axes: frequency %d on axis %d of %d", i, axis_of[i], axes);
    p.axis_of[i >> 4] |= (uint32_t)axis_of[i] << (2 * (i & 15));
  }
  p.qkv = (const bf16*)qkv; p.positions = positions; p.slots = slot_mapping; p.table = rope_table;
  p.q_norm_w = (const bf16*)q_norm_w; p.k_norm_w = (const bf16*)k_norm_w; p.eps = norm_eps;
  p.q = (bf16*)q_out; p.k_cache = (bf16*)k_cache; p.v_cache = (bf16*)v_cache;
  p.top = max_pos; p.num_slots = num_slots; p.M = M; p.heads = heads; p.kv_heads = kv_heads; p.rot = rot_dim; p.axes = axes;
  Launcher L = launcher(stream);
  if (head_dim == 64) return launch_rope_axes<64>(L, p);
  if (head_dim == 128) return launch_rope_axes<128>(L, p);
  return launch_rope_axes<256>(L, p);
}

int ssdk_span_bounds(const void* k_cache, const int32_t* block_tables, const int32_t* context_lens, void* bounds, int batch,
                     int new_tokens, int kv_heads, int head_dim, int block_size, int max_blocks_per_seq, int64_t num_blocks,
                     int span, void* stream) {
  CKI(check_pages("span_bounds", batch, block_size, max_blocks_per_seq, num_blocks));
  CKI(check_spans("span_bounds", kv_heads, kv_heads, head_dim, block_size, span));
  if (new_tokens < 1) return fail("span_bounds: %d new tokens", new_tokens);
  if (!k_cache || !block_tables || !context_lens || !bounds) return fail("span_bounds: null argument");
  if (off16(k_cache, bounds)) return fail("span_bounds: arrays must start at multiples of 16 bytes");
  const int64_t token = 2ll * kv_heads * head_dim, n_spans = num_blocks * (block_size / span);
  CKI(check_apart("span_bounds", {{"bounds", bounds, n_spans * 2 * token}},
                  {{"k_cache", k_cache, num_blocks * block_size * token}, {"block_tables", block_tables, 4ll * batch * max_blocks_per_seq}, {"context_lens", context_lens, 4ll * batch}}));
  SpanBoundsParams p;
  p.k_cache = (const bf16*)k_cache; p.tables = block_tables; p.lens = context_lens; p.bounds = (bf16*)bounds; p.num_blocks = num_blocks;
  p.B = batch; p.max_blocks = max_blocks_per_seq; p.block_size = block_size; p.span = span; p.kv_heads = kv_heads; p.head_dim = head_dim;
  p.fresh = (int)std::min<int64_t>(new_tokens, (int64_t)max_blocks_per_seq * block_size);
  const int cols = kv_heads * head_dim / 8;
  p.width = cols >= 32 ? 32 : cols >= 16 ? 16 : 8;
  const int64_t units = (((int64_t)p.fresh + span - 2) / span + 1) * ((cols + p.width - 1) / p.width);
  if (units >= (1ll << 31) - 8) return fail("span_bounds: %d new tokens of %d heads", new_tokens, kv_heads);
  Launcher L = launcher(stream);
  // a block to a span's columns while the blocks fit the SMs at once, else a warp
  if (units * batch <= 8 * kSms) return L.go(span_bounds_kernel<true>, dim3((unsigned)units, batch), dim3(kBoundsThreads), 0, p);
  return L.go(span_bounds_kernel<false>, dim3((unsigned)((units + kBoundsThreads / 32 - 1) / (kBoundsThreads / 32)), batch), dim3(kBoundsThreads), 0, p);
}

int64_t ssdk_select_spans_scratch_bytes(int batch, int kv_heads, int block_size, int max_blocks_per_seq, int span) {
  if (batch < 1 || kv_heads < 1 || block_size < 1 || max_blocks_per_seq < 1 || span < 1) return 0;
  const int64_t spans = (int64_t)max_blocks_per_seq * (block_size / span);
  return (spans + (spans + 127) / 128 * (kEstimateThreads / 32)) * 4 * batch * kv_heads;
}

int ssdk_select_spans(const void* q, const void* bounds, const int32_t* block_tables, const int32_t* context_lens, int32_t* selected,
                      void* scratch, int batch, int q_len, int heads, int kv_heads, int head_dim, int block_size,
                      int max_blocks_per_seq, int64_t num_blocks, int span, int count, int first, int last, void* stream) {
  CKI(check_pages("select_spans", batch, block_size, max_blocks_per_seq, num_blocks));
  CKI(check_spans("select_spans", heads, kv_heads, head_dim, block_size, span));
  if (q_len < 1 || count < 1 || count > kMaxListed || first < 0 || last < 0 || (int64_t)first + last > count)
    return fail("select_spans: q_len=%d, %d spans (at most %d), of them the first %d and the last %d", q_len, count, kMaxListed, first, last);
  if ((int64_t)batch * q_len >= (1ll << 31)) return fail("select_spans: %d rows of %d sequences", q_len, batch);
  if (!q || !bounds || !block_tables || !context_lens || !selected || !scratch) return fail("select_spans: null argument");
  if (off16(q, bounds, scratch)) return fail("select_spans: arrays must start at multiples of 16 bytes");
  const int64_t max_spans = (int64_t)max_blocks_per_seq * (block_size / span);
  if (max_spans > kMaxSpans) return fail("select_spans: tables of %lld spans (at most %d)", (long long)max_spans, kMaxSpans);
  const int64_t rows = (int64_t)q_len * (heads / kv_heads);
  if (rows > 4096 || pick_smem((int)max_spans, rows, head_dim) > kMaxSmem || estimate_smem(rows, head_dim) > kMaxSmem)
    return fail("select_spans: %lld query rows to a key head beside tables of %lld spans pass the shared memory", (long long)rows, (long long)max_spans);
  CKI(check_apart("select_spans", {{"selected", selected, 4ll * batch * kv_heads * count},
                                   {"scratch", scratch, ssdk_select_spans_scratch_bytes(batch, kv_heads, block_size, max_blocks_per_seq, span)}},
                  {{"q", q, 2ll * batch * q_len * heads * head_dim}, {"bounds", bounds, num_blocks * (block_size / span) * kv_heads * 4ll * head_dim},
                   {"block_tables", block_tables, 4ll * batch * max_blocks_per_seq}, {"context_lens", context_lens, 4ll * batch}}));
  SelectParams p;
  p.sub_magic = ((1ull << 32) + block_size / span - 1) / (block_size / span);
  p.q = (const bf16*)q; p.bounds = (const bf16*)bounds; p.tables = block_tables; p.lens = context_lens; p.out = selected;
  p.num_blocks = num_blocks; p.B = batch; p.Q = q_len; p.heads = heads; p.kv_heads = kv_heads;
  p.block_size = block_size; p.span = span; p.max_blocks = max_blocks_per_seq; p.max_spans = (int)max_spans;
  p.count = count; p.first = first; p.last = last;
  p.warps = select_warps(batch, kv_heads, max_spans, rows > 8);
  p.estimates = (uint32_t*)scratch; p.wide = p.estimates + (size_t)batch * kv_heads * max_spans;
  Launcher L = launcher(stream);
  return head_dim == 64 ? launch_select<64>(L, p) : launch_select<128>(L, p);
}

int ssdk_span_attn(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables, const int32_t* context_lens,
                   const int32_t* selected, void* out, int batch, int q_len, int heads, int kv_heads, int head_dim, int block_size,
                   int max_blocks_per_seq, int64_t num_blocks, int span, int count, float scale, void* stream) {
  CKI(check_pages("span_attn", batch, block_size, max_blocks_per_seq, num_blocks));
  CKI(check_spans("span_attn", heads, kv_heads, head_dim, block_size, span));
  const int G = heads / kv_heads;
  const float scale_log2 = fabsf(scale) * 1.4426950408889634f;
  if (q_len < 1 || count < 1 || count > kMaxListed || G > 32 || !std::isfinite(scale_log2))
    return fail("span_attn: q_len=%d, %d spans (at most %d), %d query heads to a key head (at most 32), scale %g (finite, log2(e) times it too)", q_len, count, kMaxListed, G, (double)scale);
  if ((int64_t)count * span >= (1ll << 31) || (int64_t)batch * q_len >= (1ll << 31)) return fail("span_attn: %d spans of %d tokens, %d rows of %d sequences", count, span, q_len, batch);
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !selected || !out) return fail("span_attn: null argument");
  if (off16(q, k_cache, v_cache, out)) return fail("span_attn: arrays must start at multiples of 16 bytes");
  // (a row's query is read before its output is written, by the blocks that write it: out may be q itself)
  const int64_t rows = 2ll * batch * q_len * heads * head_dim, cache = num_blocks * block_size * kv_heads * 2ll * head_dim;
  CKI(check_apart("span_attn", {{"out", out, rows}},
                  {{"q", out == q ? nullptr : q, rows}, {"k_cache", k_cache, cache}, {"v_cache", v_cache, cache}, {"block_tables", block_tables, 4ll * batch * max_blocks_per_seq},
                   {"context_lens", context_lens, 4ll * batch}, {"selected", selected, 4ll * batch * kv_heads * count}}));
  SpanAttnParams p;
  p.q = (const bf16*)q; p.k_cache = (const bf16*)k_cache; p.v_cache = (const bf16*)v_cache; p.tables = block_tables; p.lens = context_lens;
  p.spans = selected; p.out = (bf16*)out; p.num_blocks = num_blocks; p.B = batch; p.Q = q_len; p.heads = heads; p.kv_heads = kv_heads;
  p.block_size = block_size; p.span = span; p.max_blocks = max_blocks_per_seq; p.count = count; p.scale_log2 = scale == 0.f ? 1.f : scale_log2;
  p.q_sign = scale < 0.f ? 0x80008000u : 0u; p.zero_scale = scale == 0.f;
  Launcher L = launcher(stream);
  if (G * (int64_t)q_len <= 16) return head_dim == 64 ? launch_span_attn<64>(L, p) : launch_span_attn<128>(L, p);
  return head_dim == 64 ? launch_span_tiles<64>(L, p) : launch_span_tiles<128>(L, p);
}

}  // extern "C"
