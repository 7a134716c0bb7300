// Runs the SOURCE of place_tokens_kernel, rope_axes_kernel and span_bounds_kernel (csrc/cache_ops.cuh) on host threads.  TEST INFRASTRUCTURE.
// run_cache_ops <place|rope|bounds> <in> <out>.  Arrays end where they are said to: built with AddressSanitizer a read or write outside one is an error.
#include "cuda_emu.h"
#define SSDK_HOST_EMU 1
inline int atomicMax(int* p, int v) {
  int old = __atomic_load_n(p, __ATOMIC_SEQ_CST);
  while (old < v && !__atomic_compare_exchange_n(p, &old, v, false, __ATOMIC_SEQ_CST, __ATOMIC_SEQ_CST)) {}
  return old;
}
#include "pairs_emu.h"
#include "../../ssd_b200/csrc/cache_ops.cuh"

#include <fstream>
#include <string>

using bf16 = __nv_bfloat16;
template <typename T>
struct Exact {   // an array of its own allocation, so that its end is the allocator's
  T* p;
  size_t n;
  explicit Exact(size_t n) : p(static_cast<T*>(aligned_alloc(16, (n * sizeof(T) + 15) / 16 * 16))), n(n) { std::memset((void*)p, 0, n * sizeof(T)); }
};
template <typename T>
static Exact<T> rd(std::ifstream& f, size_t n) {
  Exact<T> v(n);
  f.read(reinterpret_cast<char*>(v.p), (std::streamsize)(n * sizeof(T)));
  if (!f && n) std::exit(2);
  return v;
}
template <typename T>
static void wr(std::ofstream& o, const Exact<T>& v) { o.write(reinterpret_cast<const char*>(v.p), (std::streamsize)(v.n * sizeof(T))); }

int main(int argc, char** argv) {
  if (argc != 4) return 2;
  const std::string mode = argv[1];
  std::ifstream f(argv[2], std::ios::binary);
  std::ofstream o(argv[3], std::ios::binary);
  if (mode == "place") {
    auto h = rd<int32_t>(f, 7);   // B max_blocks n_free rows block_size num_blocks blocks
    ssdk::PlaceParams p;
    p.B = h.p[0]; p.max_blocks = h.p[1]; p.n_free = h.p[2]; p.rows = h.p[3]; p.block_size = h.p[4]; p.num_blocks = h.p[5];
    auto ctx = rd<int32_t>(f, p.B), fresh = rd<int32_t>(f, p.B), tables = rd<int32_t>(f, (size_t)p.B * p.max_blocks), free_blocks = rd<int32_t>(f, p.n_free), used = rd<int32_t>(f, 1);
    Exact<int64_t> positions(p.rows);
    Exact<int32_t> slots(p.rows), seqs(p.rows), cu(p.B + 1), lens(p.B), out(1);
    p.ctx = ctx.p; p.fresh = fresh.p; p.tables = tables.p; p.free_blocks = free_blocks.p; p.free_used = used.p;
    p.positions = positions.p; p.slots = slots.p; p.seqs = seqs.p; p.cu = cu.p; p.lens = lens.p; p.used = out.p;
    dim3 grid;
    grid.x = (unsigned)h.p[6];
    emu::launch(ssdk::place_tokens_kernel, p, grid, ssdk::kPlaceThreads, ssdk::place_smem(p.B), 2);
    wr(o, positions); wr(o, slots); wr(o, seqs); wr(o, cu); wr(o, lens); wr(o, out); wr(o, tables);
    return 0;
  }
  if (mode == "rope") {
    auto h = rd<int32_t>(f, 10);   // M H KV hd rot axes top num_slots norm most-warps
    auto eps = rd<float>(f, 1);
    const int hd = h.p[3], rot = h.p[4];
    ssdk::RopeAxesParams p;
    std::memset(&p, 0, sizeof(p));
    p.M = h.p[0]; p.heads = h.p[1]; p.kv_heads = h.p[2]; p.rot = rot; p.axes = h.p[5]; p.top = h.p[6]; p.num_slots = h.p[7]; p.eps = eps.p[0];
    auto axis_of = rd<int32_t>(f, rot / 2);
    for (int i = 0; i < rot / 2; ++i) p.axis_of[i >> 4] |= (uint32_t)axis_of.p[i] << (2 * (i & 15));
    auto positions = rd<int64_t>(f, (size_t)p.axes * p.M);
    auto slots = rd<int32_t>(f, p.M);
    auto table = rd<float>(f, (size_t)p.top * rot);
    auto qn = rd<bf16>(f, hd), kn = rd<bf16>(f, hd), qkv = rd<bf16>(f, (size_t)p.M * (p.heads + 2 * p.kv_heads) * hd);
    Exact<bf16> q((size_t)p.M * p.heads * hd), kc((size_t)p.num_slots * p.kv_heads * hd), vc((size_t)p.num_slots * p.kv_heads * hd);
    p.qkv = qkv.p; p.positions = positions.p; p.slots = slots.p; p.table = table.p; p.q = q.p; p.k_cache = kc.p; p.v_cache = vc.p;
    p.q_norm_w = h.p[8] ? qn.p : nullptr; p.k_norm_w = h.p[8] ? kn.p : nullptr;
    const int n = p.heads + 2 * p.kv_heads, at_once = ssdk::rope_axes_heads(hd);
    p.batches = (n + at_once - 1) / at_once;
    p.warps = std::min(p.M * p.batches, h.p[9]);
    p.each = p.M * p.batches / p.warps;
    p.longer = p.M * p.batches % p.warps;
    dim3 grid;
    grid.x = (unsigned)((p.warps + 3) / 4);
    const auto kernel = hd == 64 ? (h.p[8] ? ssdk::rope_axes_kernel<64, true> : ssdk::rope_axes_kernel<64, false>)
                                 : (h.p[8] ? ssdk::rope_axes_kernel<128, true> : ssdk::rope_axes_kernel<128, false>);
    emu::launch(kernel, p, grid, ssdk::kRopeAxesThreads, 0, 8);
    wr(o, q); wr(o, kc); wr(o, vc);
    return 0;
  }
  if (mode == "bounds") {
    auto h = rd<int32_t>(f, 9);   // B max_blocks num_blocks block_size span KV hd fresh split
    ssdk::SpanBoundsParams p;
    p.B = h.p[0]; p.max_blocks = h.p[1]; p.num_blocks = h.p[2]; p.block_size = h.p[3]; p.span = h.p[4]; p.kv_heads = h.p[5]; p.head_dim = h.p[6]; p.fresh = h.p[7];
    auto tables = rd<int32_t>(f, (size_t)p.B * p.max_blocks), lens = rd<int32_t>(f, p.B);
    auto keys = rd<bf16>(f, (size_t)p.num_blocks * p.block_size * p.kv_heads * p.head_dim);
    auto bounds = rd<bf16>(f, (size_t)p.num_blocks * (p.block_size / p.span) * p.kv_heads * 2 * p.head_dim);
    p.k_cache = keys.p; p.tables = tables.p; p.lens = lens.p; p.bounds = bounds.p;
    dim3 grid;
    const int cols = p.kv_heads * p.head_dim / 8;
    p.width = cols >= 32 ? 32 : cols >= 16 ? 16 : 8;
    const int units = ((p.fresh + p.span - 2) / p.span + 1) * ((cols + p.width - 1) / p.width);
    grid.x = (unsigned)(h.p[8] ? units : (units + 7) / 8);
    grid.y = (unsigned)p.B;
    if (h.p[8]) emu::launch(+[](ssdk::SpanBoundsParams q) { ssdk::span_bounds_kernel<true>(q); }, p, grid, ssdk::kBoundsThreads, 0, 4);
    else emu::launch(+[](ssdk::SpanBoundsParams q) { ssdk::span_bounds_kernel<false>(q); }, p, grid, ssdk::kBoundsThreads, 0, 4);
    wr(o, bounds);
    return 0;
  }
  return 2;
}
