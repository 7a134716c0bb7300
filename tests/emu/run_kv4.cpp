// Runs the SOURCE of kv4_store_kernel and kv4_load_kernel (csrc/kv4.cuh) on host threads.  TEST INFRASTRUCTURE.
// run_kv4 <store|rope|load> <in> <out>.  Arrays end where they are said to: built with AddressSanitizer a read or write outside one is an error.
#include "cuda_emu.h"
#define SSDK_HOST_EMU 1
inline float __uint_as_float(uint32_t u) {
  float f;
  std::memcpy(&f, &u, 4);
  return f;
}
inline uint32_t __float_as_uint(float f) {
  uint32_t u;
  std::memcpy(&u, &f, 4);
  return u;
}
template <typename T>
inline void __stcs(T* p, const T& v) { *p = v; }
#include "pairs_emu.h"
namespace ssdk {
inline float one_if_ge(float a, float b) { return a >= b ? 1.f : 0.f; }
inline uint32_t and_or(uint32_t x, uint32_t a, uint32_t b) { return (x & a) | b; }
}  // namespace ssdk
#include "../../ssd_b200/csrc/kv4.cuh"

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

template <int HD, bool ROPE, bool VALUES>
static void store(ssdk::Kv4StoreParams p, int most) {
  constexpr int SIDE = ssdk::kv4_store_heads(HD);
  p.groups = (p.heads + 2 * p.kv_heads + SIDE - 1) / SIDE;
  const int units = p.M * p.groups;
  p.warps = std::min(units, most);
  p.each = units / p.warps;
  p.longer = units % p.warps;
  dim3 grid;
  grid.x = (unsigned)((p.warps + 3) / 4);
  emu::launch(+[](ssdk::Kv4StoreParams q) { ssdk::kv4_store_kernel<HD, ROPE, VALUES>(q); }, p, grid, ssdk::kKv4StoreThreads, 0, 4);
}
template <int HD>
static void store(const ssdk::Kv4StoreParams& p, bool rope, bool values, int most) {
  if (rope) values ? store<HD, true, true>(p, most) : store<HD, true, false>(p, most);
  else values ? store<HD, false, true>(p, most) : store<HD, false, false>(p, most);
}

int main(int argc, char** argv) {
  if (argc != 4) return 2;
  const std::string mode = argv[1];
  std::ifstream f(argv[2], std::ios::binary);
  std::ofstream o(argv[3], std::ios::binary);
  if (mode == "load") {
    auto h = rd<int32_t>(f, 6);   // M KV hd block_size num_blocks blocks
    ssdk::Kv4LoadParams p;
    const int hd = h.p[2];
    p.M = h.p[0]; p.kv_heads = h.p[1]; p.block_size = h.p[3]; p.num_slots = (int64_t)h.p[3] * h.p[4];
    const size_t bytes = (size_t)p.num_slots * p.kv_heads * (hd / 2 + 4), n = (size_t)p.M * p.kv_heads * hd;
    auto kc = rd<uint8_t>(f, bytes), vc = rd<uint8_t>(f, bytes);
    auto slots = rd<int32_t>(f, p.M);
    Exact<bf16> k(n), v(n);
    p.k_cache = kc.p; p.v_cache = vc.p; p.slots = slots.p; p.k = k.p; p.v = v.p;
    dim3 grid;
    grid.x = (unsigned)h.p[5];
    emu::launch(hd == 64 ? ssdk::kv4_load_kernel<64> : ssdk::kv4_load_kernel<128>, p, grid, ssdk::kKv4LoadThreads, 0, 2);
    wr(o, k); wr(o, v);
    return 0;
  }
  auto h = rd<int32_t>(f, 11);   // M H KV hd rot top block_size num_blocks norm values most-warps
  auto eps = rd<float>(f, 1);
  const bool rope = mode == "rope";
  const int hd = h.p[3];
  ssdk::Kv4StoreParams p;
  std::memset(&p, 0, sizeof(p));
  p.M = h.p[0]; p.heads = rope ? h.p[1] : 0; p.kv_heads = h.p[2]; p.rot = rope ? h.p[4] : 0; p.top = h.p[5]; p.block_size = h.p[6]; p.num_slots = (int64_t)h.p[6] * h.p[7]; p.eps = eps.p[0];
  auto positions = rd<int64_t>(f, p.M);
  auto slots = rd<int32_t>(f, p.M);
  auto table = rd<float>(f, (size_t)p.top * h.p[4]);
  auto qn = rd<bf16>(f, hd), kn = rd<bf16>(f, hd);
  const int all = h.p[1] + 2 * p.kv_heads;
  auto qkv = rd<bf16>(f, (size_t)p.M * all * hd);
  const size_t bytes = (size_t)p.num_slots * p.kv_heads * (hd / 2 + 4), n = (size_t)p.M * p.kv_heads * hd;
  auto kc = rd<uint8_t>(f, bytes), vc = rd<uint8_t>(f, bytes);
  Exact<bf16> q((size_t)p.M * p.heads * hd), kv(h.p[9] ? n : 0), vv(h.p[9] ? n : 0);
  p.q = qkv.p; p.k = qkv.p + h.p[1] * hd; p.v = p.k + p.kv_heads * hd;
  p.q_row = p.k_row = p.v_row = (int64_t)all * hd;
  p.positions = positions.p; p.slots = slots.p; p.table = table.p; p.q_out = q.p; p.k_cache = kc.p; p.v_cache = vc.p;
  p.q_norm_w = rope && h.p[8] ? qn.p : nullptr; p.k_norm_w = rope && h.p[8] ? kn.p : nullptr;
  p.k_values = h.p[9] ? kv.p : nullptr; p.v_values = h.p[9] ? vv.p : nullptr;
  hd == 64 ? store<64>(p, rope, h.p[9], h.p[10]) : store<128>(p, rope, h.p[9], h.p[10]);
  wr(o, q); wr(o, kc); wr(o, vc); wr(o, kv); wr(o, vv);
  return 0;
}
