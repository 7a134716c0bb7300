// Runs the SOURCE of span_estimate_kernel and span_pick_kernel (csrc/span_ops.cuh) on host threads.  TEST INFRASTRUCTURE.
// run_select_spans <in> <out>.  Arrays end where they are said to, and nothing may be read in front of the bounds: built with AddressSanitizer.
#include <sanitizer/asan_interface.h>

#include "cuda_emu.h"
#define SSDK_HOST_EMU 1
#include "pairs_emu.h"

struct int4 { int x, y, z, w; };
inline int4 make_int4(int x, int y, int z, int w) { return {x, y, z, w}; }
template <typename To, typename From>
To bits_as(From v) {
  static_assert(sizeof(To) == sizeof(From));
  To r;
  std::memcpy(&r, &v, sizeof(r));
  return r;
}
inline float __uint_as_float(uint32_t v) { return bits_as<float>(v); }
inline uint32_t __float_as_uint(float v) { return bits_as<uint32_t>(v); }
inline long long __double_as_longlong(double v) { return bits_as<long long>(v); }
inline double __longlong_as_double(long long v) { return bits_as<double>(v); }
inline int __popc(uint32_t v) { return __builtin_popcount(v); }
inline int __ffs(uint32_t v) { return __builtin_ffs((int)v); }
inline int atomicAdd(int* p, int v) { return __atomic_fetch_add(p, v, __ATOMIC_SEQ_CST); }
inline uint32_t atomicOr(uint32_t* p, uint32_t v) { return __atomic_fetch_or(p, v, __ATOMIC_SEQ_CST); }
template <typename T>
T atomicMax(T* p, T v) {
  T old = __atomic_load_n(p, __ATOMIC_SEQ_CST);
  while (old < v && !__atomic_compare_exchange_n(p, &old, v, false, __ATOMIC_SEQ_CST, __ATOMIC_SEQ_CST)) {}
  return old;
}
namespace emu {
// every lane's word of a warp
inline void all_words(uint32_t v, uint32_t* all) {
  Warp& w = *tctx.cta->warps[threadIdx.x >> 5];
  w.slot[threadIdx.x & 31] = v;
  w.bar.arrive_and_wait();
  std::memcpy(all, w.slot, sizeof(w.slot));
  w.bar.arrive_and_wait();
}
template <typename T, typename Op>
T folded(T v, Op op) {
  uint32_t all[32];
  all_words(bits_as<uint32_t>(v), all);
  T r = bits_as<T>(all[0]);
  for (int i = 1; i < 32; ++i) r = op(r, bits_as<T>(all[i]));
  return r;
}
template <typename T>
T xor64(T v, int mask) {
  const uint64_t u = bits_as<uint64_t>(v);
  uint32_t lo[32], hi[32];
  all_words((uint32_t)u, lo);
  all_words((uint32_t)(u >> 32), hi);
  const int from = (threadIdx.x & 31) ^ mask;
  return bits_as<T>((uint64_t)hi[from] << 32 | lo[from]);
}
}  // namespace emu
inline double __shfl_xor_sync(unsigned, double v, int mask) { return emu::xor64(v, mask); }
inline unsigned long long __shfl_xor_sync(unsigned, unsigned long long v, int mask) { return emu::xor64(v, mask); }
inline int __shfl_up_sync(unsigned, int v, int by) {
  uint32_t all[32];
  emu::all_words((uint32_t)v, all);
  const int lane = threadIdx.x & 31;
  return (int)all[lane >= by ? lane - by : lane];
}
inline uint32_t __ballot_sync(unsigned, bool v) {
  uint32_t all[32], m = 0;
  emu::all_words(v, all);
  for (int i = 0; i < 32; ++i) m |= (all[i] & 1u) << i;
  return m;
}
inline int __reduce_add_sync(unsigned, int v) { return emu::folded(v, [](int a, int b) { return a + b; }); }
inline uint32_t __reduce_max_sync(unsigned, uint32_t v) { return emu::folded(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); }
inline uint32_t __reduce_min_sync(unsigned, uint32_t v) { return emu::folded(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; }); }

#include "../../ssd_b200/csrc/span_ops.cuh"

#include <fstream>

using bf16 = __nv_bfloat16;
template <typename T>
static T* rd(std::ifstream& f, size_t n, size_t front = 0) {   // an array of its own allocation; `front` values in front of it are nobody's
  char* raw = static_cast<char*>(aligned_alloc(16, ((front + n) * sizeof(T) + 15) / 16 * 16 + 16));
  T* p = reinterpret_cast<T*>(raw) + front;
  f.read(reinterpret_cast<char*>(p), (std::streamsize)(n * sizeof(T)));
  if (!f && n) std::exit(2);
  ASAN_POISON_MEMORY_REGION(raw, front * sizeof(T));
  ASAN_POISON_MEMORY_REGION(p + n, 16);
  return p;
}

template <int HD>
static void select(const ssdk::SelectParams& p, const int32_t* later, bool own) {
  constexpr int W = ssdk::kEstimateThreads / 32;
  const int64_t rows = (int64_t)p.Q * (p.heads / p.kv_heads);
  const size_t smem = ssdk::pick_smem(p.max_spans, rows, HD);
  dim3 heads;
  heads.x = (unsigned)p.kv_heads;
  heads.y = (unsigned)p.B;
  if (own) {
    emu::launch(ssdk::span_pick_kernel<HD, true>, p, heads, ssdk::kPickThreads, smem, 1);
    return;
  }
  const bool many = rows > 8;
  const int gy = many ? p.kv_heads : 1;
  dim3 grid;
  grid.x = (unsigned)(many ? p.warps / W : (p.warps * p.kv_heads + W - 1) / W);
  grid.y = (unsigned)(gy * p.B);
  emu::launch([&](const ssdk::SelectParams& q) {
    blockIdx.z = blockIdx.y / gy;
    blockIdx.y %= gy;
    if (many) ssdk::span_estimate_kernel<HD, true>(q);
    else ssdk::span_estimate_kernel<HD, false>(q);
  }, p, grid, ssdk::kEstimateThreads, (size_t)ssdk::estimate_smem(rows, HD), 2);
  ssdk::SelectParams second = p;
  second.tables = later;
  emu::launch(ssdk::span_pick_kernel<HD, false>, second, heads, ssdk::kPickThreads, smem, 1);
}

int main(int argc, char** argv) {
  if (argc != 3) return 2;
  std::ifstream f(argv[1], std::ios::binary);
  const int32_t* h = rd<int32_t>(f, 14);   // B Q H KV hd block_size span max_blocks num_blocks count first last warps own
  ssdk::SelectParams p;
  p.B = h[0]; p.Q = h[1]; p.heads = h[2]; p.kv_heads = h[3]; p.block_size = h[5]; p.span = h[6]; p.max_blocks = h[7]; p.num_blocks = h[8];
  p.count = h[9]; p.first = h[10]; p.last = h[11]; p.warps = h[12];
  const int hd = h[4], subs = p.block_size / p.span;
  p.max_spans = p.max_blocks * subs;
  p.sub_magic = ((1ull << 32) + subs - 1) / subs;
  p.tables = rd<int32_t>(f, (size_t)p.B * p.max_blocks);
  const int32_t* later = rd<int32_t>(f, (size_t)p.B * p.max_blocks);   // the tables as the second kernel finds them
  p.lens = rd<int32_t>(f, p.B);
  p.q = rd<bf16>(f, (size_t)p.B * p.Q * p.heads * hd);
  const size_t page = (size_t)subs * p.kv_heads * 2 * hd;
  p.bounds = rd<bf16>(f, page * p.num_blocks, page);
  std::vector<int32_t> out((size_t)p.B * p.kv_heads * p.count, -7);
  std::vector<uint32_t> scratch((size_t)p.B * p.kv_heads * (p.max_spans + p.warps), 0xdeadbeefu);
  p.out = out.data();
  p.estimates = scratch.data();
  p.wide = p.estimates + (size_t)p.B * p.kv_heads * p.max_spans;
  if (hd == 64) select<64>(p, later, h[13]);
  else select<128>(p, later, h[13]);
  std::ofstream o(argv[2], std::ios::binary);
  o.write(reinterpret_cast<const char*>(out.data()), (std::streamsize)(out.size() * 4));
  return 0;
}
