// op_host.cuh — what the entry points of the operators around a paged cache share: checks of arrays and pages, attributes of kernels, launches.
#pragma once
#include <atomic>
#include <initializer_list>

#include "host.cuh"

namespace ssdk {

inline bool off16(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) != 0;
}
// An array of a call.  What is written lies apart from everything else: other blocks still read the inputs, or write the other outputs, while one writes.
struct Array {
  const char* name;
  const void* at;
  int64_t bytes;
};
inline bool overlap(const Array& a, const Array& b) {
  return a.at && b.at && (uintptr_t)a.at < (uintptr_t)b.at + (uintptr_t)b.bytes && (uintptr_t)b.at < (uintptr_t)a.at + (uintptr_t)a.bytes;
}
inline int check_apart(const char* who, std::initializer_list<Array> written, std::initializer_list<Array> read) {
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
inline int check_pages(const char* who, int batch, int block_size, int max_blocks, int64_t num_blocks) {
  if (batch < 1 || batch > 65535 || block_size < 1 || max_blocks < 1 || num_blocks < 1)
    return fail("%s: batch=%d, pages of %d, %d to a sequence, %lld in all", who, batch, block_size, max_blocks, (long long)num_blocks);
  if ((int64_t)max_blocks * block_size >= (1ll << 31) - 65536 || num_blocks * block_size >= (1ll << 31))
    return fail("%s: tables of %d pages or a cache of %lld of %d tokens pass 32 bits", who, max_blocks, (long long)num_blocks, block_size);
  return 0;
}
// The attributes that a kernel needs, once per device.  The large carve-out is for kernels whose blocks are to share an SM: loads into registers wait in the cache
// that it takes (span_estimate_kernel for sixteen rows, 24 contexts of 64000: 67 us with it, 37 without).
enum { kSmemOnly = 0, kSmemCarveout = 1, kSmemClusters = 3 };
template <typename Kernel>
inline int with_smem(Kernel* kernel, int bytes, int what, std::atomic<bool>* done) {
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
// successor be scheduled only behind that wait.  (So two kernels may read before their wait what the kernel right in front of them has waited for and does not write: span_pick_kernel behind span_estimate_kernel, and
// kv4_join_kernel, which reads the lengths, behind kv4_attn_kernel or kv4_tile_kernel.  Nothing may be launched between the two.)  us a call, back to back
// on one stream, without and with: 4003 rows rotated 22.5 -> 20.7, four prompts' bounds 25.6 -> 24.3, 24 selections 44.4 -> 40.0, 8 x 7 rows' attention 38.0 -> 36.8.
inline Launcher launcher(void* stream) {
  Launcher L;
  L.st = (cudaStream_t)stream;
  L.pdl = L.prev_kernel = true;
  return L;
}

}  // namespace ssdk
