// host.cuh — what the host sides of libssdk share: the text of the last error of a thread, checks that return it, kernel launches, maps of heads for TMA, the word
// that bounded waits set.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <nccl.h>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <string>

namespace ssdk {

// ------------------------------------------------------------------------------------------
// errors
// ------------------------------------------------------------------------------------------
inline thread_local std::string g_err;
inline int fail(const char* fmt, ...) {
  char buf[1024];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_err = buf;
  return -1;
}
#define CK(expr)                                                                              \
  do {                                                                                        \
    cudaError_t _e = (expr);                                                                  \
    if (_e != cudaSuccess) return fail("%s:%d %s -> %s", __FILE__, __LINE__, #expr, cudaGetErrorString(_e)); \
  } while (0)
#define CKN(expr)                                                                             \
  do {                                                                                        \
    ncclResult_t _e = (expr);                                                                 \
    if (_e != ncclSuccess) return fail("%s:%d %s -> nccl error %d", __FILE__, __LINE__, #expr, (int)_e); \
  } while (0)
#define CKI(expr)                 \
  do {                            \
    int _r = (expr);              \
    if (_r != 0) return _r;       \
  } while (0)

inline int env_int(const char* name, int dflt) {
  const char* s = getenv(name);
  return (s && *s) ? atoi(s) : dflt;
}

// ------------------------------------------------------------------------------------------
// launch helper (optional programmatic dependent launch)
// ------------------------------------------------------------------------------------------
struct Launcher {
  cudaStream_t st = nullptr;
  unsigned* gave_up = nullptr;   // the engine's word for waits that run out (WaitWord)
  bool pdl = false;       // PDL enabled at all
  bool prev_kernel = false;  // the previous op on the stream was one of our kernels
  int64_t count = 0;
  int cluster = 1;        // blocks (along x) of a cluster

  template <typename... KArgs, typename... Args>
  int go(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (pdl && prev_kernel) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs].val.clusterDim.x = cluster;
      attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
      ++cfg.numAttrs;
    }
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
    if (e != cudaSuccess) return fail("kernel launch failed: %s", cudaGetErrorString(e));
    prev_kernel = true;
    ++count;
    return 0;
  }
  void barrier_op() { prev_kernel = false; }  // memcpy / NCCL / anything that is not our kernel
};

// ------------------------------------------------------------------------------------------
// TMA descriptors of heads
// ------------------------------------------------------------------------------------------
inline PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
inline int get_encode() {
  if (g_encode) return 0;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult qres;
  cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
  if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !fn)
    return fail("cuTensorMapEncodeTiled unavailable (%s)", cudaGetErrorString(e));
  g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  return 0;
}
// rows [rows][heads][hd] as {column, head, row}; box: 64 columns x box_heads x box_rows
inline int make_tmap_heads(CUtensorMap* tm, const void* ptr, int64_t rows, int64_t heads, int hd, int box_heads, int box_rows) {
  CKI(get_encode());
  if (hd % 64 != 0 || ((uintptr_t)ptr & 15) != 0) return fail("TMA: heads of %d", hd);
  cuuint64_t gdim[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t gstride[2] = {(cuuint64_t)hd * 2, (cuuint64_t)heads * hd * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows}, estr[3] = {1, 1, 1};
  CUresult r = g_encode(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), gdim, gstride, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail("cuTensorMapEncodeTiled failed (%d) rows of %lld heads of %d x %lld", (int)r, (long long)heads, hd, (long long)rows);
  return 0;
}

// ------------------------------------------------------------------------------------------
// bounded waits
// ------------------------------------------------------------------------------------------
// Word in host memory that the kernels of one engine set when a bounded wait of theirs runs out.  Read wherever a call has waited for the
// stream: a call that does not wait (prompt passes without a token) leaves its report to the next one that does.
struct WaitWord {
  unsigned* word = nullptr;   // (unified addressing: the host pointer is the device's too)
  WaitWord() = default;
  WaitWord(const WaitWord&) = delete;
  ~WaitWord() { if (word) cudaFreeHost(word); }
  bool make() {
    if (cudaHostAlloc(&word, sizeof(unsigned), cudaHostAllocMapped | cudaHostAllocPortable) != cudaSuccess) { word = nullptr; return false; }
    *word = 0;
    return true;
  }
  int check(const char* whose = "this engine's calls left since the last check is not complete") {
    volatile unsigned* w = word;
    if (!*w) return 0;
    *w = 0;
    return fail("a bounded wait in a tile-pair product, the prompt attention or the streaming kernel ran out: what %s", whose);
  }
};
// The same for calls without an engine, which do not wait for the stream: rows whose waits ran out are NaN, and the next such call reports it.  One word for the
// process that is never freed (a kernel in flight may still write to it); made under relaxed capture rules, since the first such call may be a captured one.
inline WaitWord* op_waits() {
  static WaitWord* const w = [] {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    (void)cudaThreadExchangeStreamCaptureMode(&mode);
    WaitWord* made = new WaitWord;
    if (!made->make()) { delete made; made = nullptr; }
    (void)cudaThreadExchangeStreamCaptureMode(&mode);
    return made;
  }();
  return w;
}

}  // namespace ssdk
