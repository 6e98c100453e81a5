// Status plumbing of the C ABI: per-host-thread last-error message and version.
#include "common.cuh"
#include "tmap.cuh"

#include <atomic>
#include <mutex>
#include <stdarg.h>
#include <stdio.h>

namespace verace {

static thread_local char g_last_error[512] = "no error";
static std::atomic<unsigned long long> g_launches{0};

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
}

int check_launch(const char* what) {
  g_launches.fetch_add(1, std::memory_order_relaxed);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("%s: kernel launch failed: %s", what, cudaGetErrorString(e));
    return VERACE_ERR_CUDA;
  }
  return VERACE_OK;
}

static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

// The driver's entry point wants a current context, which a thread has from its first call of the runtime that needs one.
// Neither cudaGetDevice nor a block out of torch's cache is such a call, so a thread's first product may come here without
// (autograd's own thread, a server's worker): the current device's context is bound then, and the map asked for again.
static CUresult CUDAAPI encode_here(CUtensorMap* map, CUtensorMapDataType type, cuuint32_t rank, void* base,
                                    const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                                    const cuuint32_t* steps, CUtensorMapInterleave interleave, CUtensorMapSwizzle swizzle,
                                    CUtensorMapL2promotion promotion, CUtensorMapFloatOOBfill fill) {
  CUresult r = g_encode(map, type, rank, base, dims, strides, box, steps, interleave, swizzle, promotion, fill);
  int dev = 0;
  if (r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess)
    r = g_encode(map, type, rank, base, dims, strides, box, steps, interleave, swizzle, promotion, fill);
  return r;
}

PFN_cuTensorMapEncodeTiled_v12000 tmap_encoder() {
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) == cudaSuccess &&
        qr == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return g_encode ? encode_here : nullptr;
}

}  // namespace verace

extern "C" int verace_version(void) { return 1 * 10000 + 0 * 100 + 0; }

extern "C" const char* verace_last_error(void) { return verace::g_last_error; }

extern "C" unsigned long long verace_kernel_launches(void) {
  return verace::g_launches.load(std::memory_order_relaxed);
}
