// C-ABI plumbing: error text, device queries, version.
#include <stdarg.h>
#include <stdio.h>

#include <atomic>

#include "common.cuh"

namespace smaq {

static thread_local char g_err[512] = "";

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int cuda_status(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return SMAQ_OK;
  return fail(SMAQ_ERR_CUDA, "%s: %s", where, cudaGetErrorString(e));
}

int num_sms() {
  static std::atomic<int> known[64];  // by device: the count does not change
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

int allow_smem(const void* kernel, int bytes, const char* where) {
  struct Grant {
    const void* kernel;
    int dev, bytes;
  };
  static thread_local Grant known[64];  // one more question to the driver a thread costs nothing; a lock would
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, where);
  Grant* slot = nullptr;
  for (Grant& g : known) {
    if (g.kernel == kernel && g.dev == dev && g.bytes >= bytes) return SMAQ_OK;
    if (!slot && (!g.kernel || (g.kernel == kernel && g.dev == dev))) slot = &g;
  }
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_status(e, where);
  if (slot) *slot = {kernel, dev, bytes};
  return SMAQ_OK;
}

}  // namespace smaq

extern "C" int smaq_abi_version(void) { return SMAQ_ABI_VERSION; }
extern "C" size_t smaq_args_size(int which) {
  return which == 0 ? sizeof(smaq_append_args)
       : which == 1 ? sizeof(smaq_decode_args)
       : which == 2 ? sizeof(smaq_scores_args)
       : which == 3 ? sizeof(smaq_attend_args)
                    : 0;
}
extern "C" size_t smaq_paged_args_size(int which) {
  return which == 0 ? sizeof(smaq_tables_args)
       : which == 1 ? sizeof(smaq_norm_rope_args)
       : which == 2 ? sizeof(smaq_paged_args)
                    : 0;
}
extern "C" const char* smaq_last_error(void) { return smaq::g_err; }
