// Library-level C ABI: version, last-error text, launch counter.
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "common.cuh"

namespace qk {

namespace {
thread_local char g_last_error[512] = "";
std::atomic<uint64_t> g_launches{0};
int g_sm_count[64] = {0};
}  // namespace

int set_error(int status, const char* fmt, ...) {
  va_list args;
  va_start(args, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, args);
  va_end(args);
  return status;
}

int cuda_error(cudaError_t err, const char* where) {
  return set_error(QK_ERR_CUDA, "%s: %s", where, cudaGetErrorString(err));
}

void count_launch(int n) { g_launches.fetch_add(static_cast<uint64_t>(n)); }

int sm_count() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (g_sm_count[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
    g_sm_count[dev] = n;
  }
  return g_sm_count[dev];
}

int allow_smem(const void* kernel, size_t bytes) {
  // The attribute is per (kernel, device) and is a ceiling: remember the largest value set so far and raise it when a
  // launch needs more (never lower it). One memory for all host threads: with one each, a thread's first call of a
  // kernel lowered the ceiling that another had raised.
  struct Ceiling {
    const void* kernel;
    int dev;
    size_t bytes;
  };
  static std::mutex mutex;
  static Ceiling done[512];
  static int n_done = 0;
  if (bytes <= 48 * 1024) return QK_OK;  // below the default limit: nothing to opt into
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mutex);
  Ceiling* slot = nullptr;
  for (int i = 0; i < n_done && !slot; ++i)
    if (done[i].kernel == kernel && done[i].dev == dev) slot = &done[i];
  if (slot && slot->bytes >= bytes) return QK_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(bytes));
  if (e != cudaSuccess) return cuda_error(e, "cudaFuncSetAttribute");
  if (!slot && n_done < 512) slot = &done[n_done++];
  if (slot) *slot = Ceiling{kernel, dev, bytes};
  return QK_OK;
}

void* tensor_map_encoder() {
  static void* fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return p;
  }();
  return fn;
}

}  // namespace qk

extern "C" {

const char* qk_version(void) { return "qk_b200 0.1 sm_100a"; }

const char* qk_last_error(void) { return qk::g_last_error; }

uint64_t qk_launch_count(void) { return qk::g_launches.load(); }

}  // extern "C"
