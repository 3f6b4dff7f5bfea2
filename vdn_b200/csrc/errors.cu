// Thread-local last-error message and library metadata entry points.
#include "common.cuh"

#include <string.h>

#include <atomic>

namespace vdn {

static thread_local char g_last_error[1024] = "";

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return code;
}

void clear_error() { g_last_error[0] = '\0'; }

}  // namespace vdn

extern "C" {

const char* vdn_last_error(void) { return vdn::g_last_error; }

int vdn_abi_version(void) { return VDN_ABI_VERSION; }

int vdn_device_supported(int device, int* supported) {
  if (!supported) return vdn::set_error(VDN_ERR_VALUE, "supported must not be null");
  int major = 0, minor = 0;
  VDN_CUDA_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
  VDN_CUDA_TRY(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device));
  *supported = (major == 10 && minor == 0) ? 1 : 0;
  return VDN_OK;
}

// One word a device, 64 bytes apart, in one block of pinned host memory that lives as long as the
// process: captured graphs keep its address, and the host reads it without waiting for the GPU.
int vdn_status_word(int device, int** word) {
  static std::atomic<int*> words{nullptr};
  constexpr int kDevices = 64, kStep = 16;
  VDN_CHECK_ARG(word, "word must not be null");
  VDN_CHECK_ARG(device >= 0 && device < kDevices, "device index out of range");
  int* base = words.load();
  if (!base) {
    // a capture under way on this thread must not be broken by the allocation, which is not part of it
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    VDN_CUDA_TRY(cudaThreadExchangeStreamCaptureMode(&mode));
    void *host = nullptr, *seen = nullptr;
    cudaError_t err = cudaHostAlloc(&host, kDevices * kStep * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
    if (err == cudaSuccess) err = cudaHostGetDevicePointer(&seen, host, 0);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (err == cudaSuccess && seen != host) err = cudaErrorNotSupported;   // one address for both: unified addressing
    if (err != cudaSuccess) {
      if (host) cudaFreeHost(host);
      return vdn::set_error(VDN_ERR_RUNTIME, "status words: %s", cudaGetErrorString(err));
    }
    memset(host, 0, kDevices * kStep * sizeof(int));
    if (words.compare_exchange_strong(base, static_cast<int*>(host))) base = static_cast<int*>(host);
    else cudaFreeHost(host);                         // another thread was first
  }
  *word = base + device * kStep;
  return VDN_OK;
}

}  // extern "C"
