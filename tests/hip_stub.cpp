// A HIP runtime with two pretended gfx950 devices and no kernels, for CPU tests of what the library's entry points do on
// the host.  Loaded into the global scope of a process before libclpeak_mi355.so, its functions are the ones that the library
// calls.  It keeps the calling thread's current device, which kernels have been allowed how much LDS on which device, and counts
// launches that ask for more than they may (64 KiB where nothing was said).
#include <hip/hip_runtime_api.h>
#include <cstring>
#include <map>
#include <utility>

namespace {

constexpr int kDevices = 2;
thread_local int current = 0;
struct Config {
  dim3 grid, block;
  size_t lds;
  hipStream_t stream;
};
thread_local Config config;
std::map<std::pair<int, const void *>, int> allowed;
int launches = 0, refused = 0, wrong_device = 0, big_lds = 0;
alignas(4096) char memory[1 << 16];
int stream_of[kDevices] = {0, 1};

int device_of(hipStream_t s) { return s ? *reinterpret_cast<int *>(s) : current; }

}  // namespace

extern "C" {

void stub_counts(int *out) { out[0] = launches; out[1] = refused; out[2] = wrong_device; out[3] = big_lds; }
int stub_current() { return current; }
void stub_make_current(int device) { current = device; }
void stub_forget() { allowed.clear(); }   // (as a new process would start)
void *stub_stream(int device) { return &stream_of[device]; }

hipError_t hipGetDeviceCount(int *n) { *n = kDevices; return hipSuccess; }
hipError_t hipGetDevice(int *d) { *d = current; return hipSuccess; }
hipError_t hipSetDevice(int d) {
  if (d < 0 || d >= kDevices) return hipErrorInvalidDevice;
  current = d;
  return hipSuccess;
}
hipError_t hipGetDeviceProperties(hipDeviceProp_t *p, int) {
  memset(p, 0, sizeof(*p));
  strcpy(p->name, "pretended");
  strcpy(p->gcnArchName, "gfx950");
  p->multiProcessorCount = 256;
  p->warpSize = 64;
  p->maxThreadsPerBlock = 1024;
  return hipSuccess;
}
hipError_t hipDriverGetVersion(int *v) { *v = 0; return hipSuccess; }
hipError_t hipRuntimeGetVersion(int *v) { *v = 0; return hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) { *s = reinterpret_cast<hipStream_t>(&stream_of[current]); return hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t s, hipDevice_t *d) { *d = device_of(s); return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t *e) { *e = reinterpret_cast<hipEvent_t>(memory); return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float *ms, hipEvent_t, hipEvent_t) { *ms = 1.0f; return hipSuccess; }
hipError_t hipGetSymbolAddress(void **p, const void *) { *p = memory; return hipSuccess; }
hipError_t hipMalloc(void **p, size_t) { *p = memory; return hipSuccess; }
hipError_t hipFree(void *) { return hipSuccess; }
hipError_t hipHostMalloc(void **p, size_t, unsigned) { *p = memory; return hipSuccess; }
hipError_t hipHostFree(void *) { return hipSuccess; }
hipError_t hipMemcpyAsync(void *, const void *, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipMemsetAsync(void *, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "an error"; }

hipError_t hipFuncSetAttribute(const void *f, hipFuncAttribute a, int value) {
  if (a == hipFuncAttributeMaxDynamicSharedMemorySize) allowed[{current, f}] = value;
  return hipSuccess;
}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t s) { config = {grid, block, lds, s}; return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *s) {
  *grid = config.grid; *block = config.block; *lds = config.lds; *s = config.stream;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void *f, dim3, dim3, void **, size_t lds, hipStream_t s) {
  launches++;
  const auto it = allowed.find({current, f});
  if (lds > 65536u) {
    big_lds++;
    if (it == allowed.end() || (size_t)it->second < lds) refused++;
  }
  if (device_of(s) != current) wrong_device++;
  return hipSuccess;
}

}
