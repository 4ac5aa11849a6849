/* A HIP runtime of host memory that launches nothing, for tests of the
 * library's host code without a GPU: loaded with RTLD_GLOBAL before
 * libmitok.so, its functions take the place of the runtime's.  Device memory
 * is calloc'd, copies happen at once, kernels are only counted.
 *   host_hip_calls(name)      calls of a runtime function so far
 *   host_hip_launches(part)   launches of kernels whose name contains `part`
 *   host_hip_fail(name, k)    the k-th call of `name` from now fails (0: none)
 *   host_hip_pinned(bytes)    the pinned allocation of that size
 */
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

namespace {
std::map<std::string, long> g_calls, g_fail;
std::map<const void*, std::string> g_kernels;
std::map<std::string, long> g_launches;
std::map<char*, size_t> g_memory;  // device allocations
std::map<void*, size_t> g_pinned;
std::map<const void*, void*> g_symbols;
hipError_t g_last = hipSuccess;

bool fails(const char* name, hipError_t e) {
  ++g_calls[name];
  auto it = g_fail.find(name);
  if (it == g_fail.end() || --it->second) return false;
  g_fail.erase(it);
  g_last = e;
  return true;
}
hipError_t launch(const void* f) {
  if (fails("launch", hipErrorLaunchFailure)) return g_last;
  ++g_launches[g_kernels[f]];
  return hipSuccess;
}
struct Config {
  dim3 grid, block;
  size_t shared;
  hipStream_t stream;
} g_config;
int g_handle;
}  // namespace

#define CALL(name)                                              \
  do {                                                          \
    if (fails(name, hipErrorInvalidValue)) return hipErrorInvalidValue; \
  } while (0)

extern "C" {
long host_hip_calls(const char* name) { return g_calls[name]; }
long host_hip_launches(const char* part) {
  long n = 0;
  for (auto& k : g_launches)
    if (k.first.find(part) != std::string::npos) n += k.second;
  return n;
}
void host_hip_fail(const char* name, long k) {
  g_fail.erase(name);
  if (k > 0) g_fail[name] = k;
}
void* host_hip_pinned(size_t n) {
  for (auto& m : g_pinned)
    if (m.second == n) return m.first;
  return nullptr;
}

void** __hipRegisterFatBinary(const void*) { return (void**)&g_handle; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* f, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
  g_kernels[f] = name;
}
void __hipRegisterVar(void**, void* var, char*, const char*, int, size_t size, int, int) { g_symbols[var] = calloc(1, size); }
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t s, hipStream_t st) {
  g_config = {g, b, s, st};
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* s, hipStream_t* st) {
  *g = g_config.grid, *b = g_config.block, *s = g_config.shared, *st = g_config.stream;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3, dim3, void**, size_t, hipStream_t) { return launch(f); }
hipError_t hipLaunchCooperativeKernel(const void* f, dim3, dim3, void**, unsigned, hipStream_t) { return launch(f); }
hipError_t hipExtLaunchKernel(const void* f, dim3, dim3, void**, size_t, hipStream_t, hipEvent_t, hipEvent_t, int) { return launch(f); }

hipError_t hipGetDeviceCount(int* n) { return *n = 1, hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int d) {
  if (d) return g_last = hipErrorInvalidDevice;
  return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
  memset(p, 0, sizeof *p);
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void*, int, size_t) { return *n = 1, hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "host_hip"; }
hipError_t hipGetLastError() {
  const hipError_t e = g_last;
  g_last = hipSuccess;
  return e;
}

hipError_t hipMalloc(void** p, size_t n) {
  if (fails("hipMalloc", hipErrorOutOfMemory)) return hipErrorOutOfMemory;
  *p = calloc(1, n);
  g_memory[(char*)*p] = n;
  return hipSuccess;
}
hipError_t hipFree(void* p) {
  g_memory.erase((char*)p);
  free(p);
  return hipSuccess;
}
hipError_t hipHostMalloc(void** p, size_t n, unsigned) {
  if (fails("hipHostMalloc", hipErrorOutOfMemory)) return hipErrorOutOfMemory;
  *p = calloc(1, n);
  g_pinned[*p] = n;
  return hipSuccess;
}
hipError_t hipHostFree(void* p) {
  g_pinned.erase(p);
  free(p);
  return hipSuccess;
}
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) {
  CALL("hipMemcpy");
  memmove(d, s, n);
  return hipSuccess;
}
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t) {
  CALL("hipMemcpyAsync");
  memmove(d, s, n);
  return hipSuccess;
}
hipError_t hipMemset(void* d, int v, size_t n) { return memset(d, v, n), hipSuccess; }
hipError_t hipMemsetAsync(void* d, int v, size_t n, hipStream_t) { return memset(d, v, n), hipSuccess; }
hipError_t hipMemGetAddressRange(hipDeviceptr_t* base, size_t* size, hipDeviceptr_t p) {
  auto it = g_memory.upper_bound((char*)p);
  if (it == g_memory.begin() || (char*)p >= (--it)->first + it->second) return g_last = hipErrorNotFound;
  *base = it->first, *size = it->second;
  return hipSuccess;
}
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* a, const void* p) {
  hipDeviceptr_t base;
  size_t size;
  memset(a, 0, sizeof *a);
  if (hipMemGetAddressRange(&base, &size, (hipDeviceptr_t)p) != hipSuccess) return g_last = hipErrorInvalidValue;
  a->type = hipMemoryTypeDevice;
  return hipSuccess;
}
hipError_t hipGetSymbolAddress(void** p, const void* s) { return *p = g_symbols[s], hipSuccess; }

hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = (hipStream_t)&g_handle, hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamQuery(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) {
  CALL("hipStreamSynchronize");
  return hipSuccess;
}
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
hipError_t hipStreamBeginCapture(hipStream_t, hipStreamCaptureMode) { return hipSuccess; }
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t* g) { return *g = (hipGraph_t)&g_handle, hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { return *e = (hipEvent_t)&g_handle, hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return *e = (hipEvent_t)&g_handle, hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { return *ms = 0.f, hipSuccess; }
hipError_t hipGraphInstantiate(hipGraphExec_t* e, hipGraph_t, hipGraphNode_t*, char*, size_t) {
  CALL("hipGraphInstantiate");
  return *e = (hipGraphExec_t)&g_handle, hipSuccess;
}
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t) {
  CALL("hipGraphLaunch");
  return hipSuccess;
}
hipError_t hipGraphDestroy(hipGraph_t) { return hipSuccess; }
hipError_t hipGraphExecDestroy(hipGraphExec_t) { return hipSuccess; }
}
