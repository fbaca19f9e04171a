// The HIP entry points that libnva.so calls, over host memory and without a device: kernel launches
// only count, copies are memcpy, streams and events are dummies.  Loaded before the library, it lets
// the CPU tests run the library's own host side (checks, plans, uploads, errors) anywhere.  Host and
// device allocations can be told to fail from the n-th on.
#include <cstddef>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <new>

namespace {
struct Dim3 {
  uint32_t x, y, z;
};
constexpr int kOk = 0, kOutOfMemory = 2;
long host_left = -1, device_left = -1;  // allocations until they fail; < 0: never
long launches = 0;
int capturing = 0, last_error = kOk;
bool spent(long &left) { return left >= 0 && (left == 0 || left-- == 0); }
struct Config {
  Dim3 grid, block;
  size_t shared;
  void *stream;
} config;
void *symbol_memory = nullptr;
}  // namespace

void *operator new(size_t n) {
  if (spent(host_left)) throw std::bad_alloc();
  void *p = malloc(n ? n : 1);
  if (!p) throw std::bad_alloc();
  return p;
}
void operator delete(void *p) noexcept { free(p); }
void operator delete(void *p, size_t) noexcept { free(p); }

extern "C" {
void stub_fail_host_after(long n) { host_left = n; }
void stub_fail_device_after(long n) { device_left = n; }
long stub_host_left() { return host_left; }
long stub_device_left() { return device_left; }
long stub_launches() { return launches; }
void stub_set_capturing(int on) { capturing = on; }

void *__hipRegisterFatBinary(const void *) {
  static void *module;
  return &module;
}
void __hipUnregisterFatBinary(void *) {}
void __hipRegisterFunction(void *, const void *, char *, const char *, unsigned, void *, void *,
                           void *, void *, int *) {}
void __hipRegisterVar(void *, void *, char *, char *, int, size_t, int, int) {}
int __hipPushCallConfiguration(Dim3 grid, Dim3 block, size_t shared, void *stream) {
  config = {grid, block, shared, stream};
  return kOk;
}
int __hipPopCallConfiguration(Dim3 *grid, Dim3 *block, size_t *shared, void **stream) {
  *grid = config.grid;
  *block = config.block;
  *shared = config.shared;
  *stream = config.stream;
  return kOk;
}
int hipLaunchKernel(const void *, Dim3, Dim3, void **, size_t, void *) {
  launches++;
  return kOk;
}
int hipOccupancyMaxActiveBlocksPerMultiprocessor(int *blocks, const void *, int, size_t) {
  *blocks = 2;
  return kOk;
}

int hipGetDeviceCount(int *n) { return *n = 1, kOk; }
int hipGetDevice(int *d) { return *d = 0, kOk; }
int hipSetDevice(int) { return kOk; }
int hipGetDevicePropertiesR0600(void *, int) { return 1; }  // the library's defaults
const char *hipGetErrorString(int e) { return e == kOutOfMemory ? "out of memory" : "error"; }
int hipGetLastError() {  // of a call that failed, once
  const int e = last_error;
  last_error = kOk;
  return e;
}

static int allocate(void **p, size_t n) {
  *p = nullptr;
  if (spent(device_left)) return last_error = kOutOfMemory;
  *p = calloc(1, n ? n : 1);
  return *p ? kOk : kOutOfMemory;
}
int hipMalloc(void **p, size_t n) { return allocate(p, n); }
int hipHostMalloc(void **p, size_t n, unsigned) { return allocate(p, n); }
int hipFree(void *p) { return free(p), kOk; }
int hipHostFree(void *p) { return free(p), kOk; }
int hipMemGetInfo(size_t *f, size_t *t) { return *f = *t = (size_t)1 << 34, kOk; }
int hipMemcpy(void *d, const void *s, size_t n, int) { return memcpy(d, s, n), kOk; }
int hipMemcpyAsync(void *d, const void *s, size_t n, int, void *) { return memcpy(d, s, n), kOk; }
int hipMemset(void *d, int v, size_t n) { return memset(d, v, n), kOk; }
int hipMemsetAsync(void *d, int v, size_t n, void *) { return memset(d, v, n), kOk; }
int hipGetSymbolAddress(void **p, const void *) {
  if (!symbol_memory) symbol_memory = calloc(1, (size_t)128 << 20);
  return *p = symbol_memory, kOk;
}

int hipStreamCreateWithFlags(void **s, unsigned) { return *s = malloc(1), kOk; }
int hipStreamDestroy(void *s) { return free(s), kOk; }
int hipStreamSynchronize(void *) { return kOk; }
int hipStreamWaitEvent(void *, void *, unsigned) { return kOk; }
int hipStreamIsCapturing(void *, int *status) { return *status = capturing, kOk; }
int hipEventCreate(void **e) { return *e = malloc(1), kOk; }
int hipEventCreateWithFlags(void **e, unsigned) { return *e = malloc(1), kOk; }
int hipEventDestroy(void *e) { return free(e), kOk; }
int hipEventRecord(void *, void *) { return kOk; }
int hipEventSynchronize(void *) { return kOk; }
int hipEventElapsedTime(float *ms, void *, void *) { return *ms = 0.001f, kOk; }
}
