// A stand-in for the part of the HIP runtime that the C ABI's host code calls,
// for checks without a GPU: a few devices whose memory is host memory. Every
// allocation remembers the device that was current, so that a check can ask
// where a pointer lives. Streams hold no work: calls are done when they return.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <map>

#define __host__
#define __device__
#define __forceinline__ inline
#define __align__(n) __attribute__((aligned(n)))
#define HIP_SYMBOL(x) (&(x))

enum hipError_t { hipSuccess = 0, hipErrorInvalidValue = 1, hipErrorOutOfMemory = 2 };
enum hipMemcpyKind { hipMemcpyHostToDevice = 1, hipMemcpyDeviceToDevice = 3 };
enum hipStreamCaptureStatus { hipStreamCaptureStatusNone = 0, hipStreamCaptureStatusActive = 1 };
enum hipDeviceAttribute_t { hipDeviceAttributeMultiprocessorCount };
constexpr unsigned hipHostMallocCoherent = 1, hipEventDisableTiming = 2;
struct hipDeviceProp_t {
  char gcnArchName[64];
};
typedef struct fakeStream* hipStream_t;
typedef struct fakeEvent* hipEvent_t;

namespace fake_hip {

struct Alloc {
  std::size_t bytes;
  int device;  // -1: pinned host memory
};
struct State {
  int device = 0, devices = 2;
  bool capturing = false;
  std::map<const char*, Alloc> live;
};
inline State& state() {
  static State s;
  return s;
}
// The device of the allocation that holds `p`: -1 pinned, -2 none.
inline int owner(const void* p) {
  const char* c = static_cast<const char*>(p);
  auto it = state().live.upper_bound(c);
  if (it == state().live.begin()) return -2;
  --it;
  return c < it->first + it->second.bytes ? it->second.device : -2;
}
inline hipError_t alloc(void** p, std::size_t n, int device) {
  *p = std::malloc(n ? n : 1);
  if (!*p) return hipErrorOutOfMemory;
  state().live[static_cast<char*>(*p)] = Alloc{n, device};
  return hipSuccess;
}
inline hipError_t release(void* p) {
  state().live.erase(static_cast<char*>(p));
  std::free(p);
  return hipSuccess;
}

}  // namespace fake_hip

inline const char* hipGetErrorString(hipError_t) { return "stand-in error"; }
inline hipError_t hipGetLastError() { return hipSuccess; }
inline hipError_t hipGetDeviceCount(int* n) { return *n = fake_hip::state().devices, hipSuccess; }
inline hipError_t hipGetDevice(int* d) { return *d = fake_hip::state().device, hipSuccess; }
inline hipError_t hipSetDevice(int d) { return fake_hip::state().device = d, hipSuccess; }
inline hipError_t hipDeviceSynchronize() { return hipSuccess; }
inline hipError_t hipGetDeviceProperties(hipDeviceProp_t* p, int) {
  return std::strcpy(p->gcnArchName, "gfx950"), hipSuccess;
}
inline hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
inline hipError_t hipMalloc(void** p, std::size_t n) { return fake_hip::alloc(p, n, fake_hip::state().device); }
template <class T>
hipError_t hipMalloc(T** p, std::size_t n) {
  return hipMalloc(reinterpret_cast<void**>(p), n);
}
inline hipError_t hipFree(void* p) { return p ? fake_hip::release(p) : hipSuccess; }
inline hipError_t hipHostMalloc(void** p, std::size_t n, unsigned) { return fake_hip::alloc(p, n, -1); }
inline hipError_t hipHostFree(void* p) { return p ? fake_hip::release(p) : hipSuccess; }
inline hipError_t hipHostGetDevicePointer(void** d, void* h, unsigned) { return *d = h, hipSuccess; }
inline hipError_t hipMemset(void* p, int v, std::size_t n) { return std::memset(p, v, n), hipSuccess; }
inline hipError_t hipMemsetAsync(void* p, int v, std::size_t n, hipStream_t) { return hipMemset(p, v, n); }
inline hipError_t hipMemcpyAsync(void* d, const void* s, std::size_t n, hipMemcpyKind, hipStream_t) {
  return std::memmove(d, s, n), hipSuccess;
}
inline hipError_t hipMemcpy2DAsync(void* d, std::size_t dp, const void* s, std::size_t sp, std::size_t w, std::size_t h,
                                   hipMemcpyKind, hipStream_t) {
  for (std::size_t i = 0; i < h; ++i) std::memmove(static_cast<char*>(d) + i * dp, static_cast<const char*>(s) + i * sp, w);
  return hipSuccess;
}
inline hipError_t hipGetSymbolAddress(void** p, const void* symbol) {
  return *p = const_cast<void*>(symbol), hipSuccess;
}
inline hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
  return *s = fake_hip::state().capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess;
}
inline hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
inline hipError_t hipEventCreate(hipEvent_t* e) {
  return *e = static_cast<hipEvent_t>(std::malloc(1)), *e ? hipSuccess : hipErrorOutOfMemory;
}
inline hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return hipEventCreate(e); }
inline hipError_t hipEventDestroy(hipEvent_t e) { return std::free(e), hipSuccess; }
inline hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
inline hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
inline hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { return *ms = 0.0f, hipSuccess; }
