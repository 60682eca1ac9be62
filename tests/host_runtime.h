// A stand-in for the HIP runtime, for programs that link the library on a machine without a GPU: memory is addresses that nobody may
// touch, a launch is a line in a list.  The library's calls land here because a program's own symbols go before those of the
// libraries it loads.
#pragma once

#include <cxxabi.h>

#include <cstdlib>
#include <map>
#include <string>
#include <vector>

#include "../burn_dragon_amd/csrc/bdh_internal.h"

namespace host_runtime {

struct Launch {
  std::string kernel;  // as it is written, e.g. "k_packed_few<2, 0, 1, 4, 1, false>"
  dim3 grid, block;
};
// (made where they are first asked for: the library registers its kernels before this program's own objects exist)
inline std::map<const void *, std::string> &kernels() {
  static std::map<const void *, std::string> m;
  return m;
}
inline std::vector<Launch> &launches() {
  static std::vector<Launch> v;
  return v;
}
inline std::map<char *, size_t> &memory() {  // what is allocated
  static std::map<char *, size_t> m;
  return m;
}
inline bool &capturing() {  // streams other than the null stream are
  static bool c = false;
  return c;
}
inline hipStream_t stream() { return reinterpret_cast<hipStream_t>(64); }
inline void *device_address(size_t bytes) {
  static char *next = reinterpret_cast<char *>(size_t(1) << 44);
  char *at = next;
  next += bdh_align_up(bytes, 4096) + 4096;
  return at;
}
inline std::string plain_name(const char *mangled) {
  int status = 0;
  char *text = abi::__cxa_demangle(mangled, nullptr, nullptr, &status);
  std::string s = status == 0 ? text : mangled;
  free(text);
  for (const char *gone : {"(anonymous namespace)::", "void "})
    for (size_t at; (at = s.find(gone)) != std::string::npos;) s.erase(at, strlen(gone));
  int depth = 0;  // the arguments
  for (size_t i = 0; i < s.size(); ++i) {
    if (s[i] == '<') ++depth;
    if (s[i] == '>') --depth;
    if (s[i] == '(' && depth == 0) return s.substr(0, i);
  }
  return s;
}

}  // namespace host_runtime

extern "C" {

hipError_t hipMalloc(void **p, size_t bytes) {
  *p = host_runtime::device_address(bytes);
  host_runtime::memory()[static_cast<char *>(*p)] = bytes;
  return hipSuccess;
}
hipError_t hipFree(void *p) { return !p || host_runtime::memory().erase(static_cast<char *>(p)) ? hipSuccess : hipErrorInvalidValue; }
hipError_t hipMemcpy(void *, const void *, size_t, hipMemcpyKind) { return hipSuccess; }
hipError_t hipMemcpyAsync(void *, const void *, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t s) {
  return s && host_runtime::capturing() ? hipErrorStreamCaptureUnsupported : hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus *status) {
  *status = s && host_runtime::capturing() ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGetDeviceCount(int *n) {
  *n = 1;
  return hipSuccess;
}
hipError_t hipGetDevice(int *d) {
  *d = 0;
  return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDeviceProperties(hipDeviceProp_t *p, int) {
  memset(p, 0, sizeof(*p));
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipGetSymbolAddress(void **p, const void *) {
  *p = host_runtime::device_address(size_t(1) << 26);
  return hipSuccess;
}
hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipLaunchKernel(const void *f, dim3 grid, dim3 block, void **, size_t, hipStream_t) {
  host_runtime::launches().push_back({host_runtime::kernels()[f], grid, block});
  return hipSuccess;
}
void **__hipRegisterFatBinary(const void *) {
  static void *module;
  return &module;
}
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *f, char *, const char *name, unsigned int, void *, void *, void *, void *, int *) {
  host_runtime::kernels()[f] = host_runtime::plain_name(name);
}
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
static dim3 pushed_grid, pushed_block;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t, hipStream_t) {
  pushed_grid = grid;
  pushed_block = block;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *s) {
  *grid = pushed_grid;
  *block = pushed_block;
  *lds = 0;
  *s = nullptr;
  return hipSuccess;
}

}  // extern "C"
