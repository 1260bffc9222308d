// host_util.cuh — host-side helpers shared by the C ABI's translation units:
// error messages, the exception guard of the entry points, and the driver's
// tensor-map encoder.
#pragma once

#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <exception>
#include <mutex>
#include <new>

#include "../../include/futon_cuda.h"

namespace {

int set_err(char* err, size_t errlen, int code, const char* fmt, ...) {
  if (err && errlen) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(err, errlen, fmt, ap);
    va_end(ap);
  }
  return code;
}

// The tail of every C entry point: no C++ exception crosses the ABI (a cgo
// or ctypes caller cannot take one); host allocation failure is
// FUTON_ENOMEM, anything else FUTON_ECUDA with its message.
#define FUTON_CATCH(err, errlen)                                                         \
  catch (const std::bad_alloc&) {                                                        \
    return set_err(err, errlen, FUTON_ENOMEM, "native: out of host memory");             \
  }                                                                                      \
  catch (const std::exception& ex_) {                                                    \
    return set_err(err, errlen, FUTON_ECUDA, "native: host exception: %s", ex_.what());  \
  }                                                                                      \
  catch (...) {                                                                          \
    return set_err(err, errlen, FUTON_ECUDA, "native: host exception");                  \
  }

#define CU_TRY(call)                                                                     \
  do {                                                                                   \
    cudaError_t e_ = (call);                                                             \
    if (e_ != cudaSuccess)                                                               \
      return set_err(err, errlen, e_ == cudaErrorMemoryAllocation ? FUTON_ENOMEM : FUTON_ECUDA, \
                     "native: cuda %s (%s:%d)", cudaGetErrorString(e_), __FILE__, __LINE__); \
  } while (0)

// ---------------------------------------------------------------------------
// Tensor maps (TMA descriptors)
// ---------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

}  // namespace
