// host_common.hpp -- host helpers shared by the C entry points that launch
// work: the device scope, HIP error reporting, the device check and the
// library-owned workspaces.
#pragma once

#include <hip/hip_runtime_api.h>

#include <string>

#include "abi_common.hpp"

namespace ullm {

// Makes `device` current for the scope and restores the caller's device.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (hipGetDevice(&prev_) != hipSuccess) {
      prev_ = -1;
    }
    err_ = prev_ == device ? hipSuccess : hipSetDevice(device);
    if (prev_ == device) {
      prev_ = -1;  // nothing to restore
    }
  }
  ~DeviceScope() {
    if (prev_ >= 0) {
      (void)hipSetDevice(prev_);
    }
  }
  hipError_t error() const { return err_; }

 private:
  int prev_ = -1;
  hipError_t err_ = hipSuccess;
};

inline ullm_status_t hip_fail(ullm_error_sink_t *sink, const char *what,
                              hipError_t err) {
  const ullm_status_t st = err == hipErrorOutOfMemory
                               ? ULLM_STATUS_OUT_OF_MEMORY
                               : ULLM_STATUS_HIP_RUNTIME_ERROR;
  return write_errorf(sink, st,
                      std::string(what) + ": " + hipGetErrorName(err));
}

#define HIP_TRY(sink, what, expr)              \
  do {                                         \
    const hipError_t e_ = (expr);              \
    if (e_ != hipSuccess) {                    \
      return ::ullm::hip_fail(sink, what, e_); \
    }                                          \
  } while (0)

inline ullm_status_t check_device(int device, ullm_error_sink_t *sink) {
  int count = 0;
  const hipError_t err = hipGetDeviceCount(&count);
  if (err != hipSuccess || count == 0) {
    return write_error(sink, ULLM_STATUS_HIP_UNAVAILABLE,
                       "no HIP device is visible");
  }
  if (device < 0 || device >= count) {
    return write_error(sink, ULLM_STATUS_INVALID_ARGUMENT,
                       "device ordinal is out of range");
  }
  hipDeviceProp_t prop;
  HIP_TRY(sink, "hipGetDeviceProperties", hipGetDeviceProperties(&prop, device));
  if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0) {
    return write_errorf(sink, ULLM_STATUS_UNSUPPORTED,
                        std::string("device architecture ") + prop.gcnArchName +
                            " is not gfx950");
  }
  return ULLM_STATUS_OK;
}

// The library-owned workspace of at least `need` bytes for a call on `device`
// and `stream` (linear_api.cpp).
ullm_status_t library_workspace(int device, const void *stream, bool zeroed,
                                uint64_t need, void **out,
                                ullm_error_sink_t *error_sink);

}  // namespace ullm
