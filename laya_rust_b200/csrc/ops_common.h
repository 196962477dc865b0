// Host helpers shared by the operators on caller-owned device buffers:
// status-code guards, argument checks and the device switch.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <exception>
#include <new>
#include <stdexcept>
#include <string>

#include "../../include/laya_ops.h"

namespace laya {

void set_last_error(const char* msg);

struct OpError : std::runtime_error {
  int code;
  OpError(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

inline void op_check(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return;
  cudaGetLastError();  // a failed call leaves nothing behind for the next one
  throw OpError(LAYA_E_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

inline void op_require(bool ok, const char* msg) {
  if (!ok) throw OpError(LAYA_E_INVALID, msg);
}

// Runs f; an exception becomes a status and the thread's last error.
template <class F>
int op_guard(F&& f) {
  try {
    f();
    set_last_error("");
    return LAYA_OK;
  } catch (const OpError& e) {
    set_last_error(e.what());
    return e.code;
  } catch (const std::bad_alloc&) {
    set_last_error("out of host memory");
    return LAYA_E_INVALID;
  } catch (const std::exception& e) {
    set_last_error(e.what());
    return LAYA_E_INVALID;
  }
}

// The number of devices, asked once it is known (a failed query is repeated).
inline int device_count() {
  static std::atomic<int> known{0};
  int n = known.load(std::memory_order_relaxed);
  if (n > 0) return n;
  op_check(cudaGetDeviceCount(&n), "cudaGetDeviceCount");
  known.store(n, std::memory_order_relaxed);
  return n;
}

// SMs of a device (one that exists), asked once.
inline int device_sms(int device) {
  static std::atomic<int> known[64] = {};
  int n = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  op_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device), "device query");
  if (device < 64) known[device].store(n, std::memory_order_relaxed);
  return n;
}

// Makes `device` current and restores the caller's device on the way out.
struct DeviceScope {
  int prev = -1;
  explicit DeviceScope(int device) {
    if (device < 0 || device >= device_count()) throw OpError(LAYA_E_INVALID, "device out of range");
    op_check(cudaGetDevice(&prev), "cudaGetDevice");
    if (prev == device) {
      prev = -1;
      return;
    }
    op_check(cudaSetDevice(device), "cudaSetDevice");
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
};

// Refuses an address that is not memory of `device` (a host address would
// fault the GPU, another device's would be read over the link).
inline void require_device_ptr(const void* p, int device, const char* what) {
  cudaPointerAttributes a{};
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    throw OpError(LAYA_E_INVALID, std::string(what) + ": not a device address");
  }
  if (a.type == cudaMemoryTypeManaged) return;
  if (a.type != cudaMemoryTypeDevice) throw OpError(LAYA_E_INVALID, std::string(what) + ": not a device address");
  if (a.device != device) throw OpError(LAYA_E_INVALID, std::string(what) + ": memory of another device");
}

}  // namespace laya
