// Host-side helpers shared by the files that hold entry points: the error text, the per-device record
// of launch planning, occupancy queries and kernel launches.  Defined in norm_abi.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>
#include <unordered_map>

#include "b200norm.h"

namespace b200norm {

constexpr int64_t kMaxRowBytes = 65536;          // the reference's limit (layernorm.py:69-72)
constexpr size_t kMaxSmemPerCta = 227 * 1024;  // opt-in dynamic + static shared memory of one sm_100 CTA

// Stores the thread's error text and returns `code`.
int fail(int code, const char* fmt, ...);

// Whether a buffer (or none) starts on a boundary of its elements, `size` bytes each, a power of two.
inline bool on_element(const void* p, size_t size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) == 0; }
inline int fail_off_element() { return fail(B200NORM_ERR_ARG, "a buffer starts inside an element: its address is no multiple of their size"); }
inline size_t dtype_size(int dtype) { return dtype == B200NORM_F64 ? 8 : dtype == B200NORM_F32 ? 4 : 2; }

struct DeviceState {
  // Launch planning: SM count, occupancies, shared-memory allowances.  Set up without allocating
  // anything, and shared by every entry point -- a kernel's shared-memory allowance is a property
  // of the device, so there must be exactly one record of it per device.
  std::once_flag once;
  cudaError_t init_err = cudaSuccess;
  int sm_count = 0;
  std::mutex mu;
  std::unordered_map<unsigned long long, int> occupancy;  // (kernel, dyn smem) -> CTAs per SM
  std::unordered_map<const void*, size_t> smem_limit;     // kernel -> dynamic shared memory it has been allowed
  // Status word: pinned, mapped host memory where kernels report a timed-out wait.  Allocated by the
  // first call of an entry point that reports through it (never by b200norm_rms_bwd_static).
  std::once_flag status_once;
  cudaError_t status_err = cudaSuccess;
  int* status_host = nullptr;
  int* status_dev = nullptr;
};

// The launch-planning part of the current device's state; allocates nothing.
int device_caches(DeviceState** out);

// The same with the device's status word for bounded waits; the first call on a device allocates it.
int device_state(DeviceState** out);

// Resident CTAs per SM of `fn` at this block size and dynamic shared memory (cluster == 1), or
// resident clusters on the whole device (cluster > 1); cached.
int occupancy(DeviceState& s, const void* fn, int threads, size_t smem, int* out, int cluster = 1);

// `pdl`: launch with programmatic stream serialization (the kernel calls grid_dependency_sync()
// before its first global access).
int launch(const void* fn, dim3 grid, dim3 block, size_t smem, void* params, cudaStream_t stream, bool pdl = true,
           int cluster = 1);

}  // namespace b200norm
