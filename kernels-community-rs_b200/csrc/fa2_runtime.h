// What the host files of the C ABI share: the error message, the state of a device, and the scope of a call's device.
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace fa2 {

// Message of the last failed call on this thread.
extern thread_local char g_error[512];
// Keeps the message, returns the code.
int fail(int code, const char* fmt, ...);

constexpr int kMaxDevices = 64;

// Per-device state, created on first use (the reference keeps the same kind of lazily built,
// never-freed per-device runtime: flash-attn2-rs/src/host/runtime.rs:68-84).
struct Runtime {
  bool ready = false;
  int sm_count = 0;
  int cc_major = 0;
  int* status = nullptr;  // device status word
};
int get_runtime(int device, Runtime** out);

// A tensor map over [batch][rows][heads][D] of 16-bit (dtype 2: fp32) elements; strides in elements, boxes of box_inner columns and
// box_rows rows, 128-byte swizzle. `wide`: L2 fetches 256 bytes at a time, which
// brings a neighbour's data too where a row's columns are not a multiple of that. The runtime has to be there.
int make_map(CUtensorMap* m, const void* ptr, int dtype, int esize, int64_t d, int64_t heads, int64_t rows, int64_t batch, int64_t head_stride,
             int64_t row_stride, int64_t batch_stride, int box_inner, int box_rows, const char* name, bool wide = true);

// Makes the device that owns `ptr` current for the lifetime of the object and restores the caller's
// device afterwards, as the reference binds the context of q before every launch
// (flash-attn2-rs/src/host/forward/mod.rs:716-718). A pointer the runtime does not know (or a null
// one) leaves the current device as it is.
class DeviceScope {
 public:
  explicit DeviceScope(const void* ptr);
  ~DeviceScope();
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  int device() const { return device_; }

 private:
  int prev_ = 0, device_ = 0;
};

}  // namespace fa2
