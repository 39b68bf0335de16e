// az_ops.hip.h -- what the operator files (az_sample.hip, az_norm.hip, az_ortho.hip) share: element types, the launch device,
// wave reductions.  Everything is static / inline: no device code crosses a file.
#ifndef AZ_OPS_HIP_H
#define AZ_OPS_HIP_H

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/az_engine.h"

void tower_set_error(const std::string &msg);     // az_tower.hip (az_tower_last_error)
int tower_device(hipStream_t stream, int *dev);  // az_tower.hip: the device that owns the stream (current device for the NULL stream)

namespace azops {

// launches belong to the stream's GPU, whatever device the calling thread has current
struct DeviceGuard {
  int dev = -1, back = -1;
  bool ok = false;
  explicit DeviceGuard(hipStream_t s) {
    int cur = 0;
    if (tower_device(s, &dev) != 0 || dev < 0 || hipGetDevice(&cur) != hipSuccess) return;
    if (dev != cur) {
      if (hipSetDevice(dev) != hipSuccess) return;
      back = cur;
    }
    ok = true;
  }
  ~DeviceGuard() { if (back >= 0) (void)hipSetDevice(back); }
};

// nothing may leave a C entry point but its status: a message that cannot be stored is dropped
inline int fail(int code, const char *msg) noexcept {
  try { tower_set_error(msg); } catch (...) {}
  return code;
}

inline int launched(const char *what) noexcept {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return AZ_OK;
  try { tower_set_error(std::string(what) + " launch: " + hipGetErrorString(e)); } catch (...) {}
  return AZ_EHIP;
}

inline bool misaligned(const void *p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

// 16-bit formats as raw bits: the widening is exact, the narrowing rounds to nearest even (half a step: at most 2^-8 of a bf16's value, 2^-11 of an f16's)
struct bf16_t { uint16_t b; };
struct f16_t { _Float16 h; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float((uint32_t)v.b << 16); }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)v.h; }
__device__ __forceinline__ void from_f32(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f32(float v, bf16_t &o) { o.b = __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ void from_f32(float v, f16_t &o) { o.h = (_Float16)v; }

// one 32-bit register of a tensor as floats and back: one f32, or two 16-bit elements (they stay packed in registers)
template <class T> struct Word;
template <> struct Word<float> {
  static constexpr int N = 1;
  static __device__ __forceinline__ float get(uint32_t w, int) { return __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t put(const float *v) { return __float_as_uint(v[0]); }
};
template <> struct Word<bf16_t> {
  static constexpr int N = 2;
  static __device__ __forceinline__ float get(uint32_t w, int i) { return __uint_as_float(i ? w & 0xFFFF0000u : w << 16); }
  static __device__ __forceinline__ uint32_t put(const float *v) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, b2{(__bf16)v[0], (__bf16)v[1]});
  }
};
template <> struct Word<f16_t> {
  static constexpr int N = 2;
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ float get(uint32_t w, int i) { return (float)__builtin_bit_cast(h2, w)[i]; }
  static __device__ __forceinline__ uint32_t put(const float *v) { return __builtin_bit_cast(uint32_t, h2{(_Float16)v[0], (_Float16)v[1]}); }
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

}  // namespace azops

#endif
