// Element types of the serving operators (MB_F32, MB_BF16, MB_F16) and their
// 16-byte vectors: every operator computes in FP32 and rounds once on output.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "host.h"

namespace mb {

template <class T>
struct Element;

template <>
struct Element<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float to(float x) { return x; }
  static __device__ __forceinline__ float from(float x) { return x; }
  static __device__ __forceinline__ void unpack(uint4 v, float* x) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};

template <>
struct Element<__nv_bfloat16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ void unpack(uint4 v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a bfloat16 is the high half of its FP32 value
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <>
struct Element<__half> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ void unpack(uint4 v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <class T>
struct TypeTag {
  using type = T;
};

// Calls f with a TypeTag of the element type that `dtype` names.
template <class F>
void with_dtype(uint32_t dtype, F&& f) {
  switch (dtype) {
    case MB_F32: return f(TypeTag<float>{});
    case MB_BF16: return f(TypeTag<__nv_bfloat16>{});
    case MB_F16: return f(TypeTag<__half>{});
  }
  throw Error(MB_ERR_INVALID, "dtype must be MB_F32, MB_BF16 or MB_F16");
}

inline void aligned_to(const void* p, size_t bytes, const char* message) {
  require(reinterpret_cast<uintptr_t>(p) % bytes == 0, message);
}

constexpr int kMaxDevices = 64;

inline int current_device() {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  require(e == cudaSuccess && dev < kMaxDevices, "no usable CUDA device", MB_ERR_CUDA);
  return dev;
}

// SMs of the current device.
inline int sm_count() {
  static std::atomic<int> known[kMaxDevices];
  const int dev = current_device();
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    const cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    require(e == cudaSuccess, "no usable CUDA device", MB_ERR_CUDA);
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// A kernel attribute, set once on each device.
class DeviceOnce {
 public:
  template <class F>
  void operator()(F&& set) {
    const uint64_t bit = 1ull << current_device();
    if (done_.load(std::memory_order_acquire) & bit) return;
    const cudaError_t e = set();
    if (e != cudaSuccess) throw Error(MB_ERR_CUDA, std::string("kernel attribute: ") + cudaGetErrorString(e));
    done_.fetch_or(bit, std::memory_order_release);
  }

 private:
  std::atomic<uint64_t> done_{0};
};

inline void launched(const char* what, cudaError_t e = cudaGetLastError()) {
  if (e != cudaSuccess) throw Error(MB_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace mb
