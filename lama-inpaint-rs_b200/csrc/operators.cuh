// What the token-mixer operators share: element types, error text, the CUDA
// device guard and the device status word of their bounded waits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <mutex>

#include "lama_b200.h"

namespace lama {
namespace ops {

inline int fail(char* err, int err_len, int code, const char* fmt, ...) {
  if (err && err_len > 0) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(err, (size_t)err_len, fmt, ap);
    va_end(ap);
  }
  return code;
}

// Makes `device` current for the duration of a call and restores the caller's.
// `bind`: the calling thread has the device's context afterwards.  A thread that has
// made no CUDA call yet has none (the device is current all the same, and a launch would bind
// it), and the driver encodes no tensor map for it.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device, bool bind = false) {
    if ((status = cudaGetDevice(&prev_)) == cudaSuccess && (bind || prev_ != device)) {
      status = cudaSetDevice(device);
      moved_ = status == cudaSuccess && prev_ != device;
    }
    if (status != cudaSuccess) cudaGetLastError();  // not sticky: keep it from the caller's next call
  }
  ~DeviceGuard() {
    if (moved_) cudaSetDevice(prev_);
  }
  cudaError_t status = cudaSuccess;

 private:
  int prev_ = 0;
  bool moved_ = false;
};

// The status word of the operators' bounded waits on the current device
// (0: no wait ran out).
cudaError_t status_word(int** p);

// Sets a kernel's dynamic shared-memory limit once per device (`done`: one per
// kernel; the limit only ever has to be at least `bytes`).
constexpr int MAX_DEVICES = 64;
struct SmemLimit {
  std::atomic<int> set[MAX_DEVICES] = {};
  template <class K>
  cudaError_t reach(K* kernel, int bytes) {
    int dev = 0;
    cudaError_t ce = cudaGetDevice(&dev);
    if (ce != cudaSuccess) return ce;
    if (dev < MAX_DEVICES && set[dev].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
    std::lock_guard<std::mutex> lock(mutex);  // two threads' limits: the larger stays
    if (dev < MAX_DEVICES && set[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    ce = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (ce == cudaSuccess && dev < MAX_DEVICES) set[dev].store(bytes, std::memory_order_release);
    return ce;
  }
  std::mutex mutex;
};

// Launch with programmatic stream serialisation: the kernel may start, up to
// its pdl_wait(), while the one before it on the stream ends.  Every kernel of
// the operators calls pdl_launch_dependents() first and pdl_wait() before it
// touches global memory, so the chain of kernels stays ordered.
template <class... KArgs, class... Args>
cudaError_t launch_chained(void (*kernel)(KArgs...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st,
                           const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// Whether any of the pointers is off a multiple of `bytes` (a null pointer is not).
template <class... P>
bool misaligned(int bytes, P... p) {
  return (((uintptr_t)p | ...) & (uintptr_t)(bytes - 1)) != 0;
}
constexpr int WORKSPACE_ALIGN = 16;  // the kernels' widest access

inline int dtype_size(int t) { return t == LAMA_F32 ? 4 : 2; }
inline bool dtype_ok(int t) { return t == LAMA_F32 || t == LAMA_F16 || t == LAMA_BF16; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// N consecutive elements as floats; N * sizeof(T) is 8 or a multiple of 16
// and p is aligned to min(16, N * sizeof(T)).
template <class T, int N>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  constexpr int BYTES = N * (int)sizeof(T);
  if constexpr (BYTES >= 16) {
    constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < BYTES / 16; i++) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[i];
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int j = 0; j < PER; j++) v[i * PER + j] = to_float(e[j]);
    }
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int j = 0; j < N; j++) v[j] = to_float(e[j]);
  }
}
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  constexpr int BYTES = N * (int)sizeof(T);
  if constexpr (BYTES >= 16) {
    constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < BYTES / 16; i++) {
      uint4 u;
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int j = 0; j < PER; j++) e[j] = from_float<T>(v[i * PER + j]);
      reinterpret_cast<uint4*>(p)[i] = u;
    }
  } else {
    uint2 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int j = 0; j < N; j++) e[j] = from_float<T>(v[j]);
    *reinterpret_cast<uint2*>(p) = u;
  }
}

// 8 elements of a row as they are in memory.
template <class T>
struct alignas(16) Raw8 {
  T e[8];
  __device__ __forceinline__ void to(float* v) const {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = to_float(e[i]);
  }
};
template <class T, bool VEC>  // VEC: p is 16-byte aligned, and n is 8 or not positive
__device__ __forceinline__ Raw8<T> load_raw(const T* p, int n) {
  Raw8<T> r;
  if (VEC) {
    if (n > 0)
      r = *reinterpret_cast<const Raw8<T>*>(p);
    else
      memset(&r, 0, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) r.e[i] = i < n ? p[i] : from_float<T>(0.f);
  }
  return r;
}

// Pairs of fp32 in one instruction: (x, y) *= (a, b); (x, y) += (a, b);
// (x, y) = (a, b) * (c, d) + (x, y).  Each element is rounded as by itself.
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 p, q;\n\t"
      "mov.b64 p, {%0, %1};\n\t"
      "mov.b64 q, {%2, %3};\n\t"
      "mul.rn.f32x2 p, p, q;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 p, q;\n\t"
      "mov.b64 p, {%0, %1};\n\t"
      "mov.b64 q, {%2, %3};\n\t"
      "add.rn.f32x2 p, p, q;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float c, float d) {
  asm("{\n\t.reg .b64 p, q, r;\n\t"
      "mov.b64 p, {%0, %1};\n\t"
      "mov.b64 q, {%2, %3};\n\t"
      "mov.b64 r, {%4, %5};\n\t"
      "fma.rn.f32x2 p, q, r, p;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b), "f"(c), "f"(d));
}

}  // namespace ops
}  // namespace lama
