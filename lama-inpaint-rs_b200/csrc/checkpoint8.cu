// Storing and restoring an activation in 8 bits (the format is in
// checkpoint8.cuh).  Both are one pass bound by memory: a half-warp takes a
// group of 128 channels, a lane 8 of them (16 bytes of a 16-bit type).
#include <algorithm>
#include <type_traits>

#include "checkpoint8.cuh"
#include "ptx.cuh"

namespace lama {
namespace ops {

namespace {

constexpr int THREADS = 256;
constexpr int PER_CTA = THREADS / 16;  // groups a CTA takes at a time

template <class T>
__global__ void __launch_bounds__(THREADS) k_store(const T* x, long long stride, int8_t* codes, float* scales,
                                                   long long rows, int c, int groups, bool vec) {
  pdl_launch_dependents();
  pdl_wait();
  const long long total = rows * groups;
  const int lane = threadIdx.x & 15;
  // every lane of a warp stays in the loop together: encode8 shuffles
  for (long long g0 = (long long)blockIdx.x * PER_CTA; g0 < total; g0 += (long long)gridDim.x * PER_CTA) {
    const long long g = g0 + (threadIdx.x >> 4);
    const bool on = g < total;
    const long long row = on ? g / groups : 0;
    const int grp = (int)(g - row * groups), c0 = grp * GROUP8 + lane * 8;
    const int n = on ? min(8, c - c0) : 0;
    float v[8], scale;
    const Raw8<T> raw = vec ? load_raw<T, true>(x + row * stride + c0, n) : load_raw<T, false>(x + row * stride + c0, n);
    raw.to(v);
    const uint2 code = encode8(raw, v, scale);
    store_codes(codes + row * c + c0, n, vec, code);
    if (on && lane == 0) scales[g] = scale;
  }
}

template <class T>
__global__ void __launch_bounds__(THREADS) k_restore(const int8_t* codes, const float* scales, T* x, long long stride,
                                                     long long rows, int c, int groups, bool vec) {
  pdl_launch_dependents();
  pdl_wait();
  const long long total = rows * groups;
  const int lane = threadIdx.x & 15;
  for (long long g = (long long)blockIdx.x * PER_CTA + (threadIdx.x >> 4); g < total;
       g += (long long)gridDim.x * PER_CTA) {
    const long long row = g / groups;
    const int grp = (int)(g - row * groups), c0 = grp * GROUP8 + lane * 8;
    const int n = min(8, c - c0);
    float v[8];
    decode8(load_codes(codes + row * c + c0, n, vec), scales[g], v);
    store8(x + row * stride + c0, n, vec, v);
  }
}

int check(const void* x, const void* codes, const void* scales, int dtype, long long rows, int c, long long stride,
          char* err, int err_len) {
  if (err && err_len > 0) err[0] = 0;
  if (!x || !codes || !scales) return fail(err, err_len, LAMA_EINVAL, "null tensor, codes or scales");
  if (!dtype_ok(dtype)) return fail(err, err_len, LAMA_EINVAL, "unknown element type %d", dtype);
  if (rows < 1 || c < 1) return fail(err, err_len, LAMA_EINVAL, "rows and channels must be positive");
  if (stride < c) return fail(err, err_len, LAMA_EINVAL, "row stride %lld is below %d channels", stride, c);
  if ((uintptr_t)x % dtype_size(dtype) || (uintptr_t)scales % 4)
    return fail(err, err_len, LAMA_EINVAL, "the tensor or the scales are not aligned to their elements");
  return LAMA_OK;
}

bool vectors(const void* x, const void* codes, int dtype, int c, long long stride) {
  return c % 8 == 0 && ((uintptr_t)x & 15) == 0 && (stride * dtype_size(dtype)) % 16 == 0 && ((uintptr_t)codes & 7) == 0;
}

}  // namespace
}  // namespace ops
}  // namespace lama

using namespace lama::ops;

extern "C" int lama_checkpoint_store(const void* x, int dtype, long long rows, int channels, long long row_stride,
                                     int8_t* codes, float* scales, int device, void* stream, char* err, int err_len) {
  const int rc = check(x, codes, scales, dtype, rows, channels, row_stride, err, err_len);
  if (rc != LAMA_OK) return rc;
  const int groups = (channels + GROUP8 - 1) / GROUP8;
  const unsigned grid = (unsigned)std::min<long long>((rows * groups + PER_CTA - 1) / PER_CTA, 148 * 64);
  const bool vec = vectors(x, codes, dtype, channels, row_stride);
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto* p) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    return launch_chained(k_store<T>, dim3(grid), THREADS, 0, st, p, row_stride, codes, scales, rows, channels, groups, vec);
  };
  if (ce == cudaSuccess)
    ce = dtype == LAMA_F32   ? run(static_cast<const float*>(x))
         : dtype == LAMA_F16 ? run(static_cast<const __half*>(x))
                             : run(static_cast<const __nv_bfloat16*>(x));
  if (ce != cudaSuccess) return fail(err, err_len, LAMA_ECUDA, "checkpoint store: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}

extern "C" int lama_checkpoint_restore(const int8_t* codes, const float* scales, int dtype, long long rows, int channels,
                                       long long row_stride, void* x, int device, void* stream, char* err,
                                       int err_len) {
  const int rc = check(x, codes, scales, dtype, rows, channels, row_stride, err, err_len);
  if (rc != LAMA_OK) return rc;
  const int groups = (channels + GROUP8 - 1) / GROUP8;
  const unsigned grid = (unsigned)std::min<long long>((rows * groups + PER_CTA - 1) / PER_CTA, 148 * 64);
  const bool vec = vectors(x, codes, dtype, channels, row_stride);
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    return launch_chained(k_restore<T>, dim3(grid), THREADS, 0, st, codes, scales, p, row_stride, rows, channels, groups, vec);
  };
  if (ce == cudaSuccess)
    ce = dtype == LAMA_F32   ? run(static_cast<float*>(x))
         : dtype == LAMA_F16 ? run(static_cast<__half*>(x))
                             : run(static_cast<__nv_bfloat16*>(x));
  if (ce != cudaSuccess) return fail(err, err_len, LAMA_ECUDA, "checkpoint restore: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}
