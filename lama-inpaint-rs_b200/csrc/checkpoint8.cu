// Storing and restoring an activation in 8 bits (the format is in
// checkpoint8.cuh).  Both are one pass bound by memory: a half-warp takes a
// group of 128 channels, a lane 8 of them (16 bytes of a 16-bit type), four
// groups at a time so that their loads are in flight together.  Measured:
// 65536 x 512 bf16 stored in 24 us (4.2 TB/s; two divisions and the packing
// take 63 % of the issue slots) and restored in 14.7 us (6.9 TB/s, part of it
// from L2).
#include <algorithm>
#include <type_traits>

#include "checkpoint8.cuh"
#include "ptx.cuh"

namespace lama {
namespace ops {

namespace {

constexpr int THREADS = 256;
constexpr int PER = 4;                        // groups of a half-warp at a time: their loads go out together
constexpr int PER_CTA = THREADS / 16 * PER;

// Where lane `lane` of group g reads and writes.  FLAT: rows follow one another
// and hold whole groups, so no division is needed (a 64-bit one costs more than the rest).
template <bool FLAT>
struct Place {
  long long x, code;  // offsets of its 8 channels in the tensor and in the codes
  int n;              // how many of them are in the row
  __device__ __forceinline__ Place(long long g, bool on, int lane, long long stride, int c, int groups) {
    if (FLAT) {
      x = code = g * GROUP8 + lane * 8;
      n = on ? 8 : 0;
    } else {
      const long long row = on ? (g >> 31 ? g / groups : (long long)((uint32_t)g / (uint32_t)groups)) : 0;
      const int c0 = on ? (int)(g - row * groups) * GROUP8 + lane * 8 : 0;
      x = row * stride + c0;
      code = row * c + c0;
      n = on ? min(8, c - c0) : 0;
    }
  }
};

template <class T, bool VEC, bool FLAT>
__global__ void __launch_bounds__(THREADS) k_store(const T* x, long long stride, int8_t* codes, float* scales,
                                                   long long rows, int c, int groups) {
  pdl_launch_dependents();
  pdl_wait();
  const long long total = rows * groups;
  const int lane = threadIdx.x & 15, half = threadIdx.x >> 4;
  // every lane of a warp stays in the loop together: encode8 shuffles
  for (long long g0 = (long long)blockIdx.x * PER_CTA; g0 < total; g0 += (long long)gridDim.x * PER_CTA) {
    Raw8<T> raw[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const long long g = g0 + i * (THREADS / 16) + half;
      const Place<FLAT> at(g, g < total, lane, stride, c, groups);
      raw[i] = load_raw<T, VEC>(x + at.x, at.n);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const long long g = g0 + i * (THREADS / 16) + half;
      const Place<FLAT> at(g, g < total, lane, stride, c, groups);
      float v[8], scale;
      raw[i].to(v);
      const uint2 code = encode8(raw[i], v, scale);
      store_codes(codes + at.code, at.n, VEC, code);
      if (g < total && lane == 0) scales[g] = scale;
    }
  }
}

template <class T, bool VEC, bool FLAT>
__global__ void __launch_bounds__(THREADS) k_restore(const int8_t* codes, const float* scales, T* x, long long stride,
                                                     long long rows, int c, int groups) {
  pdl_launch_dependents();
  pdl_wait();
  const long long total = rows * groups;
  const int lane = threadIdx.x & 15, half = threadIdx.x >> 4;
  for (long long g0 = (long long)blockIdx.x * PER_CTA; g0 < total; g0 += (long long)gridDim.x * PER_CTA) {
    uint2 code[PER];
    float scale[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const long long g = g0 + i * (THREADS / 16) + half;
      const Place<FLAT> at(g, g < total, lane, stride, c, groups);
      code[i] = at.n > 0 ? load_codes(codes + at.code, at.n, VEC) : make_uint2(0, 0);
      scale[i] = g < total ? scales[g] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const long long g = g0 + i * (THREADS / 16) + half;
      const Place<FLAT> at(g, g < total, lane, stride, c, groups);
      float v[8];
      decode8(code[i], scale[i], v);
      store8(x + at.x, at.n, VEC, v);
    }
  }
}

// The grid of both, and f(VEC, FLAT).
template <class F>
cudaError_t by_layout(bool vec, int c, long long stride, F&& f) {
  const std::true_type yes;
  const std::false_type no;
  if (!vec) return f(no, no);
  return stride == c && c % GROUP8 == 0 ? f(yes, yes) : f(yes, no);
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
  const unsigned grid = (unsigned)std::min<long long>((rows * groups + PER_CTA - 1) / PER_CTA, 148 * 16);
  const bool vec = vectors(x, codes, dtype, channels, row_stride);
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto* p) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    return by_layout(vec, channels, row_stride, [&](auto v, auto flat) {
      return launch_chained(k_store<T, decltype(v)::value, decltype(flat)::value>, dim3(grid), THREADS, 0, st, p, row_stride,
                            codes, scales, rows, channels, groups);
    });
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
  const unsigned grid = (unsigned)std::min<long long>((rows * groups + PER_CTA - 1) / PER_CTA, 148 * 16);
  const bool vec = vectors(x, codes, dtype, channels, row_stride);
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    return by_layout(vec, channels, row_stride, [&](auto v, auto flat) {
      return launch_chained(k_restore<T, decltype(v)::value, decltype(flat)::value>, dim3(grid), THREADS, 0, st, codes, scales, p,
                            row_stride, rows, channels, groups);
    });
  };
  if (ce == cudaSuccess)
    ce = dtype == LAMA_F32   ? run(static_cast<float*>(x))
         : dtype == LAMA_F16 ? run(static_cast<__half*>(x))
                             : run(static_cast<__nv_bfloat16*>(x));
  if (ce != cudaSuccess) return fail(err, err_len, LAMA_ECUDA, "checkpoint restore: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}
