// 8-bit checkpoints of activations: per row and group of 128 channels, with
// a = max |x| over the group,
//
//   code = rint(x * (127 / a)),  scale = a / 127,  value = code * scale,
//
// each operation one rounding in fp32, so the codes are the same wherever they
// are made.  A group with a < 2^-96 (127 / a would overflow) is stored as
// zeros; a group that holds an infinity or a NaN restores to NaN throughout,
// so that a step that has blown up stays visible.
//
// A half-warp holds a group: 16 lanes with 8 consecutive channels each.
#pragma once

#include "operators.cuh"

namespace lama {
namespace ops {

constexpr int GROUP8 = 128;

// Codes (packed, 8 bytes) of this lane's 8 values and the group's scale; every
// lane of the half-warp takes part.  Channels past the row's end hold zeros.
// Integers up to 127 are rounded (half to even) and read off by adding
// 1.5 * 2^23, whose last place is 1: the conversion instructions run at a
// sixteenth of the rate.
// `raw`: the same values as they are in memory (16-bit types are compared as
// such, two a word).
template <class T>
__device__ __forceinline__ uint2 encode8(const Raw8<T>& raw, const float* v, float& scale) {
  uint32_t a = 0;
  if constexpr (sizeof(T) == 2) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; i++) a = __vmaxu2(a, w[i] & 0x7fff7fffu);  // NaN compares above infinity
    a = max(a & 0xffffu, a >> 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) a = max(a, __float_as_uint(v[i]) & 0x7fffffffu);
  }
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) a = max(a, __shfl_xor_sync(~0u, a, m));
  if constexpr (sizeof(T) == 2) {
    const uint16_t h = (uint16_t)a;
    a = __float_as_uint(to_float(*reinterpret_cast<const T*>(&h)));
  }
  const float amax = __uint_as_float(a);
  float inv = 0.f;
  scale = 0.f;
  if (a >= 0x7f800000u) {
    scale = __uint_as_float(0x7fffffffu);
  } else if (amax >= 1.2621774483536189e-29f) {  // 2^-96
    inv = __fdiv_rn(127.f, amax);
    scale = __fdiv_rn(amax, 127.f);
  }
  constexpr float MAGIC = 12582912.f;
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = __fadd_rn(__fmul_rn(v[i + j], inv), MAGIC);  // mul2 and add2 may become one fma
    const uint32_t lo = __byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(x[2]), __float_as_uint(x[3]), 0x0040);
    w[i >> 2] = __byte_perm(lo, hi, 0x5410);
  }
  if (inv == 0.f) w[0] = w[1] = 0;  // zeros, or a group that restores to NaN
  return make_uint2(w[0], w[1]);
}

// The 8 codes times `scale`, rounded once: a byte c + 128 below the exponent
// of 2^23 is the number 2^23 + 128 + c.
__device__ __forceinline__ void decode8(uint2 c, float scale, float* v) {
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const uint32_t w = (i ? c.y : c.x) ^ 0x80808080u;
#pragma unroll
    for (int j = 0; j < 4; j++) v[i + j] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + j));
    add2(v[i], v[i + 1], -8388736.f, -8388736.f);
    add2(v[i + 2], v[i + 3], -8388736.f, -8388736.f);
    mul2(v[i], v[i + 1], scale, scale);
    mul2(v[i + 2], v[i + 3], scale, scale);
  }
}

// 8 elements to p (or n < 8 where the row ends); `vec`: p is 16-byte (fp32:
// two 16-byte words) aligned and n is 8.
template <class T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float* v) {
  if (vec && n >= 8) {
    store_vec<T, 8>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) p[i] = from_float<T>(v[i]);
  }
}
__device__ __forceinline__ uint2 load_codes(const int8_t* p, int n, bool vec) {
  if (vec && n >= 8) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < n) w[i >> 2] |= ((uint32_t)p[i] & 255u) << ((i & 3) * 8);
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(int8_t* p, int n, bool vec, uint2 c) {
  if (vec && n >= 8) {
    *reinterpret_cast<uint2*>(p) = c;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) p[i] = (int8_t)(((i < 4 ? c.x : c.y) >> ((i & 3) * 8)) & 255u);
  }
}

}  // namespace ops
}  // namespace lama
