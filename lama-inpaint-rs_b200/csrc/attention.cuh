// What the whole-sequence kernels of linear attention share: a run of the
// recurrence (roles, strides, cut into segments) and operand descriptors.
#pragma once

#include <cudaTypedefs.h>
#include <type_traits>

#include "operators.cuh"
#include "ptx.cuh"

namespace lama {
namespace ops {

constexpr int CH = 128;         // tokens of a chunk (the MMA's M)
constexpr int FINE = 4 * CH;    // tokens up to which the pipelined kernel keeps scores in two parts
constexpr uint32_t TILE = 128 * 128;  // bytes of 128 rows x 64 bf16, 128-byte swizzle
constexpr uint32_t ETILE = 64 * 128;  // 64 rows x 64 bf16

// One operand: element (token, d) of the head's row at
// p + batch * sb + token * st + head * sh + d.
struct Operand {
  const void* p;
  long long sb, st, sh;
  int per;  // heads of the run that share one head of the operand
  int vec;  // rows are 16-byte aligned and a multiple of 16 bytes long
  int hs, bs;  // 0 where all heads or batches are the same memory
};

struct Run {
  Operand a, b, c;
  void* out;  // element (token, d) of head h at out + batch * ob + token * ot + h * oh + d
  long long ob, ot, oh;
  int out_f32;  // out is fp32 whatever the inputs are
  int out_vec;
  const float* log_decay;
  const int* lengths;
  const float* init;  // [batch][heads] of [da][dc], element (r, c) at r * ir + c * ic
  float* fin;
  long long ir, ic, fr, fc;
  float* seg;  // [batch*heads][nseg][slabs*64][blocks*64]: states of the segments, element (r, c) of one
  long long sr, sc;  // at r * sr + c * sc (another run's states may be read transposed)
  int* status;
  float inter, intra, update;  // scales of a E, of the scores, of b c^T
  int batch, tokens, heads, da, dc;
  int reverse;     // walk backwards in time; the initial state is not decayed, the final one is
  int nseg, chunks;  // segments of a sequence, chunks of a segment
  int pipe;        // attention_pipe.cu runs it: segments stay where they are when it runs backwards
  int staged;      // the segments' states are made first and scanned
  int fine;        // scores in two parts (attention_pipe.cu)
  int blocks;      // 64-column blocks of c
  int slabs;       // 64-column slabs of a and b
};

__device__ __forceinline__ float power(float g, int n) { return n == 0 ? 1.f : expf(g * (float)n); }

__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t lbo) {
  // MN-major, 128-byte swizzle: 64-element blocks `lbo` bytes apart, groups of 8 k-rows 1024 apart
  return smem_desc(saddr, 1024, 2) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16);
}

// true in one lane of the (converged) warp
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void sts16(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t swz(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(a, b);
  }
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (std::is_same_v<T, __half>)
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  else
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));  // bf16: the upper half of an fp32
}
// v[0..7] into N parts of type T, 16 bytes each (part p holds what parts 0..p-1 left over)
template <int N, class T>
__device__ __forceinline__ void split8(const float* v, uint4* out) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; i++) r[i] = v[i];
#pragma unroll
  for (int p = 0; p < N; p++) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w[i] = pack2<T>(r[2 * i], r[2 * i + 1]);
      if (p + 1 < N) {
        const float2 h = unpack2<T>(w[i]);
        r[2 * i] -= h.x;
        r[2 * i + 1] -= h.y;
      }
    }
    out[p] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// 8 results of a row, `left` of them inside it
template <class T>
__device__ __forceinline__ void store_row(T* dst, const float* v, int left, int vec) {
  if (vec && left >= 8) {
    store_vec<T, 8>(dst, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < left) dst[i] = from_float<T>(v[i]);
  }
}

constexpr uint32_t A_MN = 1u << 15, B_MN = 1u << 16;

// Runs that go through the kernels together, one after another in the grid:
// up to three of one sequence length, cut alike.
struct Maps {
  CUtensorMap a, b, c, o;
};
struct Set {
  Run run[3];
  Maps maps[3];
  int n;
};
// The run of this CTA; `id` becomes its number within the run.
__device__ __forceinline__ int run_of(const Set& set, int segs, int& id) {
  int w = 0;
  for (; w + 1 < set.n; w++) {
    const int n = set.run[w].batch * set.run[w].heads * set.run[w].blocks * segs;
    if (id < n) break;
    id -= n;
  }
  return w;
}
inline long long ctas(const Set& set, int segs) {
  long long n = 0;
  for (int w = 0; w < set.n; w++) n += (long long)set.run[w].batch * set.run[w].heads * set.run[w].blocks * segs;
  return n;
}

// The pipelined kernel of attention_pipe.cu.  encode_maps: false where TMA
// cannot address the operands.  The runs of a set have one direction and one
// number of slabs.  `states`: only the states that the segments add, into seg.
bool encode_maps(Run& r, Maps& m);
cudaError_t launch_pipe(const Set& set, int dtype, bool states, cudaStream_t st);

}  // namespace ops
}  // namespace lama
