// Kernels of residual_norm.cuh, instantiated for one type in each of
// residual_norm_bf16.cu, residual_norm_f16.cu and residual_norm_f32.cu.
#pragma once

#include "residual_norm.cuh"

namespace lama {
namespace ops {

// Sum over the W warps that share a row.  Two slots take turns, so one barrier a sum is enough.
template <int W>
__device__ __forceinline__ float row_sum(float v, float* slots, int& turn, int team, int warp) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(~0u, v, m);
  if (W == 1) return v;
  float* s = slots + turn * W;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) s[warp] = v;
  named_sync(1 + team, W * 32);
  v = 0.f;
#pragma unroll
  for (int i = 0; i < W; i++) v += s[i];
  return v;
}

template <int W>
constexpr int team_threads = W < 4 ? 128 : W * 32;

// How rows are read.  SCALAR: element by element (odd widths, unaligned rows).
// VECTOR: 16 bytes a lane, the next row's into registers.  RING: whole rows by
// bulk copies into a ring of STAGES rows for each team, so that the bytes in flight take
// no registers (bf16, 131072 x 512 with 8-bit checkpoints: forward 180 us,
// backward 319 us with VECTOR).
enum Mode { SCALAR = 0, VECTOR = 1, RING = 2 };
constexpr int STAGES = 3;

// channel of element 0 of part i of this lane
#define LAMA_CH(i) (((i)*W * 32 + warp * 32 + lane) * 8)

// The per-channel factors of a CTA's rows, in shared memory: [0] s and, where
// the rows share a gate row, that; [1] w_pre; [2] w_post.  FOLDED: [0] times
// w_post, no [2].
template <class T, bool FOLDED, class P>
__device__ __forceinline__ void fill_factors(const P& p, int set, bool set_gate, float* f) {
  for (int c = threadIdx.x; c < p.c; c += blockDim.x) {
    float a = p.s ? p.s[c] : p.s0;
    const float w = p.w_post ? p.w_post[c] : 1.f;
    if (FOLDED) a *= w;
    if (set_gate) a *= to_float(static_cast<const T*>(p.gate)[set * p.gs + c]);
    f[c] = a;
    f[p.c + c] = p.w_pre ? p.w_pre[c] : 1.f;
    if (!FOLDED) f[2 * p.c + c] = w;
  }
}
__device__ __forceinline__ void factors8(const float* f, int c0, int c, float* v) {
  if ((c & 3) == 0) {  // the rows of the table stay 16-byte aligned
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c0 + 4 * h < c) x = *reinterpret_cast<const float4*>(f + c0 + 4 * h);
      v[4 * h] = x.x, v[4 * h + 1] = x.y, v[4 * h + 2] = x.z, v[4 * h + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = c0 + j < c ? f[c0 + j] : 0.f;
  }
}

// A CTA's rows: part `part` of set `set` (sets: runs of rows with one gate row
// where the gate has several for many rows, else all rows).
struct Span {
  int set;
  long long r0, r1;
};
template <class P>
__device__ __forceinline__ Span rows_of(const P& p) {
  Span s;
  s.set = blockIdx.x / p.parts;
  const int part = blockIdx.x % p.parts;
  const long long n = p.sets > 1 ? p.per : p.rows, each = (n + p.parts - 1) / p.parts;
  s.r0 = s.set * n + part * each;
  s.r1 = min(s.r0 + each, min((s.set + 1) * n, p.rows));
  return s;
}

// The rows of a team in flight: row k of the team in stage k % STAGES.
//
// A stage is filled again only once the loads that read it have been performed,
// which each warp reports on a second barrier of the stage.  A named barrier or
// __syncwarp is not enough: it orders the warps' own accesses, which go through one
// pipe, but a load can still be queued there when a bulk copy, which does not go through it,
// lands (with those, rows of 5453 x 2048 fp32 were seen with wrong values).
constexpr int BARS = 2 * STAGES;  // of a team
template <int W>
struct Ring {
  uint32_t bars, base, bytes;  // the team's barriers and stages in shared memory, bytes of a stage
  bool leader;     // this thread's warp issues the team's copies
  int issued = 0;  // leader: rows
  __device__ __forceinline__ void init(uint64_t* b, uint32_t data, uint32_t n, int t, bool lead, int arrivals) {
    bars = smem_u32(b + t * BARS);
    base = data + (uint32_t)t * STAGES * n;
    bytes = n;
    leader = lead;
    if (leader && (threadIdx.x & 31) == 0) {
      for (int i = 0; i < STAGES; i++) {
        mbar_init(bars + 8 * i, arrivals);
        mbar_init(bars + 8 * (STAGES + i), W);
      }
      fence_mbar_init();
    }
    __syncwarp();
  }
  __device__ __forceinline__ uint32_t stage(int k) const { return base + (k % STAGES) * bytes; }
  __device__ __forceinline__ uint32_t bar(int k) const { return bars + 8 * (k % STAGES); }
  // A wait that runs out is recorded and the row computed from what is there: the
  // team's warps stay together at their barriers.
  __device__ __forceinline__ void wait(int k, int* failed) const {
    mbar_wait(bar(k), (uint32_t)(k / STAGES) & 1, failed, 31);
    __syncwarp();
  }
  // this warp has read row k
  __device__ __forceinline__ void release(int k) const {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar(k) + 8 * STAGES);
  }
  // leader: every warp of the team has
  __device__ __forceinline__ void wait_read(int k, int* failed) const {
    mbar_wait(bar(k) + 8 * STAGES, (uint32_t)(k / STAGES) & 1, failed, 32);
    __syncwarp();
  }
  // leader, at the end: where a wait ran out, the copies in flight land before the CTA leaves
  __device__ __forceinline__ void drain() const {
    for (int k = issued > STAGES ? issued - STAGES : 0; k < issued; k++)
      mbar_wait_drain(bar(k), (uint32_t)(k / STAGES) & 1);
  }
};
__device__ __forceinline__ void copy4(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// one of the barrier's arrivals, once this thread's copies so far have landed
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float shared_float(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}
template <class T>
__device__ __forceinline__ Raw8<T> shared_raw(uint32_t at, int n) {
  Raw8<T> r;
  uint4* q = reinterpret_cast<uint4*>(&r);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r) / 16); i++) {
    q[i] = make_uint4(0, 0, 0, 0);
    if (n > 0)
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(q[i].x), "=r"(q[i].y), "=r"(q[i].z), "=r"(q[i].w)
                   : "r"(at + 16 * i));
  }
  return r;
}
__device__ __forceinline__ uint2 shared_codes(uint32_t at, int n) {
  uint2 c = make_uint2(0, 0);
  if (n > 0) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(c.x), "=r"(c.y) : "r"(at));
  return c;
}

template <class T, int W, int NI, bool SAVE8, int MODE, bool TOKEN>  // TOKEN: a gate for each row
__global__ void __launch_bounds__(team_threads<W>, W <= 4 ? 5 : 1) k_norm(const __grid_constant__ Fwd p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int TEAMS = team_threads<W> / (W * 32);
  __shared__ float slots[TEAMS][2 * W];
  extern __shared__ __align__(16) float factors[];
  const int lane = threadIdx.x & 31, team = threadIdx.x / (W * 32), warp = (threadIdx.x >> 5) % W;
  int turn = 0;
  const float inv_c = 1.f / (float)p.c;
  const Span span = rows_of(p);
  constexpr bool token_gate = TOKEN;
  constexpr bool VEC = MODE != SCALAR;
  __shared__ uint64_t bars[MODE == RING ? TEAMS * BARS : 1];
  __shared__ int failed;
  if (threadIdx.x == 0) failed = 0;
  Raw8<T> rx[NI], ry_[NI], rg[NI];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int n = p.c - LAMA_CH(i);
      ry_[i] = load_raw<T, VEC>(static_cast<const T*>(p.y) + row * p.ys + LAMA_CH(i), n);
      rx[i] = load_raw<T, VEC>(static_cast<const T*>(p.x) + row * p.xs + LAMA_CH(i), n);
      if (token_gate) rg[i] = load_raw<T, VEC>(static_cast<const T*>(p.gate) + row * p.gs + LAMA_CH(i), n);
    }
  };
  long long row = span.r0 + team;
  Ring<W> ring;
  const uint32_t rb = (uint32_t)p.c * sizeof(T);  // bytes of a row
  auto issue = [&](long long r) {  // leader: a row into the ring
    const uint32_t at = ring.stage(ring.issued), bar = ring.bar(ring.issued);
    if (lane == 0) {
      mbar_arrive_expect_tx(bar, token_gate ? 3 * rb : 2 * rb);
      bulk_load(at, static_cast<const T*>(p.y) + r * p.ys, rb, bar);
      bulk_load(at + rb, static_cast<const T*>(p.x) + r * p.xs, rb, bar);
      if (token_gate) bulk_load(at + 2 * rb, static_cast<const T*>(p.gate) + r * p.gs, rb, bar);
    }
    ring.issued++;
  };
  if (MODE == RING) {
    ring.init(bars, smem_u32(factors) + 12 * p.c, (token_gate ? 3 : 2) * rb, team, warp == 0, 1);
    if (ring.leader)
      for (int k = 0; k < STAGES && row + k * TEAMS < span.r1; k++) issue(row + k * TEAMS);
  } else if (row < span.r1) {
    fetch(row);
  }
  fill_factors<T, false>(p, span.set, p.gate && !token_gate, factors);
  __syncthreads();
  int k = 0;  // rows of the team so far
  const int left = p.c - LAMA_CH(0);  // of this lane's row from its first channel on
  const long long at0 = row * p.c + LAMA_CH(0);
  const int step = TEAMS * p.c;
  T *pu = static_cast<T*>(p.u) + at0, *pn = static_cast<T*>(p.n) + at0;
  int8_t *cy = p.cy + at0, *cu = p.cu + at0;
  float *sy = p.sy + row * p.groups + LAMA_CH(0) / GROUP8, *su = p.su + row * p.groups + LAMA_CH(0) / GROUP8;
  auto codes = [&](const Raw8<T>* raw, const float (*v)[8], int8_t* codes, float* scales) {
#pragma unroll
    for (int i = 0; i < NI; i++) {
      float scale;
      const uint2 code = encode8(raw[i], v[i], scale);
      store_codes(codes + i * W * 256, left - i * W * 256, VEC, code);
      if ((lane & 15) == 0 && left > i * W * 256) scales[i * W * 2] = scale;
    }
  };
  for (; row < span.r1; row += TEAMS, k++, pu += step, pn += step, cy += step, cu += step, sy += TEAMS * p.groups,
                        su += TEAMS * p.groups) {
    float x[NI][8], y[NI][8];
    if (MODE == RING) {
      ring.wait(k, &failed);
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const uint32_t at = ring.stage(k) + LAMA_CH(i) * sizeof(T);
        const int n = p.c - LAMA_CH(i);
        ry_[i] = shared_raw<T>(at, n);
        rx[i] = shared_raw<T>(at + rb, n);
        if (token_gate) rg[i] = shared_raw<T>(at + 2 * rb, n);
      }
    }
#pragma unroll
    for (int i = 0; i < NI; i++) {
      rx[i].to(x[i]);
      ry_[i].to(y[i]);
    }
    if (MODE == RING) ring.release(k);
    float ry = 1.f;
    if (p.w_post) {
      float q0 = 0.f, q1 = 0.f;
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 8; j += 2) fma2(q0, q1, y[i][j], y[i][j + 1], y[i][j], y[i][j + 1]);
      ry = rsqrtf(row_sum<W>(q0 + q1, slots[team], turn, team, warp) * inv_c + p.eps);
    }
    if (MODE == RING && ring.leader && row + STAGES * TEAMS < span.r1) {
      ring.wait_read(k, &failed);
      issue(row + STAGES * TEAMS);
    }
    if (SAVE8) codes(ry_, y, cy, sy);
    Raw8<T> u[NI];
    float q0 = 0.f, q1 = 0.f;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      float f[8], w[8];
      factors8(factors, LAMA_CH(i), p.c, f);
      factors8(factors + 2 * p.c, LAMA_CH(i), p.c, w);
      if (token_gate) {
        float g[8];
        rg[i].to(g);
#pragma unroll
        for (int j = 0; j < 8; j += 2) mul2(f[j], f[j + 1], g[j], g[j + 1]);
      }
      // each operation of x + (s g) ((y r_y) w_post) rounded by itself: u decides codes that a contracted sum would flip
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        mul2(y[i][j], y[i][j + 1], ry, ry);
        mul2(y[i][j], y[i][j + 1], w[j], w[j + 1]);
        x[i][j] = __fadd_rn(x[i][j], __fmul_rn(f[j], y[i][j]));
        x[i][j + 1] = __fadd_rn(x[i][j + 1], __fmul_rn(f[j + 1], y[i][j + 1]));
        u[i].e[j] = from_float<T>(x[i][j]);
        u[i].e[j + 1] = from_float<T>(x[i][j + 1]);
      }
      u[i].to(x[i]);  // the stream carries the rounded sum
#pragma unroll
      for (int j = 0; j < 8; j += 2) fma2(q0, q1, x[i][j], x[i][j + 1], x[i][j], x[i][j + 1]);
      store8(pu + i * W * 256, left - i * W * 256, VEC, x[i]);
    }
    if (MODE != RING && row + TEAMS < span.r1) fetch(row + TEAMS);  // in flight during the second half
    if (SAVE8 && p.cu) codes(u, x, cu, su);
    if (p.w_pre) {
      const float ru = rsqrtf(row_sum<W>(q0 + q1, slots[team], turn, team, warp) * inv_c + p.eps);
#pragma unroll
      for (int i = 0; i < NI; i++) {
        float f[8];
        factors8(factors + p.c, LAMA_CH(i), p.c, f);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          mul2(x[i][j], x[i][j + 1], ru, ru);
          mul2(x[i][j], x[i][j + 1], f[j], f[j + 1]);
        }
        store8(pn + i * W * 256, left - i * W * 256, VEC, x[i]);
      }
      if (p.ru && warp == 0 && lane == 0) p.ru[row] = ru;
    }
    if (p.ry && p.w_post && warp == 0 && lane == 0) p.ry[row] = ry;
  }
  if (MODE == RING && ring.leader && failed) {
    ring.drain();
    if (lane == 0) atomicCAS(p.status, 0, failed);
  }
}

// y or u of the backward pass, as such or as codes with their scale
template <class T, bool SAVE8>
struct Saved {
  Raw8<T> raw;
  uint2 code;
  float scale;
  __device__ __forceinline__ void to(float r, float* v) const {  // times r
    if (SAVE8) {
      decode8(code, scale * r, v);
    } else {
      raw.to(v);
#pragma unroll
      for (int j = 0; j < 8; j += 2) mul2(v[j], v[j + 1], r, r);
    }
  }
};

template <class T, int W, int NI, bool SAVE8, int MODE, bool TOKEN>  // TOKEN: a gate for each row
__global__ void __launch_bounds__(team_threads<W>, W <= 4 ? 4 : 1) k_norm_grad(const __grid_constant__ Bwd p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int TEAMS = team_threads<W> / (W * 32);
  __shared__ float slots[TEAMS][2 * W];
  __shared__ float sums[TEAMS > 1 ? TEAMS : 1][TEAMS > 1 ? W * NI * 256 : 1];
  extern __shared__ __align__(16) float factors[];
  const int lane = threadIdx.x & 31, team = threadIdx.x / (W * 32), warp = (threadIdx.x >> 5) % W;
  int turn = 0;
  const float inv_c = 1.f / (float)p.c;
  const Span span = rows_of(p);
  constexpr bool token_gate = TOKEN;
  const bool pre = p.w_pre && p.gn;
  float sa[NI][8], sb[NI][8];
#pragma unroll
  for (int i = 0; i < NI; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) sa[i][j] = sb[i][j] = 0.f;
  constexpr bool VEC = MODE != SCALAR;
  __shared__ uint64_t bars[MODE == RING ? TEAMS * BARS : 1];
  __shared__ int failed;
  if (threadIdx.x == 0) failed = 0;
  Raw8<T> rd[NI], rn[NI], rg[NI];
  Saved<T, SAVE8> sy[NI], su[NI];
  float ry = 1.f, ru = 0.f;
  auto saved = [&](Saved<T, SAVE8>& s, const void* x, long long stride, const int8_t* codes, const float* scales,
                   long long row, int c0) {
    const int n = p.c - c0;
    if (SAVE8) {
      s.code = load_codes(codes + row * p.c + c0, n, VEC);
      s.scale = n > 0 ? scales[row * p.groups + c0 / GROUP8] : 0.f;
    } else {
      s.raw = load_raw<T, VEC>(static_cast<const T*>(x) + row * stride + c0, n);
    }
  };
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int c0 = LAMA_CH(i), n = p.c - c0;
      if (pre) saved(su[i], p.u, p.us, p.cu, p.su, row, c0);
      saved(sy[i], p.y, p.ys, p.cy, p.sy, row, c0);
      if (pre) rn[i] = load_raw<T, VEC>(static_cast<const T*>(p.gn) + row * p.gns + c0, n);
      rd[i] = load_raw<T, VEC>(static_cast<const T*>(p.gu) + row * p.gus + c0, p.gu ? n : 0);
      if (token_gate) rg[i] = load_raw<T, VEC>(static_cast<const T*>(p.gate) + row * p.gs + c0, n);
    }
    if (p.w_post) ry = p.ry[row];
    if (pre) ru = p.ru[row];
  };
  long long row = span.r0 + team;
  Ring<W> ring;
  const uint32_t rb = (uint32_t)p.c * sizeof(T), sb8 = SAVE8 ? (uint32_t)p.c : rb;  // bytes of a row, of a saved row
  // a stage: y, then grad_u, grad_n, u and the gate as far as they are there
  const uint32_t o_d = sb8, o_n = o_d + (p.gu ? rb : 0), o_u = o_n + (pre ? rb : 0), o_g = o_u + (pre ? sb8 : 0),
                 o_end = o_g + (token_gate ? rb : 0);
  // then the two statistics and, of codes, the scales of y and of u: 4-byte copies by the leader's lanes
  // (loaded a row ahead into registers they were waited for: 316 us at 131072 x 512)
  const uint32_t extras = 2 + (SAVE8 ? 2 * (uint32_t)p.groups : 0), o_stage = o_end + (4 * extras + 15) / 16 * 16;
  auto issue = [&](long long r) {
    const uint32_t at = ring.stage(ring.issued), bar = ring.bar(ring.issued);
    for (uint32_t i = lane; i < extras; i += 32) {
      const float* src = nullptr;
      if (i == 0)
        src = p.w_post ? p.ry + r : nullptr;
      else if (i == 1)
        src = pre ? p.ru + r : nullptr;
      else if (i < 2 + (uint32_t)p.groups)
        src = p.sy + r * p.groups + (i - 2);
      else if (pre)
        src = p.su + r * p.groups + (i - 2 - p.groups);
      if (src) copy4(at + o_end + 4 * i, src);
    }
    copies_arrive(bar);
    ring.issued++;
    if (lane != 0) return;
    mbar_arrive_expect_tx(bar, o_end);
    auto kept = [&](uint32_t dst, const void* x, long long stride, const int8_t* codes) {
      if (SAVE8)
        bulk_load(dst, codes + r * p.c, sb8, bar);
      else
        bulk_load(dst, static_cast<const T*>(x) + r * stride, rb, bar);
    };
    if (pre) {
      bulk_load(at + o_n, static_cast<const T*>(p.gn) + r * p.gns, rb, bar);
      kept(at + o_u, p.u, p.us, p.cu);
    }
    if (p.gu) bulk_load(at + o_d, static_cast<const T*>(p.gu) + r * p.gus, rb, bar);
    kept(at, p.y, p.ys, p.cy);
    if (token_gate) bulk_load(at + o_g, static_cast<const T*>(p.gate) + r * p.gs, rb, bar);
  };
  if (MODE == RING) {
    ring.init(bars, smem_u32(factors) + 8 * p.c, o_stage, team, warp == 0, 33);
    if (ring.leader)
      for (int k = 0; k < STAGES && row + k * TEAMS < span.r1; k++) issue(row + k * TEAMS);
  }
  if (MODE != RING && row < span.r1) fetch(row);
  fill_factors<T, true>(p, span.set, p.gate && !token_gate, factors);
  __syncthreads();
  int k = 0;  // rows of the team so far
  T *dx = static_cast<T*>(p.dx) + row * p.c + LAMA_CH(0), *dy = static_cast<T*>(p.dy) + row * p.c + LAMA_CH(0);
  const int left = p.c - LAMA_CH(0);  // of this lane's row from its first channel on
  for (; row < span.r1; row += TEAMS, k++, dx += TEAMS * p.c, dy += TEAMS * p.c) {
    if (MODE == RING) ring.wait(k, &failed);
    auto from_ring = [&](Saved<T, SAVE8>& s, uint32_t at, uint32_t scales, int c0) {
      if (SAVE8) {
        s.code = shared_codes(at + c0, p.c - c0);
        s.scale = c0 < p.c ? shared_float(scales + 4 * (c0 / GROUP8)) : 0.f;
      } else {
        s.raw = shared_raw<T>(at + c0 * sizeof(T), p.c - c0);
      }
    };
    if (MODE == RING) {
      if (p.w_post) ry = shared_float(ring.stage(k) + o_end);
      if (pre) ru = shared_float(ring.stage(k) + o_end + 4);
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const uint32_t at = ring.stage(k);
        const int c0 = LAMA_CH(i), n = p.c - c0;
        if (pre) {
          from_ring(su[i], at + o_u, at + o_end + 8 + 4 * p.groups, c0);
          rn[i] = shared_raw<T>(at + o_n + c0 * sizeof(T), n);
        }
      }
    }
    float d[NI][8];  // D
    auto stream = [&] {  // grad_u
#pragma unroll
      for (int i = 0; i < NI; i++) {
        if (MODE == RING) rd[i] = shared_raw<T>(ring.stage(k) + o_d + LAMA_CH(i) * sizeof(T), p.gu ? p.c - LAMA_CH(i) : 0);
        rd[i].to(d[i]);
      }
    };
    if (!pre) {
      stream();
    } else {
      float uh[NI][8], t[NI][8], q0 = 0.f, q1 = 0.f;
#pragma unroll
      for (int i = 0; i < NI; i++) {
        float f[8];
        factors8(factors + p.c, LAMA_CH(i), p.c, f);
        su[i].to(ru, uh[i]);
        rn[i].to(t[i]);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          fma2(sb[i][j], sb[i][j + 1], t[i][j], t[i][j + 1], uh[i][j], uh[i][j + 1]);
          mul2(t[i][j], t[i][j + 1], f[j], f[j + 1]);
          fma2(q0, q1, t[i][j], t[i][j + 1], uh[i][j], uh[i][j + 1]);
        }
      }
      const float q = -ru * (row_sum<W>(q0 + q1, slots[team], turn, team, warp) * inv_c);
      stream();
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          fma2(d[i][j], d[i][j + 1], t[i][j], t[i][j + 1], ru, ru);
          fma2(d[i][j], d[i][j + 1], uh[i][j], uh[i][j + 1], q, q);
        }
    }
#pragma unroll
    for (int i = 0; i < NI; i++) store8(dx + i * W * 256, left - i * W * 256, VEC, d[i]);
    float y[NI][8], q0 = 0.f, q1 = 0.f;
    if (MODE == RING) {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const uint32_t at = ring.stage(k);
        from_ring(sy[i], at, at + o_end + 8, LAMA_CH(i));
        if (token_gate) rg[i] = shared_raw<T>(at + o_g + LAMA_CH(i) * sizeof(T), p.c - LAMA_CH(i));
      }
      ring.release(k);
    }
#pragma unroll
    for (int i = 0; i < NI; i++) {
      float f[8], g[8];
      factors8(factors, LAMA_CH(i), p.c, f);
      sy[i].to(ry, y[i]);
      if (token_gate) {
        float dg[8];
        rg[i].to(g);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float a0 = d[i][j], a1 = d[i][j + 1];
          mul2(a0, a1, y[i][j], y[i][j + 1]);
          fma2(sa[i][j], sa[i][j + 1], a0, a1, g[j], g[j + 1]);
          mul2(a0, a1, f[j], f[j + 1]);
          dg[j] = a0, dg[j + 1] = a1;
          mul2(f[j], f[j + 1], g[j], g[j + 1]);
        }
        if (p.dgate) store8(static_cast<T*>(p.dgate) + row * p.c + LAMA_CH(i), p.c - LAMA_CH(i), VEC, dg);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j += 2) fma2(sa[i][j], sa[i][j + 1], d[i][j], d[i][j + 1], y[i][j], y[i][j + 1]);
      }
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        mul2(d[i][j], d[i][j + 1], f[j], f[j + 1]);  // w_post dp
        fma2(q0, q1, d[i][j], d[i][j + 1], y[i][j], y[i][j + 1]);
      }
    }
    const float r = ry;
    if (MODE != RING && row + TEAMS < span.r1) fetch(row + TEAMS);  // in flight during the last sum and the stores
    if (MODE == RING && ring.leader && row + STAGES * TEAMS < span.r1) {
      ring.wait_read(k, &failed);
      issue(row + STAGES * TEAMS);
    }
    if (p.w_post) {
      const float q = -r * (row_sum<W>(q0 + q1, slots[team], turn, team, warp) * inv_c);
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          mul2(d[i][j], d[i][j + 1], r, r);
          fma2(d[i][j], d[i][j + 1], y[i][j], y[i][j + 1], q, q);
        }
    }
#pragma unroll
    for (int i = 0; i < NI; i++) store8(dy + i * W * 256, left - i * W * 256, VEC, d[i]);
  }
  if (MODE == RING && ring.leader && failed) {
    ring.drain();
    if (lane == 0) atomicCAS(p.status, 0, failed);
  }
  // this CTA's column sums: part[cta][0] = sum D yh (times the gate where each token has one), [1] = sum dn uh
  float* dst = p.part + (long long)blockIdx.x * 2 * p.c;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    if (TEAMS == 1) {
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (LAMA_CH(i) + j < p.c) dst[k * p.c + LAMA_CH(i) + j] = k ? sb[i][j] : sa[i][j];
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) sums[team][LAMA_CH(i) + j] = k ? sb[i][j] : sa[i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < p.c; c += team_threads<W>) {
        float v = 0.f;
#pragma unroll
        for (int t = 0; t < TEAMS; t++) v += sums[t][c];
        dst[k * p.c + c] = v;
      }
    }
  }
}

// The vector gradients from the partial rows.  32 channels a CTA; its 32 warps
// are split between sets and parts, added up in a fixed order.
template <class T>
__global__ void __launch_bounds__(1024) k_norm_sums(const __grid_constant__ Bwd p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float sa[32][33], sb[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  int ps = 1;  // warps that share a set
  while (ps * 2 * p.sets <= 32) ps *= 2;
  const int ns = 32 / ps, si = warp / ps, pi = warp % ps;
  const bool set_gate = p.gate && p.per > 1, on = c < p.c;
  float s = 0.f, w = 0.f, ta = 0.f, tb = 0.f;
  if (on) {
    s = p.s ? p.s[c] : p.s0;
    w = p.w_post ? p.w_post[c] : 1.f;
  }
  for (int s0 = 0; s0 < p.sets; s0 += ns) {
    const int set = s0 + si;
    float a = 0.f, b = 0.f;
    if (on && set < p.sets) {
      const float* src = p.part + (long long)set * p.parts * 2 * p.c + c;
      constexpr int BATCH = 10;  // rows whose loads are in flight together
      for (int i0 = pi; i0 < p.parts; i0 += BATCH * ps) {
        float x[BATCH], y[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
          const int i = i0 + k * ps;
          x[k] = i < p.parts ? src[(long long)i * 2 * p.c] : 0.f;
          y[k] = i < p.parts ? src[(long long)i * 2 * p.c + p.c] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
          a += x[k];
          b += y[k];
        }
      }
    }
    sa[warp][lane] = a;
    sb[warp][lane] = b;
    __syncthreads();
    if (pi == 0 && on && set < p.sets) {
      for (int i = 1; i < ps; i++) {
        a += sa[warp + i][lane];
        b += sb[warp + i][lane];
      }
      if (set_gate) {
        if (p.dgate) static_cast<T*>(p.dgate)[(long long)set * p.c + c] = from_float<T>(a * s * w);
        a *= to_float(static_cast<const T*>(p.gate)[set * p.gs + c]);
      }
      ta += a;
      tb += b;
    }
    __syncthreads();
  }
  sa[warp][lane] = ta;
  sb[warp][lane] = tb;
  __syncthreads();
  if (warp == 0 && on) {
    ta = tb = 0.f;
    for (int i = 0; i < 32; i++) {
      ta += sa[i][lane];
      tb += sb[i][lane];
    }
    if (p.dw_post) p.dw_post[c] = s * ta;
    if (p.ds) p.ds[c] = w * ta;
    if (p.dw_pre) p.dw_pre[c] = tb;
  }
}

// Warps that share a row: a lane holds 8 channels (rows up to 256) or 16.
template <class F>
cudaError_t by_width(int c, F&& f) {
  using std::integral_constant;
  if (c <= 256) return f(integral_constant<int, 1>(), integral_constant<int, 1>());
  if (c <= 512) return f(integral_constant<int, 1>(), integral_constant<int, 2>());
  if (c <= 1024) return f(integral_constant<int, 2>(), integral_constant<int, 2>());
  if (c <= 2048) return f(integral_constant<int, 4>(), integral_constant<int, 2>());
  if (c <= 4096) return f(integral_constant<int, 8>(), integral_constant<int, 2>());
  if (c <= 8192) return f(integral_constant<int, 16>(), integral_constant<int, 2>());
  return f(integral_constant<int, 32>(), integral_constant<int, 2>());
}
constexpr int STATIC_SMEM = 12 * 1024;  // the kernels' static arrays, at most

template <auto KERNEL, class P>
cudaError_t start(unsigned grid, int threads, size_t smem, cudaStream_t st, const P& p) {
  static SmemLimit limit;
  if (smem > 48 * 1024 - STATIC_SMEM) {
    const cudaError_t e = limit.reach(KERNEL, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return launch_chained(KERNEL, dim3(grid), (unsigned)threads, smem, st, p);
}

// Adds a CTA's rings to its factors' bytes, if they leave room for a second
// CTA of four warps, or for one of more.
template <int W>
bool ring_fits(size_t row_bytes, size_t& smem) {
  constexpr int TEAMS = team_threads<W> / (W * 32);
  const size_t with = smem + TEAMS * STAGES * row_bytes;
  if (with + STATIC_SMEM > (size_t)(W <= 4 ? 227 * 1024 / 2 : 227 * 1024)) return false;
  smem = with;
  return true;
}

template <class T>
cudaError_t run_forward(const Fwd& f, cudaStream_t st) {
  return by_width(f.c, [&](auto w, auto ni) {
    constexpr int W = decltype(w)::value, NI = decltype(ni)::value, TH = team_threads<W>;
    const unsigned grid = (unsigned)(f.sets * f.parts);
    size_t smem = 3 * sizeof(float) * (size_t)f.c;
    const size_t row = (size_t)f.c * sizeof(T) * (f.gate && f.per == 1 ? 3 : 2);
    const int mode = !f.vec ? SCALAR : ring_fits<W>(row, smem) ? RING : VECTOR;
    auto go = [&](auto save8, auto token) {
      constexpr bool S = decltype(save8)::value, G = decltype(token)::value;
      return mode == RING     ? start<k_norm<T, W, NI, S, RING, G>>(grid, TH, smem, st, f)
             : mode == VECTOR ? start<k_norm<T, W, NI, S, VECTOR, G>>(grid, TH, smem, st, f)
                              : start<k_norm<T, W, NI, S, SCALAR, G>>(grid, TH, smem, st, f);
    };
    const std::true_type yes;
    const std::false_type no;
    const bool token = f.gate && f.per == 1;
    return f.cy ? (token ? go(yes, yes) : go(yes, no)) : (token ? go(no, yes) : go(no, no));
  });
}

template <class T>
cudaError_t run_backward(const Bwd& b, cudaStream_t st) {
  const cudaError_t e = by_width(b.c, [&](auto w, auto ni) {
    constexpr int W = decltype(w)::value, NI = decltype(ni)::value, TH = team_threads<W>;
    const unsigned grid = (unsigned)(b.sets * b.parts);
    size_t smem = 2 * sizeof(float) * (size_t)b.c;
    const bool codes = b.cy != nullptr, pre = b.w_pre && b.gn;
    const size_t kept = (size_t)b.c * (codes ? 1 : sizeof(T)), full = (size_t)b.c * sizeof(T);
    const size_t row = kept * (pre ? 2 : 1) + full * ((b.gu != nullptr) + pre + (b.gate && b.per == 1)) +
                       (8 + (codes ? 8 * (size_t)b.groups : 0) + 15) / 16 * 16;
    const int mode = !b.vec ? SCALAR
                     : (!codes || ((uintptr_t)b.cy | (uintptr_t)b.cu | b.c) % 16 == 0) && ring_fits<W>(row, smem) ? RING
                                                                                                                  : VECTOR;
    auto go = [&](auto save8, auto token) {
      constexpr bool S = decltype(save8)::value, G = decltype(token)::value;
      return mode == RING     ? start<k_norm_grad<T, W, NI, S, RING, G>>(grid, TH, smem, st, b)
             : mode == VECTOR ? start<k_norm_grad<T, W, NI, S, VECTOR, G>>(grid, TH, smem, st, b)
                              : start<k_norm_grad<T, W, NI, S, SCALAR, G>>(grid, TH, smem, st, b);
    };
    const std::true_type yes;
    const std::false_type no;
    const bool token = b.gate && b.per == 1;
    return codes ? (token ? go(yes, yes) : go(yes, no)) : (token ? go(no, yes) : go(no, no));
  });
  if (e != cudaSuccess) return e;
  return launch_chained(k_norm_sums<T>, dim3((b.c + 31) / 32), 1024, 0, st, b);
}

}  // namespace ops
}  // namespace lama
