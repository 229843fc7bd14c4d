// The norm after a block, its gate and residual scale, the residual sum and
// the norm before the next block, in one pass; and its gradients.
//
//   p = w_post y r_y,   r_y = 1 / sqrt(mean y^2 + eps)
//   u = x + s g p       (rounded to the stream's type, which is what is normed next)
//   n = w_pre u r_u,    r_u = 1 / sqrt(mean u^2 + eps)
//
// With D the whole gradient of u, yh = y r_y and uh = u r_u:
//
//   D   = du + r_u (w_pre dn - uh mean(uh w_pre dn)),  dx = D
//   dp  = D s g,   dy = r_y (w_post dp - yh mean(yh w_post dp))
//   dg  = D s w_post yh
//   dw_post = s sum(g D yh),  ds = w_post sum(g D yh),  dw_pre = sum(dn uh)   (sums over rows)
//
// so two sums per channel give every vector gradient, and where the gate is
// one row for many tokens, sum(D yh) over those tokens gives its gradient and,
// times g, the other two.
//
// Both passes are bound by memory: every tensor is read or written once, in 16-byte
// accesses, a row's values staying in registers between its two statistics
// and its outputs.  W warps share a row so that a lane holds at most 16
// channels; the vectors stay in registers over a CTA's rows.  The backward
// pass walks a contiguous range of rows per CTA, keeps the two column sums in
// registers and leaves one partial row per CTA, which a second kernel adds in
// a fixed order: results do not change from run to run.
//
// Checkpoints in 8 bits: the forward pass can store y and u as codes, made
// from the registers it holds anyway, and the backward pass read the codes in their
// place; the statistics r_y and r_u are kept as computed.
#include <algorithm>

#include "checkpoint8.cuh"
#include "ptx.cuh"

namespace lama {
namespace ops {

namespace {

struct Fwd {
  const void *x, *y, *gate;
  void *u, *n;
  const float *w_post, *w_pre, *s;
  float *ry, *ru;
  int8_t *cy, *cu;
  float *sy, *su;
  long long rows, xs, ys, gs, per;  // row strides of x, y and the gate; rows of one gate row
  int c, groups;
  float s0, eps;
  int vec;
};

struct Bwd {
  const void *gu, *gn, *u, *y, *gate;
  const int8_t *cy, *cu;
  const float *sy, *su;
  void *dx, *dy, *dgate;
  const float *w_post, *w_pre, *s, *ry, *ru;
  float *dw_post, *dw_pre, *ds, *part;
  long long rows, gus, gns, us, ys, gs, per;
  int c, groups;   // channels, 128-channel groups of a checkpoint
  int sets, parts;  // gate rows that are summed apart, CTAs of each
  float s0;
  int vec;
};

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

// channel of element 0 of part i of this lane
#define LAMA_CH(i) (((i)*W * 32 + warp * 32 + lane) * 8)

__device__ __forceinline__ void load_vector(const float* w, int c0, int c, float other, float* v) {
#pragma unroll
  for (int j = 0; j < 8; j++) v[j] = c0 + j < c ? (w ? w[c0 + j] : other) : 0.f;
}

template <class T, int W, int NI, bool SAVE8>
__global__ void __launch_bounds__(team_threads<W>) k_norm(const __grid_constant__ Fwd p) {
  constexpr int TEAMS = team_threads<W> / (W * 32);
  __shared__ float slots[TEAMS][2 * W];
  const int lane = threadIdx.x & 31, team = threadIdx.x / (W * 32), warp = (threadIdx.x >> 5) % W;
  int turn = 0;
  float wp[NI][8], wn[NI][8], sc[NI][8];
#pragma unroll
  for (int i = 0; i < NI; i++) {
    load_vector(p.w_post, LAMA_CH(i), p.c, 1.f, wp[i]);
    load_vector(p.w_pre, LAMA_CH(i), p.c, 1.f, wn[i]);
    load_vector(p.s, LAMA_CH(i), p.c, p.s0, sc[i]);
  }
  const float inv_c = 1.f / (float)p.c;
  for (long long row = (long long)blockIdx.x * TEAMS + team; row < p.rows; row += (long long)gridDim.x * TEAMS) {
    float x[NI][8], y[NI][8], g[NI][8];
    const T* px = static_cast<const T*>(p.x) + row * p.xs;
    const T* py = static_cast<const T*>(p.y) + row * p.ys;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      load8(py + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, y[i]);
      load8(px + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, x[i]);
    }
    if (p.gate) {
      const T* pg = static_cast<const T*>(p.gate) + (row / p.per) * p.gs;
#pragma unroll
      for (int i = 0; i < NI; i++) load8(pg + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, g[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) g[i][j] = 1.f;
    }
    if (SAVE8) {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        float scale;
        const uint2 code = encode8(y[i], scale);
        const int n = p.c - LAMA_CH(i);
        store_codes(p.cy + row * p.c + LAMA_CH(i), n, p.vec, code);
        if ((lane & 15) == 0 && n > 0) p.sy[row * p.groups + LAMA_CH(i) / GROUP8] = scale;
      }
    }
    float ry = 1.f;
    if (p.w_post) {
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) q += y[i][j] * y[i][j];
      ry = 1.f / sqrtf(row_sum<W>(q, slots[team], turn, team, warp) * inv_c + p.eps);
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NI; i++) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        x[i][j] += sc[i][j] * g[i][j] * (y[i][j] * ry * wp[i][j]);
        x[i][j] = to_float(from_float<T>(x[i][j]));
        q += x[i][j] * x[i][j];
      }
      store8(static_cast<T*>(p.u) + row * p.c + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, x[i]);
    }
    if (SAVE8 && p.cu) {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        float scale;
        const uint2 code = encode8(x[i], scale);
        const int n = p.c - LAMA_CH(i);
        store_codes(p.cu + row * p.c + LAMA_CH(i), n, p.vec, code);
        if ((lane & 15) == 0 && n > 0) p.su[row * p.groups + LAMA_CH(i) / GROUP8] = scale;
      }
    }
    if (p.w_pre) {
      const float ru = 1.f / sqrtf(row_sum<W>(q, slots[team], turn, team, warp) * inv_c + p.eps);
#pragma unroll
      for (int i = 0; i < NI; i++) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[i][j] *= ru * wn[i][j];
        store8(static_cast<T*>(p.n) + row * p.c + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, x[i]);
      }
      if (p.ru && warp == 0 && lane == 0) p.ru[row] = ru;
    }
    if (p.ry && p.w_post && warp == 0 && lane == 0) p.ry[row] = ry;
  }
}

template <class T, int W, int NI, bool SAVE8>
__global__ void __launch_bounds__(team_threads<W>) k_norm_grad(const __grid_constant__ Bwd p) {
  constexpr int TEAMS = team_threads<W> / (W * 32);
  __shared__ float slots[TEAMS][2 * W];
  __shared__ float sums[TEAMS > 1 ? TEAMS : 1][TEAMS > 1 ? W * NI * 256 : 1];
  const int lane = threadIdx.x & 31, team = threadIdx.x / (W * 32), warp = (threadIdx.x >> 5) % W;
  int turn = 0;
  const float inv_c = 1.f / (float)p.c;
  const int set = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const long long set_rows = p.sets > 1 ? p.per : p.rows;
  const long long each = (set_rows + p.parts - 1) / p.parts;
  const long long r0 = set * set_rows + part * each, r1 = min(r0 + each, min((set + 1) * set_rows, p.rows));
  const bool token_gate = p.gate && p.per == 1;
  float wp[NI][8], wn[NI][8], sc[NI][8], sa[NI][8], sb[NI][8];
#pragma unroll
  for (int i = 0; i < NI; i++) {
    load_vector(p.w_post, LAMA_CH(i), p.c, 1.f, wp[i]);
    load_vector(p.w_pre, LAMA_CH(i), p.c, 1.f, wn[i]);
    load_vector(p.s, LAMA_CH(i), p.c, p.s0, sc[i]);
    if (p.gate && !token_gate) {
      float g[8];
      load8(static_cast<const T*>(p.gate) + set * p.gs + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, g);
#pragma unroll
      for (int j = 0; j < 8; j++) sc[i][j] *= g[j];  // s g, the same for all rows of the set
    }
#pragma unroll
    for (int j = 0; j < 8; j++) sa[i][j] = sb[i][j] = 0.f;
  }
  for (long long row = r0 + team; row < r1; row += TEAMS) {
    float d[NI][8], t[NI][8], y[NI][8];
    float ry = 1.f;
    // y first: its loads are in flight during the first sum
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int n = p.c - LAMA_CH(i);
      if (p.gu) {
        load8(static_cast<const T*>(p.gu) + row * p.gus + LAMA_CH(i), n, p.vec, d[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) d[i][j] = 0.f;
      }
      if (SAVE8)
        decode8(load_codes(p.cy + row * p.c + LAMA_CH(i), n, p.vec),
                n > 0 ? p.sy[row * p.groups + LAMA_CH(i) / GROUP8] : 0.f, y[i]);
      else
        load8(static_cast<const T*>(p.y) + row * p.ys + LAMA_CH(i), n, p.vec, y[i]);
    }
    if (p.w_post) ry = p.ry[row];
    if (p.w_pre && p.gn) {
      const float ru = p.ru[row];
      float uh[NI][8], q = 0.f;
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int n = p.c - LAMA_CH(i);
        load8(static_cast<const T*>(p.gn) + row * p.gns + LAMA_CH(i), n, p.vec, t[i]);
        if (SAVE8)
          decode8(load_codes(p.cu + row * p.c + LAMA_CH(i), n, p.vec),
                  n > 0 ? p.su[row * p.groups + LAMA_CH(i) / GROUP8] : 0.f, uh[i]);
        else
          load8(static_cast<const T*>(p.u) + row * p.us + LAMA_CH(i), n, p.vec, uh[i]);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          uh[i][j] *= ru;
          sb[i][j] += t[i][j] * uh[i][j];
          t[i][j] *= wn[i][j];
          q += uh[i][j] * t[i][j];
        }
      }
      q = row_sum<W>(q, slots[team], turn, team, warp) * inv_c;
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) d[i][j] += ru * (t[i][j] - uh[i][j] * q);
    }
#pragma unroll
    for (int i = 0; i < NI; i++) store8(static_cast<T*>(p.dx) + row * p.c + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, d[i]);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      float g[8];
      if (token_gate) load8(static_cast<const T*>(p.gate) + row * p.gs + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, g);
      float dg[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        y[i][j] *= ry;
        const float a = d[i][j] * y[i][j];
        sa[i][j] += token_gate ? a * g[j] : a;
        dg[j] = a * sc[i][j] * wp[i][j];
        t[i][j] = d[i][j] * sc[i][j] * (token_gate ? g[j] : 1.f) * wp[i][j];  // w_post dp
        q += y[i][j] * t[i][j];
      }
      if (token_gate && p.dgate)
        store8(static_cast<T*>(p.dgate) + row * p.c + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, dg);
    }
    if (p.w_post) {
      q = row_sum<W>(q, slots[team], turn, team, warp) * inv_c;
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) t[i][j] = ry * (t[i][j] - y[i][j] * q);
    }
#pragma unroll
    for (int i = 0; i < NI; i++) store8(static_cast<T*>(p.dy) + row * p.c + LAMA_CH(i), p.c - LAMA_CH(i), p.vec, t[i]);
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
#pragma unroll 8
      for (int i = pi; i < p.parts; i += ps) {
        a += src[(long long)i * 2 * p.c];
        b += src[(long long)i * 2 * p.c + p.c];
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
constexpr int MAX_C = 16384;

int teams(int c) { return c <= 512 ? 4 : c <= 1024 ? 2 : 1; }

// CTAs of a set of rows in the backward pass: about four CTAs a SM in all.
void split(const lama_norm* p, int& sets, int& parts) {
  const bool set_gate = p->gate && p->gate_rows > 1;
  sets = set_gate ? (int)((p->rows + p->gate_rows - 1) / p->gate_rows) : 1;
  const long long rows = set_gate ? std::min(p->gate_rows, p->rows) : p->rows;
  const long long most = (rows + teams(p->channels) - 1) / teams(p->channels);
  parts = (int)std::max<long long>(1, std::min<long long>(most, 148 * 4 / sets));
}

int check(const lama_norm* p, char* err, int err_len) {
  if (err && err_len > 0) err[0] = 0;
  if (!p) return fail(err, err_len, LAMA_EINVAL, "null arguments");
  if (!dtype_ok(p->dtype)) return fail(err, err_len, LAMA_EINVAL, "unknown element type %d", p->dtype);
  if (p->rows < 1 || p->channels < 1) return fail(err, err_len, LAMA_EINVAL, "rows and channels must be positive");
  if (p->channels > MAX_C)
    return fail(err, err_len, LAMA_EUNSUPPORTED, "%d channels exceed %d", p->channels, MAX_C);
  if (p->rows > 0x7fffffffLL) return fail(err, err_len, LAMA_EUNSUPPORTED, "rows exceed 2^31 - 1");
  if (p->gate && p->gate_rows < 1) return fail(err, err_len, LAMA_EINVAL, "gate_rows must be positive");
  if (!(p->eps >= 0.f)) return fail(err, err_len, LAMA_EINVAL, "eps must not be negative");
  return LAMA_OK;
}

bool aligned(const void* p, long long stride, int dtype) {
  return ((uintptr_t)p & 15) == 0 && (stride * dtype_size(dtype)) % 16 == 0;
}

}  // namespace
}  // namespace ops
}  // namespace lama

using namespace lama::ops;

extern "C" int lama_gated_residual_norm(const lama_norm* p, const void* x, long long x_stride, const void* y,
                                        long long y_stride, void* u, void* n, float* post_rstd, float* pre_rstd,
                                        int8_t* y_codes, float* y_scales, int8_t* u_codes, float* u_scales, int device,
                                        void* stream, char* err, int err_len) {
  const int rc = check(p, err, err_len);
  if (rc != LAMA_OK) return rc;
  if (!x || !y || !u || (p->pre_weight && !n)) return fail(err, err_len, LAMA_EINVAL, "x, y, u or n is null");
  if (x_stride < p->channels || y_stride < p->channels)
    return fail(err, err_len, LAMA_EINVAL, "a row stride is below %d channels", p->channels);
  if ((y_codes && !y_scales) || (u_codes && !u_scales) || (u_codes && !y_codes))
    return fail(err, err_len, LAMA_EINVAL, "codes without scales, or of u without those of y");
  Fwd f{};
  f.x = x, f.xs = x_stride, f.y = y, f.ys = y_stride, f.u = u, f.n = n;
  f.gate = p->gate, f.gs = p->gate_stride, f.per = p->gate ? p->gate_rows : 1;
  f.w_post = p->post_weight, f.w_pre = p->pre_weight, f.s = p->residual_scales, f.s0 = p->residual_scale;
  f.ry = post_rstd, f.ru = pre_rstd;
  f.cy = y_codes, f.sy = y_scales, f.cu = u_codes, f.su = u_scales;
  f.rows = p->rows, f.c = p->channels, f.groups = (p->channels + GROUP8 - 1) / GROUP8;
  f.eps = p->eps;
  f.vec = p->channels % 8 == 0 && aligned(x, x_stride, p->dtype) && aligned(y, y_stride, p->dtype) &&
          aligned(u, 0, p->dtype) && aligned(n, 0, p->dtype) && aligned(p->gate, p->gate_stride, p->dtype) &&
          (((uintptr_t)y_codes | (uintptr_t)u_codes) & 7) == 0;
  const int t = teams(f.c);
  const unsigned grid = (unsigned)std::min<long long>((f.rows + t - 1) / t, 148 * 8);
  const cudaStream_t st = (cudaStream_t)stream;
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  auto run = [&](auto tag) {
    using T = decltype(tag);
    return by_width(f.c, [&](auto w, auto ni) {
      constexpr int W = decltype(w)::value, NI = decltype(ni)::value;
      if (f.cy)
        k_norm<T, W, NI, true><<<grid, team_threads<W>, 0, st>>>(f);
      else
        k_norm<T, W, NI, false><<<grid, team_threads<W>, 0, st>>>(f);
      return cudaGetLastError();
    });
  };
  if (ce == cudaSuccess)
    ce = p->dtype == LAMA_F32 ? run(0.f) : p->dtype == LAMA_F16 ? run(__half()) : run(__nv_bfloat16());
  if (ce != cudaSuccess) return fail(err, err_len, LAMA_ECUDA, "gated residual norm: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}

extern "C" long long lama_gated_residual_norm_workspace(const lama_norm* p, char* err, int err_len) {
  const int rc = check(p, err, err_len);
  if (rc != LAMA_OK) return rc;
  int sets, parts;
  split(p, sets, parts);
  return (long long)sets * parts * 2 * p->channels * 4;
}

extern "C" int lama_gated_residual_norm_backward(const lama_norm* p, const lama_norm_grads* g, void* workspace,
                                                 long long workspace_bytes, int device, void* stream, char* err,
                                                 int err_len) {
  const long long need = lama_gated_residual_norm_workspace(p, err, err_len);
  if (need < 0) return (int)need;
  if (!g || !g->grad_x || !g->grad_y) return fail(err, err_len, LAMA_EINVAL, "grad_x or grad_y is null");
  if (!workspace || workspace_bytes < need)
    return fail(err, err_len, LAMA_EINVAL, "workspace of %lld bytes, %lld needed", workspace_bytes, need);
  const bool codes = g->y_codes != nullptr, pre = p->pre_weight && g->grad_n;
  if (codes ? !g->y_scales : !g->y) return fail(err, err_len, LAMA_EINVAL, "neither y nor its checkpoint is given");
  if (pre && (codes ? !g->u_codes || !g->u_scales : !g->u))
    return fail(err, err_len, LAMA_EINVAL, "neither u nor its checkpoint is given");
  if ((p->post_weight && !g->post_rstd) || (pre && !g->pre_rstd))
    return fail(err, err_len, LAMA_EINVAL, "a norm's saved statistics are missing");
  if ((g->grad_u && g->grad_u_stride < p->channels) || (pre && g->grad_n_stride < p->channels) ||
      (!codes && g->y_stride < p->channels) || (pre && !codes && g->u_stride < p->channels))
    return fail(err, err_len, LAMA_EINVAL, "a row stride is below %d channels", p->channels);
  Bwd b{};
  b.gu = g->grad_u, b.gus = g->grad_u_stride, b.gn = g->grad_n, b.gns = g->grad_n_stride;
  b.u = g->u, b.us = g->u_stride, b.y = g->y, b.ys = g->y_stride;
  b.cy = g->y_codes, b.sy = g->y_scales, b.cu = g->u_codes, b.su = g->u_scales;
  b.gate = p->gate, b.gs = p->gate_stride, b.per = p->gate ? p->gate_rows : 1;
  b.w_post = p->post_weight, b.w_pre = p->pre_weight, b.s = p->residual_scales, b.s0 = p->residual_scale;
  b.ry = g->post_rstd, b.ru = g->pre_rstd;
  b.dx = g->grad_x, b.dy = g->grad_y, b.dgate = g->grad_gate;
  b.dw_post = g->grad_post_weight, b.dw_pre = g->grad_pre_weight, b.ds = g->grad_residual_scales;
  b.part = static_cast<float*>(workspace);
  b.rows = p->rows, b.c = p->channels, b.groups = (p->channels + GROUP8 - 1) / GROUP8;
  split(p, b.sets, b.parts);
  const int d = p->dtype;
  b.vec = p->channels % 8 == 0 && aligned(b.gu, b.gus, d) && aligned(b.gn, b.gns, d) &&
          (codes ? (((uintptr_t)b.cy | (uintptr_t)b.cu) & 7) == 0 : aligned(b.u, b.us, d) && aligned(b.y, b.ys, d)) &&
          aligned(b.gate, b.gs, d) && aligned(b.dx, 0, d) && aligned(b.dy, 0, d) && aligned(b.dgate, 0, d);
  const unsigned grid = (unsigned)(b.sets * b.parts);
  const cudaStream_t st = (cudaStream_t)stream;
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  auto run = [&](auto tag) {
    using T = decltype(tag);
    const cudaError_t e = by_width(b.c, [&](auto w, auto ni) {
      constexpr int W = decltype(w)::value, NI = decltype(ni)::value;
      if (codes)
        k_norm_grad<T, W, NI, true><<<grid, team_threads<W>, 0, st>>>(b);
      else
        k_norm_grad<T, W, NI, false><<<grid, team_threads<W>, 0, st>>>(b);
      return cudaGetLastError();
    });
    if (e != cudaSuccess) return e;
    k_norm_sums<T><<<(b.c + 31) / 32, 1024, 0, st>>>(b);
    return cudaGetLastError();
  };
  if (ce == cudaSuccess)
    ce = d == LAMA_F32 ? run(0.f) : d == LAMA_F16 ? run(__half()) : run(__nv_bfloat16());
  if (ce != cudaSuccess)
    return fail(err, err_len, LAMA_ECUDA, "gated residual norm backward: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}
