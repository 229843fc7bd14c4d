// Entry points of the gated residual norm (the operator is described in
// residual_norm.cuh).
#include <algorithm>

#include "residual_norm.cuh"

namespace lama {
namespace ops {

namespace {

constexpr int MAX_C = 16384;

int teams(int c) { return c <= 512 ? 4 : c <= 1024 ? 2 : 1; }

// CTAs of a set of rows: `most_ctas` in all where there are rows enough, fewer
// of the wide ones, which a SM holds fewer of and which fill longer tables of
// factors (2000 x 8000, bf16, forward and backward: 169 us, 247 with as many).
void split(const lama_norm* p, int most_ctas, int& sets, int& parts) {
  const bool set_gate = p->gate && p->gate_rows > 1;
  sets = set_gate ? (int)((p->rows + p->gate_rows - 1) / p->gate_rows) : 1;
  const long long rows = set_gate ? std::min<long long>(p->gate_rows, p->rows) : p->rows;
  const long long most = (rows + teams(p->channels) - 1) / teams(p->channels);
  if (p->channels > 4096)
    most_ctas = 148;
  else if (p->channels > 2048)
    most_ctas = 148 * 2;
  parts = (int)std::max<long long>(1, std::min<long long>(most, most_ctas / sets));
}
constexpr int FWD_CTAS = 148 * 5, BWD_CTAS = 148 * 4;

int check(const lama_norm* p, char* err, int err_len) {
  if (err && err_len > 0) err[0] = 0;
  if (!p) return fail(err, err_len, LAMA_EINVAL, "null arguments");
  if (!dtype_ok(p->dtype)) return fail(err, err_len, LAMA_EINVAL, "unknown element type %d", p->dtype);
  if (p->rows < 1 || p->channels < 1) return fail(err, err_len, LAMA_EINVAL, "rows and channels must be positive");
  if (p->channels > MAX_C)
    return fail(err, err_len, LAMA_EUNSUPPORTED, "%d channels exceed %d", p->channels, MAX_C);
  if (p->rows > 0x7fffffffLL) return fail(err, err_len, LAMA_EUNSUPPORTED, "rows exceed 2^31 - 1");
  if (p->gate && p->gate_rows < 1) return fail(err, err_len, LAMA_EINVAL, "gate_rows must be positive");
  if (misaligned(dtype_size(p->dtype), p->gate) || misaligned(4, p->post_weight, p->pre_weight, p->residual_scales))
    return fail(err, err_len, LAMA_EINVAL, "the gate, a weight or residual_scales is not aligned to its elements");
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
  if (misaligned(dtype_size(p->dtype), x, y, u, n) || misaligned(4, post_rstd, pre_rstd, y_scales, u_scales))
    return fail(err, err_len, LAMA_EINVAL, "a tensor, a statistic or a checkpoint's scales are not aligned to their elements");
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
  split(p, FWD_CTAS, f.sets, f.parts);
  const cudaStream_t st = (cudaStream_t)stream;
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  if (ce == cudaSuccess) ce = status_word(&f.status);
  if (ce == cudaSuccess)
    ce = p->dtype == LAMA_F32   ? run_forward<float>(f, st)
         : p->dtype == LAMA_F16 ? run_forward<__half>(f, st)
                                : run_forward<__nv_bfloat16>(f, st);
  if (ce != cudaSuccess) return fail(err, err_len, LAMA_ECUDA, "gated residual norm: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}

extern "C" long long lama_gated_residual_norm_workspace(const lama_norm* p, char* err, int err_len) {
  const int rc = check(p, err, err_len);
  if (rc != LAMA_OK) return rc;
  int sets, parts;
  split(p, BWD_CTAS, sets, parts);
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
  if (misaligned(WORKSPACE_ALIGN, workspace))
    return fail(err, err_len, LAMA_EINVAL, "the workspace is not aligned to %d bytes", WORKSPACE_ALIGN);
  if (misaligned(dtype_size(p->dtype), g->grad_u, g->grad_n, g->y, g->u, g->grad_x, g->grad_y, g->grad_gate) ||
      misaligned(4, g->y_scales, g->u_scales, g->post_rstd, g->pre_rstd, g->grad_post_weight, g->grad_pre_weight,
                 g->grad_residual_scales))
    return fail(err, err_len, LAMA_EINVAL, "a tensor, a statistic or a vector's gradient is not aligned to its elements");
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
  split(p, BWD_CTAS, b.sets, b.parts);
  const int d = p->dtype;
  b.vec = p->channels % 8 == 0 && aligned(b.gu, b.gus, d) && aligned(b.gn, b.gns, d) &&
          (codes ? (((uintptr_t)b.cy | (uintptr_t)b.cu) & 7) == 0 : aligned(b.u, b.us, d) && aligned(b.y, b.ys, d)) &&
          aligned(b.gate, b.gs, d) && aligned(b.dx, 0, d) && aligned(b.dy, 0, d) && aligned(b.dgate, 0, d);
  const cudaStream_t st = (cudaStream_t)stream;
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  if (ce == cudaSuccess) ce = status_word(&b.status);
  if (ce == cudaSuccess)
    ce = d == LAMA_F32   ? run_backward<float>(b, st)
         : d == LAMA_F16 ? run_backward<__half>(b, st)
                         : run_backward<__nv_bfloat16>(b, st);
  if (ce != cudaSuccess)
    return fail(err, err_len, LAMA_ECUDA, "gated residual norm backward: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}
