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
// channels.  A CTA walks a contiguous range of rows with its per-channel
// factors in shared memory and loads the next row while it finishes one; the
// backward pass keeps the two column sums in registers and leaves one partial
// row per CTA, which a second kernel adds in a fixed order: results do not
// change from run to run.
//
// Measured: 131072 x 512 bf16 with 8-bit checkpoints, forward 157 us (4.3
// TB/s), backward 147 us (4.6 TB/s) and 10 us for the vectors; 4096 x 512
// forward 6.8 us.  Four or five CTAs of four one-row teams a SM; two warps a
// row of 512 channels (half the registers) measured 1.4-1.8 times slower.
//
// Checkpoints in 8 bits: the forward pass can store y and u as codes, made
// from the registers it holds anyway, and the backward pass read the codes in their
// place; the statistics r_y and r_u are kept as computed.
#pragma once

#include <algorithm>
#include <type_traits>

#include "checkpoint8.cuh"
#include "ptx.cuh"

namespace lama {
namespace ops {

struct Fwd {
  const void *x, *y, *gate;
  void *u, *n;
  const float *w_post, *w_pre, *s;
  float *ry, *ru;
  int8_t *cy, *cu;
  float *sy, *su;
  long long rows, xs, ys, gs, per;  // row strides of x, y and the gate; rows of one gate row
  int c, groups;
  int sets, parts;
  float s0, eps;
  int vec;
  int *status;
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
  int *status;
};

// One translation unit a type (residual_norm_*.cu).
template <class T>
cudaError_t run_forward(const Fwd& f, cudaStream_t st);
template <class T>
cudaError_t run_backward(const Bwd& b, cudaStream_t st);

}  // namespace ops
}  // namespace lama
