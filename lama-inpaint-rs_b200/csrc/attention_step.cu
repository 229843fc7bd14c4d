// Linear attention for single tokens: one step of the recurrence on a state
// that stays on the device,
//
//   S <- exp(g) S + k v^T,   o = scale q S.
//
// Bound by the state's bytes (read once, written once, fp32): 8 dk dv bytes a
// row and head against 5 dk dv operations.  A CTA takes 32 columns of one state
// (128-byte runs of every row), 16 groups of 8 threads share its rows, and a
// thread issues all its loads before the first use; the products with q are
// summed over the groups by shuffles and one pass through shared memory.
// Splitting the columns gives a single stream 4 * heads CTAs at dv = 128.
// Measured: 256 rows x 8 heads x 128 x 128 in 43.5 us (6.2 TB/s, 95 % of the
// measured copy bandwidth); one row x 8 x 64 x 64 in 2.8 us.
#include "operators.cuh"
#include "ptx.cuh"

namespace lama {
namespace ops {

namespace {

constexpr int THREADS = 128;
constexpr int COLS = 32;
constexpr int GROUPS = THREADS / (COLS / 4);  // groups of threads that share the state's rows

struct Step {
  const void *q, *k, *v;
  void* out;
  long long qb, qh, kb, kh, vb, vh, ob, oh;
  int q_per, k_per, v_per;
  const float* log_decay;
  const float* state;
  float* out_state;
  const int* slots;
  int num_slots, heads, dk, dv;
  float scale;
};

template <class T, int ROWS, bool VEC>  // ROWS * GROUPS >= dk
__global__ void __launch_bounds__(THREADS) k_step(const __grid_constant__ Step p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float sq[128], sk[128];
  __shared__ float part[THREADS / 32][COLS];
  const int blocks = (p.dv + COLS - 1) / COLS;
  const int blk = blockIdx.x % blocks, bh = blockIdx.x / blocks, head = bh % p.heads, row = bh / p.heads;
  const int tid = threadIdx.x, col = blk * COLS + (tid & 7) * 4, grp = tid >> 3;
  T* out = static_cast<T*>(p.out) + row * p.ob + head * p.oh;
  const long long slot = p.slots ? p.slots[row] : row;
  if (slot < 0 || slot >= p.num_slots) {  // an unused row
    if (tid < COLS && blk * COLS + tid < p.dv) out[blk * COLS + tid] = from_float<T>(0.f);
    return;
  }
  const long long base = (slot * p.heads + head) * p.dk * p.dv;
  float s[ROWS][4];
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const int r = i * GROUPS + grp;
    const float* src = p.state + base + (long long)r * p.dv + col;
    if (VEC) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < p.dk && col < p.dv) x = *reinterpret_cast<const float4*>(src);
      s[i][0] = x.x, s[i][1] = x.y, s[i][2] = x.z, s[i][3] = x.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) s[i][j] = r < p.dk && col + j < p.dv ? src[j] : 0.f;
    }
  }
  if (tid < p.dk) {
    sq[tid] = to_float(static_cast<const T*>(p.q)[row * p.qb + (head / p.q_per) * p.qh + tid]);
    sk[tid] = to_float(static_cast<const T*>(p.k)[row * p.kb + (head / p.k_per) * p.kh + tid]);
  }
  float v[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; j++)
    v[j] = col + j < p.dv ? to_float(static_cast<const T*>(p.v)[row * p.vb + (head / p.v_per) * p.vh + col + j]) : 0.f;
  const float lam = expf(p.log_decay[head]);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const int r = i * GROUPS + grp;
    if (r >= p.dk) break;
    const float kr = sk[r], qr = sq[r];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      s[i][j] = lam * s[i][j] + kr * v[j];
      o[j] += qr * s[i][j];
    }
    float* dst = p.out_state + base + (long long)r * p.dv + col;
    if (VEC) {
      if (col < p.dv) *reinterpret_cast<float4*>(dst) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (col + j < p.dv) dst[j] = s[i][j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    o[j] += __shfl_xor_sync(~0u, o[j], 8);
    o[j] += __shfl_xor_sync(~0u, o[j], 16);
    if ((tid & 31) < 8) part[tid >> 5][(tid & 7) * 4 + j] = o[j];
  }
  __syncthreads();
  if (tid < COLS && blk * COLS + tid < p.dv) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) x += part[w][tid];
    out[blk * COLS + tid] = from_float<T>(x * p.scale);
  }
}

template <class T>
cudaError_t go(const Step& p, unsigned grid, bool vec, cudaStream_t st) {
  const dim3 g(grid);
  if (p.dk <= 4 * GROUPS)
    return vec ? launch_chained(k_step<T, 4, true>, g, THREADS, 0, st, p)
               : launch_chained(k_step<T, 4, false>, g, THREADS, 0, st, p);
  return vec ? launch_chained(k_step<T, 8, true>, g, THREADS, 0, st, p)
             : launch_chained(k_step<T, 8, false>, g, THREADS, 0, st, p);
}

}  // namespace
}  // namespace ops
}  // namespace lama

using namespace lama::ops;

extern "C" int lama_linear_attention_step(const lama_attention* a, const lama_rows* out, const float* state,
                                          float* out_state, int num_slots, const int* slots, int device, void* stream,
                                          char* err, int err_len) {
  if (err && err_len > 0) err[0] = 0;
  if (!a || !out || !state || !out_state || !a->log_decay) return fail(err, err_len, LAMA_EINVAL, "null argument");
  if (!dtype_ok(a->dtype)) return fail(err, err_len, LAMA_EINVAL, "unknown element type %d", a->dtype);
  if (misaligned(4, a->log_decay, state, out_state, slots))
    return fail(err, err_len, LAMA_EINVAL, "log_decay, a state or slots is not aligned to its elements");
  if (a->batch < 1 || a->heads < 1 || a->dk < 1 || a->dv < 1 || num_slots < 1)
    return fail(err, err_len, LAMA_EINVAL, "batch, heads, dk, dv and num_slots must be positive");
  if (a->tokens != 1) return fail(err, err_len, LAMA_EINVAL, "a step takes one token, not %d", a->tokens);
  if (a->dk > 128 || a->dv > 128)
    return fail(err, err_len, LAMA_EUNSUPPORTED, "head sizes %d and %d exceed 128", a->dk, a->dv);
  if (a->initial_state || a->lengths)
    return fail(err, err_len, LAMA_EINVAL, "a step takes no initial_state and no lengths");
  if (!slots && num_slots < a->batch)
    return fail(err, err_len, LAMA_EINVAL, "%d slots for %d rows", num_slots, a->batch);
  const uintptr_t from = (uintptr_t)state, to = (uintptr_t)out_state;
  if (from != to && (from < to ? to - from : from - to) < (uintptr_t)num_slots * a->heads * a->dk * a->dv * 4)
    return fail(err, err_len, LAMA_EINVAL, "out_state overlaps state");
  const lama_rows* rows[4] = {&a->q, &a->k, &a->v, out};
  const char* names[4] = {"q", "k", "v", "out"};
  for (int i = 0; i < 4; i++) {
    if (!rows[i]->data || (uintptr_t)rows[i]->data % dtype_size(a->dtype))
      return fail(err, err_len, LAMA_EINVAL, "%s is null or not aligned to its elements", names[i]);
    if (rows[i]->heads < 1 || a->heads % rows[i]->heads)
      return fail(err, err_len, LAMA_EINVAL, "%s has %d heads, which do not divide the %d heads of log_decay", names[i],
                  rows[i]->heads, a->heads);
  }
  if (out->heads != a->heads) return fail(err, err_len, LAMA_EINVAL, "out has %d heads, not %d", out->heads, a->heads);
  const long long grid = (long long)a->batch * a->heads * ((a->dv + COLS - 1) / COLS);
  if (grid > 0x7fffffffLL) return fail(err, err_len, LAMA_EUNSUPPORTED, "batch * heads too large");
  Step p{};
  p.q = a->q.data, p.qb = a->q.batch_stride, p.qh = a->q.head_stride, p.q_per = a->heads / a->q.heads;
  p.k = a->k.data, p.kb = a->k.batch_stride, p.kh = a->k.head_stride, p.k_per = a->heads / a->k.heads;
  p.v = a->v.data, p.vb = a->v.batch_stride, p.vh = a->v.head_stride, p.v_per = a->heads / a->v.heads;
  p.out = out->data, p.ob = out->batch_stride, p.oh = out->head_stride;
  p.log_decay = a->log_decay;
  p.state = state, p.out_state = out_state;
  p.slots = slots, p.num_slots = num_slots;
  p.heads = a->heads, p.dk = a->dk, p.dv = a->dv;
  p.scale = a->scale;
  const bool vec = a->dv % 4 == 0 && (((uintptr_t)state | (uintptr_t)out_state) & 15) == 0;
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  const cudaStream_t st = (cudaStream_t)stream;
  if (ce == cudaSuccess)
    ce = a->dtype == LAMA_F32   ? go<float>(p, (unsigned)grid, vec, st)
         : a->dtype == LAMA_F16 ? go<__half>(p, (unsigned)grid, vec, st)
                                : go<__nv_bfloat16>(p, (unsigned)grid, vec, st);
  if (ce != cudaSuccess) return fail(err, err_len, LAMA_ECUDA, "linear attention step: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}
