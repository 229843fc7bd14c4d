// Linear attention with a decay for each head: whole sequences and gradients.
//
//   S_t = lam S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   lam = exp(g_head)
//
// Chunked form.  For a chunk of n tokens with the entering state E (the state
// of the tokens before it, decayed to its first token),
//
//   o_i = scale ( lam^i q_i E + sum_{j<=i} lam^{i-j} (q_i . k_j) v_j ),  i = 0..n-1
//   X   = lam^{n-1} E + sum_j lam^{n-1-j} k_j v_j^T      (state after its last token)
//   E'  = lam X                                          (enters the next chunk)
//
// so every power of lam has an exponent >= 0: no decay overflows, lam = 0
// (g = -inf) included.  Gradients are the same recurrence on other operands:
//
//   dq: forward in time on  (do; v, k), state S^T
//   dv: backward in time on (k; q, do), state D_t = lam D_{t+1} + scale q_t do_t^T (+ dS_T)
//   dk: backward in time on (v; do, q), state D^T
//
// So one kernel computes all of them: it takes roles (a; b, c) with
// S = sum b c^T and out = a S, a direction in time, and strides.  A CTA walks
// the chunks of one segment of one (sequence, head, 64 columns of c); the
// chunk products run on the tensor core (tcgen05, fp32 accumulators in TMEM),
// the state stays in registers in fp32.  A sequence long enough to be cut into
// several segments takes three launches: the state each segment adds (the
// kernel without outputs), the scan over segments, the outputs.
//
// This file has the general kernel, `k_chunks` (fp32, and 16-bit rows that are
// not 16-byte aligned), the scan and the host side; 16-bit aligned rows go
// through the pipelined kernel of attention_pipe.cu.  In k_chunks eight warps load
// and convert one chunk after another, and a warp of its own issues the products,
// since an issue waits for the products before it: the decayed operand is made
// during the scores' products, the scores are rounded during those of the state
// (one warp doing both: 91.7 -> 85.9 us for 2 x 1521 tokens of 4 heads of 64, fp32, forward
// and backward).  What bounds it is a chunk's chain: loads, conversions, and for
// fp32 six bf16 products for one (8000 clocks of MMAs of 21500 for one chunk).
//
// Precision (k_chunks).  Operands are carried as sums of bf16 parts, as in the
// generator's convolutions: bf16 inputs are one part (exact), fp16 inputs two
// (exact), fp32 inputs three (24 bits), and a product keeps the pairs of
// parts above the last part's size.  What the kernel computes itself and
// feeds back as an operand is rounded: the decayed b to three parts always
// (the state is an fp32 result), the scores and the entering state to two
// (three for fp32 inputs).  Scores in one part would add an error of the size of a
// bf16 output's own rounding.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "attention.cuh"

namespace lama {
namespace ops {

namespace {

__device__ int g_status;

constexpr int THREADS = 256;          // that work on tiles
constexpr int ALL = THREADS + 128;    // with the warpgroup one warp of which issues k_chunks' products
// Registers a thread: at launch, of the workers, of the other warpgroup.
constexpr int LAUNCH_REGS = 168, WORK_REGS = 232, ISSUE_REGS = 40;
static_assert(THREADS * WORK_REGS + (ALL - THREADS) * ISSUE_REGS <= ALL * LAUNCH_REGS, "registers");

template <class T>
struct Parts {
  static constexpr int N = 1;
};
template <>
struct Parts<__half> {
  static constexpr int N = 2;
};
template <>
struct Parts<float> {
  static constexpr int N = 3;
};

// 64 columns from d0 of the chunk's rows, as parts, zeros past the sequence
// and past the head's size.  Row r of the chunk is token first + r * step.
// Loops here and below stay loops: unrolled, the kernel is 150 KB of code that is
// fetched again for every chunk.
// Aligned rows are fetched into registers a tile ahead (Fetch), so that their
// latency passes during the products of the tile before; other rows are read
// element by element when their place is free.
template <class T>
struct Fetch {
  Raw8<T> r[CH * 8 / THREADS];
  __device__ __forceinline__ void load(const T* base, long long stride, int n, int left) {
#pragma unroll
    for (int it = 0; it < CH * 8 / THREADS; it++) {
      const int c = it * THREADS + (int)threadIdx.x, row = c >> 3, ck = c & 7;
      r[it] = load_raw<T, true>(base + row * stride + ck * 8, row < n ? left - ck * 8 : 0);
    }
  }
  __device__ __forceinline__ void store(uint32_t dst) const {
#pragma unroll
    for (int it = 0; it < CH * 8 / THREADS; it++) {
      const int c = it * THREADS + (int)threadIdx.x, row = c >> 3, ck = c & 7;
      float v[8];
      uint4 parts[Parts<T>::N];
      r[it].to(v);
      split8<Parts<T>::N, __nv_bfloat16>(v, parts);
#pragma unroll
      for (int p = 0; p < Parts<T>::N; p++) sts16(dst + p * TILE + swz(row, ck), parts[p]);
    }
  }
};
template <class T>
__device__ __noinline__ void load_elements(uint32_t dst, const T* base, long long stride, int n, int left) {
  // one at a time, 4 heads of 33, 8192 tokens, fp32, forward and backward took 420 us, not 247; inlined
  // and with the issuing warp, bf16 takes 315 us, not 224
  constexpr int BATCH = 16;  // loads in flight
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < CH * 64; i0 += BATCH * THREADS) {
    float v[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; k++) {
      const int i = i0 + k * THREADS, row = i >> 6, col = i & 63;
      v[k] = row < n && col < left ? to_float(base[row * stride + col]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < BATCH; k++) {
      const int i = i0 + k * THREADS, row = i >> 6, col = i & 63;
#pragma unroll
      for (int p = 0; p < Parts<T>::N; p++) {
        const __nv_bfloat16 h = __float2bfloat16_rn(v[k]);
        asm volatile("st.shared.b16 [%0], %1;" ::"r"(dst + p * TILE + swz(row, col >> 3) + (col & 7) * 2),
                     "h"(__bfloat16_as_ushort(h))
                     : "memory");
        v[k] -= __bfloat162float(h);
      }
    }
  }
}

// D (+)= A B over K, the pairs of parts (x, y) with x + y < max(NA, NB), the
// smallest first: the tensor core truncates each sum to fp32, so what is
// added while the accumulator is still small loses less (fp32 inputs measured
// 2e-6 off with the largest pair first).  K in `blocks` of four 16-wide steps,
// `ka` and `kb` bytes apart, the blocks `ba` and `bb`.
template <int NA, int NB>
__device__ __forceinline__ void mma_parts(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int blocks, uint32_t ka,
                                          uint32_t ba, uint32_t pa, uint32_t kb, uint32_t bb, uint32_t pb,
                                          bool accumulate) {
  constexpr int LIM = NA > NB ? NA : NB;
  uint32_t acc = accumulate;
#pragma unroll 1
  for (int z = LIM - 1; z >= 0; z--)
#pragma unroll 1
    for (int x = max(0, z - NB + 1); x < NA && x <= z; x++) {
      uint64_t ax = a + ((x * pa) >> 4), by = b + (((z - x) * pb) >> 4);
#pragma unroll 1
      for (int k = 0; k < blocks; k++, ax += ba >> 4, by += bb >> 4)
#pragma unroll
        for (int s = 0; s < 4; s++) {
          mma_bf16(d, ax + ((s * ka) >> 4), by + ((s * kb) >> 4), idesc, acc);
          acc = 1;
        }
    }
}

template <class T>
struct Plan {
  static constexpr int NP = Parts<T>::N;
  static constexpr int EP = NP == 1 ? 2 : NP;  // parts of the entering state and of the scores
  // a, b, c: NP tiles each; the decayed b: 3 tiles; the entering state.  The
  // scores' 2 * EP tiles and then the chunk's outputs take the place of a and b.
  static constexpr uint32_t A = 0, B = NP * TILE, C = 2 * EP * TILE;
  static constexpr uint32_t P = A, O = A;
  static constexpr uint32_t BD = C + NP * TILE;
  static constexpr uint32_t E = BD + 3 * TILE;
  static constexpr uint32_t bytes() { return E + EP * ETILE + 1024; }
  static_assert(bytes() <= 227 * 1024 && CH * 64 * 4 <= C, "shared memory");
};

// ALIGNED: all of a, b and c come in groups of 8.  A kernel of its own, since
// the call for single elements takes registers from the others (4 heads of 64,
// 8192 tokens, fp32, forward and backward: 159 us against 184 before the issuing warp).
template <class T, bool OUT, bool ALIGNED>
__global__ void __launch_bounds__(ALL, 1) k_chunks(const __grid_constant__ Set set) {
  using PL = Plan<T>;
  constexpr int NP = PL::NP, EP = PL::EP;
  constexpr int MAXS = 2;
  extern __shared__ uint8_t raw[];
  __shared__ float pw[CH + 1];
  __shared__ uint64_t bar_mem[5];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const uint32_t smem = (smem_u32(raw) + 1023u) & ~1023u;
  // products done, and operands ready for them (an arrival a warp)
  const uint32_t bar_p = smem_u32(&bar_mem[0]), bar_u = smem_u32(&bar_mem[1]);
  const uint32_t rdy_s = smem_u32(&bar_mem[2]), rdy_u = smem_u32(&bar_mem[3]), rdy_p = smem_u32(&bar_mem[4]);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_launch_dependents();
  if (warp == 0) tmem_alloc(smem_u32(&tmem_slot), 256);
  if (tid == 0) {
    mbar_init(bar_p, 1);
    mbar_init(bar_u, 1);
    mbar_init(rdy_s, THREADS / 32);
    mbar_init(rdy_u, THREADS / 32);
    mbar_init(rdy_p, THREADS / 32);
    fence_mbar_init();
    failed = 0;
  }
  pdl_wait();

  const int segs = OUT ? set.run[0].nseg : set.run[0].nseg - 1;
  int id = blockIdx.x;
  const Run& r = set.run[run_of(set, segs, id)];
  const int seg = id % segs;
  id /= segs;
  const int blk = id % r.blocks;
  id /= r.blocks;
  const int head = id % r.heads, batch = id / r.heads;

  const float g = r.log_decay[head];
  int len = r.tokens;
  if (r.lengths) len = min(max(r.lengths[batch], 0), r.tokens);
  const int seg_tokens = r.chunks * CH;
  const int p0 = seg * seg_tokens;

  if (tid <= CH) pw[tid] = power(g, tid);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t t_p = tmem, t_o = tmem + 128, t_u = tmem + 192;
  const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
  const int row = (warp & 3) * 32 + lane;            // TMEM lane: token row, or state row (twice)
  const int srow = row & 63;                         // state row of a slab
  const int scol = ((warp >> 2) * 2 + (row >> 6)) * 16;  // its 16 columns

  bool ok = true;
  if (warp >= THREADS / 32) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(ISSUE_REGS));
  if (warp == THREADS / 32) {
    // The issuing warp: a product's issue waits for the products before it, and
    // the other warps' conversions pass meanwhile.
    const int chunks = min(r.chunks, (max(len - p0, 0) + CH - 1) / CH);
    uint32_t phase_s = 0, phase_p = 0;
    const bool leader = elect_one();
    auto ready = [&](uint32_t bar, uint32_t phase, int code) {
      ok = __all_sync(~0u, mbar_wait(bar, phase, &failed, code));
      tc_fence_after();
      return ok;
    };
#pragma unroll 1
    for (int i = 0, s = 0; i < chunks * r.slabs; i++) {
      const bool last_slab = s + 1 == r.slabs;
      if (!ready(rdy_s, phase_s, 4)) break;
      if (OUT && leader) {  // the scores and a E
        mma_parts<NP, NP>(t_p, smem_desc(smem + PL::A, 1024, 2), smem_desc(smem + PL::B, 1024, 2), idesc_bf16_f32(128),
                          1, 32, 0, TILE, 32, 0, TILE, s > 0);
        mma_parts<NP, EP>(t_o, smem_desc(smem + PL::A, 1024, 2), desc_mn(smem + PL::E, 0), idesc_bf16_f32(64) | B_MN, 1,
                          32, 0, TILE, 2048, 0, ETILE, s > 0);
        if (last_slab) mma_commit(bar_p);
      }
      __syncwarp();
      if (!ready(rdy_u, phase_s, 5)) break;
      if (leader) {
        // both 64-row halves of the MMA's 128 rows read the slab's 64 columns
        mma_parts<3, NP>(t_u, desc_mn(smem + PL::BD, 0), desc_mn(smem + PL::C, 0), idesc_bf16_f32(64) | A_MN | B_MN, 2,
                         2048, 8192, TILE, 2048, 8192, TILE, false);
        mma_commit(bar_u);
      }
      __syncwarp();
      phase_s ^= 1;
      if (OUT && last_slab) {
        if (!ready(rdy_p, phase_p, 6)) break;
        if (leader) {
          mma_parts<EP, NP>(t_p, smem_desc(smem + PL::P, 1024, 2), desc_mn(smem + PL::C, 0), idesc_bf16_f32(64) | B_MN, 2,
                            32, TILE, 2 * TILE, 2048, 8192, TILE, false);
          mma_commit(bar_p);
        }
        __syncwarp();
        phase_p ^= 1;
      }
      s = last_slab ? 0 : s + 1;
    }
  } else if (warp < THREADS / 32) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(WORK_REGS));
    uint32_t phase_p = 0, phase_u = 0;
    bool pending_p = false, pending_u = false;  // products committed and not waited for
    int done = 0;  // tokens of this segment so far
    const int step = r.reverse ? -1 : 1;
    auto wait = [&](uint32_t bar, uint32_t& phase, bool& pending, int code) {
      ok = named_sync_and(1, THREADS, mbar_wait(bar, phase, &failed, code));
      if (ok) phase ^= 1, pending = false;
      tc_fence_after();
      return ok;
    };
    // what this thread wrote (and its TMEM loads) before products that the other warp issues
    auto hand_over = [&](uint32_t bar) {
      tc_fence_before();
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto first_of = [&](int pos) { return r.reverse ? (long long)len - 1 - pos : (long long)pos; };
    auto at_tile = [&](const Operand& o, long long first, int d0) {
      return static_cast<const T*>(o.p) + batch * o.sb + (head / o.per) * o.sh + first * o.st + d0;
    };
    auto vec = [](const Operand& o) { return ALIGNED || o.vec; };
    Fetch<T> fa, fb, fc;
    auto fetch = [&](int pos, int s) {  // the tiles of the chunk at pos and slab s
      const int n = min(CH, len - pos);
      if (n <= 0) return;
      const long long first = first_of(pos);
      if (OUT && vec(r.a)) fa.load(at_tile(r.a, first, s * 64), step * r.a.st, n, r.da - s * 64);
      if (vec(r.b)) fb.load(at_tile(r.b, first, s * 64), step * r.b.st, n, r.da - s * 64);
      if (s == 0 && vec(r.c)) fc.load(at_tile(r.c, first, blk * 64), step * r.c.st, n, r.dc - blk * 64);
    };
    fetch(p0, 0);

    // the carried state: 16 columns of row srow of each slab
    float E[MAXS][16];
    const int ld = r.blocks * 64;
    const float lam = pw[1];
    const long long bh = (long long)batch * r.heads + head;
#pragma unroll
    for (int s = 0; s < MAXS; s++) {
      const int er = s * 64 + srow, ec = blk * 64 + scol;
      const float* src = nullptr;
      long long step = 1;
      int cols = 0;
      float f = 1.f;
      if (OUT && s < r.slabs) {
        if (r.staged) {
          src = r.seg + (bh * r.nseg + seg) * (r.slabs * 64 * ld) + er * r.sr + ec * r.sc;
          step = r.sc;
          cols = 16;
        } else if (r.init && er < r.da) {
          src = r.init + bh * r.da * r.dc + er * r.ir + ec * r.ic;
          step = r.ic;
          cols = r.dc - ec;
          if (!r.reverse) f = lam;
        }
      }
      if (cols == 16 && step == 1 && r.staged) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) load_vec<float, 4>(src + i, &E[s][i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; i++, src += step) E[s][i] = i < cols ? f * *src : 0.f;
      }
    }

#pragma unroll 1
    for (int ch = 0; ok && ch < r.chunks; ch++) {
      const int pos = p0 + ch * CH;
      const int n = min(CH, len - pos);
      if (n <= 0) break;
      const bool last = pos + n == len;
      const long long first = first_of(pos);
      if (vec(r.c))
        fc.store(smem + PL::C);
      else
        load_elements<T>(smem + PL::C, at_tile(r.c, first, blk * 64), step * r.c.st, n, r.dc - blk * 64);
#pragma unroll 1
      for (int s = 0; s < r.slabs; s++) {
        if (OUT) {
          float e[16];
#pragma unroll
          for (int i = 0; i < 16; i++) e[i] = s ? E[1][i] : E[0][i];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint4 parts[EP];
            split8<EP, __nv_bfloat16>(e + h * 8, parts);
#pragma unroll
            for (int p = 0; p < EP; p++) sts16(smem + PL::E + p * ETILE + swz(srow, (scol >> 3) + h), parts[p]);
          }
          if (vec(r.a))
            fa.store(smem + PL::A);
          else
            load_elements<T>(smem + PL::A, at_tile(r.a, first, s * 64), step * r.a.st, n, r.da - s * 64);
        }
        if (vec(r.b))
          fb.store(smem + PL::B);
        else
          load_elements<T>(smem + PL::B, at_tile(r.b, first, s * 64), step * r.b.st, n, r.da - s * 64);
        if (s + 1 < r.slabs)
          fetch(pos, s + 1);
        else if (ch + 1 < r.chunks)
          fetch(pos + CH, 0);
        const bool last_slab = s + 1 == r.slabs;
        hand_over(rdy_s);
        pending_p = OUT && last_slab;
        if (!vec(r.b)) named_sync(1, THREADS);  // below, a thread reads groups of b, those that it stored itself
        // decayed b: row j times lam^{n-1-j}, three parts
#pragma unroll 2
        for (int it = 0; it < CH * 8 / THREADS; it++) {
          const int c = it * THREADS + tid, j = c >> 3, ck = c & 7;
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] = 0.f;
#pragma unroll
          for (int p = 0; p < NP; p++) {
            const uint4 u = lds16(smem + PL::B + p * TILE + swz(j, ck));
            const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
            for (int i = 0; i < 4; i++) {
              v[2 * i] += __low2float(x[i]);
              v[2 * i + 1] += __high2float(x[i]);
            }
          }
          const float w = j < n ? pw[n - 1 - j] : 0.f;
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] = j < n ? v[i] * w : 0.f;
          uint4 parts[3];
          split8<3, __nv_bfloat16>(v, parts);
#pragma unroll
          for (int p = 0; p < 3; p++) sts16(smem + PL::BD + p * TILE + swz(j, ck), parts[p]);
        }
        hand_over(rdy_u);
        pending_u = true;
        if (OUT && last_slab) {
          // scores: decay and causal mask, rounded to EP parts
          if (!wait(bar_p, phase_p, pending_p, 1)) break;
#pragma unroll 1
          for (int h = 0; h < 2; h++) {
            const int col0 = (warp >> 2) * 64 + h * 32;
            float v[32];
            tmem_ld32(t_p + lane_base + col0, v);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; j++) {
              const int dist = row - (col0 + j);
              v[j] = dist >= 0 ? v[j] * pw[max(dist, 0)] : 0.f;
            }
#pragma unroll
            for (int q = 0; q < 4; q++) {
              uint4 parts[EP];
              split8<EP, __nv_bfloat16>(v + q * 8, parts);
#pragma unroll
              for (int p = 0; p < EP; p++)
                sts16(smem + PL::P + (p * 2 + (warp >> 2)) * TILE + swz(row, h * 4 + q), parts[p]);
            }
          }
          hand_over(rdy_p);
          pending_p = true;
        }
        if (!wait(bar_u, phase_u, pending_u, 2)) break;
        float e[16], u[16];
#pragma unroll
        for (int i = 0; i < 16; i++) e[i] = s ? E[1][i] : E[0][i];
        tmem_ld16(t_u + lane_base + scol, u);
        tmem_wait_ld();
        const float dn1 = pw[n - 1];
#pragma unroll
        for (int i = 0; i < 16; i++) e[i] = dn1 * e[i] + r.update * u[i];  // the state after the chunk
        if (OUT && last && r.fin) {
          const int er = s * 64 + srow, ec = blk * 64 + scol;
          float* dst = r.fin + bh * r.da * r.dc + er * r.fr + ec * r.fc;
#pragma unroll
          for (int i = 0; i < 16; i++, dst += r.fc)
            if (er < r.da && ec + i < r.dc) *dst = r.reverse ? lam * e[i] : e[i];
        }
        const float f = OUT || ch + 1 < r.chunks ? lam : 1.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
          e[i] *= f;
          if (s)
            E[1][i] = e[i];
          else
            E[0][i] = e[i];
        }
      }
      if (!ok) break;
      done = pos + n - p0;
      if (OUT) {
        if (!wait(bar_p, phase_p, pending_p, 3)) break;
        const float di = pw[row] * r.inter;
        // through shared memory, so that eight threads write a row's 64 columns
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
          const int col0 = (warp >> 2) * 32 + h * 16;
          float x[16], y[16];
          tmem_ld16(t_o + lane_base + col0, x);
          tmem_ld16(t_p + lane_base + col0, y);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            uint4 w;
            w.x = __float_as_uint(di * x[i] + r.intra * y[i]);
            w.y = __float_as_uint(di * x[i + 1] + r.intra * y[i + 1]);
            w.z = __float_as_uint(di * x[i + 2] + r.intra * y[i + 2]);
            w.w = __float_as_uint(di * x[i + 3] + r.intra * y[i + 3]);
            sts16(smem + PL::O + row * 256 + ((((col0 + i) >> 2) ^ (row & 7)) << 4), w);
          }
        }
        named_sync(1, THREADS);
#pragma unroll 1
        for (int it = 0; it < CH * 8 / THREADS; it++) {
          const int c = it * THREADS + tid, j = c >> 3, ck = c & 7, left = r.dc - blk * 64 - ck * 8;
          if (j >= n) break;
          float v[8];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint4 w = lds16(smem + PL::O + j * 256 + (((ck * 2 + h) ^ (j & 7)) << 4));
            v[4 * h] = __uint_as_float(w.x), v[4 * h + 1] = __uint_as_float(w.y);
            v[4 * h + 2] = __uint_as_float(w.z), v[4 * h + 3] = __uint_as_float(w.w);
          }
          const long long at = batch * r.ob + (first + (long long)j * step) * r.ot + head * r.oh + blk * 64 + ck * 8;
          if (r.out_f32)
            store_row(static_cast<float*>(r.out) + at, v, left, r.out_vec);
          else
            store_row(static_cast<T*>(r.out) + at, v, left, r.out_vec);
        }
        named_sync(1, THREADS);  // the next chunk's tiles
      }
    }

    if (ok && OUT) {
      // tokens past the sequence's end
      const int end = min(p0 + seg_tokens, r.tokens);
      const int width = min(64, r.dc - blk * 64);
#pragma unroll 1
      for (int i = tid; i < (end - p0 - done) * 64; i += THREADS) {
        const int t = p0 + done + (i >> 6), c = i & 63;
        if (c >= width) continue;
        const long long at = batch * r.ob + (long long)t * r.ot + head * r.oh + blk * 64 + c;
        if (r.out_f32)
          static_cast<float*>(r.out)[at] = 0.f;
        else
          static_cast<T*>(r.out)[at] = from_float<T>(0.f);
      }
      if (len == 0 && seg == 0 && r.fin) {
#pragma unroll 1
        for (int i = tid; i < r.da * 64; i += THREADS) {
          const int er = i >> 6, ec = blk * 64 + (i & 63);
          const long long base = bh * r.da * r.dc;
          if (ec < r.dc) r.fin[base + er * r.fr + ec * r.fc] = r.init ? r.init[base + er * r.ir + ec * r.ic] : 0.f;
        }
      }
    }
    if (ok && !OUT) {
#pragma unroll
      for (int s = 0; s < MAXS; s++) {
        if (s >= r.slabs) break;
        float* dst = r.seg + ((bh * r.nseg + seg) * (r.slabs * 64) + s * 64 + srow) * ld + blk * 64 + scol;
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(E[s][i], E[s][i + 1], E[s][i + 2], E[s][i + 3]);
      }
    }
    if (!ok) {
      // the products still in flight
      if (pending_p) mbar_wait_drain(bar_p, phase_p);
      if (pending_u) mbar_wait_drain(bar_u, phase_u);
      if (tid == 0) atomicCAS(r.status, 0, failed);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) {
    tmem_relinquish();
    tmem_dealloc(tmem, 256);
  }
}

// seg[s]: the state segment s adds -> the state that enters it (segments in
// the order of the recurrence).  The pipelined kernel leaves the final state
// to this kernel.
__global__ void k_scan(const __grid_constant__ Set set) {
  pdl_launch_dependents();
  pdl_wait();
  const Run& r = set.run[blockIdx.z];
  const int rows = r.slabs * 64, cols = r.blocks * 64;
  const long long per = (long long)rows * cols;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= per) return;
  const int bh = blockIdx.y, head = bh % r.heads, batch = bh / r.heads;
  const int er = (int)(i / cols), ec = (int)(i % cols);
  const bool inside = er < r.da && ec < r.dc;
  float* p = r.seg + (long long)bh * r.nseg * per + i;
  const int made = r.pipe && r.fin ? r.nseg : r.nseg - 1;  // segments whose states are there
  // A batch is loaded before anything waits for a load, the next one before
  // this one's places are written: the kernel is nothing but that latency.
  constexpr int BATCH = 16;
  float x[BATCH], next[BATCH];
  auto load = [&](int s0, float* v) {
#pragma unroll
    for (int k = 0; k < BATCH; k++) v[k] = s0 + k < made ? p[(s0 + k) * per] : 0.f;
  };
  load(0, x);
  float e = 0.f;  // the state that enters a segment
  if (r.init && inside) e = r.init[(long long)bh * r.da * r.dc + er * r.ir + ec * r.ic];
  const float g = r.log_decay[head];
  int len = r.tokens;
  if (r.lengths) len = min(max(r.lengths[batch], 0), r.tokens);
  const float lam = power(g, 1);
  const int seg_tokens = r.chunks * CH;
  const float through = power(g, seg_tokens - 1);
  float after = e;  // the state after the last token
  if (!r.reverse) e *= lam;
  for (int s0 = 0; s0 < r.nseg; s0 += BATCH) {
    if (s0 + BATCH < r.nseg) load(s0 + BATCH, next);
#pragma unroll
    for (int k = 0; k < BATCH; k++) {
      const int s = s0 + k;
      if (s >= r.nseg) break;
      const int seg = r.pipe && r.reverse ? r.nseg - 1 - s : s;
      const int n = min(max(len - seg * seg_tokens, 0), seg_tokens);
      p[s * per] = e;
      if (n > 0) {
        after = x[k] + (n == seg_tokens ? through : power(g, n - 1)) * e;
        e = lam * after;
        if (r.reverse) after = e;
      }
    }
#pragma unroll
    for (int k = 0; k < BATCH; k++) x[k] = next[k];
  }
  if (r.pipe && r.fin && inside) r.fin[(long long)bh * r.da * r.dc + er * r.fr + ec * r.fc] = after;
}

// Sum over the heads that share one head of an operand: src fp32
// [batch][tokens][heads][d] -> dst [batch][tokens][heads / per][d] with
// strides; one operand a blockIdx.y.
struct Share {
  struct {
    const float* src;
    void* dst;
    long long sb, st, sh;
    int per, d;
  } of[3];
  long long rows;  // batch * tokens
  int tokens, heads, n;
};
template <class T>
__global__ void k_share(const __grid_constant__ Share s) {
  pdl_launch_dependents();
  pdl_wait();
  const auto& o = s.of[blockIdx.y];
  const int nh = s.heads / o.per, row_size = nh * o.d;
  for (long long row = blockIdx.x; row < s.rows; row += gridDim.x) {
    const long long batch = row / s.tokens, token = row - batch * s.tokens;
    T* dst = static_cast<T*>(o.dst) + batch * o.sb + token * o.st;
    for (int i = threadIdx.x; i < row_size; i += blockDim.x) {
      const int h = i / o.d, c = i - h * o.d;
      const float* src = o.src + (row * s.heads + (long long)h * o.per) * o.d + c;
      float v = 0.f;
      for (int k = 0; k < o.per; k++) v += src[(long long)k * o.d];
      dst[h * o.sh + c] = from_float<T>(v);
    }
  }
}

template <class T, bool OUT, bool ALIGNED>
cudaError_t launch_chunks(const Set& set, cudaStream_t st) {
  const uint32_t bytes = Plan<T>::bytes();
  static SmemLimit limit;
  const cudaError_t ce = limit.reach(k_chunks<T, OUT, ALIGNED>, (int)bytes);
  if (ce != cudaSuccess) return ce;
  // setmaxnreg.inc takes from the registers of the launch, and would wait for
  // more than those for good
  static const bool fits = [] {
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, k_chunks<T, OUT, ALIGNED>) == cudaSuccess && a.numRegs >= LAUNCH_REGS;
  }();
  if (!fits) return cudaErrorLaunchOutOfResources;
  const int nseg = set.run[0].nseg;
  const dim3 grid((unsigned)ctas(set, OUT ? nseg : nseg - 1));
  return launch_chained(k_chunks<T, OUT, ALIGNED>, grid, ALL, bytes, st, set);
}
template <bool OUT>
cudaError_t launch_chunks(const Set& set, int dtype, cudaStream_t st) {
  bool vec = true;
  for (int w = 0; w < set.n; w++) vec = vec && (!OUT || set.run[w].a.vec) && set.run[w].b.vec && set.run[w].c.vec;
  if (dtype == LAMA_F16) return launch_chunks<__half, OUT, false>(set, st);
  if (dtype == LAMA_BF16) return launch_chunks<__nv_bfloat16, OUT, false>(set, st);
  return vec ? launch_chunks<float, OUT, true>(set, st) : launch_chunks<float, OUT, false>(set, st);
}
cudaError_t launch_scan(const Set& set, cudaStream_t st) {
  int per = 0;
  for (int w = 0; w < set.n; w++) per = std::max(per, set.run[w].slabs * 64 * set.run[w].blocks * 64);
  const Run& r = set.run[0];
  return launch_chained(k_scan, dim3((per + 255) / 256, r.batch * r.heads, set.n), 256, 0, st, set);
}

// How the sequences of a call are cut: one segment reads everything once,
// several read b and c twice but fill the GPU.  Takes the least time on the
// busiest SM, counted in chunk steps, for `rows` (sequence, head, 64 columns)
// that run together.  Pipelined (16-bit types): a CTA costs 4 beside its
// chunks (set-up, the first loads, the last products), the pass that makes the
// states 0.6 a chunk and, with the scan, two launches of 3 each.  The other
// kernel's steps are several times longer and do not overlap; 16-bit rows that go
// through it are cut by the first costs all the same, since a workspace is sized before the output's
// place is known.
struct Cut {
  int nseg = 1, chunks = 1;
};
Cut cut(const lama_attention* p, long long rows) {
  const bool pipe = p->dtype != LAMA_F32;
  const double cta = pipe ? 4 : 1, pass = pipe ? 6 : 1;
  const int slots = 148;
  const int chunks = (p->tokens + CH - 1) / CH;
  double best = 1e300;
  Cut r;
  for (int c = chunks;;) {
    const int nseg = (chunks + c - 1) / c;
    const double waves = (double)((rows * nseg + slots - 1) / slots);
    const double cost = nseg == 1 ? waves * (c + cta) : waves * (1.6 * c + 2 * cta) + pass + 0.05 * nseg;
    if (cost < best) {
      best = cost;
      r.nseg = nseg;
      r.chunks = c;
    }
    if (c == 1) break;
    c = std::max(1, std::min(c - 1, (chunks + nseg) / (nseg + 1)));
  }
  return r;
}
int blocks_of(int d) { return (d + 63) / 64; }
Cut cut_forward(const lama_attention* p) { return cut(p, (long long)p->batch * p->heads * blocks_of(p->dv)); }
// The gradients' runs: dq and dk have blocks of dk, dv those of dv.  The
// pipelined kernel takes dk and dv together, the other all three.
Cut cut_backward(const lama_attention* p) {
  const int k = blocks_of(p->dk), v = blocks_of(p->dv);
  return cut(p, (long long)p->batch * p->heads * (p->dtype != LAMA_F32 ? k + v : 2 * k + v));
}

// Room for the segments' states of one run, whatever its alignment turns out
// to be and whether or not the final state is asked for.
long long seg_bytes(const lama_attention* p, const Cut& c) {
  if (c.nseg == 1 && p->dtype == LAMA_F32) return 0;
  return (long long)p->batch * p->heads * c.nseg * blocks_of(p->dk) * blocks_of(p->dv) * 64 * 64 * 4;
}

Operand operand(const lama_rows& x, int heads, int d, int dtype) {
  const int e = dtype_size(dtype);
  Operand o;
  o.p = x.data;
  o.sb = x.batch_stride;
  o.st = x.token_stride;
  o.sh = x.head_stride;
  o.per = heads / x.heads;
  const long long bits = (long long)(uintptr_t)x.data | (x.batch_stride * e) | (x.token_stride * e) | (x.head_stride * e);
  o.vec = (bits & 15) == 0 && d % 8 == 0;
  return o;
}

void output(Run& r, const lama_rows& x, int d, int dtype) {
  const Operand o = operand(x, x.heads, d, dtype);
  r.out = x.data;
  r.ob = o.sb;
  r.ot = o.st;
  r.oh = o.sh;
  r.out_vec = o.vec;
  r.out_f32 = 0;
}

void roles(Run& r, const Operand& a, const Operand& b, const Operand& c, int da, int dc) {
  r.a = a;
  r.b = b;
  r.c = c;
  r.da = da;
  r.dc = dc;
  r.slabs = blocks_of(da);
  r.blocks = blocks_of(dc);
  r.sr = r.blocks * 64;
  r.sc = 1;
}

bool aligned(const Run& r) { return r.a.vec && r.b.vec && r.c.vec && r.out_vec; }

const char* check_rows(const lama_rows& x, const lama_attention* p, const char* what, char* buf, size_t n) {
  if (!x.data) {
    snprintf(buf, n, "%s is null", what);
    return buf;
  }
  if ((uintptr_t)x.data % dtype_size(p->dtype)) {
    snprintf(buf, n, "%s is not aligned to its elements", what);
    return buf;
  }
  if (x.heads < 1 || p->heads % x.heads) {
    snprintf(buf, n, "%s has %d heads, which do not divide the %d heads of log_decay", what, x.heads, p->heads);
    return buf;
  }
  return nullptr;
}

int check_workspace(const void* workspace, long long bytes, long long need, char* err, int err_len) {
  if (bytes < need || (need && !workspace))
    return fail(err, err_len, LAMA_EINVAL, "workspace of %lld bytes, %lld needed", bytes, need);
  if (need && misaligned(WORKSPACE_ALIGN, workspace))
    return fail(err, err_len, LAMA_EINVAL, "the workspace is not aligned to %d bytes", WORKSPACE_ALIGN);
  return LAMA_OK;
}

int check(const lama_attention* p, char* err, int err_len) {
  if (!p) return fail(err, err_len, LAMA_EINVAL, "null arguments");
  if (!dtype_ok(p->dtype)) return fail(err, err_len, LAMA_EINVAL, "unknown element type %d", p->dtype);
  if (p->batch < 1 || p->tokens < 1 || p->heads < 1 || p->dk < 1 || p->dv < 1)
    return fail(err, err_len, LAMA_EINVAL, "batch, tokens, heads, dk and dv must be positive");
  if (p->dk > 128 || p->dv > 128)
    return fail(err, err_len, LAMA_EUNSUPPORTED, "head sizes %d and %d exceed 128", p->dk, p->dv);
  if (p->tokens > (1 << 30) || (long long)p->batch * p->heads > 65535)
    return fail(err, err_len, LAMA_EUNSUPPORTED, "tokens exceed 2^30 or batch * heads exceeds 65535");
  if (!p->log_decay) return fail(err, err_len, LAMA_EINVAL, "log_decay is null");
  if (misaligned(4, p->log_decay, p->initial_state, p->lengths))
    return fail(err, err_len, LAMA_EINVAL, "log_decay, initial_state or lengths is not aligned to its elements");
  char buf[160];
  const char* m = check_rows(p->q, p, "q", buf, sizeof(buf));
  if (!m) m = check_rows(p->k, p, "k", buf, sizeof(buf));
  if (!m) m = check_rows(p->v, p, "v", buf, sizeof(buf));
  if (m) return fail(err, err_len, LAMA_EINVAL, "%s", m);
  return LAMA_OK;
}

Run common(const lama_attention* p, const Cut& c) {
  Run r{};
  r.nseg = c.nseg;
  r.chunks = c.chunks;
  r.staged = c.nseg > 1;
  r.fine = p->tokens <= FINE;
  r.log_decay = p->log_decay;
  r.lengths = p->lengths;
  r.batch = p->batch;
  r.tokens = p->tokens;
  r.heads = p->heads;
  return r;
}

Run forward_run(const lama_attention* p, float* final_state) {
  Run r = common(p, cut_forward(p));
  roles(r, operand(p->q, p->heads, p->dk, p->dtype), operand(p->k, p->heads, p->dk, p->dtype),
        operand(p->v, p->heads, p->dv, p->dtype), p->dk, p->dv);
  r.fin = final_state;
  r.inter = r.intra = p->scale;
  r.update = 1.f;
  r.init = p->initial_state;
  r.ir = r.fr = p->dv;
  r.ic = r.fc = 1;
  return r;
}

// The three gradient runs: 0 dq, 1 dk, 2 dv.
Run gradient_run(const lama_attention* p, const lama_attention_grads* g, const Cut& c, int which) {
  Run r = common(p, c);
  const Operand q = operand(p->q, p->heads, p->dk, p->dtype), k = operand(p->k, p->heads, p->dk, p->dtype),
                v = operand(p->v, p->heads, p->dv, p->dtype), d = operand(g->grad_out, p->heads, p->dv, p->dtype);
  if (which == 0) {
    roles(r, d, v, k, p->dv, p->dk);
    r.inter = r.intra = p->scale;
    r.update = 1.f;
    r.init = p->initial_state;
  } else {
    if (which == 1) {
      roles(r, v, d, q, p->dv, p->dk);
    } else {
      roles(r, k, q, d, p->dk, p->dv);
      r.fin = g->grad_initial_state;
    }
    r.inter = 1.f;
    r.intra = r.update = p->scale;
    r.reverse = 1;
    r.init = g->grad_final_state;
  }
  r.ir = r.fr = which == 2 ? p->dv : 1;  // states are [dk][dv]; dq and dk use them transposed
  r.ic = r.fc = which == 2 ? 1 : p->dv;
  return r;
}

constexpr long long ALIGN = 256;
long long up(long long b) { return (b + ALIGN - 1) / ALIGN * ALIGN; }

}  // namespace

cudaError_t status_word(int** p) {
  static std::atomic<int*> known[MAX_DEVICES] = {};
  int dev = 0;
  cudaError_t ce = cudaGetDevice(&dev);
  if (ce != cudaSuccess) return ce;
  if (dev < MAX_DEVICES && (*p = known[dev].load(std::memory_order_acquire))) return cudaSuccess;
  ce = cudaGetSymbolAddress((void**)p, g_status);
  if (ce == cudaSuccess && dev < MAX_DEVICES) known[dev].store(*p, std::memory_order_release);
  return ce;
}

}  // namespace ops
}  // namespace lama

using namespace lama::ops;

extern "C" long long lama_linear_attention_workspace(const lama_attention* p, int backward, char* err, int err_len) {
  if (err && err_len > 0) err[0] = 0;
  const int rc = check(p, err, err_len);
  if (rc != LAMA_OK) return rc;
  if (!backward) return up(seg_bytes(p, cut_forward(p)));
  // the states of dq's run and of dv's, then the unsummed gradients of shared heads
  long long bytes = 2 * up(seg_bytes(p, cut_backward(p)));
  const int heads[3] = {p->q.heads, p->k.heads, p->v.heads}, d[3] = {p->dk, p->dk, p->dv};
  for (int w = 0; w < 3; w++)
    if (heads[w] != p->heads) bytes += up((long long)p->batch * p->tokens * p->heads * d[w] * 4);
  return bytes;
}

extern "C" int lama_linear_attention(const lama_attention* p, const lama_rows* out, float* final_state, void* workspace,
                                     long long workspace_bytes, int device, void* stream, char* err, int err_len) {
  const long long need = lama_linear_attention_workspace(p, 0, err, err_len);
  if (need < 0) return (int)need;
  if (!out) return fail(err, err_len, LAMA_EINVAL, "null output");
  char buf[160];
  if (const char* m = check_rows(*out, p, "out", buf, sizeof(buf))) return fail(err, err_len, LAMA_EINVAL, "%s", m);
  if (out->heads != p->heads) return fail(err, err_len, LAMA_EINVAL, "out has %d heads, not %d", out->heads, p->heads);
  if (misaligned(4, final_state)) return fail(err, err_len, LAMA_EINVAL, "final_state is not aligned to its elements");
  if (const int rc = check_workspace(workspace, workspace_bytes, need, err, err_len)) return rc;
  DeviceGuard dev(device, true);
  cudaError_t ce = dev.status;
  const cudaStream_t st = (cudaStream_t)stream;
  Set set;
  set.n = 1;
  Run& r = set.run[0];
  r = forward_run(p, final_state);
  output(r, *out, p->dv, p->dtype);
  r.seg = static_cast<float*>(workspace);
  if (ce == cudaSuccess) ce = status_word(&r.status);
  r.pipe = p->dtype != LAMA_F32 && aligned(r) && encode_maps(r, set.maps[0]);
  if (r.pipe && r.fin) r.staged = 1;
  if (ce == cudaSuccess && r.staged) {
    ce = r.pipe ? launch_pipe(set, p->dtype, true, st) : launch_chunks<false>(set, p->dtype, st);
    if (ce == cudaSuccess) ce = launch_scan(set, st);
  }
  if (ce == cudaSuccess) ce = r.pipe ? launch_pipe(set, p->dtype, false, st) : launch_chunks<true>(set, p->dtype, st);
  if (ce != cudaSuccess) return fail(err, err_len, LAMA_ECUDA, "linear attention: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}

extern "C" int lama_linear_attention_backward(const lama_attention* p, const lama_attention_grads* g, void* workspace,
                                              long long workspace_bytes, int device, void* stream, char* err,
                                              int err_len) {
  const long long need = lama_linear_attention_workspace(p, 1, err, err_len);
  if (need < 0) return (int)need;
  if (!g) return fail(err, err_len, LAMA_EINVAL, "null gradients");
  char buf[160];
  const lama_rows* rows[4] = {&g->grad_out, &g->grad_q, &g->grad_k, &g->grad_v};
  const char* names[4] = {"grad_out", "grad_q", "grad_k", "grad_v"};
  const int heads[4] = {p->heads, p->q.heads, p->k.heads, p->v.heads};
  for (int i = 0; i < 4; i++) {
    if (const char* m = check_rows(*rows[i], p, names[i], buf, sizeof(buf))) return fail(err, err_len, LAMA_EINVAL, "%s", m);
    if (rows[i]->heads != heads[i])
      return fail(err, err_len, LAMA_EINVAL, "%s has %d heads, not %d", names[i], rows[i]->heads, heads[i]);
  }
  if (misaligned(4, g->grad_final_state, g->grad_initial_state))
    return fail(err, err_len, LAMA_EINVAL, "a state's gradient is not aligned to its elements");
  if (const int rc = check_workspace(workspace, workspace_bytes, need, err, err_len)) return rc;
  DeviceGuard dev(device, true);
  cudaError_t ce = dev.status;
  int* status = nullptr;
  if (ce == cudaSuccess) ce = status_word(&status);
  const cudaStream_t st = (cudaStream_t)stream;
  const Cut c = cut_backward(p);
  char* room = static_cast<char*>(workspace) + 2 * up(seg_bytes(p, c));
  Share share{};
  share.rows = (long long)p->batch * p->tokens;
  share.tokens = p->tokens, share.heads = p->heads;
  Run run[3];  // dq, dk, dv
  bool pipe = p->dtype != LAMA_F32;
  for (int w = 0; w < 3; w++) {
    Run& r = run[w] = gradient_run(p, g, c, w);
    const lama_rows& o = *rows[1 + w];
    const int d = w == 2 ? p->dv : p->dk;
    r.status = status;
    r.seg = reinterpret_cast<float*>(static_cast<char*>(workspace) + (w ? up(seg_bytes(p, c)) : 0));
    if (o.heads == p->heads) {
      output(r, o, d, p->dtype);
    } else {
      r.out = room;
      r.out_f32 = 1;
      r.oh = d;
      r.ot = (long long)p->heads * d;
      r.ob = r.ot * p->tokens;
      r.out_vec = d % 8 == 0;
      auto& s = share.of[share.n++];
      s.src = reinterpret_cast<float*>(room);
      s.dst = o.data, s.sb = o.batch_stride, s.st = o.token_stride, s.sh = o.head_stride;
      s.per = p->heads / o.heads, s.d = d;
      room += up((long long)p->batch * p->tokens * p->heads * d * 4);
    }
    pipe = pipe && aligned(r);
  }
  // dk's carried state is dv's transposed
  run[1].sr = 1, run[1].sc = run[2].sr;
  Set set;
  auto take = [&](std::initializer_list<int> which) {
    set.n = 0;
    for (int w : which) set.run[set.n++] = run[w];
  };
  Maps maps[3];
  for (int w = 0; w < 3 && pipe; w++) pipe = encode_maps(run[w], maps[w]);
  for (Run& r : run) {
    r.pipe = pipe;
    r.staged = r.staged || (pipe && g->grad_initial_state);
  }
  if (ce == cudaSuccess && pipe) {
    auto pass = [&](std::initializer_list<int> which, bool states) {
      if (ce != cudaSuccess) return;
      take(which);
      int i = 0;
      for (int w : which) set.maps[i++] = maps[w];
      ce = launch_pipe(set, p->dtype, states, st);
    };
    // one set per direction and number of slabs
    if (run[0].staged) {
      if (run[0].nseg > 1) pass({0}, true);
      pass({2}, true);
      take({0, 2});
      if (ce == cudaSuccess) ce = launch_scan(set, st);
    }
    pass({0}, false);
    if (run[1].slabs == run[2].slabs) {
      pass({1, 2}, false);
    } else {
      pass({1}, false);
      pass({2}, false);
    }
  } else if (ce == cudaSuccess) {
    if (run[0].staged) {
      take({0, 2});
      ce = launch_chunks<false>(set, p->dtype, st);
      if (ce == cudaSuccess) ce = launch_scan(set, st);
    }
    take({0, 1, 2});
    if (ce == cudaSuccess) ce = launch_chunks<true>(set, p->dtype, st);
  }
  if (ce == cudaSuccess && share.n) {
    const dim3 grid((unsigned)std::min<long long>(share.rows, 148 * 16), share.n);
    ce = p->dtype == LAMA_F32   ? launch_chained(k_share<float>, grid, 128, 0, st, share)
         : p->dtype == LAMA_F16 ? launch_chained(k_share<__half>, grid, 128, 0, st, share)
                                : launch_chained(k_share<__nv_bfloat16>, grid, 128, 0, st, share);
  }
  if (ce != cudaSuccess) return fail(err, err_len, LAMA_ECUDA, "linear attention backward: %s", cudaGetErrorString(ce));
  return LAMA_OK;
}

extern "C" int lama_operator_status(int device, char* err, int err_len) {
  if (err && err_len > 0) err[0] = 0;
  DeviceGuard dev(device);
  cudaError_t ce = dev.status;
  int *p = nullptr, code = 0;
  const int zero = 0;
  if (ce == cudaSuccess) ce = status_word(&p);
  if (ce == cudaSuccess) ce = cudaDeviceSynchronize();
  if (ce == cudaSuccess) ce = cudaMemcpy(&code, p, sizeof(int), cudaMemcpyDeviceToHost);
  if (ce == cudaSuccess && code) ce = cudaMemcpy(p, &zero, sizeof(int), cudaMemcpyHostToDevice);
  if (ce != cudaSuccess) return fail(err, err_len, LAMA_ECUDA, "operator status: %s", cudaGetErrorString(ce));
  if (code) return fail(err, err_len, LAMA_EDEVICE, "a kernel wait timed out (code %d)", code);
  return LAMA_OK;
}
