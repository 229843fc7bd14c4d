// Linear attention over whole sequences for 16-bit inputs and outputs with
// 16-byte-aligned rows (head sizes are then multiples of 8): the recurrence of
// linear_attention.cu (roles (a; b, c), S = sum b c^T, out = a S) as one pipeline per CTA.
//
// A CTA takes one segment of one (sequence, head, 64 columns of c) and walks
// its 128-token chunks; the chunks overlap, each step by its own warps:
//
//   warp  12      loads a, b, c (TMA, zeros past the tokens and the head) into
//                 a ring of stages
//   warps  8..11  state: b decayed to the chunk's end, rounded, as an MMA
//                 operand; U = c^T b~ back from TMEM; the state in registers
//                 (fp32), E' = lam^n E + lam U, and E as two bf16 parts
//   warps 14, 15  with two slabs, half of the decayed b
//   warp  13      issues the MMAs: U = c^T b~, S = a b^T, O = a E, O += P c
//   warps  0..7   two groups that take chunks in turn: scores S from TMEM,
//                 decay and causal mask, rounded to bf16 P in S's place (the
//                 A operand of O += P c comes from TMEM); O's rows times
//                 lam^i in place before that product; O to memory
//
// U and S need no state, so only O = a E waits for the chunk before; the
// two groups hide the latency of each other's products.  A chunk's own tokens
// run forward or, for the gradients of b and c, backward in time (REV: the
// mask and every power of lam mirrored, the chunks taken last to first).
//
// Rounding (bf16; fp16 below): P and, where U only feeds the outputs of the same segment, the
// decayed b to one bf16 part (both errors are of the size of the output's own
// rounding and do not add up on one term), E to two.  The states that segments
// hand on, and the final state, come from the kernel without outputs, with the
// decayed b in three parts (24 bits): they are fp32 results.  So a final state
// costs a pass over b and c, and outputs do not depend on asking for it.
//
// Sequences of up to FINE tokens take P in two parts: a choice of precision for
// strips and crops, whose calls are cheapest.  Error against 64 bits in units
// of the results' own rounding (bf16 or fp16, 4 heads of 64 with memories of two to 3000 tokens),
// P in one part and in two: 1.41 and 1.00 up to 128 tokens, 1.41 and 1.28 at 512, 1.41 and
// 1.33 at 1024 (b~'s one part is most of it there), 1.07 and 1.00 from 2048 on (cut into
// segments, whose states are exact); heads that forget within a few tokens: 1.41 and 1.00 at any length.
// Time (bf16, 8 heads of 64, forward; forward and backward): 512 tokens 15.4 and 17.4 us;
// 38 and 42; 128 x 512 tokens 91 and 99; 338 and 369; 4096 tokens 28.7 and 29.7; 81 and 85;
// 16 x 4096 tokens 64.5 and 70.7; 240 and 266.
//
// fp16 has 3 more bits and a narrow range, so what the kernel rounds to it is
// scaled by powers of two first: the rows of P by the row's largest decayed
// score, the columns of E by the column's largest entry, b~ by the chunk's
// largest: a factor is kept to 2^-38 of the largest it is summed with, however
// strong the decay.  Two parts of b~ (22 bits) make the states.
//
// TMEM: two chunks' S (128 columns, P over them) and O (64), and U.
#include <type_traits>

#include "attention.cuh"

namespace lama {
namespace ops {

namespace {


template <int N>
using num_of = std::integral_constant<int, N>;

template <class T, int NS, bool OUT>
struct Lay {
  static constexpr int UP = OUT ? 1 : std::is_same_v<T, __half> ? 2 : 3;  // parts of b~
  // stages of (a, b), free once S and a E are made, and of c, free after P c;
  // buffers of b~ (of a chunk, or without outputs of half a chunk), of U and of E
  static constexpr int AS = OUT ? (NS == 1 ? 3 : 2) : (NS == 1 ? 5 : 2), CS = OUT ? (NS == 1 ? 4 : 2) : (NS == 1 ? 5 : 4);
  static constexpr int KB = OUT && NS == 2 ? 1 : 2, UB = KB, ES = NS == 1 ? 2 : 1;
  static constexpr uint32_t B = OUT ? NS * TILE : 0, AB = B + NS * TILE;  // a stage's b, its size
  static constexpr uint32_t BTILE = OUT ? TILE : ETILE;                   // one slab and part of b~
  static constexpr uint32_t C = AS * AB, BD = C + CS * TILE, BD_BUF = UP * NS * BTILE;
  static constexpr uint32_t E = BD + KB * BD_BUF, E_BUF = 2 * NS * ETILE;
  static constexpr uint32_t BYTES = E + (OUT ? ES * E_BUF : 0);
  // Two more warps make half of b~ where a chunk has two slabs (350 -> 310 us at
  // 2 x 65536 x 4 x 128); with one the state warps keep up, and the two would
  // be in the way (train step of 16 x 4096 x 8 x 64: 240 -> 299 us).
  static constexpr bool MORE = OUT && NS == 2;
  static constexpr int CONV = OUT ? (MORE ? 6 : 4) : 8;  // warps that make b~
  static constexpr int THREADS = (MORE ? 16 : 14) * 32;  // 4 warps a scheduler at most: 128 registers a thread
  static constexpr uint32_t T_U = OUT ? 384 : 0;  // TMEM column of U; buffer i of S at 192 i, of O at 192 i + 128
  static_assert(T_U + UB * 64 * NS <= 512, "TMEM columns");
};

constexpr int MAX_STAGES = 5;
struct Bars {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], cfull[MAX_STAGES], cempty[MAX_STAGES], bd[2], u[2], e[2], s[2], p[2], o[2], oe[2];
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

template <class T>
__device__ __forceinline__ void unpack8(uint4 x, float* v) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = unpack2<T>(w[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}

// A from TMEM (128 lanes, two 16-bit elements a column), B from shared memory
__device__ __forceinline__ void mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The roles' loops share the instruction cache: what is rare stays out of line,
// and what repeats is a loop (unrolled throughout, the kernel was 143 KB of
// code and took 5.8 us a chunk).
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t phase, int* err, int code) {
  return mbar_wait(bar, phase, err, code);
}

template <class T, int NS, bool OUT, bool REV>
__global__ void __launch_bounds__(Lay<T, NS, OUT>::THREADS, 1) k_pipe(const __grid_constant__ Set set, int segs) {
  using L = Lay<T, NS, OUT>;
  constexpr int UP = L::UP, THREADS = L::THREADS;
  constexpr bool HALF = std::is_same_v<T, __half>;
  // Results leave through the stage that held c (one TMA store a chunk; per-row
  // stores kept the load/store unit busy: 70 -> 59 us at 128 x 4096 tokens of
  // 64).  With two slabs c has two stages only, and holding them longer costs
  // more (195 -> 213 us): there the rows are stored directly.
  constexpr bool STAGED_OUT = NS == 1;
  static_assert(L::AS <= MAX_STAGES && L::CS <= MAX_STAGES && L::KB <= 2 && L::UB <= 2 && L::ES <= 2, "barriers");
  extern __shared__ uint8_t raw[];
  __shared__ __align__(16) float pw[CH + 4];
  // fp16: factors 2^e of the columns of E (bf16, chunk c in row c % 4: a group is done with its chunk
  // before E of the fourth next is made), exponents on their way between threads, 1 / the scale of b~
  // (chunk c in entry c % 4: b~ is made at most three chunks ahead of the states)
  __shared__ __align__(16) uint16_t ef[HALF && OUT ? 4 : 1][64];
  __shared__ uint8_t ex[HALF && OUT ? 128 : 1];
  __shared__ float bs[HALF ? 4 : 1];
  __shared__ uint32_t tops[HALF ? 2 : 1][2][8];  // the largest b~ of each warp of a team, two chunks in turn
  __shared__ __align__(16) float rv[32];  // lam^{31-j}
  __shared__ Bars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const uint32_t smem = (smem_u32(raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_launch_dependents();
  if (warp == 0) tmem_alloc(smem_u32(&tmem_slot), 512);
  if (tid == 32) {
    failed = 0;
    for (int i = 0; i < MAX_STAGES; i++) {
      mbar_init(smem_u32(&bars.full[i]), 1);
      mbar_init(smem_u32(&bars.empty[i]), 1);
      mbar_init(smem_u32(&bars.cfull[i]), 1);
      mbar_init(smem_u32(&bars.cempty[i]), 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(smem_u32(&bars.bd[i]), L::CONV);
      mbar_init(smem_u32(&bars.u[i]), 1);
      mbar_init(smem_u32(&bars.e[i]), 4);
      mbar_init(smem_u32(&bars.s[i]), 1);
      mbar_init(smem_u32(&bars.p[i]), OUT ? 4 : 1);
      mbar_init(smem_u32(&bars.o[i]), 1);
      mbar_init(smem_u32(&bars.oe[i]), 4);
    }
    fence_mbar_init();
  }
  pdl_wait();

  int id = blockIdx.x;
  const int which = run_of(set, segs, id);
  const Run& r = set.run[which];
  const Maps& maps = set.maps[which];
  const int slot = id % segs;  // in the order of the recurrence
  id /= segs;
  const int blk = id % r.blocks;
  id /= r.blocks;
  const int head = id % r.heads, batch = id / r.heads;
  const float g = r.log_decay[head];
  const int tokens = r.tokens;
  const bool ragged = r.lengths, out_f32 = r.out_f32, fine = r.fine;
  int len = tokens;
  if (ragged) len = min(max(r.lengths[batch], 0), tokens);
  const int seg_tokens = r.chunks * CH;
  const int seg = REV ? r.nseg - 1 - slot : slot;
  const int p0 = seg * seg_tokens;
  const int mine = min(max(len - p0, 0), seg_tokens);  // tokens of this segment
  const int live = (mine + CH - 1) / CH;
  // the c-th chunk of the recurrence starts at token p0 + at(c) and has num(c) tokens
  auto at = [&](int c) { return (REV ? live - 1 - c : c) * CH; };
  auto num = [&](int c) { return min(CH, mine - at(c)); };

  for (int i = tid; i <= CH; i += THREADS) pw[i] = power(g, i);
  for (int i = tid; i < 32; i += THREADS) rv[i] = power(g, 31 - i);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // Barrier i of a set of n for the c-th chunk: its phase ends once every n
  // chunks.  Where a wait runs out, the roles that share named barriers go on
  // with what is there (every later wait gives up at once, the loops end), so
  // that none is left waiting for another; the other two roles stop.
  auto wait = [&](uint64_t* set, int n, int c, int code) {
    const uint32_t bar = smem_u32(&set[c % n]), ph = (uint32_t)(c / n) & 1;
    return mbar_try_wait(bar, ph) || wait_long(bar, ph, &failed, code);
  };
  auto arrive = [&](uint64_t* set, int n, int c) {  // once a warp, after all its lanes
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&set[c % n]));
  };

  auto wait_stage = [&](int c) {  // b, and c where its rows may have to be cleared
    return wait(bars.full, L::AS, c, 13) && (!ragged || wait(bars.cfull, L::CS, c, 22));
  };
  // b~ of chunk c: row j times lam to the chunk's end, in UP parts; ROWS rows (half h
  // of them, or all) by a team of TH threads, t one of them.
  float up = 1.f;  // fp16: the scale of b~
  auto make_rows = [&](int c, int h, int t, auto team, auto rows) {
    constexpr int TH = decltype(team)::value, ROWS = decltype(rows)::value, LOG = ROWS == 128 ? 7 : 6;
    const uint32_t ab = smem + (c % L::AS) * L::AB, ct = smem + L::C + (c % L::CS) * TILE;
    const uint32_t src = ab + L::B;
    const uint32_t dst = smem + L::BD + (OUT ? c % L::KB : h) * L::BD_BUF;
    const int n = num(c), ck = t & 7;
    if (ragged && n < CH) {  // the boxes hold tokens past the sequence's end
#pragma unroll 1
      for (uint32_t i = t; i < (L::AB + TILE) / TILE * ROWS * 8; i += TH) {
        const uint32_t at = (i >> (LOG + 3)) * TILE + h * (TILE / 2) + (i & (ROWS * 8 - 1)) * 16;  // its rows, tile after tile
        if ((int)((at >> 7) & 127) >= n) sts16(at < L::AB ? ab + at : ct + (at - L::AB), make_uint4(0, 0, 0, 0));
      }
    }
    // a batch's loads go out before its first use: loads and stores of shared memory stay in program order
    constexpr int ALL = NS * ROWS * 8 / TH, MOST = UP == 1 ? 8 : 4, BATCH = ALL < MOST ? ALL : MOST;
    if (HALF && (OUT || h == 0)) {
      // b~ = b lam^m in fp16's range: the chunk's largest |b~| to 2^14..2^15 (not more than 2^100 times as large)
      uint32_t top = 0;  // as bits: an infinity or NaN is above every number
#pragma unroll 4
      for (int i = 0; i < NS * CH * 8 / TH; i++) {
        const int k = i * (TH / 8) + (t >> 3), j = k & (CH - 1);
        const uint4 x = lds16(src + (k >> 7) * TILE + swz(j, ck));
        const uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                                    __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
        const float most = __half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16)));
        if (j < n) top = max(top, __float_as_uint(most * pw[REV ? j : n - 1 - j]) & 0x7fffffffu);
      }
      top = __reduce_max_sync(~0u, top);
      uint32_t* all = tops[TH == 64][c & 1];
      if (lane == 0) all[t >> 5] = top;
      named_sync(3 + 2 * (TH == 64), TH);
#pragma unroll
      for (int i = 0; i < TH / 32; i++) top = max(top, all[i]);
      const int e = (int)(top >> 23), shift = e == 255 ? -1 : min(max(141 - e, -1), 100);  // 2^(14 - (e - 127))
      up = __uint_as_float((uint32_t)(127 + shift) << 23);
      if (t == 0 && h == 0) bs[c & 3] = __uint_as_float((uint32_t)(127 - shift) << 23);
    }
#pragma unroll 1
    for (int i0 = 0; i0 < ALL; i0 += BATCH) {
      uint4 x[BATCH];
      float w[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; i++) {
        const int k = (i0 + i) * (TH / 8) + (t >> 3), j = h * 64 + (k & (ROWS - 1));  // the slabs' rows one after another
        x[i] = lds16(src + (k >> LOG) * TILE + swz(j, ck));
        w[i] = pw[REV ? j : max(n - 1 - j, 0)];
        if (HALF) w[i] *= up;
      }
#pragma unroll
      for (int i = 0; i < BATCH; i++) {
        const int k = (i0 + i) * (TH / 8) + (t >> 3), j = h * 64 + (k & (ROWS - 1));
        if (j >= n) x[i] = make_uint4(0, 0, 0, 0);
        float v[8];
        unpack8<T>(x[i], v);
#pragma unroll
        for (int q = 0; q < 8; q += 2) mul2(v[q], v[q + 1], w[i], w[i]);
        uint4 parts[UP];
        split8<UP, T>(v, parts);
#pragma unroll
        for (int p = 0; p < UP; p++) sts16(dst + (p * NS + (k >> LOG)) * L::BTILE + swz(OUT ? j : j & 63, ck), parts[p]);
      }
    }
    fence_async_smem();
    arrive(bars.bd, L::KB, OUT ? c : 2 * c + h);
  };

  if (warp == 12) {
    // ------------------------------------------------------------ loads
    if (elect_one()) {
      bool ok = true;
      const int ha = head / r.a.per * r.a.hs, hb = head / r.b.per * r.b.hs, hc = head / r.c.per * r.c.hs;
      const int ba = batch * r.a.bs, bb = batch * r.b.bs, bc = batch * r.c.bs;
      int issued = 0, cissued = 0;
#pragma unroll 1
      for (int c = 0; c < live; c++) {
        auto tile = [&](uint32_t dst, const CUtensorMap* map, int h, int b, int d0, uint32_t bar) {
          tma_load_4d(dst, map, d0, p0 + at(c), h, b, bar);
        };
        // boxes count in full, past the tensor's end too
        if (c >= L::AS && !(ok = wait(bars.empty, L::AS, c - L::AS, 11))) break;
        const uint32_t ab = smem + (c % L::AS) * L::AB, bar = smem_u32(&bars.full[c % L::AS]);
        mbar_arrive_expect_tx(bar, L::AB);
#pragma unroll 1
        for (int s = 0; s < NS; s++) {
          if (OUT) tile(ab + s * TILE, &maps.a, ha, ba, s * 64, bar);
          tile(ab + L::B + s * TILE, &maps.b, hb, bb, s * 64, bar);
        }
        issued = c + 1;
        if (c >= L::CS && !(ok = wait(bars.cempty, L::CS, c - L::CS, 21))) break;
        const uint32_t cbar = smem_u32(&bars.cfull[c % L::CS]);
        mbar_arrive_expect_tx(cbar, TILE);
        tile(smem + L::C + (c % L::CS) * TILE, &maps.c, hc, bc, blk * 64, cbar);
        cissued = c + 1;
      }
      // after a wait that ran out, the copies in flight end before the CTA does
      for (int c = max(0, issued - L::AS); !ok && c < issued; c++)
        mbar_wait_drain(smem_u32(&bars.full[c % L::AS]), (uint32_t)(c / L::AS) & 1);
      for (int c = max(0, cissued - L::CS); !ok && c < cissued; c++)
        mbar_wait_drain(smem_u32(&bars.cfull[c % L::CS]), (uint32_t)(c / L::CS) & 1);
    }
  } else if (warp >= 8 && warp < 12) {
    // ------------------------------------------------------------ state
    const int t = tid - 8 * 32;            // TMEM lane: column t % 64 of c, half t / 64 of the rows of b
    const int ec = blk * 64 + (t & 63), half = t >> 6;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    constexpr int W = 32 * NS;             // state elements of a thread
    const long long bh = (long long)batch * r.heads + head;
    const float lam = pw[1];
    float E[W];
    {
      const float* src = nullptr;
      long long step = 0;
      int rows = 0;  // of this thread's state rows, how many are read
      float f = 1.f;
      if (OUT && r.staged) {
        src = r.seg + (bh * r.nseg + slot) * (NS * 64 * r.blocks * 64) + half * W * r.sr + ec * r.sc;
        step = r.sr;
        rows = W;
      } else if (OUT && r.init && ec < r.dc) {
        src = r.init + bh * r.da * r.dc + half * W * r.ir + ec * r.ic;
        step = r.ir;
        rows = r.da - half * W;
        if (!REV) f = lam;
      }
#pragma unroll
      for (int i = 0; i < W; i++, src += step) E[i] = i < rows ? f * *src : 0.f;
    }
    const float update = r.update;
    auto take = [&](int c) {  // E: the state after chunk c, and unless it is the last one decayed to the next
      wait(bars.u, L::UB, c, 12);
      __syncwarp();
      tc_fence_after();
      const float d = pw[num(c) - 1], f = c + 1 < live ? lam : 1.f;
      const float fe = f * d, fu = f * update * (HALF ? bs[c & 3] : 1.f);
#pragma unroll
      for (int i = 0; i < W; i += 32) {
        float u[32];
        tmem_ld32(tmem + L::T_U + (c % L::UB) * (64 * NS) + lane_base + half * W + i, u);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          mul2(u[j], u[j + 1], fu, fu);
          mul2(E[i + j], E[i + j + 1], fe, fe);
          E[i + j] += u[j];
          E[i + j + 1] += u[j + 1];
        }
      }
      tc_fence_before();
      if (!OUT) arrive(bars.e, L::UB, c);  // U's buffer is free
    };
#pragma unroll 1
    for (int c = 0; c < live; c++) {
      if (OUT) {
        wait_stage(c);
        __syncwarp();
      }
      if (L::KB == 1 && c > 0) take(c - 1);  // the products that read b~'s only buffer
      if (OUT) make_rows(c, 0, t, num_of<128>(), num_of<L::MORE ? 64 : 128>());
      if (L::KB == 2 && c > 0) take(c - 1);
      if (OUT) {
        // E's buffer is free once the products of chunk c - ES are done
        if (c >= L::ES) wait(bars.s, 2, c - L::ES, 14);
        __syncwarp();
        const uint32_t eb = smem + L::E + (c % L::ES) * L::E_BUF;
        float fe = 1.f;
        if (HALF) {
          // E in fp16's range: the row's largest magnitude (the other half's thread has a say) to 2^14..2^15
          float m = 0.f;
#pragma unroll
          for (int i = 0; i < W; i++) m = fmaxf(m, fabsf(E[i]));
          ex[t] = (uint8_t)(__float_as_uint(m) >> 23);
          named_sync(4, 128);
          const int e = max((int)max(ex[t], ex[t ^ 64]), 28);  // below 2^-99 as zero
          fe = __uint_as_float((uint32_t)(268 - min(e, 254)) << 23);   // 2^(14 - (e - 127))
          if (half == 0) ef[c & 3][t] = (uint16_t)((uint32_t)(min(e, 254) - 14) << 7);  // 1 / fe, as bf16
          named_sync(4, 128);
        }
#pragma unroll
        for (int i = 0; i < W; i += 8) {
          uint4 parts[2];
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = E[i + j];
          if (HALF)
#pragma unroll
            for (int j = 0; j < 8; j += 2) mul2(x[j], x[j + 1], fe, fe);
          split8<2, T>(x, parts);
          const int er = half * W + i;
#pragma unroll
          for (int p = 0; p < 2; p++) sts16(eb + (p * NS + (er >> 6)) * ETILE + swz(t & 63, (er & 63) >> 3), parts[p]);
        }
        fence_async_smem();
        arrive(bars.e, L::ES, c);
      }
    }
    if (live) take(live - 1);
    if (!OUT) {
      float* dst = r.seg + ((bh * r.nseg + slot) * (NS * 64) + half * W) * (r.blocks * 64) + ec;
#pragma unroll
      for (int i = 0; i < W; i++, dst += r.blocks * 64) *dst = E[i];
    }
  } else if (warp == 13) {
    // ------------------------------------------------------------ MMAs
    // The whole warp walks the loop and one elected lane issues: in a branch
    // on the lane number the compiler takes 88 clocks an MMA, elected 51 (what
    // 128 x 64 x 16 from shared memory takes).
    const bool leader = elect_one();
    constexpr uint32_t F = HALF ? (1u << 7) | (1u << 10) : 0;  // the format fields: 1 bf16, 0 fp16
    constexpr uint32_t ID_U = (idesc_bf16_f32(64 * NS) ^ F) | A_MN | B_MN, ID_S = idesc_bf16_f32(128) ^ F,
                       ID_E = idesc_bf16_f32(64) ^ F, ID_P = (idesc_bf16_f32(64) ^ F) | B_MN;
    bool ok = true;
    auto ready = [&](uint64_t* set, int n, int c, int code) {
      ok = __all_sync(~0u, wait(set, n, c, code));
      tc_fence_after();
      return ok;
    };
    auto second = [&](int c) {  // O += P c of chunk c
      if (!ready(bars.p, 2, c, 15)) return;
      if (leader) {
        const uint32_t t = tmem + (c & 1) * 192;
        const uint64_t dc = desc_mn(smem + L::C + (c % L::CS) * TILE, 0);
#pragma unroll 1
        for (int p = fine; p >= 0; p--)
#pragma unroll 4
          for (int k = 0; k < 8; k++)
            mma_ta(t + 128, t + (k >> 2) * 64 + p * 32 + (k & 3) * 8, dc + ((2048 * k) >> 4), ID_P, 1);
        mma_commit(smem_u32(&bars.o[c & 1]));
        if (!STAGED_OUT) mma_commit(smem_u32(&bars.cempty[c % L::CS]));
      }
      __syncwarp();
    };
#pragma unroll 1
    for (int c = 0; c < live; c++) {
      const uint32_t st = smem + (c % L::AS) * L::AB;
      if (!ready(bars.cfull, L::CS, c, 23)) break;
      if (!OUT && c >= L::UB && !ready(bars.e, L::UB, c - L::UB, 25)) break;
      const uint32_t tu = tmem + L::T_U + (c % L::UB) * (64 * NS);
      constexpr int HALVES = OUT ? 1 : 2, STEPS = 8 / HALVES;  // b~ comes in halves without outputs
#pragma unroll 1
      for (int h = 0; h < HALVES; h++) {
        const int u = c * HALVES + h;
        if (!ready(bars.bd, L::KB, u, 16)) break;  // b~ is made from a full stage
        if (leader) {
          // 64 columns, read twice to fill the MMA's 128 rows
          const uint64_t dc = desc_mn(smem + L::C + (c % L::CS) * TILE + h * (TILE / 2), 0);
#pragma unroll 1
          for (int p = UP - 1; p >= 0; p--) {
            const uint64_t db = desc_mn(smem + L::BD + (u % L::KB) * L::BD_BUF + p * NS * L::BTILE, L::BTILE);
#pragma unroll 4
            for (int k = 0; k < STEPS; k++)
              mma_bf16(tu, dc + ((2048 * k) >> 4), db + ((2048 * k) >> 4), ID_U, h > 0 || p < UP - 1 || k > 0);
          }
          if (!OUT) mma_commit(smem_u32(&bars.p[h]));
        }
        __syncwarp();
      }
      if (!ok) break;
      if (leader) {
        mma_commit(smem_u32(&bars.u[c % L::UB]));
        if (!OUT) {
          mma_commit(smem_u32(&bars.empty[c % L::AS]));
          mma_commit(smem_u32(&bars.cempty[c % L::CS]));
        }
      }
      __syncwarp();
      if (!OUT) continue;
      // S and O of this chunk: the group has read O of chunk c - 2, and P c of that chunk was issued before
      if (c >= 2 && !ready(bars.oe, 2, c - 2, 17)) break;
      const uint32_t t = tmem + (c & 1) * 192;
      if (leader) {
#pragma unroll 1
        for (int s = 0; s < NS; s++) {
          const uint64_t da = smem_desc(st + s * TILE, 1024, 2), db = smem_desc(st + L::B + s * TILE, 1024, 2);
#pragma unroll
          for (int k = 0; k < 4; k++) mma_bf16(t, da + 2 * k, db + 2 * k, ID_S, s > 0 || k > 0);
        }
      }
      __syncwarp();
      if (!ready(bars.e, L::ES, c, 18)) break;
      if (leader) {
#pragma unroll 1
        for (int i = 2 * NS - 1; i >= 0; i--) {  // the small part of E first
          const uint64_t da = smem_desc(st + (i % NS) * TILE, 1024, 2),
                         de = smem_desc(smem + L::E + (c % L::ES) * L::E_BUF + i * ETILE, 1024, 2);
#pragma unroll
          for (int k = 0; k < 4; k++) mma_bf16(t + 128, da + 2 * k, de + 2 * k, ID_E, i < 2 * NS - 1 || k > 0);
        }
        mma_commit(smem_u32(&bars.s[c & 1]));
        mma_commit(smem_u32(&bars.empty[c % L::AS]));
      }
      __syncwarp();
      if (c > 0) second(c - 1);
      if (!ok) break;
    }
    if (OUT && ok && live) second(live - 1);
    // leave only when every product issued has completed
    __shared__ uint64_t drain;
    if (leader) {
      mbar_init(smem_u32(&drain), 1);
      fence_mbar_init();
      mma_commit(smem_u32(&drain));
      mbar_wait_drain(smem_u32(&drain), 0);
    }
  } else if (!OUT && warp < 8) {
    // ------------------------------------------------------------ b~ of the kernel without outputs
#pragma unroll 1
    for (int u = 0; u < 2 * live; u++) {
      if ((u & 1) == 0) wait_stage(u >> 1);
      if (u >= 2) wait(bars.p, 2, u - 2, 24);
      __syncwarp();
      make_rows(u >> 1, u & 1, tid, num_of<256>(), num_of<64>());
    }
  } else if (L::MORE && warp >= 14) {
    // ------------------------------------------------------------ the second half of b~
#pragma unroll 1
    for (int c = 0; c < live; c++) {
      wait_stage(c);
      if (c >= L::KB) wait(bars.u, L::UB, c - L::KB, 24);
      __syncwarp();
      make_rows(c, 1, tid - 14 * 32, num_of<64>(), num_of<64>());
    }
  } else if (OUT && warp < 8) {
    // ------------------------------------------------------------ scores and outputs
    const int grp = warp >> 2, rb = warp & 3, row = rb * 32 + lane;
    const uint32_t t = tmem + grp * 192 + ((uint32_t)(rb * 32) << 16);
    const long long hb = batch * r.ob + head * r.oh + blk * 64;
    const float intra = r.intra, inter = r.inter;
    const int width = min(64, r.dc - blk * 64);
#pragma unroll 1
    for (int c = grp; c < live; c += 2) {
      wait(bars.s, 2, c, 19);
      __syncwarp();
      tc_fence_after();
      const int n = num(c);
      float rowf = intra, back = 1.f;  // factors of the row's scores, and of its results
      float m = 0.f;                   // fp16: the row's largest score, decayed
#pragma unroll 1
      for (int pass = HALF; pass >= 0; pass--) {  // fp16: once for the largest, once for P
        if (HALF && pass == 0) {
          // P in fp16's range: its largest to 2^13..2^14 (fp16 keeps its precision over 2^28 below).  The limits: scores
          // below 2^-60 are nothing in fp16 results, and what is carried in the same sum stays within fp32.
          const int shift = min(max((int)(__float_as_uint(m) >> 23) - 140, -60), 100);
          rowf *= __uint_as_float((uint32_t)(127 - shift) << 23);
          back = __uint_as_float((uint32_t)(127 + shift) << 23);
        }
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
          float v[64];
          const bool some = REV ? 2 * h + 1 >= rb : 2 * h <= rb;
          if (some) {
            tmem_ld32(t + h * 64, v);
            tmem_ld32(t + h * 64 + 32, v + 32);
            tmem_wait_ld();
          }
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const int b = 2 * h + k;
            float* x = v + k * 32;
            uint32_t w[16];
            if (REV ? b < rb : b > rb) {
              if (HALF && pass) continue;
#pragma unroll
              for (int i = 0; i < 16; i++) w[i] = 0;
              tmem_st16(t + h * 64 + k * 16, w);
              if (fine) tmem_st16(t + h * 64 + 32 + k * 16, w);
              continue;
            }
            if (b == rb) {
#pragma unroll
              for (int j = 0; j < 32; j++) {
                const int d = REV ? j - lane : lane - j;
                x[j] = d >= 0 ? x[j] * (rowf * pw[max(d, 0)]) : 0.f;
              }
            } else {
              const float base = rowf * pw[REV ? b * 32 - row : row - b * 32 - 31];
              const float4* f = reinterpret_cast<const float4*>(REV ? pw : rv);
#pragma unroll
              for (int j = 0; j < 8; j++) {
                float4 y = f[j];
                mul2(y.x, y.y, base, base);
                mul2(y.z, y.w, base, base);
                mul2(x[4 * j], x[4 * j + 1], y.x, y.y);
                mul2(x[4 * j + 2], x[4 * j + 3], y.z, y.w);
              }
            }
            if (HALF && pass) {
#pragma unroll
              for (int i = 0; i < 32; i++) m = fmaxf(m, fabsf(x[i]));
              continue;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
            // over this half's columns, which have been read: 32 of the first parts, 32 of the second
            tmem_st16(t + h * 64 + k * 16, w);
            if (fine) {
#pragma unroll
              for (int i = 0; i < 16; i++) {
                const float2 f = unpack2<T>(w[i]);
                w[i] = pack2<T>(x[2 * i] - f.x, x[2 * i + 1] - f.y);
              }
              tmem_st16(t + h * 64 + 32 + k * 16, w);
            }
          }
        }
      }
      const int dist = REV ? n - 1 - row : row;
      float di = dist >= 0 ? inter * pw[dist] : 0.f;
      if (HALF) di *= 1.f / back;
#pragma unroll 1
      for (int h = 0; h < 2; h++) {
        float v[32];
        tmem_ld32(t + 128 + h * 32, v);
        tmem_wait_ld();
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          mul2(v[i], v[i + 1], di, di);
          if (HALF) {
            const uint32_t f = *reinterpret_cast<const uint32_t*>(&ef[c & 3][h * 32 + i]);
            mul2(v[i], v[i + 1], __uint_as_float(f << 16), __uint_as_float(f & 0xffff0000u));
          }
          w[i] = __float_as_uint(v[i]);
          w[i + 1] = __float_as_uint(v[i + 1]);
        }
        tmem_st16(t + 128 + h * 32, w);
        tmem_st16(t + 144 + h * 32, w + 16);
      }
      tmem_wait_st();
      tc_fence_before();
      arrive(bars.p, 2, c);
      wait(bars.o, 2, c, 20);
      __syncwarp();
      tc_fence_after();
      const int tok = p0 + at(c) + row;
      // the tile of c has been read: the results take its place on their way out
      const uint32_t ct = smem + L::C + (c % L::CS) * TILE;
#pragma unroll 1
      for (int h = 0; h < 2; h++) {
        float v[32];
        tmem_ld32(t + 128 + h * 32, v);
        tmem_wait_ld();
        if (h == 1) {
          tc_fence_before();
          arrive(bars.oe, 2, c);
        }
        if (HALF)
#pragma unroll
          for (int i = 0; i < 32; i += 2) mul2(v[i], v[i + 1], back, back);
        if (row >= n)
#pragma unroll
          for (int i = 0; i < 32; i++) v[i] = 0.f;
        if (out_f32 || !STAGED_OUT) {
          if (tok < tokens) {
            const long long dst = hb + (long long)tok * r.ot + h * 32;
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              if (h * 32 + i >= width) break;
              if (out_f32)
                store_vec<float, 8>(static_cast<float*>(r.out) + dst + i, v + i);
              else
                store_vec<T, 8>(static_cast<T*>(r.out) + dst + i, v + i);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            uint4 x;
            split8<1, T>(v + i * 8, &x);
            sts16(ct + swz(row, h * 4 + i), x);
          }
        }
      }
      if (!STAGED_OUT) continue;
      if (!out_f32) fence_async_smem();
      named_sync(1 + grp, 128);
      if (rb == (REV ? 3 : 0) && lane == 0) {  // the warp with the fewest scores
        if (!out_f32) {
          tma_store_4d(&maps.o, ct, blk * 64, p0 + at(c), head, batch);
          bulk_commit();
          bulk_wait_read0();
        }
        mbar_arrive(smem_u32(&bars.cempty[c % L::CS]));
      }
      __syncwarp();
    }
    bulk_wait0();
    // tokens past the sequence's end
    const int end = min(p0 + seg_tokens, tokens);
    for (int i = tid; i < (end - p0 - live * CH) * 64; i += 256) {
      const int c = i & 63;
      if (c >= width) continue;
      const long long dst = hb + (long long)(p0 + live * CH + (i >> 6)) * r.ot + c;
      if (out_f32)
        static_cast<float*>(r.out)[dst] = 0.f;
      else
        static_cast<T*>(r.out)[dst] = from_float<T>(0.f);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && failed) atomicCAS(r.status, 0, failed);
  if (warp == 0) {
    tmem_relinquish();
    tmem_dealloc(tmem, 512);
  }
}

template <class T, int NS, bool OUT, bool REV>
cudaError_t launch(const Set& set, int segs, cudaStream_t st) {
  constexpr int bytes = Lay<T, NS, OUT>::BYTES + 1024;
  static_assert(bytes + 2048 <= 227 * 1024, "shared memory");
  static SmemLimit limit;
  const cudaError_t ce = limit.reach(k_pipe<T, NS, OUT, REV>, bytes);
  if (ce != cudaSuccess) return ce;
  return launch_chained(k_pipe<T, NS, OUT, REV>, dim3((unsigned)ctas(set, segs)), Lay<T, NS, OUT>::THREADS, bytes, st, set, segs);
}

template <class T, int NS, bool REV>
cudaError_t launch(const Set& set, bool states, cudaStream_t st) {
  const Run& r = set.run[0];
  if (states)  // the last segment's state is needed only where the final state is
    return launch<T, NS, false, REV>(set, r.fin ? r.nseg : r.nseg - 1, st);
  return launch<T, NS, true, REV>(set, r.nseg, st);
}
template <class T>
cudaError_t launch(const Set& set, bool states, cudaStream_t st) {
  const bool rev = set.run[0].reverse;
  if (set.run[0].slabs == 1) return rev ? launch<T, 1, true>(set, states, st) : launch<T, 1, false>(set, states, st);
  return rev ? launch<T, 2, true>(set, states, st) : launch<T, 2, false>(set, states, st);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return (PFN_cuTensorMapEncodeTiled_v12000)p;
  }();
  return fn;
}

// [batch][heads][tokens][d] in boxes of 128 tokens x 64 columns.  A dimension
// with stride 0 has one element (its coordinate is multiplied by hs or bs = 0).
bool encode(CUtensorMap* m, Operand& o, const Run& r, int d) {
  const cuuint64_t heads = (cuuint64_t)(r.heads / o.per);
  o.hs = o.sh != 0, o.bs = o.sb != 0;
  if (!encode_fn() || o.st <= 0 || o.sh < 0 || o.sb < 0) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)r.tokens, o.hs ? heads : 1, o.bs ? (cuuint64_t)r.batch : 1};
  const cuuint64_t row = (cuuint64_t)o.st * 2;
  const cuuint64_t strides[3] = {row, o.hs ? (cuuint64_t)o.sh * 2 : row, o.bs ? (cuuint64_t)o.sb * 2 : row};
  for (cuuint64_t s : strides)
    if (s >> 40) return false;
  const cuuint32_t box[4] = {64, CH, 1, 1}, one[4] = {1, 1, 1, 1};
  return encode_fn()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(o.p), dims, strides, box, one,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool encode_maps(Run& r, Maps& m) {
  if (!encode(&m.a, r.a, r, r.da) || !encode(&m.b, r.b, r, r.da) || !encode(&m.c, r.c, r, r.dc)) return false;
  if (r.out_f32) return true;
  Operand o{r.out, r.ob, r.ot, r.oh, 1, 1, 0, 0};
  // a row of results has one place: no dimension may fold onto itself
  return (r.oh != 0 || r.heads == 1) && (r.ob != 0 || r.batch == 1) && encode(&m.o, o, r, r.dc);
}

cudaError_t launch_pipe(const Set& set, int dtype, bool states, cudaStream_t st) {
  return dtype == LAMA_F16 ? launch<__half>(set, states, st) : launch<__nv_bfloat16>(set, states, st);
}

}  // namespace ops
}  // namespace lama
