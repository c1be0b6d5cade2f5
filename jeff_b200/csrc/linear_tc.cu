// The chunked form of linear.cu's recurrence on tcgen05: chunks of C = 64 tokens, with gc the log-decays summed within
// the chunk and gl their total,
//   O = scale ((e^gc Q) S + (Q K^T ∘ Γ, causal) V),   Γ_ij = e^{gc_i - gc_j},
//   S <- e^gl S + (e^{gl - gc} K)^T V,
// every product an M = 128 MMA with the transposed state S^T (lanes: value columns) in tensor memory:
//   MMA1  D = bf16(S^T) Q^T           (A in tensor memory)
//   MMA2  E = [K; Q] K^T              (lanes 64-127: Q K^T; the stacked A is the K and Q tiles laid out back to back)
//   MMA3  E = V^T P^T                 (P = bf16(Q K^T ∘ Γ)); O^T = e^gc D + E, a factor for each of D's columns
//   MMA4  S^T += V^T Kd               (Kd = e^{gl - gc} K in bf16 parts, S^T scaled by e^gl beforehand)
// Rounding: the state is fp32 and what enters it keeps 24 bits (three bf16 parts of a decayed key, the value exact).
// Ahead of an output's own rounding its terms are rounded once, by P for the tokens of its chunk, by the state's bf16
// copy for those before (where the state itself is another launch's, two parts of Kd, 16 bits, serve that copy): errors
// of 0.0023 of the outputs' norm, where their own rounding makes 0.0017. A second part of P and of the copy would be 12
// more products a chunk (some 600 of its cycles by the figures below) and twice their places and stores. Sums of decays
// are fp64, their differences rounded to fp32 once, so that a strong decay early in a chunk takes no accuracy from the
// tokens behind it (-inf is held as -10000, whose exponential is 0). A value that is not finite would reach earlier
// tokens of its chunk through the zeros of P: where an output is not finite it is formed again without them.
//
// Tensor memory, 256 columns: S^T 0-127, its bf16 copy 128-191 (E once MMA1 has read it), D 192-255. Shared memory 108
// KB: two CTAs per SM, whose phases (TMA, tensor core, CUDA cores) fill each other's waits. Within a chunk Kd and the
// next chunk's gates are formed while MMA1 and MMA2 run, P by the warps of lanes 64-127 (of Γ's four 32 x 32 blocks one
// is zero, one a product of two vectors, two need exponentials), and the outputs leave while MMA4 runs; the next tiles
// are fetched as soon as theirs have been read. A (row, head) is one CTA, or, where those are fewer than the CTAs that
// fit, is cut into segments of whole chunks: a first launch leaves each segment's own contribution to the state in
// scratch (states_kernel), a second turns these into the state ahead of each segment and the final one, the third
// computes the outputs.
//
// What bounds it: a chunk's chain of phases (a batch of products waited for costs 540 cycles beside its 65 for an M128
// N128 K16 product and 49 for N64, the gates' sums and exponentials 1200; 5100 in all with outputs, so 2550 an SM) and,
// close behind, shared memory, which the operands (8 KB a product), the copies and Kd keep busy for 2300 cycles a chunk
// with outputs and 1540 without; two CTAs an SM take 8600 each. HBM would need 2000. Measured on a B200: 64 rows of 128
// tokens 64 us (231 MB with the states, 55% of the copy rate), two rows of 8,192 108 us (272 MB, 38%; 42 the states, 8
// the join, 66 the outputs, whose starts overlap), one row of 1,001 22 us (23 where the second and third launch read
// nothing ahead of their waits). Not kept: MMA2 into D as soon as the outputs have left it, P formed under MMA1 (a chunk
// shorter by the state's update on paper, 6% slower: Q and K are then needed sooner than they come).
//
// Waits are bounded (%globaltimer, 2 s): on expiry the CTA records JB_DEV_TIMEOUT | 50.. in the device status word and
// returns.

namespace jb {
namespace lintc {

using gdnt::A_MN;
using gdnt::B_MN;
using gdnt::mn_desc;
using gdnt::swz;
using gdnt::tc_wait_st;
using gdnt::tmem_st32;
using lin::Args;
using lin::D;

constexpr int C = 64, THREADS = 256;
constexpr uint32_t TILE = C * D * 2;   // 16 KB: two 64-column atoms of 64 rows x 128 B
constexpr int OFF_KQ = 0;              // atom a: K at a * 16384, Q at + 8192
constexpr int OFF_K0 = 32768;          // Kd's first part (atoms 8192 apart), then the output tile
constexpr int OFF_K1 = OFF_K0 + TILE;
constexpr int OFF_K2 = OFF_K1 + TILE;  // its third part, or with two parts the output tile
constexpr int OFF_V = OFF_K2 + TILE;
constexpr int OFF_P = OFF_V + TILE;    // 64 rows x 128 B
constexpr int OFF_G = OFF_P + TILE / 2;   // two sets of gates
constexpr int OFF_MISC = OFF_G + 2 * 7 * C * 4;
constexpr int ALLOC = OFF_MISC + 112;
static_assert(2 * (ALLOC + 1024) <= 228 * 1024, "two CTAs per SM");
constexpr uint32_t TM_S = 0, TM_B = 128, TM_D = 192, TM_SMALL = 128, TM_COLS = 256;
constexpr int FIT = 2 * 148;           // CTAs that run at once
constexpr int STATE = D * D;

enum Mode { WHOLE, OUTPUTS };

struct Seg {
  int count, chunks;   // segments of a (row, head), chunks of a segment
  float* states;       // (b * heads, count, 128, 128): a segment's contribution, then the state ahead of it
  float* decay;        // (b * heads, count): a segment's whole decay factor
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
// eight bf16 values times f, in `parts` bf16 parts
template <int PARTS>
__device__ __forceinline__ void split8(const uint4& x, float f, uint4 (&y)[PARTS]) {
  const uint32_t in[4] = {x.x, x.y, x.z, x.w};
  uint32_t out[PARTS][4];
  const uint64_t ff = pair2(f, f), minus = pair2(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint64_t v = pair2(bf_lo(in[i]), bf_hi(in[i]));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(ff));
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      float a, b;
      asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
      out[p][i] = pack_bf2(a, b);
      if (p + 1 < PARTS) {
        const uint64_t h = pair2(bf_lo(out[p][i]), bf_hi(out[p][i]));
        asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(v) : "l"(h), "l"(minus));
      }
    }
  }
#pragma unroll
  for (int p = 0; p < PARTS; ++p) y[p] = make_uint4(out[p][0], out[p][1], out[p][2], out[p][3]);
}

// 32 columns of 16 tensor-memory lanes, as matrix fragments: register 4 i + e of lane l is row l / 4 + 8 (e / 2), column
// 8 i + 2 (l % 4) + e % 2
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// four 8 x 8 matrices of such fragments, transposed: lane l gives the address of row l % 8 of matrix l / 8
__device__ __forceinline__ void st_frags_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}

// A chunk's gates, from the sums gc of its log-decays: in base 2 as two floats (their differences are the exponents
// inside the chunk), e^gc, e^{gl - gc} (and its two bf16 parts, each twice), and Γ's lower left 32 x 32 block as
// cross[32 + i] cross[j].
struct Gates {
  float hi[C], lo[C], from_start[C], to_end[C], cross[C];
  uint2 parts[C];
};

__device__ __forceinline__ float exp2_fast(float x) {   // ex2.approx: 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// a log-decay in base 2, -inf as a number whose exponential is 0
__device__ __forceinline__ double log_decay(float g) { return (g < -1e4f ? -1e4f : g) * 1.4426950408889634; }

// One of two warps' half of a chunk's gates; a, b: the log-decays of tokens lane and lane + 32. ONLY_END: `to_end` alone,
// to the segment's end, `left` being the decay (base 2) from the chunk's first token on; it shrinks by the chunk's.
template <bool ONLY_END>
__device__ __forceinline__ void form_gates(Gates& g, int half, float a, float b, int lane, volatile float* whole,
                                           double& left) {
  double x = log_decay(a), y = log_decay(b);
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double yx = __shfl_up_sync(0xffffffffu, x, off), yy = __shfl_up_sync(0xffffffffu, y, off);
    if (lane >= off) {
      x += yx;
      y += yy;
    }
  }
  const double mid = __shfl_sync(0xffffffffu, x, 31);
  y += mid;
  const double all = __shfl_sync(0xffffffffu, y, 31);
  const double z = half ? y : x;
  const int t = lane + 32 * half;
  const float f = exp2_fast((float)((ONLY_END ? left : all) - z));
  g.to_end[t] = f;
  if (!ONLY_END) {
    const float hi = (float)z;
    g.hi[t] = hi;
    g.lo[t] = (float)(z - (double)hi);
    g.from_start[t] = exp2_fast(hi);
    const uint32_t f0 = pack_bf2(f, f), f1 = pack_bf2(f - bf_lo(f0), f - bf_lo(f0));
    g.parts[t] = make_uint2(f0, f1);
    g.cross[t] = exp2_fast((float)(half ? z - mid : mid - z));
    if (lane == 0 && half == 0) *whole = exp2_fast((float)all);
  }
  left -= all;
}

// eight bf16 values x times f = f0 + f1 in two bf16 parts, on bf16 pairs: x f0 = p + r exactly (16 bits in two bf16
// values), and the second part r + x f1 rounded once: 2^-17 of the product
__device__ __forceinline__ void split8_pairs(const uint4& x, uint2 f, uint4& y0, uint4& y1) {
  const uint32_t in[4] = {x.x, x.y, x.z, x.w};
  uint32_t p0[4], p1[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t n;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(p0[i]) : "r"(in[i]), "r"(f.x));
    n = p0[i] ^ 0x80008000u;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(n) : "r"(in[i]), "r"(f.x), "r"(n));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(p1[i]) : "r"(in[i]), "r"(f.y), "r"(n));
  }
  y0 = make_uint4(p0[0], p0[1], p0[2], p0[3]);
  y1 = make_uint4(p1[0], p1[1], p1[2], p1[3]);
}
// a tile's two boxes to L2
__device__ __forceinline__ void prefetch_tile(const CUtensorMap* map, int h, int token, int row) {
#pragma unroll
  for (int x = 0; x < D; x += 64)
    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global [%0, {%1, %2, %3, %4}];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(h), "r"(token), "r"(row)
                 : "memory");
}
// an untiled copy of whole 16-byte pieces
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(reinterpret_cast<uint64_t>(dst)),
               "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}

template <int N>
struct Count {
  static constexpr int value = N;
};
template <bool B>
struct Bool {
  static constexpr bool value = B;
};

// A warp's outputs of a chunk again (32 channels of 32 tokens, in the output tile already), where MMA3 met a value that is
// not finite: above P's diagonal 0 * NaN and 0 * inf are NaN, which spoils the tokens ahead of that value. Here a token's
// sum ends at the token, P and the values from shared and global memory, and a value that is not finite goes by the
// recurrence, through each product with its key. Finding such outputs costs 1% of a long row's time (two rows of 8,192
// tokens 106.9 -> 108.1 us) and nothing of a short one's (64 rows of 128 tokens 65.0 -> 63.8).
__device__ __noinline__ void outputs_again(const Args& a, uint8_t* ot, uint8_t* pt, const Gates& gt, uint32_t ta,
                                           int row, int h, int start, int live, int qd, int ch) {
  const int lane = threadIdx.x & 31;
  const __nv_bfloat16* q = a.q + row * a.q_row + start * a.q_tok + h * D;
  const __nv_bfloat16* k = a.k + row * a.k_row + start * a.k_tok + h * D;
  const __nv_bfloat16* v = a.v + row * a.v_row + start * a.v_tok + h * D;
  const float scale = rsqrtf((float)D);
  for (int hf = 0; hf < 2; ++hf) {
    uint32_t d[16], e[16];
    tmem_ld_frag(ta + ((uint32_t)(16 * hf) << 16) + TM_D, d);
    tmem_ld_frag(ta + ((uint32_t)(16 * hf) << 16) + TM_B, e);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int t = 32 * ch + 8 * (j >> 2) + 2 * (lane & 3) + (j & 1);
      const int x = 32 * qd + 16 * hf + 8 * (j >> 1 & 1) + (lane >> 2);
      const float before = gt.from_start[t] * __uint_as_float(d[j]);
      if (t >= live || isfinite(__uint_as_float(e[j])) || !isfinite(before)) continue;
      float sum = before;
      for (int s = 0; s <= t; ++s) {
        const float vs = bf2f(v[s * a.v_tok + x]);
        if (isfinite(vs)) {
          sum += bf2f(reinterpret_cast<const __nv_bfloat16*>(swz(pt, t, s >> 3))[s & 7]) * vs;
        } else {
          float w = 0.f;
          for (int i = 0; i < D; ++i) w += bf2f(q[t * a.q_tok + i]) * (bf2f(k[s * a.k_tok + i]) * vs);
          sum += w * exp2_fast((gt.hi[t] - gt.hi[s]) + (gt.lo[t] - gt.lo[s]));
        }
      }
      reinterpret_cast<__nv_bfloat16*>(swz(ot + (x >> 6) * 8192, t, (x & 63) >> 3))[x & 7] = f2bf(sum * scale);
    }
  }
}

template <int MODE>
__global__ void __launch_bounds__(THREADS, 2)
    scan_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                const __grid_constant__ Args a, const Seg seg, int* err) {
  // The outputs' launch is let go by join_kernel's CTAs once they have seen the states' launch end, and that one began
  // when everything before it had ended: the inputs are there. Only the segments' states are waited for.
  if (MODE == WHOLE) pdl_begin();
  constexpr int PARTS = MODE == OUTPUTS ? 2 : 3;   // of Kd
  extern __shared__ __align__(1024) uint8_t sm[];
  uint8_t* kq = sm + OFF_KQ;
  uint8_t* pt = sm + OFF_P;
  // the outputs' tile: with two parts of Kd a place of its own, so that they leave while MMA4 runs
  constexpr bool EARLY = MODE == OUTPUTS;
  uint8_t* ot = sm + (EARLY ? OFF_K2 : OFF_K0);
  Gates* gates = reinterpret_cast<Gates*>(sm + OFF_G);
  uint64_t* d_bar = reinterpret_cast<uint64_t*>(sm + OFF_MISC);   // MMA1; MMA2; MMA3 (EARLY); every product
  uint64_t* p_bar = d_bar + 1;
  uint64_t* e_bar = d_bar + 2;
  uint64_t* all_bar = d_bar + 3;
  uint64_t* k_bar = d_bar + 4;
  uint64_t* q_bar = d_bar + 5;
  uint64_t* v_bar = d_bar + 6;
  uint64_t* s_bar = d_bar + 7;                                    // the state's copy
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + OFF_MISC + 64);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + OFF_MISC + 68);
  volatile float* whole = reinterpret_cast<volatile float*>(sm + OFF_MISC + 72);   // [2] the chunks' decay factors

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int qd = warp & 3, ch = warp >> 2;
  const int L = 32 * qd + lane;   // this thread's tensor-memory lane
  const uint32_t lane_bits = (uint32_t)(32 * qd) << 16;
  if (smem_u32(sm) & 1023) {         // the swizzled tiles' base
    if (tid == 0) atomicCAS(err, 0, JB_DEV_LAUNCH | 50);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < 8; ++i) mbar_init(d_bar + i, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t s_at = tmem + lane_bits + TM_S + 64 * ch, b_at = tmem + lane_bits + TM_B + 32 * ch;
  const uint32_t kq_a = smem_u32(kq), kd_a = smem_u32(sm + OFF_K0), pt_a = smem_u32(pt);
  for (int i = tid; i < 32 * 4; i += THREADS)   // P's upper right block is never anything else
    *reinterpret_cast<uint4*>(swz(pt, i >> 2, 4 + (i & 3))) = make_uint4(0, 0, 0, 0);

  int k_issued = 0, q_issued = 0, v_issued = 0;
  const int pair = blockIdx.x / seg.count, part = blockIdx.x % seg.count;
  const int row = pair / a.heads, h = pair % a.heads;
  const int stop = a.real ? min(max(a.real[row], 0), a.n) : a.n;
  const int begin = part * seg.chunks * C, end = min(begin + seg.chunks * C, a.n);
  const int work = min(end, stop);   // tokens past it are padding: zeros out, the state stays
  const int chunks = begin < work ? (work - begin + C - 1) / C : 0;
  auto start_of = [&](int i) { return begin + i * C; };   // the first token of chunk i
  // tile loads, all issued by one lane of warp 0
  auto load = [&](const CUtensorMap* map, uint8_t* to, int step, uint64_t* bar, int i, bool me) {
    if (!me) return;
    mbar_arrive_expect_tx(bar, TILE);
    tma_load_4d(to, map, bar, 0, h, start_of(i), row);
    tma_load_4d(to + step, map, bar, 64, h, start_of(i), row);
  };
  auto load_k = [&](int i, bool me) { ++k_issued, load(&tm_k, kq, 16384, k_bar, i, me); };
  auto load_q = [&](int i, bool me) { ++q_issued, load(&tm_q, kq + 8192, 16384, q_bar, i, me); };
  auto load_v = [&](int i, bool me) { ++v_issued, load(&tm_v, sm + OFF_V, 8192, v_bar, i, me); };
  const float* gp = a.g + row * a.g_row + h;
  float g0 = 0.f, g1 = 0.f;   // warps 0 and 4: the log-decays of the next chunk's tokens, 0 past the row's end
  auto gates_of = [&](int i) {
    const int t = start_of(i) + lane;
    g0 = i < chunks && t < work ? gp[t * a.g_tok] : 0.f;
    g1 = i < chunks && t + 32 < work ? gp[(t + 32) * a.g_tok] : 0.f;
  };
  double unused = 0.0;
  if (qd == 0) gates_of(0);
  // the state ahead of the segment: one copy over Kd's and V's places, which nothing needs yet
  const float* in = MODE == WHOLE ? lin::state_in(a.pool, row, h)
                                  : seg.states + ((int64_t)pair * seg.count + part) * STATE;
  float* state = reinterpret_cast<float*>(sm + OFF_K0);
  if (warp == 0 && chunks) {
    const bool me = elect_one();
    load_k(0, me);
    load_q(0, me);
    __syncwarp();
  }
  if (MODE == OUTPUTS && warp == 2) pdl_begin();
  if (warp == 2 && in && elect_one()) {
    mbar_arrive_expect_tx(s_bar, STATE * 4);
    bulk_load(state, in, STATE * 4, s_bar);
  }
  if (qd == 0) {
    form_gates<false>(gates[0], ch, g0, g1, lane, whole, unused);
    gates_of(1);
  }
  if (MODE == OUTPUTS && warp != 2) pdl_begin();
  __syncthreads();
  // lane = value column, columns = key rows: into tensor memory, scaled for the first chunk, and its bf16 copy
  auto put_state = [&](int half, uint32_t (&x)[32], float el) {
    uint32_t b[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) b[e] = pack_bf2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
    tmem_st16(b_at + 16 * half, b);
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * el);
    tmem_st32(s_at + 32 * half, x);
  };
  uint32_t r[32];
  {
    const float el = chunks ? whole[0] : 1.f;
    if (in) mbar_wait(s_bar, 0, abort_flag, err, 58);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        r[i] = in ? __float_as_uint(state[(ch * 64 + half * 32 + i) * D + L]) : 0u;
      put_state(half, r, el);
    }
    tc_wait_st();
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  if (warp == 0 && chunks) {
    load_v(0, elect_one());
    __syncwarp();
  }

  for (int c = 0; c < chunks; ++c) {
    const uint32_t phase = (uint32_t)c & 1;
    const int set = c & 1, live = min(C, work - start_of(c));
    const bool more = c + 1 < chunks;
    const Gates& gt = gates[set];
    // ---- MMA1, then, where it has read the state's copy, MMA2
    if (warp == 1) {
      mbar_wait(q_bar, phase, abort_flag, err, 53);
      __syncwarp();
      tc_fence_after();
      constexpr uint32_t id = idesc_bf16(128, 64);
      const bool issuer = elect_one();
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t b = sw128_desc(kq_a + 8192 + (kk >> 2) * 16384 + 32 * (kk & 3));
        if (issuer) w4t::tc_mma_ts(tmem + TM_D, tmem + TM_B + 8 * kk, b, id, kk != 0);
      }
      if (issuer) tc_commit(d_bar);
      __syncwarp();
      mbar_wait(k_bar, phase, abort_flag, err, 52);
      mbar_wait(d_bar, phase, abort_flag, err, 55);
      __syncwarp();
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t dsc = sw128_desc(kq_a + (kk >> 2) * 16384 + 32 * (kk & 3));
        if (issuer) tc_mma_bf16(tmem + TM_B, dsc, dsc, id, kk != 0);
      }
      if (issuer) tc_commit(p_bar);
      __syncwarp();
    }
    // ---- warps 0 and 4: the next chunk's gates, and the decays of the one after it
    if (qd == 0 && more) {
      form_gates<false>(gates[set ^ 1], ch, g0, g1, lane, whole + (set ^ 1), unused);
      gates_of(c + 2);
    }
    // values past the row's end may be anything: zeros, so that a zero weight keeps them out
    if (live < C) {
      mbar_wait(v_bar, phase, abort_flag, err, 54);
      for (int i = tid; i < (C - live) * 16; i += THREADS) {
        const int t = live + (i >> 4), x = i & 15;
        *reinterpret_cast<uint4*>(swz(sm + OFF_V + (x >> 3) * 8192, t, x & 7)) = make_uint4(0, 0, 0, 0);
      }
    }
    // ---- Kd, 16-byte pieces of the tokens' keys: five a thread of the warps that form P, six of warps 1 and 5
    auto form_kd = [&](auto count, int first, int step) {   // its loads ahead of its stores
      constexpr int N = decltype(count)::value;
      mbar_wait(k_bar, phase, abort_flag, err, 52);
      uint4 x[N];
#pragma unroll
      for (int it = 0; it < N; ++it) {
        const int i = min(first + it * step, C * 16 - 1), t = i >> 4, p = i & 15;
        x[it] = *reinterpret_cast<const uint4*>(swz(kq + (p >> 3) * 16384, t, p & 7));
      }
#pragma unroll
      for (int it = 0; it < N; ++it) {
        const int i = first + it * step, t = min(i >> 4, C - 1), p = i & 15;
        uint4 y[PARTS];
        if constexpr (PARTS == 2) split8_pairs(x[it], gt.parts[t], y[0], y[1]);
        else split8(x[it], gt.to_end[t], y);
        if (i < C * 16)
#pragma unroll
          for (int u = 0; u < PARTS; ++u)
            *reinterpret_cast<uint4*>(swz(sm + OFF_K0 + u * TILE + (p >> 3) * 8192, t, p & 7)) =
                t < live ? y[u] : make_uint4(0, 0, 0, 0);
      }
    };
    if (qd == 1) {
      form_kd(Count<6>(), 640 + ch * 32 + lane, 64);
    } else if (qd >= 2) {
      form_kd(Count<5>(), (2 * ch + qd - 2) * 32 + lane, 128);
      mbar_wait(p_bar, phase, abort_flag, err, 51);
      tc_fence_after();
      // ---- P from E's lanes 64-127: row i = L - 64; columns 16 ch .. + 15 of the left half, and for rows from 32 on
      // 32 + 16 ch .. + 15 too
      const int i = L - C;
      const float hi = gt.hi[i], lo = gt.lo[i], ci = gt.cross[i];
      const int upto = i < live ? i : -1;
      uint32_t d[2][16];
      lsh::tmem_ld16(tmem + lane_bits + TM_B + 16 * ch, d[0]);
      if (qd == 3) lsh::tmem_ld16(tmem + lane_bits + TM_B + 32 + 16 * ch, d[1]);
      tc_wait_ld();
      auto form_p = [&](const uint32_t (&e)[16], int j0, auto cross) {
#pragma unroll
        for (int c8 = 0; c8 < 2; ++c8) {
          float x[8];
#pragma unroll
          for (int e4 = 0; e4 < 2; ++e4) {
            const int j = j0 + 8 * c8 + 4 * e4;
            float f[4];
            if constexpr (decltype(cross)::value) {
              const float4 cj = *reinterpret_cast<const float4*>(&gt.cross[j]);
              f[0] = ci * cj.x; f[1] = ci * cj.y; f[2] = ci * cj.z; f[3] = ci * cj.w;
            } else {
              const float4 hj = *reinterpret_cast<const float4*>(&gt.hi[j]);
              const float4 lj = *reinterpret_cast<const float4*>(&gt.lo[j]);
              f[0] = exp2_fast((hi - hj.x) + (lo - lj.x)); f[1] = exp2_fast((hi - hj.y) + (lo - lj.y));
              f[2] = exp2_fast((hi - hj.z) + (lo - lj.z)); f[3] = exp2_fast((hi - hj.w) + (lo - lj.w));
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
              x[4 * e4 + u] = j + u <= upto ? __uint_as_float(e[8 * c8 + 4 * e4 + u]) * f[u] : 0.f;
          }
          *reinterpret_cast<uint4*>(swz(pt, i, (j0 >> 3) + c8)) = make_uint4(
              pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(x[4], x[5]), pack_bf2(x[6], x[7]));
        }
      };
      if (qd == 2) {
        form_p(d[0], 16 * ch, Bool<false>());
      } else {
        form_p(d[0], 16 * ch, Bool<true>());
        form_p(d[1], 32 + 16 * ch, Bool<false>());
      }
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) break;
    // ---- the next tiles, each once its place has been read: K by every thread and by MMA2, Q by MMA1 and MMA2
    if (warp == 0 && more) {
      const bool me = elect_one();
      load_k(c + 1, me);
      load_q(c + 1, me);
      __syncwarp();
    }
    // ---- MMA3, MMA4
    if (warp == 1) {
      mbar_wait(v_bar, phase, abort_flag, err, 54);
      __syncwarp();
      tc_fence_after();
      const bool issuer = elect_one();
      const uint32_t v_a = smem_u32(sm + OFF_V);
      constexpr uint32_t id3 = idesc_bf16(128, 64) | A_MN;
#pragma unroll
      for (int kk = 0; kk < C / 16; ++kk) {
        const uint64_t av = mn_desc(v_a + kk * 2048, 8192), b = sw128_desc(pt_a + 32 * kk);
        if (issuer) tc_mma_bf16(tmem + TM_B, av, b, id3, kk != 0);
      }
      if (EARLY && issuer) tc_commit(e_bar);
      __syncwarp();
      constexpr uint32_t id4 = idesc_bf16(128, 128) | A_MN | B_MN;
#pragma unroll
      for (int kk = 0; kk < C / 16; ++kk) {
        const uint64_t av = mn_desc(v_a + kk * 2048, 8192);
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p) {   // the small parts first
          const uint64_t b = mn_desc(kd_a + p * TILE + kk * 2048, 8192);
          if (issuer) tc_mma_bf16(tmem + TM_S, av, b, id4, 1);
        }
      }
      if (issuer) tc_commit(all_bar);
      __syncwarp();
    }
    if (EARLY) mbar_wait(e_bar, phase, abort_flag, err, 56);
    else mbar_wait(all_bar, phase, abort_flag, err, 57);
    tc_fence_after();
    if (MODE == WHOLE && warp == 0 && more) {
      load_v(c + 1, elect_one());
      __syncwarp();
    }
    // ---- O^T = e^gc D + E -> bf16 -> the output tile, laid out as the loads -> TMA store
    const float scale = rsqrtf((float)D);
    const int tq = lane & 3;
    uint32_t pk[4][4];   // 8 tokens each: the warp's four groups of 8 channels
    uint32_t zero = 0;   // the outputs times 0: NaN where one is not finite
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      uint32_t d[16], e[16];
      const uint32_t ta = tmem + lane_bits + ((uint32_t)(16 * hf) << 16) + 32 * ch;
      tmem_ld_frag(ta + TM_D, d);
      tmem_ld_frag(ta + TM_B, e);
      tc_wait_ld();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 32 * ch + 8 * i + 2 * tq;
        const float2 f = *reinterpret_cast<const float2*>(&gt.from_start[t]);
#pragma unroll
        for (int g8 = 0; g8 < 2; ++g8) {
          const float x = fmaf(f.x, __uint_as_float(d[4 * i + 2 * g8]), __uint_as_float(e[4 * i + 2 * g8])) * scale;
          const float y =
              fmaf(f.y, __uint_as_float(d[4 * i + 2 * g8 + 1]), __uint_as_float(e[4 * i + 2 * g8 + 1])) * scale;
          pk[i][2 * hf + g8] = pack_bf2(t < live ? x : 0.f, t + 1 < live ? y : 0.f);
          asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(zero) : "r"(pk[i][2 * hf + g8]), "r"(0));
        }
      }
    }
    const int x = 32 * qd + 8 * (lane >> 3);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      st_frags_trans(smem_u32(swz(ot + (x >> 6) * 8192, 32 * ch + 8 * i + (lane & 7), (x & 63) >> 3)), pk[i][0],
                     pk[i][1], pk[i][2], pk[i][3]);
    if (__any_sync(0xffffffffu, zero & 0x7fff7fffu)) {
      __syncwarp();
      outputs_again(a, ot, pt, gt, tmem + lane_bits + 32 * ch, row, h, start_of(c), live, qd, ch);
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) break;
    if (tid == 0) {
      tma_store_4d(&tm_o, ot, 0, h, start_of(c), row);
      tma_store_4d(&tm_o, ot + 8192, 64, h, start_of(c), row);
      tma_store_commit();
    }
    if (EARLY) {
      mbar_wait(all_bar, phase, abort_flag, err, 57);
      tc_fence_after();
      if (warp == 0 && more) {
        load_v(c + 1, elect_one());
        __syncwarp();
      }
    }
    if (more) {
      // ---- the next chunk's copy of the state, and the state's decay over it
      const float el = whole[set ^ 1];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        tmem_ld32(s_at + 32 * half, r);
        tc_wait_ld();
        put_state(half, r, el);
      }
      tc_wait_st();
      if (tid == 0) tma_store_wait_read();   // the output tile's place is Kd's, or the next tile's
      tc_fence_before();
      __syncthreads();
    }
  }
  const bool ok = *abort_flag == 0;
  {   // chunks that hold padding only
    const int first = max(begin, (work + C - 1) / C * C);
    uint4* o = reinterpret_cast<uint4*>(a.o + row * a.o_row + h * D);
    for (int64_t i = (int64_t)first * 16 + tid; i < (int64_t)end * 16; i += THREADS)
      o[(i >> 4) * (a.o_tok / 8) + (i & 15)] = make_uint4(0, 0, 0, 0);
  }
  float* out = MODE == WHOLE ? lin::state_out(a.pool, row, h) : nullptr;
  if (ok && out) {   // through shared memory, Kd's and V's places again, as one copy
    if (tid == 0) tma_store_wait_read();
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      tmem_ld32(s_at + 32 * half, r);
      tc_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) state[(ch * 64 + half * 32 + i) * D + L] = __uint_as_float(r[i]);
    }
    fence_proxy_async_smem();
    __syncthreads();
    if (tid == 0) {
      bulk_store(out, state, STATE * 4);
      tma_store_commit();
    }
  }
  if (tid == 0) tma_store_wait_all();
  if (!ok && warp == 0) {
    // a CTA that gave up waits (bounded) for the copies it issued before its shared memory goes away: the last tiles', the
    // others having landed before these were issued
    const uint64_t t0 = global_ns();
    auto landed = [&]() {
      return (!in || mbar_try_wait(s_bar, 0)) && (!k_issued || mbar_try_wait(k_bar, (k_issued - 1) & 1)) &&
             (!q_issued || mbar_try_wait(q_bar, (q_issued - 1) & 1)) &&
             (!v_issued || mbar_try_wait(v_bar, (v_issued - 1) & 1));
    };
    while (!landed() && global_ns() - t0 < kWaitNs) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TM_COLS);
  }
}

// A segment's own contribution to the state, and its decay: S^T += V^T Kd over its chunks, Kd with the decay to the
// segment's end (whose whole log-decay is summed first), so that the sum in tensor memory is only added to. The tensor
// core's sums truncate: the state's error at 5 rows of 3,276 tokens was 1.3e-6 from the last chunk to the first, the
// large terms at the bottom of the sum, and is 1.2e-7 so. Kd's first part and its two small ones go to accumulators of
// their own, since the small parts would make the large sum truncate three times as often. Warps 0-7 form Kd, warp 8
// fetches the tiles and issues the products, warp 9 forms the gates a chunk ahead; two halves of a chunk in turn, one's
// Kd formed while the other's products run. They meet at mbarriers only.
constexpr int ST_THREADS = 320;
constexpr int ST_K = 0;                // K tile of chunk i: atoms 16384 apart at 8192 (i % 2); Kd's first part over it
constexpr int ST_V = 32768;            // V tile: TILE (i % 2)
constexpr int ST_K1 = ST_V + 2 * TILE, ST_K2 = ST_K1 + TILE;   // Kd's other parts (atoms 8192 apart)
constexpr int ST_TOTALS = ST_K2 + TILE;
static_assert(ST_TOTALS + ST_THREADS / 32 * 8 <= OFF_G, "the sums fit ahead of the gates");

__global__ void __launch_bounds__(ST_THREADS, 2)
    states_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Args a,
                  const Seg seg, int* err) {
  pdl_begin();
  extern __shared__ __align__(1024) uint8_t sm[];
  Gates* gates = reinterpret_cast<Gates*>(sm + OFF_G);
  uint64_t* done = reinterpret_cast<uint64_t*>(sm + OFF_MISC);    // [2] a half's products
  uint64_t* k_bar = done + 2;                                     // [2] a tile's copy, by the chunk's parity
  uint64_t* v_bar = done + 4;
  uint64_t* formed = done + 6;                                    // [2] a half's Kd: eight warps
  uint64_t* g_bar = done + 8;                                     // [2] a chunk's gates, by its parity
  uint64_t* g_read = done + 10;                                   // [2] that they have been read: eight warps
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + OFF_MISC + 96);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + OFF_MISC + 100);
  double* totals = reinterpret_cast<double*>(sm + ST_TOTALS);      // [10] the warps' sums of log-decays

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(sm) & 1023) {         // the swizzled tiles' base
    if (tid == 0) atomicCAS(err, 0, JB_DEV_LAUNCH | 60);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < 12; ++i) mbar_init(done + i, i == 6 || i == 7 || i >= 10 ? 8 : 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, TM_COLS);
    tmem_relinquish();
  }
  const int pair = blockIdx.x / seg.count, part = blockIdx.x % seg.count;
  const int row = pair / a.heads, h = pair % a.heads;
  const int stop = a.real ? min(max(a.real[row], 0), a.n) : a.n;
  const int begin = part * seg.chunks * C, work = min(min(begin + seg.chunks * C, a.n), stop);
  const int chunks = begin < work ? (work - begin + C - 1) / C : 0;
  auto start_of = [&](int i) { return begin + i * C; };   // the first token of chunk i
  auto k_place = [&](int i) { return sm + ST_K + (i & 1) * 8192; };
  auto v_place = [&](int i) { return sm + ST_V + (i & 1) * TILE; };
  // the segment's whole log-decay
  const float* gp = a.g + row * a.g_row + h;
  {
    double sum = 0.0;
    for (int t = begin + tid; t < work; t += ST_THREADS) sum += log_decay(gp[t * a.g_tok]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) totals[warp] = sum;
  }
  auto odd = [](int i) { return (uint32_t)i & 1; };          // a barrier that every chunk uses: chunk i's phase
  auto odd2 = [](int i) { return (uint32_t)(i >> 1) & 1; };  // one that every other chunk uses
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 8) {
    // the accumulators' first values
    uint32_t r[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = 0u;
    const uint32_t s_at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + TM_S + 64 * (warp >> 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) tmem_st32(s_at + (i & 1) * 32 + (i >> 1) * TM_SMALL, r);
    tc_wait_st();
    for (int c = 0; c < chunks && !*abort_flag; ++c) {
      const int live = min(C, work - start_of(c));
      const Gates& gt = gates[c & 1];
      // values past the row's end may be anything: zeros, so that a zero weight keeps them out
      if (live < C) {
        mbar_wait(v_bar + (c & 1), odd2(c), abort_flag, err, 64);
        for (int i = tid; i < (C - live) * 16; i += 256) {
          const int t = live + (i >> 4), x = i & 15;
          *reinterpret_cast<uint4*>(swz(v_place(c) + (x >> 3) * 8192, t, x & 7)) = make_uint4(0, 0, 0, 0);
        }
      }
      mbar_wait(k_bar + (c & 1), odd2(c), abort_flag, err, 62);
      mbar_wait(g_bar + (c & 1), odd2(c), abort_flag, err, 63);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (c > 0) mbar_wait(done + half, odd(c - 1), abort_flag, err, 61);   // the places of this half's Kd are free
        uint4 x[2];
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          const int t = 32 * half + 16 * it + (tid >> 4), p = tid & 15;
          x[it] = *reinterpret_cast<const uint4*>(swz(k_place(c) + (p >> 3) * 16384, t, p & 7));
        }
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          const int t = 32 * half + 16 * it + (tid >> 4), p = tid & 15;
          uint4 y[3];
          split8(x[it], gt.to_end[t], y);
#pragma unroll
          for (int u = 0; u < 3; ++u)
            *reinterpret_cast<uint4*>(swz(u == 0 ? k_place(c) + (p >> 3) * 16384
                                                 : sm + (u == 1 ? ST_K1 : ST_K2) + (p >> 3) * 8192, t, p & 7)) =
                t < live ? y[u] : make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(formed + half);
      }
      if (lane == 0) mbar_arrive(g_read + (c & 1));
    }
  } else if (warp == 8) {
    const bool me = elect_one();
    int issued = 0;
    auto load = [&](int i) {
      ++issued;
      if (!me) return;
      mbar_arrive_expect_tx(k_bar + (i & 1), TILE);
      tma_load_4d(k_place(i), &tm_k, k_bar + (i & 1), 0, h, start_of(i), row);
      tma_load_4d(k_place(i) + 16384, &tm_k, k_bar + (i & 1), 64, h, start_of(i), row);
      mbar_arrive_expect_tx(v_bar + (i & 1), TILE);
      tma_load_4d(v_place(i), &tm_v, v_bar + (i & 1), 0, h, start_of(i), row);
      tma_load_4d(v_place(i) + 8192, &tm_v, v_bar + (i & 1), 64, h, start_of(i), row);
    };
    auto ahead = [&](int i) {   // to L2, since a tile's place is free only half a chunk before it is needed
      if (i < chunks && me) {
        prefetch_tile(&tm_k, h, start_of(i), row);
        prefetch_tile(&tm_v, h, start_of(i), row);
      }
    };
    if (chunks > 0) load(0);
    if (chunks > 1) load(1);
    ahead(2);
    constexpr uint32_t id = idesc_bf16(128, 128) | A_MN | B_MN;
    for (int c = 0; c < chunks && !*abort_flag; ++c) {
      mbar_wait(v_bar + (c & 1), odd2(c), abort_flag, err, 64);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (half == 1 && c > 0 && c + 1 < chunks) {   // the last chunk's products are done: its places are the next's
          mbar_wait(done + 1, odd(c - 1), abort_flag, err, 61);
          load(c + 1);
        }
        if (half == 1) ahead(c + 3);
        mbar_wait(formed + half, odd(c), abort_flag, err, 65);
        __syncwarp();
        tc_fence_after();
        const uint32_t v_a = smem_u32(v_place(c)), k_a = smem_u32(k_place(c)), p1 = smem_u32(sm + ST_K1),
                       p2 = smem_u32(sm + ST_K2);
#pragma unroll
        for (int kk = 2 * half; kk < 2 * half + 2; ++kk) {
          const uint64_t av = mn_desc(v_a + kk * 2048, 8192), b0 = mn_desc(k_a + kk * 2048, 16384),
                         b1 = mn_desc(p1 + kk * 2048, 8192), b2 = mn_desc(p2 + kk * 2048, 8192);
          if (me) {
            tc_mma_bf16(tmem + TM_SMALL, av, b2, id, 1);
            tc_mma_bf16(tmem + TM_SMALL, av, b1, id, 1);
            tc_mma_bf16(tmem + TM_S, av, b0, id, 1);
          }
        }
        if (me) tc_commit(done + half);
        __syncwarp();
      }
    }
    if (*abort_flag) {
      // a CTA that gave up waits (bounded) for the copies it issued before its shared memory goes away: the last two
      // tiles', the others having landed before these were issued
      const uint64_t t0 = global_ns();
      auto landed = [&]() {
        bool all = true;
        for (int i = max(0, issued - 2); i < issued; ++i)
          all = all && mbar_try_wait(k_bar + (i & 1), odd2(i)) && mbar_try_wait(v_bar + (i & 1), odd2(i));
        return all;
      };
      while (!landed() && global_ns() - t0 < kWaitNs) {
      }
    }
  } else {
    auto gate = [&](int i, int t) { return i < chunks && t < work ? gp[t * a.g_tok] : 0.f; };   // 0 past the row's end
    double left = 0.0;
#pragma unroll
    for (int w = 0; w < ST_THREADS / 32; ++w) left += totals[w];
    if (lane == 0) seg.decay[(int64_t)pair * seg.count + part] = exp2_fast((float)left);
    float g0 = gate(0, start_of(0) + lane), g1 = gate(0, start_of(0) + 32 + lane);
    for (int c = 0; c < chunks && !*abort_flag; ++c) {
      const float x0 = g0, x1 = g1;
      g0 = gate(c + 1, start_of(c + 1) + lane);
      g1 = gate(c + 1, start_of(c + 1) + 32 + lane);
      if (c > 1) mbar_wait(g_read + (c & 1), odd2(c - 2), abort_flag, err, 66);
      double same = left;
      form_gates<true>(gates[c & 1], 0, x0, x1, lane, nullptr, same);
      form_gates<true>(gates[c & 1], 1, x0, x1, lane, nullptr, left);
      __syncwarp();
      if (lane == 0) mbar_arrive(g_bar + (c & 1));
    }
  }
  if (chunks > 0) {
    mbar_wait(done, odd(chunks - 1), abort_flag, err, 61);
    mbar_wait(done + 1, odd(chunks - 1), abort_flag, err, 61);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*abort_flag == 0) {   // through shared memory as one copy
    float* state = reinterpret_cast<float*>(sm);
    if (warp < 8) {
      const int L = 32 * (warp & 3) + lane, ch = warp >> 2;
      const uint32_t s_at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + TM_S + 64 * ch;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t r[32], small[32];
        tmem_ld32(s_at + 32 * half, r);
        tmem_ld32(s_at + TM_SMALL + 32 * half, small);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          state[(ch * 64 + half * 32 + i) * D + L] = __uint_as_float(r[i]) + __uint_as_float(small[i]);
      }
      fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0) {
      bulk_store(seg.states + ((int64_t)pair * seg.count + part) * STATE, state, STATE * 4);
      tma_store_commit();
      tma_store_wait_all();
    }
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, TM_COLS);
  }
}

// The segments' contributions of a (row, head) -> the state ahead of each, in place, and the final state. Thread = four
// neighbouring values of the state.
__global__ void __launch_bounds__(256) join_kernel(const Args a, const Seg seg) {
  const int pair = blockIdx.x, row = pair / a.heads, h = pair % a.heads;
  const int i = blockIdx.y * 256 + threadIdx.x;
  const float* in = lin::state_in(a.pool, row, h);
  // (written before the states' launch began, and that has let this one go)
  float4 s = in ? reinterpret_cast<const float4*>(in)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
  pdl_begin();
  float4* parts = reinterpret_cast<float4*>(seg.states + (int64_t)pair * seg.count * STATE) + i;
  const float* decay = seg.decay + (int64_t)pair * seg.count;
  constexpr int AHEAD = 8;   // segments read before the first of them is overwritten
  for (int p0 = 0; p0 < seg.count; p0 += AHEAD) {
    float4 x[AHEAD];
    float e[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (p0 + j < seg.count) {
        x[j] = parts[(int64_t)(p0 + j) * (STATE / 4)];
        e[j] = decay[p0 + j];
      }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (p0 + j < seg.count) {
        parts[(int64_t)(p0 + j) * (STATE / 4)] = s;
        s = make_float4(s.x * e[j] + x[j].x, s.y * e[j] + x[j].y, s.z * e[j] + x[j].z, s.w * e[j] + x[j].w);
      }
  }
  if (float* out = lin::state_out(a.pool, row, h)) reinterpret_cast<float4*>(out)[i] = s;
}

// q, k, v or o (b, n, heads, 128) as a 4-D tensor map (channel, head, token, row), boxes of 64 x 1 x 64 x 1
int tile_map(CUtensorMap* map, const void* base, const Args& a, int b, int64_t tok, int64_t row) {
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)a.heads, (uint64_t)a.n, (uint64_t)b};
  const uint64_t strides[3] = {(uint64_t)D * 2, (uint64_t)tok * 2, (uint64_t)row * 2};
  const uint32_t box[4] = {64, 1, (uint32_t)C, 1};
  return make_tmap_nd(map, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Segments of a (row, head). Measured on a B200, in us: one segment takes 4 + 3.5 a chunk; segments of `per` chunks, all
// of them at once, 9 + 4.7 per + 0.045 for each segment of the call, whose states are written, joined, and read again.
// So 8 rows of 256 tokens stay whole (20.8 us, 30.5 in two segments a head), one row of 1,001 takes segments of two
// chunks (21.7; 66 whole), one of 8,192 as many as run at once.
inline Seg segments(int b, int heads, int n) {
  const int chunks = (n + C - 1) / C;
  const int64_t pairs = (int64_t)b * heads;
  const int64_t most = FIT / pairs;
  int64_t best = 4000 + 3500ll * chunks;   // ns
  int per = chunks;
  for (int64_t p = most ? (chunks + most - 1) / most : chunks; p < chunks && 4700 * p < best; ++p) {
    const int64_t cost = 9000 + 4700 * p + 45 * pairs * ((chunks + p - 1) / p);
    if (cost < best) {
      best = cost;
      per = (int)p;
    }
  }
  return {(chunks + per - 1) / per, per, nullptr, nullptr};
}
inline int64_t scratch_floats(int b, int heads, int n) {
  const Seg s = segments(b, heads, n);
  return s.count == 1 ? 0 : (int64_t)b * heads * s.count * (STATE + 1);
}

template <int MODE>
int launch(const CUtensorMap (&m)[4], const Args& a, const Seg& seg, int b, cudaStream_t stream) {
  if (int st = gdnc::configure(scan_kernel<MODE>, ALLOC, "linear scan_kernel")) return st;
  launch_pdl(scan_kernel<MODE>, b * a.heads * seg.count, THREADS, ALLOC, stream, m[0], m[1], m[2], m[3], a, seg,
             device_status_word());
  return check_launch("linear scan_kernel");
}

int scan(const Args& a, int b, float* scratch, cudaStream_t stream) {
  CUtensorMap m[4];   // a single row's stride may be anything
  auto row = [&](int64_t stride, int64_t tok) { return b == 1 ? tok * a.n : stride; };
  int st = tile_map(&m[0], a.q, a, b, a.q_tok, row(a.q_row, a.q_tok));
  if (!st) st = tile_map(&m[1], a.k, a, b, a.k_tok, row(a.k_row, a.k_tok));
  if (!st) st = tile_map(&m[2], a.v, a, b, a.v_tok, row(a.v_row, a.v_tok));
  if (!st) st = tile_map(&m[3], a.o, a, b, a.o_tok, row(a.o_row, a.o_tok));
  if (st) return st;
  Seg seg = segments(b, a.heads, a.n);
  if (seg.count == 1) return launch<WHOLE>(m, a, seg, b, stream);
  const int64_t parts = (int64_t)b * a.heads * seg.count;
  seg.states = scratch;
  seg.decay = scratch + parts * STATE;
  if ((st = gdnc::configure(states_kernel, ALLOC, "linear states_kernel"))) return st;
  launch_pdl(states_kernel, (unsigned)parts, ST_THREADS, ALLOC, stream, m[1], m[2], a, seg, device_status_word());
  if ((st = check_launch("linear states_kernel"))) return st;
  launch_pdl(join_kernel, dim3(b * a.heads, STATE / 4 / 256), 256, 0, stream, a, seg);
  if ((st = check_launch("linear join_kernel"))) return st;
  return launch<OUTPUTS>(m, a, seg, b, stream);
}

}  // namespace lintc
}  // namespace jb
