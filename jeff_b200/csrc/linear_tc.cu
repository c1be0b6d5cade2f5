// The chunked form of linear.cu's recurrence on tcgen05: chunks of C = 64 tokens, with gc the log-decays summed within
// the chunk and gl their total,
//   O = scale ((e^gc Q) S + (Q K^T ∘ Γ, causal) V),   Γ_ij = e^{gc_i - gc_j},
//   S <- e^gl S + (e^{gl - gc} K)^T V,
// every product an M = 128 MMA with the transposed state S^T (lanes: value columns) in tensor memory:
//   MMA1  D = [K; Q] K^T              (lanes 64-127: Q K^T; the stacked A is the K and Q tiles laid out back to back)
//   MMA2  D = bf16(S^T) Q'^T          (A in tensor memory; Q' = e^gc Q as two bf16 parts)
//   MMA3  D += V^T P^T = O^T          (P = bf16(Q K^T ∘ Γ))
//   MMA4  S^T += V^T Kd               (Kd = e^{gl - gc} K in bf16 parts, S^T scaled by e^gl beforehand)
// Rounding: the state is fp32 and what enters it keeps 24 bits (three bf16 parts of a decayed key, the value exact).
// Ahead of an output's own rounding its terms are rounded once, by P for the tokens of its chunk, by the state's bf16
// copy for those before (where the state itself is another launch's, two parts of Kd, 16 bits, serve that copy). Sums
// of decays are fp64, their differences rounded to fp32 once, so that a strong decay early in a chunk takes no accuracy
// from the tokens behind it (-inf is held as -10000, whose exponential is 0).
//
// Tensor memory, 256 columns: S^T 0-127, its bf16 copy 128-191, D 192-255. Shared memory 107 KB: two CTAs per SM, whose
// phases (TMA, tensor core, CUDA cores) fill each other's waits. Within a chunk Kd's later parts are formed while MMA1
// runs, the next chunk's gates while MMA2-4 run, and the next tiles travel during the output and the state's copy: two
// block barriers a chunk. Of Γ's four 32 x 32 blocks one is zero and one a product of two vectors, so two warps of
// eight form exponentials and the others Q'. A (row, head) is one CTA, or, where those are fewer than the CTAs that
// fit, is cut into segments of whole chunks: a first launch leaves each segment's own contribution to the state in
// scratch (no Q, no outputs), a second turns these into the state ahead of each segment and the final one, the third
// computes the outputs. Waits are bounded (%globaltimer, 2 s): on expiry the CTA records JB_DEV_TIMEOUT | 50.. in the
// device status word and returns.

namespace jb {
namespace lintc {

using gdnt::A_MN;
using gdnt::B_MN;
using gdnt::exp_neg;
using gdnt::mn_desc;
using gdnt::swz;
using gdnt::tc_wait_st;
using gdnt::tmem_st32;
using lin::Args;
using lin::D;

constexpr int C = 64, THREADS = 256;
constexpr uint32_t TILE = C * D * 2;   // 16 KB: two 64-column atoms of 64 rows x 128 B
constexpr int OFF_KQ = 0;              // atom a: K at a * 16384, Q at + 8192; then parts of Kd and Q' in place
constexpr int OFF_KM = 32768, OFF_KL = OFF_KM + TILE;   // other parts of Kd (atoms 8192 apart)
constexpr int OFF_QL = OFF_KL + TILE;  // Q's second part; then the output tile
constexpr int OFF_V = OFF_QL + TILE;
constexpr int OFF_P = OFF_V + TILE;    // 64 rows x 128 B
constexpr int OFF_G = OFF_P + TILE / 2;   // two sets of gates
constexpr int OFF_MISC = OFF_G + 2 * 5 * C * 4;
constexpr int ALLOC = OFF_MISC + 64;
static_assert(2 * (ALLOC + 1024) <= 228 * 1024, "two CTAs per SM");
constexpr uint32_t TM_S = 0, TM_B = 128, TM_D = 192, TM_COLS = 256;
constexpr int FIT = 2 * 148;           // CTAs that run at once
constexpr int STATE = D * D;

enum Mode { WHOLE, STATES, OUTPUTS };

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

// eight bf16 values times f, in `parts` bf16 parts
template <int PARTS>
__device__ __forceinline__ void split8(const uint4& x, float f, uint4 (&y)[PARTS]) {
  const uint32_t in[4] = {x.x, x.y, x.z, x.w};
  uint32_t out[PARTS][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = bf_lo(in[i]) * f, b = bf_hi(in[i]) * f;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      out[p][i] = pack_bf2(a, b);
      a -= bf_lo(out[p][i]);
      b -= bf_hi(out[p][i]);
    }
  }
#pragma unroll
  for (int p = 0; p < PARTS; ++p) y[p] = make_uint4(out[p][0], out[p][1], out[p][2], out[p][3]);
}

// A chunk's gates, from the sums gc of its log-decays: gc in two floats (their differences are the exponents inside the
// chunk), e^gc, e^{gl - gc}, and Γ's lower left 32 x 32 block as cross[32 + i] cross[j].
struct Gates {
  float hi[C], lo[C], from_start[C], to_end[C], cross[C];
};

__device__ __forceinline__ void form_gates(Gates& g, float a, float b, int lane, volatile float* whole, double& sum) {
  double x = a, y = b;   // tokens lane and lane + 32
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
  g.hi[lane] = (float)x;
  g.hi[lane + 32] = (float)y;
  g.lo[lane] = (float)(x - (double)(float)x);
  g.lo[lane + 32] = (float)(y - (double)(float)y);
  g.from_start[lane] = expf((float)x);
  g.from_start[lane + 32] = expf((float)y);
  g.to_end[lane] = expf((float)(all - x));
  g.to_end[lane + 32] = expf((float)(all - y));
  g.cross[lane] = expf((float)(mid - x));
  g.cross[lane + 32] = expf((float)(y - mid));
  if (lane == 0) *whole = expf((float)all);
  sum += all;
}

template <int MODE>
__global__ void __launch_bounds__(THREADS, 2)
    scan_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o, const Args a,
                const Seg seg, int* err) {
  pdl_begin();
  constexpr int PARTS = MODE == OUTPUTS ? 2 : 3;   // of Kd
  extern __shared__ __align__(1024) uint8_t sm[];
  uint8_t* kq = sm + OFF_KQ;
  uint8_t* km = sm + OFF_KM;
  uint8_t* kl = sm + OFF_KL;
  uint8_t* ql = sm + OFF_QL;
  uint8_t* vb = sm + OFF_V;
  uint8_t* pt = sm + OFF_P;
  Gates* gates = reinterpret_cast<Gates*>(sm + OFF_G);
  uint64_t* mma_bar = reinterpret_cast<uint64_t*>(sm + OFF_MISC);
  uint64_t* in_bar = mma_bar + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + OFF_MISC + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + OFF_MISC + 20);
  volatile float* whole = reinterpret_cast<volatile float*>(sm + OFF_MISC + 24);   // [2] the chunks' decay factors

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int qd = warp & 3, ch = warp >> 2;
  const int L = 32 * qd + lane;   // this thread's tensor-memory lane
  const uint32_t lane_bits = (uint32_t)(32 * qd) << 16;
  const int pair = blockIdx.x / seg.count, part = blockIdx.x % seg.count;
  const int row = pair / a.heads, h = pair % a.heads;
  const int stop = a.real ? min(max(a.real[row], 0), a.n) : a.n;
  const int begin = part * seg.chunks * C, end = min(begin + seg.chunks * C, a.n);
  const int work = min(end, stop);   // tokens past it are padding: zeros out, the state stays
  if (smem_u32(sm) & 1023) {         // the swizzled tiles' base
    if (tid == 0) atomicCAS(err, 0, JB_DEV_LAUNCH | 50);
    return;
  }

  if (tid == 0) {
    mbar_init(mma_bar, 1);
    mbar_init(in_bar, 2);   // the loads, and that the previous output tile has left its place
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, TM_COLS);
    tmem_relinquish();
  }
  int issued = 0;
  auto load = [&](int c0) {
    ++issued;
    mbar_arrive_expect_tx(in_bar, (MODE == STATES ? 2 : 3) * TILE);
    tma_load_4d(kq, &tm_k, in_bar, 0, h, c0, row);
    tma_load_4d(kq + 16384, &tm_k, in_bar, 64, h, c0, row);
    if (MODE != STATES) {
      tma_load_4d(kq + 8192, &tm_q, in_bar, 0, h, c0, row);
      tma_load_4d(kq + 16384 + 8192, &tm_q, in_bar, 64, h, c0, row);
    }
    tma_load_4d(vb, &tm_v, in_bar, 0, h, c0, row);
    tma_load_4d(vb + 8192, &tm_v, in_bar, 64, h, c0, row);
  };
  const float* gp = a.g + row * a.g_row + h;
  auto gate = [&](int t) {   // the log-decay of token t, 0 past the row's end, -inf as a finite number
    if (t >= work) return 0.f;
    const float x = gp[t * a.g_tok];
    return x < -1e4f ? -1e4f : x;
  };
  double decays = 0.0;   // warp 0: the segment's log-decay
  float g0 = 0.f, g1 = 0.f;
  if (warp == 0) {
    g0 = gate(begin + lane);
    g1 = gate(begin + 32 + lane);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && begin < work) load(begin);
  const uint32_t tmem = *tmem_slot;
  if (warp == 0) {
    form_gates(gates[0], g0, g1, lane, whole, decays);
    g0 = gate(begin + C + lane);
    g1 = gate(begin + C + 32 + lane);
  }
  if (MODE != STATES)   // P's upper right block is never anything else
    for (int i = tid; i < 32 * 4; i += THREADS)
      *reinterpret_cast<uint4*>(swz(pt, i >> 2, 4 + (i & 3))) = make_uint4(0, 0, 0, 0);

  // the state ahead of the segment: lane = value column, columns = key rows
  {
    const float* in = MODE == WHOLE ? lin::state_in(a.pool, row, h)
                      : MODE == OUTPUTS ? seg.states + ((int64_t)pair * seg.count + part) * STATE : nullptr;
    for (int half = 0; half < 2; ++half) {
      uint32_t r[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = in ? __float_as_uint(in[(ch * 64 + half * 32 + i) * D + L]) : 0u;
      tmem_st32(tmem + lane_bits + TM_S + ch * 64 + half * 32, r);
    }
    tc_wait_st();
  }
  // the state's bf16 copy, then its decay over the chunk
  auto turn_state = [&](float el) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t ta = tmem + lane_bits + TM_S + 64 * ch + 32 * half;
      uint32_t r[32];
      tmem_ld32(ta, r);
      tc_wait_ld();
      if (MODE != STATES) {
        uint32_t b[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) b[e] = pack_bf2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
        tmem_st16(tmem + lane_bits + TM_B + 32 * ch + 16 * half, b);
      }
#pragma unroll
      for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * el);
      tmem_st32(ta, r);
    }
    tc_wait_st();
  };
  __syncthreads();
  if (begin < work) turn_state(whole[0]);

  const uint32_t kq_a = smem_u32(kq), km_a = smem_u32(km), kl_a = smem_u32(kl), ql_a = smem_u32(ql),
                 vb_a = smem_u32(vb), pt_a = smem_u32(pt);
  uint32_t mma_phase = 0, in_phase = 0, set = 0;
  for (int c0 = begin; c0 < work; c0 += C) {
    const int live = min(C, work - c0);
    const bool more = c0 + C < work;
    const Gates& gt = gates[set];
    if (tid == 0) {
      if (MODE != STATES) tma_store_wait_read();
      mbar_arrive(in_bar);
    }
    mbar_wait(in_bar, in_phase, abort_flag, err, 52);
    in_phase ^= 1;
    // ---- MMA1
    if (MODE != STATES && warp == 1) {
      __syncwarp();
      tc_fence_after();
      constexpr uint32_t id1 = idesc_bf16(128, 64);
      const bool issuer = elect_one();
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t dsc = sw128_desc(kq_a + (kk >> 2) * 16384 + 32 * (kk & 3));
        if (issuer) tc_mma_bf16(tmem + TM_D, dsc, dsc, id1, kk != 0);
      }
      if (issuer) tc_commit(mma_bar);
      __syncwarp();
    }
    // values past the row's end may be anything: zeros, so that a zero weight keeps them out
    if (live < C)
      for (int i = tid; i < (C - live) * 16; i += THREADS) {
        const int t = live + (i >> 4), c = i & 15;
        *reinterpret_cast<uint4*>(swz(vb + (c >> 3) * 8192, t, c & 7)) = make_uint4(0, 0, 0, 0);
      }
    // ---- Kd: thread = 16-byte piece of a token; with three parts the first waits for MMA1 to have read K
    uint4 first[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int i = it * THREADS + tid, t = i >> 4, c = i & 15, at = c >> 3;
      uint4 y[PARTS];
#pragma unroll
      for (int p = 0; p < PARTS; ++p) y[p] = make_uint4(0, 0, 0, 0);
      if (t < live) split8(*reinterpret_cast<const uint4*>(swz(kq + at * 16384, t, c & 7)), gt.to_end[t], y);
      *reinterpret_cast<uint4*>(swz(km + at * 8192, t, c & 7)) = y[PARTS - 2];
      *reinterpret_cast<uint4*>(swz(kl + at * 8192, t, c & 7)) = y[PARTS - 1];
      first[it] = y[0];
    }
    if (MODE != STATES) {
      mbar_wait(mma_bar, mma_phase, abort_flag, err, 51);
      mma_phase ^= 1;
      tc_fence_after();
    }
    if (PARTS == 3) {
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int i = it * THREADS + tid, t = i >> 4, c = i & 15;
        *reinterpret_cast<uint4*>(swz(kq + (c >> 3) * 16384, t, c & 7)) = first[it];
      }
    }
    if (MODE != STATES) {
      if (qd >= 2 && !(qd == 2 && ch == 1)) {
        // ---- P from D's lanes 64-127: row i = L - 64, columns 32 ch .. + 31
        uint32_t r[32];
        tmem_ld32(tmem + lane_bits + TM_D + 32 * ch, r);
        tc_wait_ld();
        const int i = L - C;
        const float hi = gt.hi[i], lo = gt.lo[i], ci = gt.cross[i];
        const int upto = i < live ? i : -1;
#pragma unroll
        for (int c8 = 0; c8 < 4; ++c8) {
          uint32_t pk[4];
#pragma unroll
          for (int e2 = 0; e2 < 4; ++e2) {
            float x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = 32 * ch + 8 * c8 + 2 * e2 + e;
              const float f = qd == 3 && ch == 0 ? ci * gt.cross[j] : exp_neg((hi - gt.hi[j]) + (lo - gt.lo[j]));
              x[e] = j <= upto ? __uint_as_float(r[8 * c8 + 2 * e2 + e]) * f : 0.f;
            }
            pk[e2] = pack_bf2(x[0], x[1]);
          }
          *reinterpret_cast<uint4*>(swz(pt, i, 4 * ch + c8)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
      }
      if (warp != 2 && warp != 7) {
        // ---- Q' over Q, its second part behind: the six warps that form no exponentials
        const int me = (warp - (warp > 2)) * 32 + lane;
        for (int i = me; i < C * 16; i += 6 * 32) {
          const int t = i >> 4, c = i & 15, at = c >> 3;
          uint8_t* p = swz(kq + at * 16384 + 8192, t, c & 7);
          uint4 y[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
          if (t < live) split8(*reinterpret_cast<const uint4*>(p), gt.from_start[t], y);
          *reinterpret_cast<uint4*>(p) = y[0];
          *reinterpret_cast<uint4*>(swz(ql + at * 8192, t, c & 7)) = y[1];
        }
      }
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) break;
    // ---- MMA2, MMA3, MMA4
    if (warp == 1) {
      tc_fence_after();
      const bool issuer = elect_one();
      if (MODE != STATES) {
        constexpr uint32_t id2 = idesc_bf16(128, 64), id3 = idesc_bf16(128, 64) | A_MN;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t b0 = sw128_desc(kq_a + 8192 + (kk >> 2) * 16384 + 32 * (kk & 3));
          const uint64_t b1 = sw128_desc(ql_a + (kk >> 2) * 8192 + 32 * (kk & 3));
          if (issuer) {
            w4t::tc_mma_ts(tmem + TM_D, tmem + TM_B + 8 * kk, b0, id2, kk != 0);
            w4t::tc_mma_ts(tmem + TM_D, tmem + TM_B + 8 * kk, b1, id2, 1);
          }
        }
#pragma unroll
        for (int kk = 0; kk < C / 16; ++kk) {
          const uint64_t av = mn_desc(vb_a + kk * 2048, 8192), b0 = sw128_desc(pt_a + 32 * kk);
          if (issuer) tc_mma_bf16(tmem + TM_D, av, b0, id3, 1);
        }
      }
      constexpr uint32_t id4 = idesc_bf16(128, 128) | A_MN | B_MN;
#pragma unroll
      for (int kk = 0; kk < C / 16; ++kk) {
        const uint64_t av = mn_desc(vb_a + kk * 2048, 8192);
        const uint64_t b0 = mn_desc(kq_a + kk * 2048, 16384), b1 = mn_desc(km_a + kk * 2048, 8192),
                       b2 = mn_desc(kl_a + kk * 2048, 8192);
        if (issuer) {
          tc_mma_bf16(tmem + TM_S, av, b2, id4, 1);   // the small parts first
          tc_mma_bf16(tmem + TM_S, av, b1, id4, 1);
          if (PARTS == 3) tc_mma_bf16(tmem + TM_S, av, b0, id4, 1);
        }
      }
      if (issuer) tc_commit(mma_bar);
      __syncwarp();
    }
    if (warp == 0 && more) {   // the next chunk's gates, and the decays of the one after it
      form_gates(gates[set ^ 1], g0, g1, lane, whole + (set ^ 1), decays);
      g0 = gate(c0 + 2 * C + lane);
      g1 = gate(c0 + 2 * C + 32 + lane);
    }
    set ^= 1;
    mbar_wait(mma_bar, mma_phase, abort_flag, err, 51);
    mma_phase ^= 1;
    tc_fence_after();
    if (tid == 0 && more) load(c0 + C);   // every tile has been read
    if (MODE != STATES) {
      // ---- O^T -> bf16 -> the output tile over Q's second part, laid out as the loads -> TMA store
      uint32_t r[32];
      tmem_ld32(tmem + lane_bits + TM_D + 32 * ch, r);
      tc_wait_ld();
      const float scale = rsqrtf((float)D);
      __nv_bfloat16* ot = reinterpret_cast<__nv_bfloat16*>(ql + (L >> 6) * 8192);
      const int cl = L & 63;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const int t = 32 * ch + e;
        ot[(sw128_offset(t, cl >> 3) >> 1) + (cl & 7)] = f2bf(t < live ? __uint_as_float(r[e]) * scale : 0.f);
      }
      fence_proxy_async_smem();
      tc_fence_before();
    }
    __syncthreads();
    if (*abort_flag) break;
    if (MODE != STATES && tid == 0) {
      tma_store_4d(&tm_o, ql, 0, h, c0, row);
      tma_store_4d(&tm_o, ql + 8192, 64, h, c0, row);
      tma_store_commit();
    }
    if (more) turn_state(whole[set]);
  }
  const bool ok = *abort_flag == 0;
  if (tid == 0) {
    if (MODE != STATES) tma_store_wait_all();
    // a CTA that gave up waits (bounded) for the copies it issued before its shared memory goes away: without its own
    // arrival their phase may never end, so it arrives first
    if (!ok && issued) {
      mbar_arrive(in_bar);
      const uint64_t t0 = global_ns();
      while (!mbar_try_wait(in_bar, (issued - 1) & 1) && global_ns() - t0 < kWaitNs) {
      }
    }
  }
  if (MODE != STATES) {   // chunks that hold padding only
    const int first = max(begin, (work + C - 1) / C * C);
    for (int i = first * 16 + tid; i < end * 16; i += THREADS)
      reinterpret_cast<uint4*>(a.o + row * a.o_row + (int64_t)(i >> 4) * a.o_tok + h * D)[i & 15] =
          make_uint4(0, 0, 0, 0);
  }
  float* out = MODE == WHOLE ? lin::state_out(a.pool, row, h)
               : MODE == STATES ? seg.states + ((int64_t)pair * seg.count + part) * STATE : nullptr;
  if (ok && out) {
    for (int half = 0; half < 2; ++half) {
      uint32_t r[32];
      tmem_ld32(tmem + lane_bits + TM_S + 64 * ch + 32 * half, r);
      tc_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) out[(ch * 64 + half * 32 + i) * D + L] = __uint_as_float(r[i]);
    }
    if (MODE == STATES && tid == 0) seg.decay[(int64_t)pair * seg.count + part] = expf((float)decays);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, TM_COLS);
  }
}

// The segments' contributions of a (row, head) -> the state ahead of each, in place, and the final state. Thread = four
// neighbouring values of the state.
__global__ void __launch_bounds__(256) join_kernel(const Args a, const Seg seg) {
  pdl_begin();
  const int pair = blockIdx.x, row = pair / a.heads, h = pair % a.heads;
  const int i = blockIdx.y * 256 + threadIdx.x;
  const float* in = lin::state_in(a.pool, row, h);
  float4 s = in ? reinterpret_cast<const float4*>(in)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
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

// Segments of a (row, head): as many as let every CTA that fits run at once, none shorter than a chunk.
inline Seg segments(int b, int heads, int n) {
  const int chunks = (n + C - 1) / C;
  const int64_t pairs = (int64_t)b * heads;
  const int most = (int)max((int64_t)1, FIT / pairs);
  const int per = (chunks + most - 1) / most;
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
  if ((st = launch<STATES>(m, a, seg, b, stream))) return st;
  launch_pdl(join_kernel, dim3(b * a.heads, STATE / 4 / 256), 256, 0, stream, a, seg);
  if ((st = check_launch("linear join_kernel"))) return st;
  return launch<OUTPUTS>(m, a, seg, b, stream);
}

}  // namespace lintc
}  // namespace jb
