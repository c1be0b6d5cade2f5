// Linear attention with a decay for each head, each row resuming from its state in the prefix pool:
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T,   o_t = S_t^T q_t / sqrt(128)
// over (128 key, 128 value) fp32 states: a chunked form for prompts and a recurrent one for single tokens, which with
// beta is the gated delta rule (v_t replaced by beta_t (v_t - (e^{g_t} S_{t-1})^T k_t)).
//
// A state is at slot (flat head % heads_per_page) of page tables[r][flat head / heads_per_page], as in gdn.cu. A page
// outside the pool reads as zeros, and so does the sink, which a table names where no page was to be had and which holds
// what others left there; nothing is written to such pages or to the page of zeros.

namespace jb {
namespace lin {

constexpr int D = 128;
constexpr int64_t STATE_BYTES = (int64_t)D * D * 4;
constexpr int SINK = 0, RESERVED = 2;

struct Pool {
  uint8_t* base;
  int64_t pages, page_bytes;
  int heads_per_page, first_head;
  const int* tables;
  int table_stride;
  const int* out_tables;
  int out_stride;
};

__device__ __forceinline__ const float* state_in(const Pool& p, int row, int h) {
  const int flat = p.first_head + h;
  const int page = p.tables[(int64_t)row * p.table_stride + flat / p.heads_per_page];
  if (page <= SINK || page >= p.pages) return nullptr;
  return reinterpret_cast<const float*>(p.base + page * p.page_bytes + (flat % p.heads_per_page) * STATE_BYTES);
}
__device__ __forceinline__ float* state_out(const Pool& p, int row, int h) {
  if (!p.out_tables) return nullptr;
  const int flat = p.first_head + h;
  const int page = p.out_tables[(int64_t)row * p.out_stride + flat / p.heads_per_page];
  if (page < RESERVED || page >= p.pages) return nullptr;
  return reinterpret_cast<float*>(p.base + page * p.page_bytes + (flat % p.heads_per_page) * STATE_BYTES);
}

struct Args {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t q_row, k_row, v_row;   // strides in elements between rows, and between a row's tokens
  int64_t q_tok, k_tok, v_tok;
  const float* g;
  int64_t g_row, g_tok;          // both 0: a constant decay for each head
  const __nv_bfloat16* beta;     // (b, heads) or null
  const int* real;               // (b,) or null
  __nv_bfloat16* o;
  int64_t o_row, o_tok;
  int n, heads;
  Pool pool;
};

// ------------------------------------------------------------------ token by token
//
// The prompts of a few tokens: the state is read and written once (bound by HBM for many rows: 64 rows of 2 tokens 30 us),
// every token after the first adds its chain of two barriers (0.6 us for one row). One CTA per (row, head); warp w holds
// key rows [16 w, 16 w + 16) of the state in registers, lane l value columns [4 l, 4 l + 4): 16-byte accesses, 512
// contiguous bytes a warp and instruction, all 16 of a thread in flight.

// S = e S + k v (one key row, four columns), and c += q S
__device__ __forceinline__ void advance(float4& S, float e, float k, const float4& v, float q, float4& c) {
  S.x = S.x * e + k * v.x;
  S.y = S.y * e + k * v.y;
  S.z = S.z * e + k * v.z;
  S.w = S.w * e + k * v.w;
  c.x += S.x * q;
  c.y += S.y * q;
  c.z += S.z * q;
  c.w += S.w * q;
}
__device__ __forceinline__ float4 ld_bf4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(bf_lo(u.x), bf_hi(u.x), bf_lo(u.y), bf_hi(u.y));
}

__global__ void __launch_bounds__(256) recurrent_kernel(const Args a) {
  pdl_begin();
  __shared__ float sk[D], sq[D];
  __shared__ float4 part[8][32];
  const int row = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stop = a.real ? min(max(a.real[row], 0), a.n) : a.n;
  const float* in = state_in(a.pool, row, h);
  float4 S[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    S[i] = in ? reinterpret_cast<const float4*>(in + (warp * 16 + i) * D)[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
  const float scale = rsqrtf((float)D);
  for (int t = 0; t < stop; ++t) {
    if (threadIdx.x < D) sk[threadIdx.x] = bf2f(a.k[row * a.k_row + t * a.k_tok + h * D + threadIdx.x]);
    else sq[threadIdx.x - D] = bf2f(a.q[row * a.q_row + t * a.q_tok + h * D + threadIdx.x - D]);
    const float4 v = ld_bf4(a.v + row * a.v_row + t * a.v_tok + h * D + 4 * lane);
    const float e = expf(a.g[row * a.g_row + t * a.g_tok + h]);
    __syncthreads();
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) advance(S[i], e, sk[warp * 16 + i], v, sq[warp * 16 + i], c);
    part[warp][lane] = c;
    __syncthreads();
    if (threadIdx.x < D) {
      float o = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) o += reinterpret_cast<const float*>(part[w])[threadIdx.x];
      a.o[row * a.o_row + t * a.o_tok + h * D + threadIdx.x] = f2bf(o * scale);
    }
    __syncthreads();
  }
  for (int t = stop + warp; t < a.n; t += 8)
    reinterpret_cast<uint2*>(a.o + row * a.o_row + t * a.o_tok + h * D)[lane] = make_uint2(0, 0);
  float* out = state_out(a.pool, row, h);
  if (out)
#pragma unroll
    for (int i = 0; i < 16; ++i) reinterpret_cast<float4*>(out + (warp * 16 + i) * D)[lane] = S[i];
}

// ------------------------------------------------------------------ one token
//
// Reads and writes each state once (128 KB a head): bound by HBM, and for one row by its chain of reads. The columns of a
// state are independent, so a CTA takes 32 of them: 64 CTAs for one row's 16 heads, and no CTA with more than 16 KB to
// wait for. 8 lanes cover a key row's 32 columns, a warp instruction four rows; a thread's eight rows stay in registers.
// Measured on a B200 with the delta rule: 64 rows 21.3 us (135 MB: 97% of the copy rate; 24.6 with a CTA a state), one
// row 3.9 us (5.4).

template <bool DELTA>
__global__ void __launch_bounds__(128) step_kernel(const Args a) {
  pdl_begin();
  __shared__ float4 part[2][4][8];
  const int pair = blockIdx.x >> 2, row = pair / a.heads, h = pair % a.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, col = (blockIdx.x & 3) * 32 + (lane & 7) * 4;
  const float* in = state_in(a.pool, row, h);
  float4 S[8];   // key rows 32 warp + 4 i + sub
#pragma unroll
  for (int i = 0; i < 8; ++i)
    S[i] = in ? *reinterpret_cast<const float4*>(in + (32 * warp + 4 * i + sub) * D + col) : make_float4(0.f, 0.f, 0.f, 0.f);
  float kk[8], qq[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    kk[i] = bf2f(a.k[row * a.k_row + h * D + 32 * warp + 4 * i + sub]);
    qq[i] = bf2f(a.q[row * a.q_row + h * D + 32 * warp + 4 * i + sub]);
  }
  float4 v = ld_bf4(a.v + row * a.v_row + h * D + col);
  const float e = expf(a.g[row * a.g_row + h]);
  // the sum over all key rows: the lanes of a column, then the four warps
  auto total = [&](float4 c, int buf) {
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {
      c.x += __shfl_xor_sync(0xffffffffu, c.x, o);
      c.y += __shfl_xor_sync(0xffffffffu, c.y, o);
      c.z += __shfl_xor_sync(0xffffffffu, c.z, o);
      c.w += __shfl_xor_sync(0xffffffffu, c.w, o);
    }
    if (sub == 0) part[buf][warp][lane & 7] = c;
    __syncthreads();
    c = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float4 x = part[buf][w][lane & 7];
      c.x += x.x;
      c.y += x.y;
      c.z += x.z;
      c.w += x.w;
    }
    return c;
  };
  if (DELTA) {
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c.x += S[i].x * kk[i];
      c.y += S[i].y * kk[i];
      c.z += S[i].z * kk[i];
      c.w += S[i].w * kk[i];
    }
    c = total(c, 0);
    const float b = bf2f(a.beta[(int64_t)row * a.heads + h]);
    v.x = b * (v.x - e * c.x);
    v.y = b * (v.y - e * c.y);
    v.z = b * (v.z - e * c.z);
    v.w = b * (v.w - e * c.w);
  }
  float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
  float* out = state_out(a.pool, row, h);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    advance(S[i], e, kk[i], v, qq[i], c);
    if (out) *reinterpret_cast<float4*>(out + (32 * warp + 4 * i + sub) * D + col) = S[i];
  }
  c = total(c, 1);
  const float scale = rsqrtf((float)D);
  if (threadIdx.x < 8)
    *reinterpret_cast<uint2*>(a.o + row * a.o_row + h * D + col) =
        make_uint2(pack_bf2(c.x * scale, c.y * scale), pack_bf2(c.z * scale, c.w * scale));
}

inline bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

int check(const char* who, const Args& a, int b) {
  const Pool& p = a.pool;
  JB_REQUIRE(a.q && a.k && a.v && a.g && a.o && p.base && p.tables, "%s: null pointer", who);
  JB_REQUIRE(b > 0 && a.n > 0 && a.heads > 0, "%s: %d rows, %d tokens, %d heads", who, b, a.n, a.heads);
  JB_REQUIRE((int64_t)b * a.heads <= 0x7fffffff, "%s: %d rows of %d heads", who, b, a.heads);
  JB_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.o) && aligned16(p.base) &&
                 p.page_bytes % 16 == 0,
             "%s: q, k, v, o and the pages must be 16-byte aligned", who);
  JB_REQUIRE(((a.q_row | a.k_row | a.v_row | a.o_row | a.q_tok | a.k_tok | a.v_tok | a.o_tok) & 7) == 0,
             "%s: the strides of q, k, v and o must be multiples of 8", who);
  JB_REQUIRE(p.heads_per_page > 0 && p.heads_per_page * STATE_BYTES <= p.page_bytes,
             "%s: %d heads per page do not fit pages of %lld bytes", who, p.heads_per_page, (long long)p.page_bytes);
  const int last = p.first_head + a.heads - 1;
  JB_REQUIRE(p.first_head >= 0 && last / p.heads_per_page < p.table_stride &&
                 (!p.out_tables || last / p.heads_per_page < p.out_stride),
             "%s: heads %d.. reach past the block table", who, p.first_head);
  return JB_OK;
}

}  // namespace lin
}  // namespace jb
