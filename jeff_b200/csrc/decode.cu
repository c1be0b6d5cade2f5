// Single tokens over the prefix pool: block tables and slot maps from request lengths, the attention input side with
// several rotary axes writing straight into the cache, and the attention of one new token per row over its pages.

#include <atomic>

namespace jb {
namespace dec {

constexpr int PAGE = 32;   // tokens of a key/value page
// The pool's page 0 takes what belongs nowhere, and a table names it where no page was to be had: as an entry of a table
// it is no page, so that nothing that other rows left there is attended to and no two tokens get one slot.
constexpr int SINK = 0;

// ------------------------------------------------------------------ block tables and slot maps
//
// Row r holds len_r tokens and adds new_r. With pages(x) = min(ceil(x / P), table entries past kv_entry) it takes
// pages(len_r + new_r) - pages(len_r) pages (and kv_entry more for its fixed entries when it is fresh) off the free
// list, in row order: row r's first is free[T_r], T the exclusive sum of what the rows take. Token i of row r is packed
// at s_r + i (s the exclusive sum of new), and its slot is page * P + (len_r + i) % P.
//
// Bound by latency: two dependent reads (the lengths, then the tables and the free list). So one launch, in which
// every CTA repeats the two sums over all rows (8 bytes a row out of L2) instead of waiting for another's, and then
// writes its own share: a slice of the tokens and every gridDim-th group of rows. An entry that is read (held before
// the call) is never one that is written, so the CTAs need no order. Measured on a B200: 64 rows with one more token each
// 4.8 us, 256 fresh prompts of 16,384 tokens with their 50 fixed pages 6.0 us.

constexpr int TAB_THREADS = 256, TAB_ROWS = 1024, TAB_PER = TAB_ROWS / TAB_THREADS;

struct TabParams {
  const int* lengths;
  const int* added;
  int b;
  const int* free_pages;
  int free_count;
  int* tables;
  int table_stride, width, kv_entry, page, fixed, tokens;
  int64_t* slots;
  int* rows;
  int* positions;
  int* starts;
  int* taken;
};

struct TabRow {
  int len, add, held, take, head;   // pages held and taken, and how many of those fill the fixed entries
};

__device__ __forceinline__ TabRow tab_row(const TabParams& p, int r) {
  TabRow t;
  t.len = max(p.lengths[r], 0);
  t.add = min(max(p.added[r], 0), 0x7fffffff - t.len);
  const int most = p.width - p.kv_entry;
  const unsigned page = p.page;   // the sums stay below 2^32
  const int need = (int)min(((unsigned)t.len + t.add + (page - 1)) / page, (unsigned)most);
  t.held = (int)min(((unsigned)t.len + (page - 1)) / page, (unsigned)most);
  t.head = p.fixed && t.len == 0 && t.add > 0 ? p.kv_entry : 0;
  t.take = need - t.held + t.head;
  return t;
}

__global__ void __launch_bounds__(TAB_THREADS) tables_kernel(const TabParams p) {
  pdl_begin();
  __shared__ long long s_add[TAB_ROWS], s_take[TAB_ROWS];
  __shared__ long long w_add[TAB_THREADS / 32], w_take[TAB_THREADS / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (p.tokens + gridDim.x - 1) / gridDim.x;
  const int t0 = min((int)min((long long)blockIdx.x * per, (long long)p.tokens), p.tokens);
  const int t1 = min(t0 + per, p.tokens);
  long long base_add = 0, base_take = 0;
  for (int r0 = 0; r0 < p.b; r0 += TAB_ROWS) {
    const int count = min(TAB_ROWS, p.b - r0);
    TabRow mine[TAB_PER];
    long long a = 0, k = 0;
    const int rows_each = (count + TAB_THREADS - 1) / TAB_THREADS;
#pragma unroll
    for (int i = 0; i < TAB_PER; ++i) {
      const int j = tid * rows_each + i;
      mine[i].add = mine[i].take = 0;
      if (i < rows_each && j < count) mine[i] = tab_row(p, r0 + j);
      a += mine[i].add;
      k += mine[i].take;
    }
    long long ia = a, ik = k;   // inclusive sums over the warp, then over the block
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long ya = __shfl_up_sync(0xffffffffu, ia, off), yk = __shfl_up_sync(0xffffffffu, ik, off);
      if (lane >= off) {
        ia += ya;
        ik += yk;
      }
    }
    __syncthreads();   // the previous rows' sums have been read
    if (lane == 31) {
      w_add[warp] = ia;
      w_take[warp] = ik;
    }
    __syncthreads();
    long long ea = base_add + ia - a, ek = base_take + ik - k;
    long long ta = base_add, tk = base_take;
#pragma unroll
    for (int w = 0; w < TAB_THREADS / 32; ++w) {
      if (w < warp) {
        ea += w_add[w];
        ek += w_take[w];
      }
      ta += w_add[w];
      tk += w_take[w];
    }
#pragma unroll
    for (int i = 0; i < TAB_PER; ++i) {
      if (i < rows_each) {
        s_add[tid * rows_each + i] = ea;
        s_take[tid * rows_each + i] = ek;
      }
      ea += mine[i].add;
      ek += mine[i].take;
    }
    __syncthreads();
    // this CTA's tokens that belong to these rows: the row by bisection of the sums
    // (the sums may pass 32 bits, and are cut to the share ahead of that)
    const int lo = (int)min(max((long long)t0, base_add), (long long)t1), hi = (int)min((long long)t1, ta);
    for (int t = lo + tid; t < hi; t += TAB_THREADS) {
      int l = 0, h = count - 1;   // the last row whose tokens start at or before t; rows that add none share a start
      while (l < h) {
        const int m = (l + h + 1) >> 1;
        if (s_add[m] <= t) l = m;
        else h = m - 1;
      }
      const TabRow row = tab_row(p, r0 + l);
      const int pos = row.len + (int)(t - s_add[l]);
      const int j = pos / p.page;
      int page = -1;
      if (j < row.held) {
        page = p.tables[(int64_t)(r0 + l) * p.table_stride + p.kv_entry + j];
      } else if (j < p.width - p.kv_entry) {
        const long long at = s_take[l] + row.head + j - row.held;
        if (at < p.free_count) page = p.free_pages[at];
      }
      p.slots[t] = page <= SINK ? -1 : (int64_t)page * p.page + pos % p.page;
      p.rows[t] = r0 + l;
      p.positions[t] = pos;
    }
    // this CTA's rows: their sums and their new entries, a warp per row
    for (int j = blockIdx.x * (TAB_THREADS / 32) + warp; j < count; j += gridDim.x * (TAB_THREADS / 32)) {
      const TabRow row = tab_row(p, r0 + j);
      const long long at = s_take[j];
      if (lane == 0) {
        p.starts[r0 + j] = (int)min(s_add[j], 0x7fffffffLL);
        p.taken[r0 + j] = (int)min(at, 0x7fffffffLL);
      }
      int* dst = p.tables + (int64_t)(r0 + j) * p.table_stride;
      for (int i = lane; i < row.take; i += 32)
        dst[i < row.head ? i : p.kv_entry + row.held + i - row.head] = at + i < p.free_count ? p.free_pages[at + i] : SINK;
    }
    base_add = ta;
    base_take = tk;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.starts[p.b] = (int)min(base_add, 0x7fffffffLL);
    p.taken[p.b] = (int)min(base_take, 0x7fffffffLL);
  }
  for (int t = (int)max((long long)t0, min(base_add, (long long)t1)) + tid; t < t1; t += TAB_THREADS) {   // past the last row
    p.slots[t] = -1;
    p.rows[t] = -1;
    p.positions[t] = 0;
  }
}

// ------------------------------------------------------------------ attention input side, several rotary axes
//
// Per token and head: y = x rsqrt(mean(x^2) + eps) w1, then the pair (d, d + 32), d < 32, turned by the angle
// pos[axis(d)] f_d. Everything stays in fp32 and is rounded to bf16 once, at the end. The angle is formed in fp64 and
// reduced to a part of one turn before the fp32 sine and cosine. There a position of up to 29 bits times a 24-bit frequency
// is exact and past that rounded, as the factor 1 / 2 pi and its product are: in all at most 3 * 2^-53 of the angle, 7e-7 rad
// at a position of 2^31 and a frequency of 1 (the fp32 sine and cosine themselves: some 1e-7).

constexpr int NQ = 8, NKV = 2, HD = 256, ROT = 64;
// From this many tokens on a warp takes a whole token; below, a block does, a warp a head. Measured back to back, in us,
// with a warp / a block per token: 64 tokens 2.5 / 2.0, 256 2.6 / 2.7, 1,024 4.8 / 6.3, 4,096 10.2 / 18.7, 16,384
// 38.3 / 73.9 (201 MB: 80% of the copy rate / 42%).
constexpr int PREP_MANY = 256;

struct PrepParams {
  const __nv_bfloat16* pr;
  int64_t ldpr;
  int t;
  const float* q_w1;
  const float* k_w1;
  const float* inv_freq;
  const int* positions;   // (axes, t)
  int64_t axis_stride;
  unsigned long long axes;   // 2 bits a frequency
  __nv_bfloat16* q;
  __nv_bfloat16* kn;
  __nv_bfloat16* vn;
  uint8_t* kv;            // the layer's keys in page 0, or null
  int64_t pages, page_bytes;
  const int64_t* slots;
};

__device__ __forceinline__ void turn_of(const PrepParams& p, int t, int i, float& c, float& s) {
  const int axis = (int)(p.axes >> (2 * i)) & 3;
  const double turns = (double)p.positions[axis * p.axis_stride + t] * (double)p.inv_freq[i] * 0.15915494309189535;
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
}

__global__ void __launch_bounds__(384) prep_axes_kernel(const PrepParams p) {
  pdl_begin();
  const int t = blockIdx.x, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float rc[ROT / 2], rs[ROT / 2];
  if (w == 0) turn_of(p, t, lane, rc[lane], rs[lane]);
  __syncthreads();
  const __nv_bfloat16* src = p.pr + (int64_t)t * p.ldpr;
  const int base = w < NQ ? w * 2 * HD : NQ * 2 * HD + (w - NQ) * HD;   // query heads, then key heads, then value heads
  uint4 out = reinterpret_cast<const uint4*>(src + base)[lane];
  if (w < NQ + NKV) {
    const float* W = w < NQ ? p.q_w1 : p.k_w1;
    float x[8];
    ew::unpack8(out, x);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
    const float r = rsqrtf(ew::warp_sum(ss) / HD + ew::EPS);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= r * W[lane * 8 + e];
    float other[8];   // lanes 0-3 hold dims 0..31, lanes 4-7 their partners 32..63
#pragma unroll
    for (int e = 0; e < 8; ++e) other[e] = __shfl_xor_sync(0xffffffffu, x[e], 4);
    if (lane < ROT / 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = (lane & 3) * 8 + e;
        x[e] = lane < 4 ? x[e] * rc[d] - other[e] * rs[d] : x[e] * rc[d] + other[e] * rs[d];
      }
    }
    out = ew::pack8(x);
  }
  if (w < NQ) {
    reinterpret_cast<uint4*>(p.q + ((int64_t)t * NQ + w) * HD)[lane] = out;
    return;
  }
  const int head = (w - NQ) % NKV, half = (w - NQ) / NKV;   // half 0: keys, 1: values
  __nv_bfloat16* flat = half ? p.vn : p.kn;
  if (flat) reinterpret_cast<uint4*>(flat + ((int64_t)t * NKV + head) * HD)[lane] = out;
  if (p.kv) {
    const int64_t slot = p.slots[t], page = slot / PAGE;
    if (slot >= 0 && page < p.pages)
      reinterpret_cast<uint4*>(p.kv + page * p.page_bytes +
                               (((int64_t)half * PAGE + slot % PAGE) * NKV + head) * HD * 2)[lane] = out;
  }
}

// The same with a warp per token, all twelve heads of a lane's dimensions loaded at once (6 KB in flight a warp), the
// weights in registers over a warp's tokens, and no barrier. The eight query heads' sums are reduced together: each
// step of the first three halves the number of values a lane carries (9 exchanges and 8 to hand them back, not 40).
// Bound by HBM, whose reads skip the gates between the queries, every other 512 bytes: the next token's rows, positions
// and slot fetched ahead into shared memory change nothing at 16,384 tokens and cost 13% at 1,024 to 4,096.
__device__ __forceinline__ void load8(const float* w, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(w)[0], b = reinterpret_cast<const float4*>(w)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

__global__ void __launch_bounds__(128, 3) prep_tokens_kernel(const PrepParams p) {
  pdl_begin();
  constexpr int N = NQ + 2 * NKV;
  const int lane = threadIdx.x & 31;
  float wq[8], wk[8], wqo[8], wko[8];   // this lane's weights, and of the dimensions its first eight are turned with
  load8(p.q_w1 + lane * 8, wq);
  load8(p.k_w1 + lane * 8, wk);
  load8(p.q_w1 + (lane ^ 4) * 8, wqo);
  load8(p.k_w1 + (lane ^ 4) * 8, wko);
  for (int t = blockIdx.x * 4 + (threadIdx.x >> 5); t < p.t; t += gridDim.x * 4) {
    const __nv_bfloat16* src = p.pr + (int64_t)t * p.ldpr;
    uint4 x[N];
#pragma unroll
    for (int h = 0; h < N; ++h)
      x[h] = reinterpret_cast<const uint4*>(src + (h < NQ ? h * 2 * HD : NQ * 2 * HD + (h - NQ) * HD))[lane];
    float mc, ms, c[8], s[8];
    turn_of(p, t, lane, mc, ms);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = __shfl_sync(0xffffffffu, mc, (lane & 3) * 8 + e);
      s[e] = __shfl_sync(0xffffffffu, ms, (lane & 3) * 8 + e);
      if (!(lane & 4)) s[e] = -s[e];   // dimensions 0-31 subtract
    }
    float ss[NQ + NKV];
#pragma unroll
    for (int h = 0; h < NQ + NKV; ++h) {
      float f[8];
      ew::unpack8(x[h], f);
      ss[h] = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss[h] += f[e] * f[e];
    }
    float v[4];   // lanes with bit 16, 8, 4 set keep the odd heads of what is left at each step
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float keep = lane & 16 ? ss[2 * i + 1] : ss[2 * i], give = lane & 16 ? ss[2 * i] : ss[2 * i + 1];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, 16);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float keep = lane & 8 ? v[2 * i + 1] : v[2 * i], give = lane & 8 ? v[2 * i] : v[2 * i + 1];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, 8);
    }
    {
      const float keep = lane & 4 ? v[1] : v[0], give = lane & 4 ? v[0] : v[1];
      v[0] = keep + __shfl_xor_sync(0xffffffffu, give, 4);
    }
    v[0] += __shfl_xor_sync(0xffffffffu, v[0], 2);
    v[0] += __shfl_xor_sync(0xffffffffu, v[0], 1);
    const float mine = rsqrtf(v[0] / HD + ew::EPS);   // of head 4 (lane bit 4) + 2 (bit 8) + (bit 16)
#pragma unroll
    for (int h = 0; h < NQ; ++h)
      ss[h] = __shfl_sync(0xffffffffu, mine, (h & 1) * 16 + (h >> 1 & 1) * 8 + (h >> 2) * 4);
#pragma unroll
    for (int h = NQ; h < NQ + NKV; ++h) ss[h] = rsqrtf(ew::warp_sum(ss[h]) / HD + ew::EPS);
#pragma unroll
    for (int h = 0; h < NQ + NKV; ++h) {
      const uint4 o = make_uint4(__shfl_xor_sync(0xffffffffu, x[h].x, 4), __shfl_xor_sync(0xffffffffu, x[h].y, 4),
                                 __shfl_xor_sync(0xffffffffu, x[h].z, 4), __shfl_xor_sync(0xffffffffu, x[h].w, 4));
      float f[8], g[8];
      ew::unpack8(x[h], f);
      ew::unpack8(o, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] *= ss[h] * (h < NQ ? wq[e] : wk[e]);
        g[e] *= ss[h] * (h < NQ ? wqo[e] : wko[e]);
        if (lane < ROT / 8) f[e] = f[e] * c[e] + g[e] * s[e];
      }
      x[h] = ew::pack8(f);
    }
#pragma unroll
    for (int h = 0; h < NQ; ++h) reinterpret_cast<uint4*>(p.q + ((int64_t)t * NQ + h) * HD)[lane] = x[h];
    const int64_t slot = p.kv ? p.slots[t] : -1, page = slot / PAGE;
#pragma unroll
    for (int i = 0; i < 2 * NKV; ++i) {
      const int head = i % NKV, half = i / NKV;   // half 0: keys, 1: values
      __nv_bfloat16* flat = half ? p.vn : p.kn;
      if (flat) reinterpret_cast<uint4*>(flat + ((int64_t)t * NKV + head) * HD)[lane] = x[NQ + i];
      if (slot >= 0 && page < p.pages)
        reinterpret_cast<uint4*>(p.kv + page * p.page_bytes +
                                 (((int64_t)half * PAGE + slot % PAGE) * NKV + head) * HD * 2)[lane] = x[NQ + i];
    }
  }
}

// ------------------------------------------------------------------ attention of one new token per row
//
// o = sum_j softmax_j(scale q . k_j) v_j over the row's cached tokens j < lengths[r], in one pass over the pages with
// a running maximum and sum. Every key and value is read once, for all query heads of its head: 4 operations a byte
// with 4 of them, so the bound is HBM.
//
// Shares: a (row, key/value head) is cut into steps of WARPS x TILE tokens, all steps of the call into as many equal
// shares as there are CTAs (one per SM), in row order: a share's work does not depend on how the lengths are spread. A
// CTA finishes what it holds in full; of a row cut by a share's border each part leaves its unnormalised sum, maximum
// and weight in scratch, and the CTA that leaves the last of them adds the row's parts, in share order whoever it is
// (one launch instead of a second one of 5 to 7 us for the sums).
//
// In a CTA each warp takes one tile (16 or 32 tokens) of a step, with a ring of its own in shared memory (cp.async of a
// tile's keys, then its values, tokens past the row's end as zeros) and no barrier with the other warps until a row
// ends, when the warps' sums are joined in shared memory. Scores and output are taken transposed, S^T = K Q^T and
// O^T = V^T P^T on mma.sync m16n8k16: the 16 rows of the tile are keys (then 16 of the head's dimensions), the 8 columns
// the query heads, so 4 query heads cost half of what a 16-row query tile would. (tcgen05 has no use here: its 128-row
// tile would be filled with 4 rows.)
// Measured on a B200, launch included: 64 ragged rows of 1 to 8,192 tokens (8 / 2 heads of 256, 537 MB) 105 us, 78% of
// the copy rate; 33 rows of 100 to 4,096 (32 / 8 heads of 128, 283 MB) 59 us, 73%; one row of 1,000 9.8 us, latency.
// What bounds it is how its pages lie: a ring of copies alone, without lookups, arithmetic and ends of rows, takes 95 us
// for 537 MB in pages of six layers of which it reads one (5.7 TB/s), 83 us where the pages hold that layer alone, and 48
// us for 277 MB of 8 heads of 128 with one layer a page or two (5.8 TB/s: a head's keys are 256 bytes, 2 KB apart). The
// rest is the start (lengths, then tables, then keys), the ends of rows (1 us each; 3.3 with a thread a value) and SMs
// that stream slower than others. Not kept: steps of all heads of fewer tokens, so that a page is read as one contiguous
// piece (2% slower), two CTAs of four warps an SM (7%), shares in three waves (13%) or claimed by the CTAs that are done
// with theirs (21%): every share ends a row, and in waves its start waits for lengths and tables again.
//
// The weights are held as two bf16 parts, p = hi + lo to 2^-17: with at most 4 query heads the lo parts ride in
// columns 4-7, which would be empty, against the queries repeated there; with more they take a second product.

template <int D>
struct Dec {
  static constexpr int WARPS = 8;
  static constexpr int TILE = D == 256 ? 16 : 32; // tokens of a warp's tile
  static constexpr int HALVES = D == 64 ? 5 : 3;  // a warp's ring, in tiles' keys or values
  static constexpr int STEP = WARPS * TILE;       // tokens
  // bytes of a key in shared memory, its 16-byte chunk c at c ^ (key % 8): ldmatrix without conflicts, and rows on
  // 128-byte lines (with keys padded by 16 bytes instead, copies alone take 102 us for 537 MB in pages of six layers, not
  // 95, and 51 for 277 MB of 128-wide heads, not 48)
  static constexpr int PITCH = D * 2;
  static constexpr int SLOT = TILE * PITCH;       // a tile's keys or its values; eight heads' outputs at a row's end
  static constexpr int SMEM = WARPS * HALVES * SLOT;
  static_assert(8 * D * 4 <= SLOT, "eight heads' outputs fit a slot");
  static_assert(SMEM + 16384 <= 227 * 1024, "shared memory");
};

constexpr int SHARES = 148;   // one CTA per SM
__host__ __device__ constexpr int dec_part(int group, int dim) { return (group * (dim + 2) + 3) & ~3; }   // floats
inline int64_t dec_scratch(int group, int dim) { return 4 * SHARES + (int64_t)2 * SHARES * dec_part(group, dim); }
// a call's tag: 64 bits that memory does not hold by chance
inline unsigned long long dec_tag() {
  static std::atomic<unsigned long long> calls{0};
  unsigned long long x = (calls.fetch_add(1, std::memory_order_relaxed) + 1) * 0x9e3779b97f4a7c15ull;
  x ^= x >> 29;
  x *= 0xd1342543de82ef95ull;
  return x | 1;
}
constexpr int HELD = 1024;    // rows whose lengths a CTA holds

struct DecParams {
  const __nv_bfloat16* q;
  int64_t ldq;
  const uint8_t* kv;   // the layer's keys in page 0
  int64_t pages, page_bytes;
  const int* tables;
  int table_stride, kv_entry, most;   // tokens the table holds
  const int* lengths;
  int b, kv_heads, group;
  float scale_log2;
  const __nv_bfloat16* pr;
  int64_t ldpr;
  __nv_bfloat16* y;
  int64_t ldy;
  // what cut rows leave: two flags a share, then two parts a share. A part is there when its flag holds the call's tag:
  // the memory may hold anything before a call, and who joins a row's parts clears their flags, so that a replay of the
  // call (the same tag) starts without them too
  volatile unsigned long long* flags;
  unsigned long long tag;
  float* parts;
};

__device__ __forceinline__ int dec_length(const DecParams& p, int r) { return min(max(p.lengths[r], 0), p.most); }

// Units (steps of one key/value head) of all rows; warp-collective.
template <int STEP, class Len>
__device__ long long dec_units(const DecParams& p, const Len& len) {
  const int lane = threadIdx.x & 31;
  long long all = 0;
  for (int r0 = 0; r0 < p.b; r0 += 128) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 32 * i + lane;
      all += r < p.b ? (len(r) + STEP - 1) / STEP : 0;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  return all * p.kv_heads;
}

struct Cursor {   // a unit: a step of a row's head, and the row's tokens
  int row, head, step, steps, len;
};

// The unit `u` (below the total); warp-collective.
template <int STEP, class Len>
__device__ Cursor dec_find(const DecParams& p, const Len& len, long long u) {
  const int lane = threadIdx.x & 31;
  long long before = 0;
  for (int r0 = 0; r0 < p.b; r0 += 32) {
    const int n = r0 + lane < p.b ? len(r0 + lane) : 0, steps = (n + STEP - 1) / STEP;
    long long upto = (long long)steps * p.kv_heads;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    upto += before;
    const unsigned over = __ballot_sync(0xffffffffu, upto > u);
    if (over) {
      const int l = __ffs(over) - 1;
      const int ln = __shfl_sync(0xffffffffu, n, l), ls = __shfl_sync(0xffffffffu, steps, l);
      const int in = (int)(u - (__shfl_sync(0xffffffffu, upto, l) - (long long)ls * p.kv_heads));
      return {r0 + l, in / ls, in % ls, ls, ln};
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return {p.b, 0, 0, 1, 0};
}

template <int STEP, class Len>
__device__ __forceinline__ void dec_next(const DecParams& p, const Len& len, Cursor& c) {
  if (++c.step < c.steps) return;
  c.step = 0;
  if (++c.head < p.kv_heads) return;
  c.head = 0;
  do {
    ++c.row;
    c.len = c.row < p.b ? len(c.row) : 1;
    c.steps = (c.len + STEP - 1) / STEP;
  } while (c.steps == 0);
}

// the base of the exponentials while every score so far is -inf (their weights are then 0, not NaN)
__device__ __forceinline__ float finite(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The parts of a cut row's key/value head, joined in share order: share c0's part, whose slot is its first if it began
// with the row, and the following shares' first slots. A part: the group's values, then their maxima, then their sums.
// First the parts' factors, a warp a head; then the values, four of them a lane.
constexpr int WEIGHTS = 16 * (SHARES + 1);

template <int D>
__device__ void dec_join(const DecParams& p, int row, int kv_head, int c0, int count, bool first, float* s_w) {
  constexpr int EACH = (SHARES + 31) / 32, AHEAD = 8;   // parts in flight
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t stride = dec_part(p.group, D);
  auto part = [&](int i) { return p.parts + (2 * (c0 + i) + (i == 0 && !first ? 1 : 0)) * stride; };
  for (int h = warp; h < p.group; h += 8) {
    float m[EACH], l[EACH], mx = -INFINITY, sum = 0.f;   // lane i: parts i, i + 32, ...
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int i = lane + 32 * j;
      m[j] = i < count ? __ldcg(part(i) + p.group * D + h) : -INFINITY;
      l[j] = i < count ? __ldcg(part(i) + p.group * (D + 1) + h) : 0.f;
      mx = fmaxf(mx, m[j]);
    }
    mx = ew::warp_max(mx);
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      // a part without keys counts nothing; one whose scores were all NaN has that as its sum, and no maximum
      const float w = l[j] != l[j] ? l[j] : m[j] == -INFINITY ? 0.f : exp2f(m[j] - finite(mx));
      if (w != 0.f) sum += w * l[j];
      if (lane + 32 * j < SHARES) s_w[h * (SHARES + 1) + lane + 32 * j] = w;
    }
    sum = ew::warp_sum(sum);
    if (lane == 0) s_w[h * (SHARES + 1) + SHARES] = mx == -INFINITY && sum == 0.f ? INFINITY : sum;
  }
  __syncthreads();
  for (int i4 = threadIdx.x; i4 < p.group * D / 4; i4 += 256) {
    const int h = i4 * 4 / D, d = i4 * 4 % D, head = kv_head * p.group + h;
    const float* w = s_w + h * (SHARES + 1);
    uint2 gate = make_uint2(0, 0);
    if (p.pr) gate = *reinterpret_cast<const uint2*>(p.pr + row * p.ldpr + ((int64_t)2 * head + 1) * D + d);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < count; i0 += AHEAD) {
      float4 x[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        x[i] = __ldcg(reinterpret_cast<const float4*>(part(min(i0 + i, count - 1))) + i4);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (i0 + i >= count) continue;
        const float f = w[i0 + i];
        v[0] += f * x[i].x;
        v[1] += f * x[i].y;
        v[2] += f * x[i].z;
        v[3] += f * x[i].w;
      }
    }
    const float sum = w[SHARES];
    const float g[4] = {bf_lo(gate.x), bf_hi(gate.x), bf_lo(gate.y), bf_hi(gate.y)};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] /= sum;
      if (p.pr) v[e] *= ew::sigmoid(g[e]);
    }
    *reinterpret_cast<uint2*>(p.y + row * p.ldy + (int64_t)head * D + d) =
        make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
  }
}

// NT: 8-column tiles of query heads; PAIR: at most 4 query heads, the weights' lo parts in columns 4-7
template <int D, int NT, bool PAIR>
__global__ void __launch_bounds__(Dec<D>::WARPS * 32, 1) decode_kernel(const DecParams p) {
  pdl_begin();
  using L = Dec<D>;
  constexpr int KS = D / 16, CH = D / 8;   // 16-wide k steps, 16-byte chunks of a key
  constexpr int TILE = L::TILE, MT = TILE / 16, CHAINS = 4 / MT;
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ float s_m[L::WARPS][16], s_l[L::WARPS][16], s_f[16][L::WARPS], s_all[16][2];
  __shared__ float s_w[WEIGHTS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, tq = lane & 3;
  // the rows' lengths are asked for again and again: from shared memory where they fit there
  __shared__ int s_len[HELD];
  if (p.b <= HELD) {
    for (int r = threadIdx.x; r < p.b; r += L::WARPS * 32) s_len[r] = dec_length(p, r);
    __syncthreads();
  }
  auto length = [&](int r) { return p.b <= HELD ? s_len[r] : dec_length(p, r); };
  const long long total = dec_units<L::STEP>(p, length);
  for (int r = blockIdx.x; r < p.b; r += gridDim.x)   // rows without tokens
    if (length(r) == 0)
      for (int i = threadIdx.x; i < p.kv_heads * p.group * D; i += L::WARPS * 32) p.y[r * p.ldy + i] = f2bf(0.f);
  const long long shares = min((long long)SHARES, total);   // none of them empty
  if (blockIdx.x >= shares) return;
  const long long u0 = total * blockIdx.x / shares, u1 = total * (blockIdx.x + 1) / shares;
  uint8_t* ring = sm + warp * L::HALVES * L::SLOT;
  Cursor c = dec_find<L::STEP>(p, length, u0), f = c;
  const int half_bytes = PAGE * p.kv_heads * D * 2;   // a page's keys of one layer, then its values

  auto page_of = [&](const Cursor& x) -> int {   // the page of this warp's tile of a unit, -1: none
    const int j = x.step * L::STEP + warp * TILE;
    if (j >= x.len) return -1;
    const int page = p.tables[(int64_t)x.row * p.table_stride + p.kv_entry + j / PAGE];
    return page > SINK && page < p.pages ? page : -1;
  };
  // the fetches' cursor, half a tile at a time: the unit, its page (loaded one unit ahead, so that its load never stands
  // in a fetch's way), keys or values, and the slot; `valid` has a bit for each tile fetched and not yet used
  long long uf = u0;
  int page = page_of(f), value = 0, fslot = 0, ahead = 0;
  uint32_t valid = 0;
  auto fetch = [&]() {
    if (uf < u1) {
      if (page >= 0) {
        const int j0 = f.step * L::STEP + warp * TILE;
        const int live = min(TILE, f.len - j0);
        const uint8_t* src = p.kv + (int64_t)page * p.page_bytes + (int64_t)value * half_bytes +
                             ((j0 % PAGE) * p.kv_heads + f.head) * D * 2;
        const uint32_t dst = smem_u32(ring + fslot * L::SLOT);
        const int row_bytes = p.kv_heads * D * 2;
        if (live == TILE) {
#pragma unroll
          for (int i = 0; i < TILE * CH / 32; ++i) {   // TILE keys x CH chunks: consecutive lanes along a key
            const int idx = i * 32 + lane, r = idx / CH, ch = idx % CH;
            attn::cp_async16(dst + r * L::PITCH + ((ch ^ (r & 7)) << 4), src + r * row_bytes + ch * 16, true);
          }
        } else {
#pragma unroll
          for (int i = 0; i < TILE * CH / 32; ++i) {   // zeros past the row's end
            const int idx = i * 32 + lane, r = idx / CH, ch = idx % CH;
            attn::cp_async16(dst + r * L::PITCH + ((ch ^ (r & 7)) << 4),
                             r < live ? src + r * row_bytes + ch * 16 : p.kv, r < live);
          }
        }
      }
      if (value == 0) valid |= (page >= 0 ? 1u : 0u) << ahead++;
      else if (++uf < u1) {
        dec_next<L::STEP>(p, length, f);
        page = page_of(f);
      }
      value ^= 1;
      fslot = fslot + 1 == L::HALVES ? 0 : fslot + 1;
    }
    attn::cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < L::HALVES; ++s) fetch();

  uint32_t qf[NT][KS][2];
  float o[NT][KS][4], m[NT][2], l[NT][2];
  auto begin = [&]() {   // a row's head: its queries as B fragments, empty sums
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = PAIR ? (gr & 3) : nt * 8 + gr;
      const bool live = h < p.group;
      const __nv_bfloat16* src = p.q + c.row * p.ldq + ((int64_t)c.head * p.group + (live ? h : 0)) * D + 2 * tq;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        qf[nt][kk][0] = live ? *reinterpret_cast<const uint32_t*>(src + kk * 16) : 0u;
        qf[nt][kk][1] = live ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8) : 0u;
        o[nt][kk][0] = o[nt][kk][1] = o[nt][kk][2] = o[nt][kk][3] = 0.f;
      }
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
  };
  begin();
  int slot = 0;
  bool from_start = true;   // the current row's head began at the share's first unit
  int first_step = c.step;
  for (long long u = u0; u < u1; ++u) {
    const bool mine = valid & 1, ends = c.step + 1 == c.steps || u + 1 == u1;
    valid >>= 1;
    --ahead;
    uint8_t* keys = ring + slot * L::SLOT;
    const int vslot = slot + 1 == L::HALVES ? 0 : slot + 1;
    uint8_t* values = ring + vslot * L::SLOT;
    uint32_t hi[NT][MT][2], lo[NT][MT][2];
    attn::cp_async_wait<L::HALVES - 1>();
    __syncwarp();
    if (mine) {
      const int j0 = c.step * L::STEP + warp * TILE;
      const int live = c.len - j0;
      // S^T: TILE keys x 8 heads, four chains of products
      float s[NT][MT][CHAINS][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < MT * CHAINS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][i / CHAINS][i % CHAINS][e] = 0.f;
      const uint32_t ka = smem_u32(keys) + ((lane & 7) + (lane & 8)) * L::PITCH;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t a0, a1, a2, a3;
          attn::ldsm_x4(ka + mt * 16 * L::PITCH + (((kk * 2 + (lane >> 4)) ^ (lane & 7)) << 4), a0, a1, a2, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            attn::mma16816(s[nt][mt][kk % CHAINS], a0, a1, a2, a3, qf[nt][kk][0], qf[nt][kk][1]);
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[MT][4];
        float n0 = -INFINITY, n1 = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float sum = s[nt][mt][0][e];
#pragma unroll
            for (int i = 1; i < CHAINS; ++i) sum += s[nt][mt][i][e];
            x[mt][e] = mt * 16 + gr + (e >> 1) * 8 < live ? sum * p.scale_log2 : -INFINITY;
          }
          n0 = fmaxf(n0, fmaxf(x[mt][0], x[mt][2]));
          n1 = fmaxf(n1, fmaxf(x[mt][1], x[mt][3]));
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, off));
          n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, off));
        }
        if (__any_sync(0xffffffffu, n0 > m[nt][0] || n1 > m[nt][1])) {
          n0 = fmaxf(n0, m[nt][0]);
          n1 = fmaxf(n1, m[nt][1]);
          const float a0 = exp2f(m[nt][0] - finite(n0)), a1 = exp2f(m[nt][1] - finite(n1));
          m[nt][0] = n0;
          m[nt][1] = n1;
          l[nt][0] *= a0;
          l[nt][1] *= a1;
#pragma unroll
          for (int kk = 0; kk < KS; ++kk) {
            o[nt][kk][0] *= a0;
            o[nt][kk][1] *= a1;
            o[nt][kk][2] *= a0;
            o[nt][kk][3] *= a1;
          }
        }
        const float b0 = finite(m[nt][0]), b1 = finite(m[nt][1]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            const float p0 = exp2f(x[mt][2 * e2] - b0), p1 = exp2f(x[mt][2 * e2 + 1] - b1);
            l[nt][0] += p0;
            l[nt][1] += p1;
            const uint32_t h = pack_bf2(p0, p1);
            const uint32_t r = pack_bf2(p0 - bf_lo(h), p1 - bf_hi(h));
            if (PAIR) hi[nt][mt][e2] = transpose8x8(tq < 2 ? h : r);
            else {
              hi[nt][mt][e2] = transpose8x8(h);
              lo[nt][mt][e2] = transpose8x8(r);
            }
          }
        }
      }
    }
    // the keys' slot is free; at a row's end it is kept for the outputs
    __syncwarp();
    if (!ends) {
      fetch();
      attn::cp_async_wait<L::HALVES - 1>();
    } else {
      attn::cp_async_wait<L::HALVES - 2>();
    }
    __syncwarp();
    if (mine) {
      // O^T += V^T P^T, 16 dimensions at a time
      const uint32_t va = smem_u32(values) + ((lane & 7) + ((lane >> 4) << 3)) * L::PITCH;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t a0, a1, a2, a3;
          attn::ldsm_x4_trans(va + mt * 16 * L::PITCH + (((kk * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4), a0, a1, a2, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            attn::mma16816(o[nt][kk], a0, a1, a2, a3, hi[nt][mt][0], hi[nt][mt][1]);
            if (!PAIR) attn::mma16816(o[nt][kk], a0, a1, a2, a3, lo[nt][mt][0], lo[nt][mt][1]);
          }
        }
    }
    __syncwarp();
    if (ends) {
      // the warps' sums into the slots just read, eight heads each, then joined: thread = one dimension of a head
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
        }
        const int h = nt * 8 + 2 * tq;
        float* mo = reinterpret_cast<float*>(nt == 0 ? values : keys);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = o[nt][kk][e];
            if (PAIR) v += __shfl_xor_sync(0xffffffffu, v, 2);   // the lo parts' product
            if (!PAIR || tq < 2) mo[(2 * tq + (e & 1)) * D + ((kk * 16 + gr + (e >> 1) * 8) ^ (tq * 8))] = v;
          }
        }
        if (gr == 0) {
          s_m[warp][h] = m[nt][0];
          s_m[warp][h + 1] = m[nt][1];
          s_l[warp][h] = l[nt][0];
          s_l[warp][h + 1] = l[nt][1];
        }
      }
      __syncthreads();
      const bool whole = first_step == 0 && c.step + 1 == c.steps;
      float* part = p.parts + (2 * (int64_t)blockIdx.x + (from_start ? 0 : 1)) * dec_part(p.group, D);
      // each head's factors, maximum and sum over the warps: eight lanes a head
      if (threadIdx.x < 8 * NT * L::WARPS) {
        const int w = threadIdx.x % L::WARPS, h = threadIdx.x / L::WARPS;
        const float mw = s_m[w][h];
        float mx = mw;
#pragma unroll
        for (int off = 1; off < L::WARPS; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float f = mw == -INFINITY ? 0.f : exp2f(mw - mx);   // 0: a warp without keys of this row
        float sum = f * s_l[w][h];
#pragma unroll
        for (int off = 1; off < L::WARPS; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        s_f[h][w] = f;
        if (w == 0) {
          s_all[h][0] = mx;
          s_all[h][1] = sum;
        }
      }
      __syncthreads();
      for (int i4 = threadIdx.x; i4 < p.group * D / 4; i4 += L::WARPS * 32) {
        const int h = i4 * 4 / D, d = i4 * 4 % D, head = c.head * p.group + h;
        uint2 gate = make_uint2(0, 0);
        if (whole && p.pr) gate = *reinterpret_cast<const uint2*>(p.pr + c.row * p.ldpr + ((int64_t)2 * head + 1) * D + d);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < L::WARPS; ++w) {
          const float f = s_f[h][w];
          const float4 x = *reinterpret_cast<const float4*>(
              sm + (w * L::HALVES + (h < 8 ? vslot : slot)) * L::SLOT +
              ((h & 7) * D + (d ^ ((h >> 1 & 3) * 8))) * 4);
          v[0] += f * x.x;
          v[1] += f * x.y;
          v[2] += f * x.z;
          v[3] += f * x.w;
        }
        const float mx = s_all[h][0], sum = s_all[h][1];
        if (whole) {
          const float g[4] = {bf_lo(gate.x), bf_hi(gate.x), bf_lo(gate.y), bf_hi(gate.y)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = sum == 0.f ? 0.f : v[e] / sum;   // no keys: zeros
            if (p.pr) v[e] *= ew::sigmoid(g[e]);
          }
          *reinterpret_cast<uint2*>(p.y + c.row * p.ldy + (int64_t)head * D + d) =
              make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
        } else {
          reinterpret_cast<float4*>(part)[i4] = make_float4(v[0], v[1], v[2], v[3]);
          if (d == 0) {
            part[p.group * D + h] = mx;
            part[p.group * (D + 1) + h] = sum;
          }
        }
      }
      __syncthreads();   // the slots are free again, the part is written
    }
    if (ends) fetch();
    fetch();
    if (ends && !(first_step == 0 && c.step + 1 == c.steps)) {
      // a part of a row whose units are a .. z and whose shares c0 .. c1 (unit u's: the last c with total * c / shares <=
      // u): its flag, then the others' flags: of the CTAs whose fences come in this order, the last sees all of them (a
      // second one may, and then joins the same parts to the same values)
      const long long a = u - c.step, z = a + c.steps - 1;
      const int c0 = (int)(((a + 1) * shares - 1) / total), c1 = (int)(((z + 1) * shares - 1) / total);
      const int count = c1 - c0 + 1;
      const bool first = total * c0 / shares == a;
      auto slot_of = [&](int i) { return 2 * (c0 + i) + (i == 0 && !first ? 1 : 0); };
      if (threadIdx.x == 0) {
        __threadfence();
        p.flags[slot_of(blockIdx.x - c0)] = p.tag;
        __threadfence();
      }
      __syncthreads();
      bool there = true;
      for (int i = threadIdx.x; i < count; i += L::WARPS * 32) there &= p.flags[slot_of(i)] == p.tag;
      if (__syncthreads_and(there)) {
        __threadfence();
        dec_join<D>(p, c.row, c.head, c0, count, first, s_w);
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += L::WARPS * 32) p.flags[slot_of(i)] = 0;
      }
    }
    slot = vslot + 1 == L::HALVES ? 0 : vslot + 1;
    if (u + 1 < u1) {
      dec_next<L::STEP>(p, length, c);
      if (ends) {
        begin();
        from_start = false;
        first_step = 0;
      }
    }
  }
}

template <int D, int NT, bool PAIR>
int dec_launch(const DecParams& p, cudaStream_t stream) {
  if (int r = gdnc::configure(decode_kernel<D, NT, PAIR>, Dec<D>::SMEM, "decode_kernel: cudaFuncSetAttribute")) return r;
  launch_pdl(decode_kernel<D, NT, PAIR>, SHARES, Dec<D>::WARPS * 32, Dec<D>::SMEM, stream, p);
  return check_launch("decode_kernel");
}

template <int D>
int dec_launch(const DecParams& p, cudaStream_t stream) {
  if (p.group <= 4) return dec_launch<D, 1, true>(p, stream);
  if (p.group <= 8) return dec_launch<D, 1, false>(p, stream);
  return dec_launch<D, 2, false>(p, stream);
}

inline bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }

}  // namespace dec
}  // namespace jb

extern "C" int jb_block_tables(const int32_t* lengths, const int32_t* added, int b, const int32_t* free_pages,
                               int free_count, int32_t* tables, int table_stride, int width, int kv_entry,
                               int page_tokens, int fixed, int tokens, int64_t* slots, int32_t* rows,
                               int32_t* positions, int32_t* starts, int32_t* taken, void* stream) {
  using namespace jb;
  JB_REQUIRE(lengths && added && tables && slots && rows && positions && starts && taken,
             "jb_block_tables: null pointer");
  // (the kernel's indices step past the last row and token by a round of rows, a block's threads, a CTA's share)
  JB_REQUIRE(b > 0 && b <= 0x7f000000 && tokens > 0 && tokens <= 0x7f000000, "jb_block_tables: %d rows, %d tokens", b, tokens);
  JB_REQUIRE(free_count >= 0 && (free_pages || free_count == 0), "jb_block_tables: a free list of %d pages", free_count);
  JB_REQUIRE(kv_entry >= 0 && kv_entry < width && width <= table_stride && page_tokens > 0,
             "jb_block_tables: key/value entry %d of tables %d wide (stride %d), pages of %d tokens", kv_entry, width,
             table_stride, page_tokens);
  const dec::TabParams p = {lengths, added, b, free_pages, free_count, tables, table_stride, width, kv_entry,
                            page_tokens, fixed, tokens, slots, rows, positions, starts, taken};
  const int grid = min(max((tokens + 255) / 256, (b + 7) / 8), 148);
  launch_pdl(dec::tables_kernel, grid, dec::TAB_THREADS, 0, (cudaStream_t)stream, p);
  return check_launch("tables_kernel");
}

extern "C" int jb_attn_prep_axes(const uint16_t* pr, int64_t ldpr, int t, const float* q_w1, const float* k_w1,
                                 const float* inv_freq, const int32_t* positions, int64_t axis_stride, int64_t axes,
                                 uint16_t* q, uint16_t* kn, uint16_t* vn, void* kv, int64_t pages, int64_t page_bytes,
                                 int attn_layer, int attn_layers, const int64_t* slots, void* stream) {
  using namespace jb;
  JB_REQUIRE(pr && q_w1 && k_w1 && inv_freq && positions && q, "jb_attn_prep_axes: null pointer");
  if (t == 1) ldpr = dec::NQ * 2 * dec::HD + 2 * dec::NKV * dec::HD;   // a single row's stride says nothing
  JB_REQUIRE(t > 0 && ldpr >= dec::NQ * 2 * dec::HD + 2 * dec::NKV * dec::HD && ldpr % 8 == 0 && axis_stride >= 0,
             "jb_attn_prep_axes: t %d, ldpr %lld, axis stride %lld", t, (long long)ldpr, (long long)axis_stride);
  JB_REQUIRE((kn != nullptr) == (vn != nullptr) && (kv != nullptr) == (slots != nullptr) && (kn || kv),
             "jb_attn_prep_axes: keys and values go to kn and vn, to the pages that slots name, or to both");
  const int64_t layer_bytes = (int64_t)2 * dec::PAGE * dec::NKV * dec::HD * 2;
  JB_REQUIRE(!kv || (pages > 0 && attn_layer >= 0 && attn_layer < attn_layers && attn_layers * layer_bytes <= page_bytes &&
                     page_bytes % 16 == 0),
             "jb_attn_prep_axes: attention layer %d of %d does not fit pages of %lld bytes", attn_layer, attn_layers,
             (long long)page_bytes);
  JB_REQUIRE(dec::aligned16(pr) && dec::aligned16(q) && dec::aligned16(kn) && dec::aligned16(vn) && dec::aligned16(kv) &&
                 dec::aligned16(q_w1) && dec::aligned16(k_w1),
             "jb_attn_prep_axes: pr, q, kn, vn, the norms' weights and the pages must be 16-byte aligned");
  const dec::PrepParams p = {reinterpret_cast<const __nv_bfloat16*>(pr), ldpr, t, q_w1, k_w1, inv_freq, positions,
                             axis_stride, (unsigned long long)axes, reinterpret_cast<__nv_bfloat16*>(q),
                             reinterpret_cast<__nv_bfloat16*>(kn), reinterpret_cast<__nv_bfloat16*>(vn),
                             kv ? static_cast<uint8_t*>(kv) + attn_layer * layer_bytes : nullptr, pages, page_bytes,
                             slots};
  if (t >= dec::PREP_MANY) {
    launch_pdl(dec::prep_tokens_kernel, min((t + 3) / 4, 3 * dec::SHARES), 128, 0, (cudaStream_t)stream, p);
    return check_launch("prep_tokens_kernel");
  }
  launch_pdl(dec::prep_axes_kernel, t, 384, 0, (cudaStream_t)stream, p);
  return check_launch("prep_axes_kernel");
}

extern "C" int jb_decode_attention(const uint16_t* q, int64_t ldq, const void* kv, int64_t pages, int64_t page_bytes,
                                   int attn_layer, int attn_layers, const int32_t* tables, int table_stride,
                                   int width, int kv_entry, const int32_t* lengths, int b, int heads, int kv_heads,
                                   int dim, float scale, const uint16_t* pr, int64_t ldpr, uint16_t* y, int64_t ldy,
                                   float* scratch, int64_t scratch_floats, void* stream) {
  using namespace jb;
  JB_REQUIRE(q && kv && tables && lengths && y, "jb_decode_attention: null pointer");
  JB_REQUIRE(dim == 64 || dim == 128 || dim == 256, "jb_decode_attention: heads of %d (64, 128 or 256)", dim);
  JB_REQUIRE(b > 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 16,
             "jb_decode_attention: %d rows, %d query heads over %d key/value heads (a multiple, at most 16)", b, heads,
             kv_heads);
  const int64_t layer_bytes = (int64_t)2 * dec::PAGE * kv_heads * dim * 2;
  JB_REQUIRE(pages > 0 && attn_layer >= 0 && attn_layer < attn_layers && attn_layers * layer_bytes <= page_bytes &&
                 page_bytes % 16 == 0,
             "jb_decode_attention: attention layer %d of %d does not fit pages of %lld bytes", attn_layer, attn_layers,
             (long long)page_bytes);
  JB_REQUIRE(kv_entry >= 0 && kv_entry <= width && width <= table_stride,
             "jb_decode_attention: key/value entry %d of tables %d wide (stride %d)", kv_entry, width, table_stride);
  // the kernel counts a row's tokens, its steps of 128 over all heads, and a page's values in 32 bits
  const int64_t most = (int64_t)(width - kv_entry) * dec::PAGE;
  JB_REQUIRE(most <= 0x7f000000 && (most + 127) / 128 * kv_heads <= 0x7fffffff,
             "jb_decode_attention: tables of %lld tokens, %d key/value heads", (long long)most, kv_heads);
  JB_REQUIRE((int64_t)heads * dim <= 1 << 24 && b <= 0x7f000000, "jb_decode_attention: %d rows of %d heads of %d", b,
             heads, dim);
  if (b == 1) {   // a single row's strides say nothing
    ldq = ldy = heads * dim;
    ldpr = 2 * heads * dim;
  }
  JB_REQUIRE(ldq >= heads * dim && ldq % 8 == 0 && ldy >= heads * dim && ldy % 8 == 0 &&
                 (!pr || (ldpr >= 2 * heads * dim && ldpr % 8 == 0)),
             "jb_decode_attention: row strides %lld, %lld, %lld", (long long)ldq, (long long)ldy, (long long)ldpr);
  JB_REQUIRE(dec::aligned16(q) && dec::aligned16(kv) && dec::aligned16(pr) && dec::aligned16(y),
             "jb_decode_attention: q, the pages, pr and y must be 16-byte aligned");
  const int group = heads / kv_heads;
  JB_REQUIRE((int64_t)b * heads <= 0x7fffffff, "jb_decode_attention: %d rows of %d heads", b, heads);
  JB_REQUIRE(scratch && scratch_floats >= dec::dec_scratch(group, dim) && dec::aligned16(scratch),
             "jb_decode_attention: a scratch of %lld floats (16-byte aligned), %lld are needed",
             (long long)scratch_floats, (long long)dec::dec_scratch(group, dim));
  const dec::DecParams p = {reinterpret_cast<const __nv_bfloat16*>(q), ldq,
                            static_cast<const uint8_t*>(kv) + attn_layer * layer_bytes, pages, page_bytes, tables,
                            table_stride, kv_entry, (int)most, lengths, b, kv_heads, group,
                            scale * 1.4426950408889634f, reinterpret_cast<const __nv_bfloat16*>(pr), ldpr,
                            reinterpret_cast<__nv_bfloat16*>(y), ldy,
                            reinterpret_cast<unsigned long long*>(scratch), dec::dec_tag(), scratch + 4 * dec::SHARES};
  const cudaStream_t st = (cudaStream_t)stream;
  return dim == 64 ? dec::dec_launch<64>(p, st) : dim == 128 ? dec::dec_launch<128>(p, st) : dec::dec_launch<256>(p, st);
}

extern "C" int jb_decode_attention_scratch(int heads, int kv_heads, int dim) {
  return kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 16 &&
                 (dim == 64 || dim == 128 || dim == 256)
             ? (int)jb::dec::dec_scratch(heads / kv_heads, dim)
             : 0;
}
