// Single tokens over the prefix pool: block tables and slot maps from request lengths, the attention input side with
// several rotary axes writing straight into the cache, and the attention of one new token per row over its pages.

namespace jb {
namespace dec {

constexpr int PAGE = 32;   // tokens of a key/value page

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
// the call) is never one that is written, so the CTAs need no order.

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
  const int need = (int)min(((long long)t.len + t.add + p.page - 1) / p.page, (long long)most);
  t.held = (int)min(((long long)t.len + p.page - 1) / p.page, (long long)most);
  t.head = p.fixed && t.len == 0 && t.add > 0 ? p.kv_entry : 0;
  t.take = need - t.held + t.head;
  return t;
}

__global__ void __launch_bounds__(TAB_THREADS) tables_kernel(const TabParams p) {
  pdl_begin();
  __shared__ long long s_add[TAB_ROWS + 1], s_take[TAB_ROWS + 1];
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
#pragma unroll
    for (int i = 0; i < TAB_PER; ++i) {
      const int j = tid * TAB_PER + i;
      mine[i].add = mine[i].take = 0;
      if (j < count) mine[i] = tab_row(p, r0 + j);
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
      s_add[tid * TAB_PER + i] = ea;
      s_take[tid * TAB_PER + i] = ek;
      ea += mine[i].add;
      ek += mine[i].take;
    }
    if (tid == TAB_THREADS - 1) {
      s_add[TAB_ROWS] = ta;
      s_take[TAB_ROWS] = tk;
    }
    __syncthreads();
    // this CTA's tokens that belong to these rows: the row by bisection of the sums
    const int lo = (int)max((long long)t0, base_add), hi = (int)min((long long)t1, ta);
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
      p.slots[t] = page < 0 ? -1 : (int64_t)page * p.page + pos % p.page;
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
        dst[i < row.head ? i : p.kv_entry + row.held + i - row.head] = at + i < p.free_count ? p.free_pages[at + i] : 0;
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
// pos[axis(d)] f_d. Everything stays in fp32 and is rounded to bf16 once, at the end. The angle is formed in fp64 (a
// position of 31 bits times a 24-bit frequency is exact there) and reduced to a part of one turn before the fp32 sine
// and cosine, so positions of any size keep full accuracy.

constexpr int NQ = 8, NKV = 2, HD = 256, ROT = 64;

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

// ------------------------------------------------------------------ attention of one new token per row
//
// o = sum_j softmax_j(scale q . k_j) v_j over the row's cached tokens j < lengths[r], one pass with the running
// maximum and sum. CTA per (row, query head), a warp per key, fp32 throughout.

template <int D>
__global__ void __launch_bounds__(256) decode_plain_kernel(
    const __nv_bfloat16* __restrict__ q, int64_t ldq, const uint8_t* __restrict__ kv, int64_t pages,
    int64_t page_bytes, const int* __restrict__ tables, int table_stride, int width, int kv_entry,
    const int* __restrict__ lengths, int nq, int nkv, float scale_log2, const __nv_bfloat16* __restrict__ pr,
    int64_t ldpr, __nv_bfloat16* __restrict__ y, int64_t ldy) {
  pdl_begin();
  constexpr int E = D / 32;
  __shared__ float sm[8], sl[8], so[8][D];
  const int r = blockIdx.x / nq, h = blockIdx.x % nq, g = h / (nq / nkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = (int)min((long long)max(lengths[r], 0), (long long)(width - kv_entry) * PAGE);
  float qv[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qv[e] = bf2f(q[r * ldq + (int64_t)h * D + lane + 32 * e]);
    o[e] = 0.f;
  }
  for (int j = warp; j < len; j += 8) {
    const int page = tables[(int64_t)r * table_stride + kv_entry + j / PAGE];
    if (page < 0 || page >= pages) continue;
    const __nv_bfloat16* k = reinterpret_cast<const __nv_bfloat16*>(kv + page * page_bytes) +
                             ((int64_t)(j % PAGE) * nkv + g) * D;
    const __nv_bfloat16* v = k + (int64_t)PAGE * nkv * D;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += qv[e] * bf2f(k[lane + 32 * e]);
    s = ew::warp_sum(s) * scale_log2;
    const float mn = fmaxf(m, s), a = m == -INFINITY ? 0.f : exp2f(m - mn), w = exp2f(s - mn);
    l = l * a + w;
    m = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * bf2f(v[lane + 32 * e]);
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane + 32 * e] = o[e];
  __syncthreads();
  if (threadIdx.x < D) {
    float mx = -INFINITY;
    for (int w = 0; w < 8; ++w) mx = fmaxf(mx, sm[w]);
    float sum = 0.f, out = 0.f;
    if (mx != -INFINITY)
      for (int w = 0; w < 8; ++w) {
        const float a = exp2f(sm[w] - mx);
        sum += a * sl[w];
        out += a * so[w][threadIdx.x];
      }
    out = sum > 0.f ? out / sum : 0.f;
    if (pr) out *= ew::sigmoid(bf2f(pr[r * ldpr + ((int64_t)2 * h + 1) * D + threadIdx.x]));
    y[r * ldy + (int64_t)h * D + threadIdx.x] = f2bf(out);
  }
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
  JB_REQUIRE(b > 0 && tokens > 0, "jb_block_tables: %d rows, %d tokens", b, tokens);
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
  JB_REQUIRE(t > 0 && ldpr >= dec::NQ * 2 * dec::HD + 2 * dec::NKV * dec::HD && ldpr % 8 == 0 && axis_stride >= 0,
             "jb_attn_prep_axes: t %d, ldpr %lld, axis stride %lld", t, (long long)ldpr, (long long)axis_stride);
  JB_REQUIRE((kn != nullptr) == (vn != nullptr) && (kv != nullptr) == (slots != nullptr) && (kn || kv),
             "jb_attn_prep_axes: keys and values go to kn and vn, to the pages that slots name, or to both");
  const int64_t layer_bytes = (int64_t)2 * dec::PAGE * dec::NKV * dec::HD * 2;
  JB_REQUIRE(!kv || (pages > 0 && attn_layer >= 0 && attn_layer < attn_layers && attn_layers * layer_bytes <= page_bytes &&
                     page_bytes % 16 == 0),
             "jb_attn_prep_axes: attention layer %d of %d does not fit pages of %lld bytes", attn_layer, attn_layers,
             (long long)page_bytes);
  JB_REQUIRE(dec::aligned16(pr) && dec::aligned16(q) && dec::aligned16(kn) && dec::aligned16(vn) && dec::aligned16(kv),
             "jb_attn_prep_axes: pr, q, kn, vn and the pages must be 16-byte aligned");
  const dec::PrepParams p = {reinterpret_cast<const __nv_bfloat16*>(pr), ldpr, t, q_w1, k_w1, inv_freq, positions,
                             axis_stride, (unsigned long long)axes, reinterpret_cast<__nv_bfloat16*>(q),
                             reinterpret_cast<__nv_bfloat16*>(kn), reinterpret_cast<__nv_bfloat16*>(vn),
                             kv ? static_cast<uint8_t*>(kv) + attn_layer * layer_bytes : nullptr, pages, page_bytes,
                             slots};
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
  JB_REQUIRE(ldq >= heads * dim && ldq % 8 == 0 && ldy >= heads * dim && ldy % 8 == 0 &&
                 (!pr || (ldpr >= 2 * heads * dim && ldpr % 8 == 0)),
             "jb_decode_attention: row strides %lld, %lld, %lld", (long long)ldq, (long long)ldy, (long long)ldpr);
  JB_REQUIRE(dec::aligned16(q) && dec::aligned16(kv) && dec::aligned16(pr) && dec::aligned16(y),
             "jb_decode_attention: q, the pages, pr and y must be 16-byte aligned");
  auto kernel = dim == 64 ? dec::decode_plain_kernel<64> : dim == 128 ? dec::decode_plain_kernel<128>
                                                                      : dec::decode_plain_kernel<256>;
  launch_pdl(kernel, b * heads, 256, 0, (cudaStream_t)stream, reinterpret_cast<const __nv_bfloat16*>(q), ldq,
             static_cast<const uint8_t*>(kv) + attn_layer * layer_bytes, pages, page_bytes, tables, table_stride,
             width, kv_entry, lengths, heads, kv_heads, scale * 1.4426950408889634f,
             reinterpret_cast<const __nv_bfloat16*>(pr), ldpr, reinterpret_cast<__nv_bfloat16*>(y), ldy);
  return check_launch("decode_plain_kernel");
}
