// The C entries of linear.cu and linear_tc.cu.

namespace jb {
namespace lin {

// The chunked form, or token by token: that one for a few tokens, whose chunk would be mostly padding (4 tokens of 1 / 16
// / 64 rows: 5.4 / 8.4 / 38 us token by token, 8.1 / 11 / 52 as a chunk; 16 tokens: 12 / 18 / 90 against the same), and
// for strides that a tensor map does not take (one token or row standing for all).
constexpr int FEW = 7;
inline bool chunked(const Args& a, int b) {
  const bool rows = b == 1 || (a.q_row > 0 && a.k_row > 0 && a.v_row > 0);
  return a.n > FEW && rows && a.q_tok > 0 && a.k_tok > 0 && a.v_tok > 0;
}

}  // namespace lin
}  // namespace jb

extern "C" int jb_linear_scan(const uint16_t* q, int64_t q_row, int64_t q_tok, const uint16_t* k, int64_t k_row,
                              int64_t k_tok, const uint16_t* v, int64_t v_row, int64_t v_tok, const float* g,
                              int64_t g_row, int64_t g_tok, const int32_t* real, uint16_t* o, int b, int n, int heads,
                              void* state, int64_t pages, int64_t page_bytes, int heads_per_page, int first_head,
                              const int32_t* tables, int table_stride, const int32_t* out_tables, int out_stride,
                              float* scratch, int64_t scratch_floats, void* stream) {
  using namespace jb;
  if (n == 1) q_tok = k_tok = v_tok = (int64_t)heads * lin::D;   // a single token's strides say nothing, nor a single row's
  if (b == 1) q_row = k_row = v_row = (int64_t)n * heads * lin::D;
  const lin::Args a = {reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<const __nv_bfloat16*>(k),
                       reinterpret_cast<const __nv_bfloat16*>(v), q_row, k_row, v_row, q_tok, k_tok, v_tok, g, g_row,
                       g_tok, nullptr, real, reinterpret_cast<__nv_bfloat16*>(o), (int64_t)n * heads * lin::D,
                       (int64_t)heads * lin::D, n, heads,
                       {static_cast<uint8_t*>(state), pages, page_bytes, heads_per_page, first_head, tables,
                        table_stride, out_tables, out_stride}};
  if (int st = lin::check("jb_linear_scan", a, b)) return st;
  if (lin::chunked(a, b)) {
    const int64_t need = lintc::scratch_floats(b, heads, n);
    JB_REQUIRE(scratch_floats >= need && (scratch || need == 0) && lin::aligned16(scratch),
               "jb_linear_scan: a scratch of %lld floats (16-byte aligned), %lld are needed", (long long)scratch_floats,
               (long long)need);
    return lintc::scan(a, b, scratch, (cudaStream_t)stream);
  }
  launch_pdl(lin::recurrent_kernel, b * heads, 256, 0, (cudaStream_t)stream, a);
  return check_launch("linear recurrent_kernel");
}

extern "C" int jb_linear_scan_scratch(int b, int heads, int n) {
  using namespace jb;
  return b > 0 && heads > 0 && n > 0 ? (int)lintc::scratch_floats(b, heads, n) : 0;
}

extern "C" int jb_linear_step(const uint16_t* q, int64_t q_row, const uint16_t* k, int64_t k_row, const uint16_t* v,
                              int64_t v_row, const float* g, int64_t g_row, const uint16_t* beta, uint16_t* o, int b,
                              int heads, void* state, int64_t pages, int64_t page_bytes, int heads_per_page,
                              int first_head, const int32_t* tables, int table_stride, const int32_t* out_tables,
                              int out_stride, void* stream) {
  using namespace jb;
  if (b == 1) q_row = k_row = v_row = (int64_t)heads * lin::D;
  const lin::Args a = {reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<const __nv_bfloat16*>(k),
                       reinterpret_cast<const __nv_bfloat16*>(v), q_row, k_row, v_row, 0, 0, 0, g, g_row, 0,
                       reinterpret_cast<const __nv_bfloat16*>(beta), nullptr, reinterpret_cast<__nv_bfloat16*>(o),
                       (int64_t)heads * lin::D, 0, 1, heads,
                       {static_cast<uint8_t*>(state), pages, page_bytes, heads_per_page, first_head, tables,
                        table_stride, out_tables, out_stride}};
  if (int st = lin::check("jb_linear_step", a, b)) return st;
  JB_REQUIRE(out_tables, "jb_linear_step: null pointer (out_tables: where the new states go)");
  JB_REQUIRE((int64_t)b * heads <= 0x1fffffff, "jb_linear_step: %d rows of %d heads", b, heads);
  launch_pdl(beta ? lin::step_kernel<true> : lin::step_kernel<false>, 4 * b * heads, 128, 0, (cudaStream_t)stream, a);
  return check_launch("linear step_kernel");
}
