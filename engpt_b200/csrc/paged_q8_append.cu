// qkv_append_from_carried_q8: the QKV post-process with k and v quantised into the paged cache.
#include "paged_q8_store.cuh"

using namespace engpt;
using namespace engpt::paged;

extern "C" int engpt_qkv_append_q8(const void* qkv, int dtype, const float* rho, const float* cos_tab,
                                   const float* sin_tab, int rope_rows, int rope_half, const float* qk_scale,
                                   float qk_mult, float norm_eps, int64_t n, int H, int Dh, const int* positions,
                                   const int* slots, void* q_out, void* k_pages, void* v_pages, float* k_scales,
                                   float* v_scales, const int64_t* page_strides, const int64_t* scale_strides,
                                   int code, int num_pages, int page_size, int block, void* stream) {
  clear_error();
  ENGPT_REQUIRE(n >= 0 && n <= 0x7fffffffLL, ENGPT_ERR_SHAPE, "qkv_append_q8: n=%lld", (long long)n);
  ENGPT_REQUIRE(rope_half >= 0 && 2 * (int64_t)rope_half <= Dh && rope_rows >= 0, ENGPT_ERR_SHAPE,
                "qkv_append_q8: rope_half=%d rope_rows=%d Dh=%d", rope_half, rope_rows, Dh);
  ENGPT_REQUIRE(dtype == ENGPT_BF16 || dtype == ENGPT_F32, ENGPT_ERR_DTYPE, "qkv_append_q8: dtype %d", dtype);
  StoreArgs a = {};
  if (int rc = fill_q8_cache("qkv_append_q8", a.c, k_pages, v_pages, k_scales, v_scales, page_strides, scale_strides,
                             code, H, Dh, num_pages, page_size, block))
    return rc;
  if (n == 0) return ENGPT_OK;
  ENGPT_REQUIRE(qkv && rho && qk_scale && q_out && positions && slots, ENGPT_ERR_ARG, "qkv_append_q8: null pointer");
  ENGPT_REQUIRE(rope_half == 0 || (cos_tab && sin_tab), ENGPT_ERR_ARG, "qkv_append_q8: null rope table");
  a.slots = slots;
  a.n = n;
  a.qkv = qkv;
  for (int i = 0; i < 2; ++i) {                        // (k and v as rows of the projection)
    a.x[i] = static_cast<const char*>(qkv) + (size_t)(i + 1) * H * Dh * (dtype == ENGPT_BF16 ? 2 : 4);
    a.row[i] = (int64_t)3 * H * Dh;
    a.head[i] = Dh;
  }
  a.rho = rho;
  a.cos_tab = cos_tab;
  a.sin_tab = sin_tab;
  a.rope_rows = rope_rows;
  a.rope_half = rope_half;
  a.qk_scale = qk_scale;
  a.qk_mult = qk_mult;
  a.eps = norm_eps;
  a.positions = positions;
  a.q = q_out;
  const bool vec = aligned(qkv, 16) && aligned(q_out, 16) && aligned(qk_scale, 16) &&
                   (rope_half == 0 || (rope_half == Dh / 2 && aligned(cos_tab, 16) && aligned(sin_tab, 16)));
  return dtype == ENGPT_BF16 ? launch_store<__nv_bfloat16, true>(a, code, vec, "qkv_append_q8", as_stream(stream))
                             : launch_append_f32(a, code, vec, as_stream(stream));
}
