// Attention over a paged cache in 8 bits (the scheme and the kernels' frame: paged_attn.cuh; the codes: paged_q8.cuh).
//
// A key's scale multiplies its score, a value's scale its weight:
//   o = sum_j p_j vs_j vc_j / sum_j p_j,   p_j = exp(scale ks_j q.kc_j - m)
// with kc, vc the codes, so the codes themselves are what is multiplied.
#include "paged_attn.cuh"
#include "paged_q8.cuh"

namespace engpt {
namespace paged {

struct Q8AttnArgs : AttnArgs {
  const float* k_scales;
  const float* v_scales;
  int64_t kss[3], vss[3];   // element strides: page, head, block
  int block;
};

// For the CUDA-core kernel.
template <typename Type, typename C>
struct Q8Kv {
  using T = Type;
  using Code = uint8_t;
  using Args = Q8AttnArgs;
  static constexpr bool kScaled = true;
  template <int VEC>
  static __device__ __forceinline__ void load(const Code* p, float* x) {
    if constexpr (VEC == 8) {
      // (coherent: see load_vec)
      uint32_t w[2];
      asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = C::decode((uint8_t)(w[i >> 2] >> (8 * (i & 3))));
    } else {
      x[0] = C::decode(*p);
    }
  }
  static __device__ __forceinline__ float key_scale(const Args& a, int page, int h, int off) {
    return a.k_scales[page * a.kss[0] + h * a.kss[1] + off / a.block * a.kss[2]];
  }
  static __device__ __forceinline__ float value_scale(const Args& a, int page, int h, int off) {
    return a.v_scales[page * a.vss[0] + h * a.vss[1] + off / a.block * a.vss[2]];
  }
};

template <typename T, typename C>
int dispatch_simt_q8(const Q8AttnArgs& a, bool vec, cudaStream_t st) {
  using Kv = Q8Kv<T, C>;
  if (vec) {
    const int nc = (a.Dh + 63) / 64;
    if (nc <= 1) return launch_simt_heads<Kv, 8, 1, 4>(a, st);
    if (nc <= 2) return launch_simt_heads<Kv, 8, 2, 2>(a, st);
    return launch_simt<Kv, 8, 4, 1, 1>(a, st);
  }
  if (a.Dh <= 64) return launch_simt<Kv, 1, 8, 2, 1>(a, st);
  return launch_simt<Kv, 1, 32, 1, 1>(a, st);
}

}  // namespace paged
}  // namespace engpt

using namespace engpt;
using namespace engpt::paged;

extern "C" int64_t engpt_paged_attention_q8_floats(int dtype, int B, int H, int Hkv, int Dh, int table_width,
                                                   int page_size, int block) {
  (void)dtype;
  if (B <= 0 || H <= 0 || Hkv <= 0 || Dh <= 0 || table_width < 0 || page_size <= 0 || block <= 0) return 0;
  const int splits = simt_splits(B, H, (int64_t)table_width * page_size);
  return splits > kSimtCluster ? (int64_t)B * H * splits * (Dh + 2) : 0;
}

extern "C" int engpt_paged_attention_q8(const void* q, const int64_t* q_strides, const void* k_pages,
                                        const void* v_pages, const float* k_scales, const float* v_scales,
                                        const int64_t* page_strides, const int64_t* scale_strides, int dtype, int code,
                                        int B, int H, int Hkv, int Dh, int num_pages, int page_size, int block,
                                        const int* block_table, int64_t table_stride, int table_width,
                                        const int* lengths, float scale, void* o, float* workspace, void* stream) {
  clear_error();
  ENGPT_REQUIRE(B >= 0 && H > 0 && Hkv > 0 && Dh > 0 && H % Hkv == 0, ENGPT_ERR_SHAPE,
                "paged_attention_q8: B=%d H=%d Hkv=%d Dh=%d", B, H, Hkv, Dh);
  ENGPT_REQUIRE(Dh <= 256, ENGPT_ERR_UNSUPPORTED, "paged_attention_q8: head_dim %d > 256", Dh);
  ENGPT_REQUIRE(B <= 65535 && H <= 65535, ENGPT_ERR_SHAPE, "paged_attention_q8: B=%d H=%d (at most 65535)", B, H);
  ENGPT_REQUIRE(num_pages >= 0 && page_size > 0 && (int64_t)num_pages * page_size <= 0x7fffffffLL, ENGPT_ERR_SHAPE,
                "paged_attention_q8: num_pages=%d page_size=%d", num_pages, page_size);
  ENGPT_REQUIRE(block > 0 && page_size % block == 0, ENGPT_ERR_SHAPE,
                "paged_attention_q8: blocks of %d tokens in pages of %d", block, page_size);
  ENGPT_REQUIRE(table_width >= 0 && table_stride >= table_width && (int64_t)table_width * page_size <= kMostKeys,
                ENGPT_ERR_SHAPE, "paged_attention_q8: table_width=%d page_size=%d", table_width, page_size);
  ENGPT_REQUIRE(dtype == ENGPT_BF16 || dtype == ENGPT_F32, ENGPT_ERR_DTYPE, "paged_attention_q8: dtype %d", dtype);
  ENGPT_REQUIRE(code == ENGPT_CODE_INT8 || code == ENGPT_CODE_E4M3, ENGPT_ERR_DTYPE, "paged_attention_q8: code type %d",
                code);
  if (B == 0) return ENGPT_OK;
  ENGPT_REQUIRE(q && q_strides && page_strides && scale_strides && lengths && o, ENGPT_ERR_ARG,
                "paged_attention_q8: null pointer");
  ENGPT_REQUIRE((k_pages && v_pages && k_scales && v_scales) || num_pages == 0, ENGPT_ERR_ARG,
                "paged_attention_q8: null cache");
  ENGPT_REQUIRE(block_table || table_width == 0, ENGPT_ERR_ARG, "paged_attention_q8: null block table");
  const int esz = dtype == ENGPT_BF16 ? 2 : 4;
  Q8AttnArgs a;
  a.q = q;
  a.q_row = q_strides[0];
  a.q_head = q_strides[1];
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.block = block;
  a.B = B;
  a.H = H;
  a.G = H / Hkv;
  a.Dh = Dh;
  a.P = num_pages;
  a.ps = page_size;
  a.table = block_table;
  a.table_stride = table_stride;
  a.W = table_width;
  a.lengths = lengths;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.o = o;
  a.work = workspace;
  a.splits = simt_splits(B, H, (int64_t)table_width * page_size);
  ENGPT_REQUIRE(workspace || engpt_paged_attention_q8_floats(dtype, B, H, Hkv, Dh, table_width, page_size, block) == 0,
                ENGPT_ERR_ARG, "paged_attention_q8: null workspace");
  ENGPT_REQUIRE(aligned(workspace, 16), ENGPT_ERR_ALIGN, "paged_attention_q8: workspace not 16-byte aligned");
  ENGPT_REQUIRE(aligned(k_scales, 4) && aligned(v_scales, 4), ENGPT_ERR_ALIGN, "paged_attention_q8: scales not aligned");
  bool vec = aligned(q, 16) && a.q_row * esz % 16 == 0 && a.q_head * esz % 16 == 0 && aligned(k_pages, 8) &&
             aligned(v_pages, 8) && Dh % 8 == 0;
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = page_strides[i];
    a.vs[i] = page_strides[3 + i];
    a.kss[i] = scale_strides[i];
    a.vss[i] = scale_strides[3 + i];
    // the stride of an axis of one element is never used, and may be anything
    if ((i == 0 ? num_pages : i == 1 ? Hkv : page_size) == 1) a.ks[i] = a.vs[i] = Dh;
    if ((i == 0 ? num_pages : i == 1 ? Hkv : page_size / block) == 1) a.kss[i] = a.vss[i] = 1;
    vec = vec && a.ks[i] % 8 == 0 && a.vs[i] % 8 == 0;
  }
  cudaStream_t st = as_stream(stream);
  if (dtype == ENGPT_BF16)
    return code == ENGPT_CODE_INT8 ? dispatch_simt_q8<__nv_bfloat16, Int8Code>(a, vec, st)
                                   : dispatch_simt_q8<__nv_bfloat16, E4m3Code>(a, vec, st);
  return code == ENGPT_CODE_INT8 ? dispatch_simt_q8<float, Int8Code>(a, vec, st)
                                 : dispatch_simt_q8<float, E4m3Code>(a, vec, st);
}
