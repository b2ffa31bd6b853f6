// Attention over a paged cache in 8 bits: the CUDA-core kernel, the tensor-core kernel for 64 and 128 columns, and the
// entry point.
#include "paged_attn_q8.cuh"

namespace engpt {
namespace paged {

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

// (sizes and forms do not depend on the type of the codes, or of q)
template <int Pieces, bool Flat>
using AnyTile = Q8Tile<Pieces, Flat, Int8Code, __nv_bfloat16>;

// CTAs per pair of a tensor-core launch, 0 for the list form, or -1 if it cannot be one (strides and alignment apart).
inline int mma_form_q8(bool flat, int B, int H, int Hkv, int D, int table_width, int page_size, int block) {
  if (D > 128 || D % 16 != 0 || page_size % 8 != 0 || block % 8 != 0) return -1;
  auto form = [&](auto tile) {
    using F = decltype(tile);
    return list_fits(B, H, F::KT, table_width, page_size) ? pair_ctas<F>(B, H, Hkv, table_width, page_size) : -1;
  };
  if (flat) return flat_pieces(D, [&](auto n) { return form(AnyTile<n.value, true>()); });
  return mma_width(D) == 64 ? form(AnyTile<4, false>()) : form(AnyTile<8, false>());
}

template <typename T, typename C>
int dispatch_q8(const Q8AttnArgs& a, bool mma, bool flat, bool vec, int Hkv, cudaStream_t st) {
  if (!mma) return dispatch_simt_q8<T, C>(a, vec, st);
  if (flat && C::kInteger) return launch_flat_int8(a, Hkv, sizeof(T) == 4, st);
  if (flat) return launch_flat_e4m3(a, Hkv, sizeof(T) == 4, st);
  return mma_width(a.Dh) == 64 ? launch_mma_q8<Q8Tile<4, false, C, T>>(a, Hkv, st)
                               : launch_mma_q8<Q8Tile<8, false, C, T>>(a, Hkv, st);
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
  const int64_t simt = splits > kSimtCluster ? (int64_t)B * H * splits * (Dh + 2) : 0;
  if (H % Hkv != 0) return simt;
  // strides and alignment decide at the call which of the kernels runs
  int64_t mma = 0;
  for (const bool flat : {false, true})
    if (mma_form_q8(flat && Dh != 64 && Dh != 128, B, H, Hkv, Dh, table_width, page_size, block) == 0)
      mma = mma_floats(H, Hkv, Dh);
  return simt > mma ? simt : mma;
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
  // (the copies of TMA want multiples of 16 bytes; outputs are written in pieces of up to 16)
  // Rows that lie one behind the other are copied flat, but for 64 and 128 columns, which the swizzle serves better.
  const bool flat = Dh != 64 && Dh != 128 && a.ks[2] == Dh && a.vs[2] == Dh;
  bool mma = vec && aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(o, 16) && num_pages > 0 &&
             mma_form_q8(flat, B, H, Hkv, Dh, table_width, page_size, block) >= 0;
  for (int i = 0; i < 3; ++i) {
    mma = mma && a.ks[i] > 0 && a.vs[i] > 0 && a.ks[i] % 16 == 0 && a.vs[i] % 16 == 0;
    mma = mma && a.kss[i] == (int)a.kss[i] && a.vss[i] == (int)a.vss[i];   // (any scales of less than 2^31 numbers)
  }
  cudaStream_t st = as_stream(stream);
  if (dtype == ENGPT_BF16)
    return code == ENGPT_CODE_INT8 ? dispatch_q8<__nv_bfloat16, Int8Code>(a, mma, flat, vec, Hkv, st)
                                   : dispatch_q8<__nv_bfloat16, E4m3Code>(a, mma, flat, vec, Hkv, st);
  return code == ENGPT_CODE_INT8 ? dispatch_q8<float, Int8Code>(a, mma, flat, vec, Hkv, st)
                                 : dispatch_q8<float, E4m3Code>(a, mma, flat, vec, Hkv, st);
}
