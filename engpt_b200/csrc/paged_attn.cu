// Attention over a paged cache in bf16 or fp32 (the scheme and the kernels' frame: paged_attn.cuh).
#include "paged_attn.cuh"

namespace engpt {
namespace paged {

template <typename T>
int dispatch_simt(const AttnArgs& a, bool vec, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const int nc = vec ? (a.Dh + 8 * V - 1) / (8 * V) : (a.Dh + 7) / 8;
  if (vec && sizeof(T) == 4) {
    if (nc <= 1) return launch_simt_heads<PlainKv<T>, V, 1, 4>(a, st);
    if (nc <= 2) return launch_simt_heads<PlainKv<T>, V, 2, 4>(a, st);
    if (nc <= 4) return launch_simt_heads<PlainKv<T>, V, 4, 2>(a, st);
    return launch_simt<PlainKv<T>, V, 8, 1, 1>(a, st);
  }
  if (vec) {   // bf16 comes here with a head_dim above 128, or pages of an odd size
    if (nc <= 2) return launch_simt<PlainKv<T>, V, 2, 2, 1>(a, st);
    return launch_simt<PlainKv<T>, V, 4, 1, 1>(a, st);
  }
  if (nc <= 8) return launch_simt<PlainKv<T>, 1, 8, 2, 1>(a, st);
  return launch_simt<PlainKv<T>, 1, 32, 1, 1>(a, st);
}

// ------------------------------------------------------------------ tensor-core kernel (bf16, head_dim up to 128)
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// p as bf16 plus the bf16 of what that rounding left.
__device__ __forceinline__ void split_bf16x2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = sm100::pack_bf16x2(x, y);
  const float hx = __uint_as_float(hi << 16), hy = __uint_as_float(hi & 0xffff0000u);
  lo = sm100::pack_bf16x2(x - hx, y - hy);
}


// The two halves of the operand added: (sum of bf16(p) v) + (sum of (p - bf16(p)) v).  Where a value is infinite the
// first half is the result; the second one, with weights of either sign or 0, would turn it into NaN.
__device__ __forceinline__ float add_halves(float hi, float lo) { return fabsf(hi) == INFINITY ? hi : hi + lo; }

// Built for a width D of 64 or 128; a smaller head_dim is padded with zeros.
//
// Per tile, with up to 8 query heads of the kv head as rows 0-7 of the operand:
//   S = Q K^T (rows 8-15 are zero), p = 2^(S scale - m), and O += P V with P's bf16 value in rows 0-7 and the
//   remainder p - bf16(p), again as bf16, in rows 8-15: adding the two halves of O at the end gives the product
//   with weights of 16 mantissa bits for the price of the otherwise idle half of the operand.
//
// Warps and tiles are what 64 rows of up to 4096 tokens (16 heads of 64, bf16) run best with: eight warps, each of which
// idles while its 16 KB fly but has seven others beside it, 87 us; 10 or 12 such warps 90 and 89, six or four with two
// tiles in flight each 101 and 105, eight with two tiles of 8 KB 97.
template <int Width>
struct Bf16Tile {
  static constexpr int D = Width;
  static constexpr int kTile = 8192, kWarps = 8, kPairWarps = 4, kPairPerSm = 2, kTileUs = 2;
  static constexpr bool kPartsOver = false;
  static constexpr int KT = kTile / (2 * D);
  static constexpr int NT = KT / 8;     // 8-key tiles
  static constexpr int KC = KT / 16;    // 16-key steps of P V
  static constexpr int DK = D / 16;     // 16-dim steps of Q K^T
  static constexpr int DN = D / 8;      // 8-dim tiles of O
  static constexpr int kCodeBytes = 2, kBoxes = D / 64, kBoxRow = 128;
  static constexpr bool kFlat = false;
  static constexpr CUtensorMapDataType kMapType = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  static constexpr CUtensorMapSwizzle kSwizzle = CU_TENSOR_MAP_SWIZZLE_128B;
  using T = __nv_bfloat16;
  using Args = MmaArgs;
  struct Spot {};
  struct Side {};
  struct Query {
    uint32_t qa[DK][2];
  };
  static __device__ __forceinline__ Spot find(const MmaArgs&, const Cursor&, int) { return {}; }
  static __device__ __forceinline__ void fetch(const MmaArgs&, const Cursor&, const Spot&, Side&) {}

  // The running state of one pair: rows 0-7 of S and O in the mma layout (row lane / 4, columns 2 (lane % 4) + {0, 1}
  // of each 8-column tile).  m is in units of the raw product q.k.
  struct State {
    float o[DN][4];
    float m, l;
    __device__ __forceinline__ void reset() {
#pragma unroll
      for (int i = 0; i < DN; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
      m = -INFINITY;
      l = 0.f;
    }
  };

  static __device__ __forceinline__ void load_query(const MmaArgs& a, int b, int h, int lane, Query& x) {
    const int g = lane >> 2, t = lane & 3;
    const int head = (h / a.QG) * a.G + (h % a.QG) * 8 + g;
    const bool live = g < a.rows && (h % a.QG) * 8 + g < a.G;
    const uint32_t flip = a.negative ? 0x80008000u : 0u;
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + b * a.q_row + head * a.q_head + 2 * t;
#pragma unroll
    for (int k = 0; k < DK; ++k) {
      x.qa[k][0] = live && k * 16 < a.dim ? *reinterpret_cast<const uint32_t*>(q + k * 16) ^ flip : 0u;
      x.qa[k][1] = live && k * 16 + 8 < a.dim ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8) ^ flip : 0u;
    }
  }

  // One tile: scores, softmax step, P V.  WHOLE: all its keys count.  Otherwise `live` keys from the tile's start are
  // below the length, and boxes whose bit of `mask` is unset were not copied.
  template <bool WHOLE>
  static __device__ __forceinline__ void step(const MmaArgs& a, uint32_t sk, const Query& x, const Side&, State& st,
                                              int live, uint32_t mask, int lane) {
    const uint32_t sv = sk + kTile;
    const int r8 = lane & 7, q4 = lane >> 3, t = lane & 3;
    if (!WHOLE) {
      // absent values become 0: their weight 0 would not cancel a stale NaN or infinity
      for (int i = lane; i < KT * (D / 64) * 8; i += 32) {   // 16-byte pieces: half, key, piece
        const int key = (i >> 3) % KT;
        if (key >= live || !((mask >> (key >> a.r_shift)) & 1u))
          asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(sv + i * 16), "r"(0u) : "memory");
      }
      __syncwarp();
    }
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int kp = 0; kp < DK / 2; ++kp) {
      uint32_t b[NT][4];
      const int c = kp * 4 + q4;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        ldsm4(sk + (c >> 3) * (KT * 128) + (n * 8 + r8) * 128 + (((c & 7) ^ r8) << 4), b[n]);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma16816(s[n], x.qa[2 * kp][0], 0u, x.qa[2 * kp][1], 0u, b[n][0], b[n][1]);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma16816(s[n], x.qa[2 * kp + 1][0], 0u, x.qa[2 * kp + 1][1], 0u, b[n][2], b[n][3]);
    }
    if (!WHOLE) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = n * 8 + 2 * t + i;
          if (key >= live || !((mask >> (key >> a.r_shift)) & 1u)) s[n][i] = -INFINITY;
        }
    }
    float mx = st.m;
#pragma unroll
    for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(s[n][0], s[n][1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float ms = mx == -INFINITY ? 0.f : mx * a.scale_log2;
    if (__any_sync(0xffffffffu, mx > st.m)) {
      const float corr = st.m == -INFINITY ? 0.f : sm100::ex2_approx(st.m * a.scale_log2 - ms);
#pragma unroll
      for (int i = 0; i < DN; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) st.o[i][j] *= corr;
      st.l *= corr;
      st.m = mx;
    }
    uint32_t hi[KC][2], lo[KC][2];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float p[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        p[i] = sm100::ex2_approx(fmaf(s[n][i], a.scale_log2, -ms));
        if (!WHOLE && s[n][i] == -INFINITY) p[i] = 0.f;   // (the product is NaN for a scale of 0)
        sum[i] += p[i];
      }
      split_bf16x2(p[0], p[1], hi[n >> 1][n & 1], lo[n >> 1][n & 1]);
    }
    st.l += sum[0] + sum[1];
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      const int key = j * 16 + (q4 & 1) * 8 + r8;
      uint32_t b[DN / 2][4];
#pragma unroll
      for (int dp = 0; dp < DN / 2; ++dp) {
        const int c = 2 * dp + (q4 >> 1);
        ldsm4_t(sv + (c >> 3) * (KT * 128) + key * 128 + (((c & 7) ^ r8) << 4), b[dp]);
      }
#pragma unroll
      for (int dp = 0; dp < DN / 2; ++dp) {
        mma16816(st.o[2 * dp], hi[j][0], lo[j][0], hi[j][1], lo[j][1], b[dp][0], b[dp][1]);
        mma16816(st.o[2 * dp + 1], hi[j][0], lo[j][0], hi[j][1], lo[j][1], b[dp][2], b[dp][3]);
      }
    }
    if (!WHOLE) sm100::fence_proxy_async_smem();   // the zeros above, before a later copy into this memory
  }

  // The pair's sums of this lane: o (both halves) and l over the row's four lanes; m in base-2 units.
  static __device__ __forceinline__ void finish(const MmaArgs& a, State& st) {
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
    if (st.m != -INFINITY) st.m *= a.scale_log2;
#pragma unroll
    for (int i = 0; i < DN; ++i) {
      st.o[i][0] = add_halves(st.o[i][0], st.o[i][2]);
      st.o[i][1] = add_halves(st.o[i][1], st.o[i][3]);
    }
  }

  static __device__ __forceinline__ void store_part(const MmaArgs& a, const State& st, float* part, int lane) {
    const int g = lane >> 2, t = lane & 3;
    if (g >= a.rows) return;
    float* p = part + g * (D + 2);
#pragma unroll
    for (int i = 0; i < DN; ++i) *reinterpret_cast<float2*>(p + i * 8 + 2 * t) = make_float2(st.o[i][0], st.o[i][1]);
    if (t == 0) *reinterpret_cast<float2*>(p + D) = make_float2(st.m, st.l);
  }

  static __device__ __forceinline__ void store_rows(const MmaArgs& a, const State& st, int b, int h, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const int in = (h % a.QG) * 8 + g;
    if (g >= a.rows || in >= a.G) return;
    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.o) + ((int64_t)b * a.H + (h / a.QG) * a.G + in) * a.dim + 2 * t;
    const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
#pragma unroll
    for (int i = 0; i < DN; ++i)
      if (i * 8 < a.dim) *reinterpret_cast<uint32_t*>(o + i * 8) = sm100::pack_bf16x2(st.o[i][0] * inv, st.o[i][1] * inv);
  }
};

// Does a launch of these sizes go to the tensor-core kernel (strides and alignment apart)?
inline bool mma_sizes(int dtype, int B, int H, int D, int table_width, int page_size) {
  return dtype == ENGPT_BF16 && D <= 128 && D % 8 == 0 && page_size % 8 == 0 &&
         list_fits(B, H, mma_width(D) == 64 ? Bf16Tile<64>::KT : Bf16Tile<128>::KT, table_width, page_size);
}

}  // namespace paged
}  // namespace engpt

using namespace engpt;
using namespace engpt::paged;

extern "C" int64_t engpt_paged_attention_floats(int dtype, int B, int H, int Hkv, int Dh, int table_width,
                                                int page_size) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || Dh <= 0 || table_width < 0 || page_size <= 0) return 0;
  const int splits = simt_splits(B, H, (int64_t)table_width * page_size);
  const int64_t simt = splits > kSimtCluster ? (int64_t)B * H * splits * (Dh + 2) : 0;
  if (!mma_sizes(dtype, B, H, Dh, table_width, page_size)) return simt;
  // strides and alignment decide at the call which of the two kernels runs
  const int cs = mma_width(Dh) == 64 ? pair_ctas<Bf16Tile<64>>(B, H, Hkv, table_width, page_size)
                                     : pair_ctas<Bf16Tile<128>>(B, H, Hkv, table_width, page_size);
  const int64_t mma = cs == 0 ? mma_floats(H, Hkv, Dh) : 0;
  return simt > mma ? simt : mma;
}

extern "C" int engpt_paged_attention(const void* q, const int64_t* q_strides, const void* k_pages,
                                     const void* v_pages, const int64_t* page_strides, int dtype, int B, int H,
                                     int Hkv, int Dh, int num_pages, int page_size, const int* block_table,
                                     int64_t table_stride, int table_width, const int* lengths, float scale, void* o,
                                     float* workspace, void* stream) {
  clear_error();
  ENGPT_REQUIRE(B >= 0 && H > 0 && Hkv > 0 && Dh > 0 && H % Hkv == 0, ENGPT_ERR_SHAPE,
                "paged_attention: B=%d H=%d Hkv=%d Dh=%d", B, H, Hkv, Dh);
  ENGPT_REQUIRE(Dh <= 256, ENGPT_ERR_UNSUPPORTED, "paged_attention: head_dim %d > 256", Dh);
  ENGPT_REQUIRE(B <= 65535 && H <= 65535, ENGPT_ERR_SHAPE, "paged_attention: B=%d H=%d (at most 65535)", B, H);
  ENGPT_REQUIRE(num_pages >= 0 && page_size > 0 && (int64_t)num_pages * page_size <= 0x7fffffffLL, ENGPT_ERR_SHAPE,
                "paged_attention: num_pages=%d page_size=%d", num_pages, page_size);
  ENGPT_REQUIRE(table_width >= 0 && table_stride >= table_width && (int64_t)table_width * page_size <= kMostKeys,
                ENGPT_ERR_SHAPE, "paged_attention: table_width=%d page_size=%d", table_width, page_size);
  ENGPT_REQUIRE(dtype == ENGPT_BF16 || dtype == ENGPT_F32, ENGPT_ERR_DTYPE, "paged_attention: dtype %d", dtype);
  if (B == 0) return ENGPT_OK;
  ENGPT_REQUIRE(q && q_strides && page_strides && lengths && o, ENGPT_ERR_ARG, "paged_attention: null pointer");
  ENGPT_REQUIRE((k_pages && v_pages) || num_pages == 0, ENGPT_ERR_ARG, "paged_attention: null cache");
  ENGPT_REQUIRE(block_table || table_width == 0, ENGPT_ERR_ARG, "paged_attention: null block table");
  const int esz = dtype == ENGPT_BF16 ? 2 : 4;
  AttnArgs a;
  a.q = q;
  a.q_row = q_strides[0];
  a.q_head = q_strides[1];
  a.k_pages = k_pages;
  a.v_pages = v_pages;
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
  ENGPT_REQUIRE(workspace || engpt_paged_attention_floats(dtype, B, H, Hkv, Dh, table_width, page_size) == 0,
                ENGPT_ERR_ARG, "paged_attention: null workspace");
  ENGPT_REQUIRE(aligned(workspace, 16), ENGPT_ERR_ALIGN, "paged_attention: workspace not 16-byte aligned");
  bool vec = aligned(q, 16) && aligned(k_pages, 16) && aligned(v_pages, 16) && Dh * esz % 16 == 0 &&
             a.q_row * esz % 16 == 0 && a.q_head * esz % 16 == 0;
  bool positive = true;
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = page_strides[i];
    a.vs[i] = page_strides[3 + i];
    // the stride of an axis of one element is never used, and may be anything
    const bool one = (i == 0 ? num_pages : i == 1 ? Hkv : page_size) == 1;
    if (one) a.ks[i] = a.vs[i] = Dh;
    vec = vec && a.ks[i] * esz % 16 == 0 && a.vs[i] * esz % 16 == 0;
    positive = positive && a.ks[i] > 0 && a.vs[i] > 0;
  }
  cudaStream_t st = as_stream(stream);
  // (the tensor-core kernels write o in pieces of up to 16 bytes, the others element by element)
  if (vec && positive && aligned(o, 16) && num_pages > 0 && mma_sizes(dtype, B, H, Dh, table_width, page_size))
    return mma_width(Dh) == 64 ? launch_mma<Bf16Tile<64>>({}, a, Hkv, st) : launch_mma<Bf16Tile<128>>({}, a, Hkv, st);
  return dtype == ENGPT_BF16 ? dispatch_simt<__nv_bfloat16>(a, vec, st) : dispatch_simt<float>(a, vec, st);
}
