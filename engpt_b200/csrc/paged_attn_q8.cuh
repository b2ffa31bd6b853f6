// Attention over a paged cache in 8 bits (the scheme and the kernels' frame: paged_attn.cuh; the codes: paged_q8.cuh).
//
// A key's scale multiplies its score, a value's scale its weight:
//   o = sum_j p_j vs_j vc_j / sum_j p_j,   p_j = exp(scale ks_j q.kc_j - m)
// with kc, vc the codes, so the codes themselves are what is multiplied.
#pragma once

#include "paged_attn.cuh"
#include "paged_q8.cuh"

#include <type_traits>

namespace engpt {
namespace paged {

struct Q8AttnArgs : AttnArgs {
  const float* k_scales;
  const float* v_scales;
  int64_t kss[3], vss[3];   // element strides: page, head, block
  int block;
};

// ------------------------------------------------------------------ tensor-core kernel (head_dim up to 128)
//
// Scores of int8 codes are products of whole numbers (mma.sync on 8-bit integers, 32-bit sums, exact): a row of q, times a
// power of two, is rounded to 16 bits (fp32 q: 24), which are two (three) digits of 8 bits; the first two are rows 0-7
// and 8-15 of one operand, so the second one is free.  What that rounding takes from q is below 2^-15 (2^-23) of the row's
// largest element; the codes themselves are that of a number rounded to 2^-8 of a block's largest one.
//
// e4m3 codes, and all values, are exact in fp16 (4 significant bits, 2^-9 to 448; integers up to 127), so these products run
// on fp16 operands with fp32 sums:
//   S = Q K^T with q brought to [1, 2) by a power of two of its row, which the row's score factor takes back; a
//   fp32 q is two fp16 numbers, the second one (what the first left, times 2^11) in the otherwise idle rows 8-15;
//   O^T += V^T P^T with weights p vs / ref in fp16, ref the largest p vs of the head so far (it shrinks with p when the
//   running maximum of the scores rises): at most 2^15 as scaled, so that what is 2^-28 of the head's largest weight is
//   still a normal number, whatever the scales of keys that have no weight.  That rounding is 2^-11 of a weight, an
//   eighth of that of a bf16 result; for fp32 results what it left is multiplied too.  (O^T because its 16-row operand
//   is full of values, where that of O would be half empty.)
//
// The columns of a product may come in any order that both operands share, and keys and columns of O in any order at
// all: a 16-byte row of 8-bit codes that ldmatrix distributes (4 bytes a lane, in place of two 16-bit numbers) is the
// fragment of an 8-bit product, or becomes those of two steps or tiles by byte permutations, with no transposition of
// bytes.
template <typename C>
struct CodePairs;
// Two codes of w, at the bytes that SEL names in the permutation's order, as fp16.
template <>
struct CodePairs<Int8Code> {
  // With the sign bit flipped a code is c + 128, and 0x6400 + that the fp16 number 1024 + 128 + c.
  static __device__ __forceinline__ uint32_t prepare(uint32_t w) { return w ^ 0x80808080u; }
  template <int A, int B>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    const uint32_t x = __byte_perm(w, 0x64646464u, 0x4040 | A | B << 8);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&y);
  }
};
template <>
struct CodePairs<E4m3Code> {
  static __device__ __forceinline__ uint32_t prepare(uint32_t w) { return w; }
  template <int A, int B>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    uint32_t y;
    const uint16_t x = (uint16_t)__byte_perm(w, 0, A | B << 4);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(y) : "h"(x));
    return y;
  }
};

__device__ __forceinline__ void mma16816_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma16832_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_half2(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// x and y as fp16, and what that left of them.
__device__ __forceinline__ uint32_t split_half2(float& x, float& y) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  x -= f.x;
  y -= f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}

struct Q8MmaArgs : MmaArgs {
  const char* pools[2];     // k, v
  int64_t page_bytes[2], head_bytes[2];   // their strides
  const float* scales[2];
  int ss[2][3];             // element strides: page, head, block
  int block, block_shift;   // tokens of a block, a multiple of 8; its logarithm, or -1
};

// Width: of 4 or 8 pieces of 16 columns, padded by TMA and swizzled by it so that ldmatrix finds its rows in different
// banks; or, Flat, of any other number of them, exactly the head_dim: rows as they lie in the page, one behind the other
// (an odd number of 16-byte pieces has no bank conflicts, 2 and 6 have 2-way ones).  TMA takes a row of a box at a time,
// 8 to 9 cycles for 80 bytes and no fewer for 16, where it moves whole pieces of a page at the rate of memory: 64 rows
// of 2048 tokens, 8 heads of 80: 64 us padded, 38 so.
//
// A tile costs some 730 instructions of a warp (64 keys of 64: 16 products of scores, 16 of values, 96 instructions that
// make fp16 of the values' codes, 210 of the softmax, the rest its bookkeeping), and 16 warps with 8 KB each cover
// memory and each other best, although their 128 registers spill 4 to 260 bytes in nearly every form (fp32 q the most):
// 64 rows of up to 4096 tokens, 16 heads of 64, 58 us.  Measured before weights had a reference per head (57.5 then): 12
// warps with 16 KB 56.9, but 256 rows of 1 to 512 tokens 48 us there, 37 so, and eight query heads of 128 have no room; 8
// warps with 16 KB 60 and 56.  Without any arithmetic on the tiles the first is 50 us.
template <int Pieces, bool Flat, typename C, typename Type>
struct Q8Tile {
  static constexpr int DC = Pieces;                 // 16-byte pieces of a row
  static constexpr int kWidth = 16 * DC;            // bytes of a row in shared memory
  static constexpr int D = (DC + 1) / 2 * 32;       // columns of a part
  static constexpr int KT = !Flat ? 256 / DC : DC <= 2 ? 128 : DC <= 5 ? 64 : 32;
  static constexpr int kTile = KT * kWidth, kWarps = Flat && DC == 5 ? 14 : 16;
  static constexpr int kPairWarps = 8, kPairPerSm = 2, kTileUs = 2;
  // (Shared memory has room for two CTAs of the pair form per SM, with eight query heads of 128 too.  Registers have where
  // the kernel takes no more than 128: int8 codes and bf16 q at head_dim 64, and a few of the flat forms.  The others, 130 to
  // 200, run one at a time, so a launch of more CTAs than SMs is two waves: 4 rows of 1024 tokens, 16 heads of 128, 13.3 us
  // where 2 rows take 7.1.)
  static constexpr bool kPartsOver = true;
  static constexpr int NG = KT / 8;       // groups of 8 keys, which share their scales
  static constexpr int kStep = KT < 64 ? KT : 64;   // keys of a softmax step
  static constexpr int NT = kStep / 8;    // 8-key tiles of a step
  static constexpr bool kInt = C::kInteger;
  static constexpr bool kFlat = Flat;
  static constexpr int kCodeBytes = 1, kBoxes = 1, kBoxRow = kWidth;
  static constexpr CUtensorMapDataType kMapType = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  static constexpr CUtensorMapSwizzle kSwizzle = DC == 4 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  static constexpr bool kFine = sizeof(Type) == 4;   // three digits or two parts of q, two parts of a weight
  // (2^14 and 2^-112: their quotient has to be finite, as it meets scales of 0)
  static constexpr float kWeightTop = 16384.f, kLeastRef = 1.925929944387236e-34f;
  using T = Type;
  using Args = Q8MmaArgs;
  using Pairs = CodePairs<C>;
  // Lane i < NG looks after the key scale of group i of the tile, lane NG + i after its value scale.
  struct Spot {
    int page, off;   // off -1: no such key
  };
  struct Side {
    float scale;     // 0 without a key
  };
  struct Query {
    uint32_t a[DC], b[kInt || kFine ? DC : 1], c[kInt && kFine ? DC : 1];   // int8: the digits; else see load_query
    uint32_t a2[kInt ? 1 : DC], b2[!kInt && kFine ? DC : 1];
    float factor;    // base-2 score of a sum of products
  };
  struct State {
    // piece c, row of O^T: columns 16 c + 2 g and 16 c + 2 g + 1 (0, 1 and 2, 3) of heads 2 t and 2 t + 1 of the group, in
    // units of their heads' ref / kWeightTop, where g = lane / 4 and t = lane % 4.  m, l, ref and per_ref (kWeightTop / ref)
    // are those of head g.
    float o[DC][4];
    float m, l, ref, per_ref, factor;
    __device__ __forceinline__ void reset() {
#pragma unroll
      for (int i = 0; i < DC; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
      m = -INFINITY;
      l = 0.f;
      ref = kLeastRef;
      per_ref = kWeightTop / kLeastRef;
      factor = 1.f;
    }
    // Every column of O^T times its head's x.
    __device__ __forceinline__ void scale_heads(float x, int lane) {
      const float x0 = __shfl_sync(0xffffffffu, x, 8 * (lane & 3)), x1 = __shfl_sync(0xffffffffu, x, 8 * (lane & 3) + 4);
#pragma unroll
      for (int i = 0; i < DC; ++i) {
        o[i][0] *= x0;
        o[i][1] *= x1;
        o[i][2] *= x0;
        o[i][3] *= x1;
      }
    }
  };

  static __device__ __forceinline__ Spot find(const Args& a, const Cursor& c, int lane) {
    const int key = c.t * KT + lane % NG * 8;
    if (lane >= 2 * NG || key >= c.len) return Spot{0, -1};
    const int j = a.ps_shift >= 0 ? key >> a.ps_shift : key / a.ps;
    return Spot{a.table[c.b * a.table_stride + j], key - j * a.ps};
  }

  static __device__ __forceinline__ void fetch(const Args& a, const Cursor& c, const Spot& x, Side& side) {
    const int lane = threadIdx.x & 31, part = lane / NG;
    side.scale = 0.f;
    if (x.off < 0 || c.t * KT + lane % NG * 8 >= c.len || (unsigned)x.page >= (unsigned)a.P) return;
    const int block = a.block_shift >= 0 ? x.off >> a.block_shift : x.off / a.block;
    const float* p = part == 0 ? a.scales[0] : a.scales[1];
    p += (int64_t)x.page * (part == 0 ? a.ss[0][0] : a.ss[1][0]);
    p += (int64_t)c.hk * (part == 0 ? a.ss[0][1] : a.ss[1][1]);
    p += (int64_t)block * (part == 0 ? a.ss[0][2] : a.ss[1][2]);
    side.scale = *p;
  }

  static __device__ __forceinline__ void load_query(const Args& a, int b, int h, int lane, Query& x) {
    const int g = lane >> 2, t = lane & 3;
    const int head = (h / a.QG) * a.G + (h % a.QG) * 8 + g;
    const bool live = g < a.rows && (h % a.QG) * 8 + g < a.G;
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_row + head * a.q_head + 4 * t;
    float v[DC][4];
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < DC; ++k) {
      if (live && k * 16 < a.dim) {
        if constexpr (sizeof(T) == 2) {
          const uint2 r = *reinterpret_cast<const uint2*>(q + k * 16);
          v[k][0] = __uint_as_float(r.x << 16);
          v[k][1] = __uint_as_float(r.x & 0xffff0000u);
          v[k][2] = __uint_as_float(r.y << 16);
          v[k][3] = __uint_as_float(r.y & 0xffff0000u);
        } else {
          const float4 r = *reinterpret_cast<const float4*>(q + k * 16);
          v[k][0] = r.x;
          v[k][1] = r.y;
          v[k][2] = r.z;
          v[k][3] = r.w;
        }
      } else {
        v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) most = max(most, __float_as_uint(v[k][i]) & 0x7fffffffu);
    }
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    if constexpr (kInt) {
      // round(q 2^(bits - e)): the row's largest element comes to 2^bits up to 2^(bits + 1), but not so near to that that
      // its first digit would be above 127.  (Rows that are nearly zero, below 2^-100, are brought less far up.)
      constexpr int bits = kFine ? 22 : 14;
      const uint32_t e = min(max((most + 0x20000u) >> 23, 27u), 255u);
      const float up = __uint_as_float((uint32_t)(254 + bits - e) << 23);
      x.factor = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u)
                                     : a.scale_log2 * __uint_as_float((uint32_t)(e - bits) << 23);
      const float f = a.negative ? -up : up;
#pragma unroll
      for (int k = 0; k < DC; ++k) {
        int d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = __float2int_rn(v[k][i] * f);
        uint32_t* digits[3] = {&x.a[k], &x.b[k], &x.c[kFine ? k : 0]};
#pragma unroll
        for (int n = kFine ? 2 : 1; n >= 0; --n) {
          *digits[n] = __byte_perm(__byte_perm(d[0], d[1], 0x0040), __byte_perm(d[2], d[3], 0x0040), 0x5410);
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] = (d[i] - (int)(int8_t)d[i]) >> 8;
        }
      }
    } else {
      const uint32_t e = min(max(most >> 23, 1u), 253u);   // the largest |q| is in [1, 2) 2^(e - 127), for most rows
      const float down = __uint_as_float((254u - e) << 23);
      x.factor = a.scale_log2 * __uint_as_float(e << 23);
      const float f = a.negative ? -down : down;
#pragma unroll
      for (int k = 0; k < DC; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[k][i] *= f;
        x.a[k] = split_half2(v[k][0], v[k][1]);
        x.a2[k] = split_half2(v[k][2], v[k][3]);
        if constexpr (kFine) {
          x.b[k] = pack_half2(v[k][0] * 2048.f, v[k][1] * 2048.f);
          x.b2[k] = pack_half2(v[k][2] * 2048.f, v[k][3] * 2048.f);
        }
      }
    }
  }

  // Scores of the 8 keys from `key` on, as sums of products: this lane's two of head g.
  static __device__ __forceinline__ void scores(const Query& x, uint32_t sk, int key, int lane, float* s) {
    const int r8 = lane & 7, q4 = lane >> 3;
    // (four pieces at a time; behind the last one it is loaded again, and not used)
    if constexpr (kInt) {
      int c[4] = {0, 0, 0, 0}, last[4] = {0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < DC; p += 4) {
        uint32_t w[4];
        ldsm4(piece(sk, key + r8, DC % 4 ? min(p + q4, DC - 1) : p + q4), w);
#pragma unroll
        for (int i = 0; i < 4 && p + i < DC; i += 2) {
          const bool two = p + i + 1 < DC;
          const int j = two ? p + i + 1 : p + i;
          mma16832_s8(c, x.a[p + i], x.b[p + i], two ? x.a[j] : 0u, two ? x.b[j] : 0u, w[i], two ? w[i + 1] : 0u);
          if constexpr (kFine) mma16832_s8(last, x.c[p + i], 0u, two ? x.c[j] : 0u, 0u, w[i], two ? w[i + 1] : 0u);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = (float)(c[i] * 256 + c[2 + i]);     // below 2^29
        if constexpr (kFine) s[i] = fmaf(s[i], 256.f, (float)last[i]);
      }
    } else {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < DC; p += 4) {
        uint32_t w[4];
        ldsm4(piece(sk, key + r8, DC % 4 ? min(p + q4, DC - 1) : p + q4), w);
#pragma unroll
        for (int i = 0; i < 4 && p + i < DC; ++i)
          mma16816_f16(c, x.a[p + i], kFine ? x.b[p + i] : 0u, x.a2[p + i], kFine ? x.b2[p + i] : 0u,
                       Pairs::template pair<0, 1>(w[i]), Pairs::template pair<2, 3>(w[i]));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i] = kFine ? fmaf(c[2 + i], 1.f / 2048.f, c[i]) : c[i];
    }
  }

  static __device__ __forceinline__ const char* rows_at(const Args& a, int part, int page, int head, int off) {
    return a.pools[part] + page * a.page_bytes[part] + head * a.head_bytes[part] + off * kWidth;
  }

  // Address of 16-byte piece c of a key's row in shared memory (swizzled as TMA has done it).
  static __device__ __forceinline__ uint32_t piece(uint32_t base, int key, int c) {
    if (Flat) return base + key * kWidth + c * 16;
    return DC == 4 ? base + key * 64 + ((c ^ ((key >> 1) & 3)) << 4) : base + key * 128 + ((c ^ (key & 7)) << 4);
  }

  // One tile: per kStep keys scores, softmax step, P V.  WHOLE: all its keys count.  Otherwise `live` keys from the tile's
  // start are below the length, and boxes whose bit of `mask` is unset were not copied.
  template <bool WHOLE>
  static __device__ __forceinline__ void step(const Args& a, uint32_t sk, const Query& x, const Side& side, State& st,
                                              int live, uint32_t mask, int lane) {
    const uint32_t sv = sk + kTile;
    const int r8 = lane & 7, q4 = lane >> 3, t = lane & 3;
    if (!WHOLE && C::kHasNan) {
      // absent values become 0: their weight 0 would not cancel a stale NaN
      for (int i = lane; i < KT * DC; i += 32) {
        const int key = i / DC;
        if (key >= live || !((mask >> (key >> a.r_shift)) & 1u))
          asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(sv + i * 16), "r"(0u) : "memory");
      }
      __syncwarp();
    }
    st.factor = x.factor;
#pragma unroll
    for (int k0 = 0; k0 < KT; k0 += kStep) {
      float s[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        scores(x, sk, k0 + n * 8, lane, s[n]);
        const float ks = __shfl_sync(0xffffffffu, side.scale, k0 / 8 + n);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[n][i] *= ks;
          if (!WHOLE) {
            const int key = k0 + n * 8 + 2 * t + i;
            if (key >= live || !((mask >> (key >> a.r_shift)) & 1u)) s[n][i] = -INFINITY;
          }
        }
      }
      float mx = st.m;
#pragma unroll
      for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(s[n][0], s[n][1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float ms = mx == -INFINITY ? 0.f : mx * st.factor;
      const bool rises = mx > st.m;
      if (rises) {
        // (O stays as it is in its units, which shrink with the weights that are in it)
        const float corr = st.m == -INFINITY ? 0.f : sm100::ex2_approx(st.m * st.factor - ms);
        st.ref *= corr;
        st.l *= corr;
        st.m = mx;
      }
      float sum[2] = {0.f, 0.f}, most = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float vs = __shfl_sync(0xffffffffu, side.scale, NG + k0 / 8 + n);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float p = sm100::ex2_approx(fmaf(s[n][i], st.factor, -ms));
          if (!WHOLE && s[n][i] == -INFINITY) p = 0.f;      // (the product is NaN for a scale of 0)
          sum[i] += p;
          s[n][i] = p * vs;
          most = fmaxf(most, fabsf(s[n][i]));
        }
      }
      st.l += sum[0] + sum[1];
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const bool other = rises || most > 2.f * st.ref;
      if (__any_sync(0xffffffffu, other)) {
        // (a head's numbers do not depend on the others': the quotient is 1 where its ref stays)
        const float ref = other ? fmaxf(fmaxf(st.ref, most), kLeastRef) : st.ref;
        st.scale_heads(st.ref / ref, lane);
        st.ref = ref;
        st.per_ref = kWeightTop / ref;
      }
      uint32_t hi[NT], lo[kFine ? NT : 1];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n][0] *= st.per_ref;
        s[n][1] *= st.per_ref;
        if constexpr (kFine) {
          hi[n] = split_half2(s[n][0], s[n][1]);
          lo[n] = pack_half2(s[n][0], s[n][1]);
        } else {
          hi[n] = pack_half2(s[n][0], s[n][1]);
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        const int key = k0 + j * 8 + (q4 & 1) * 8 + r8;
#pragma unroll
        for (int c = 0; c < DC; c += 2) {
          uint32_t w[4];
          // keys 0-7 and 8-15 of piece c, then of piece c + 1 (or of c again, not used)
          ldsm4_t(piece(sv, key, DC % 2 ? min(c + (q4 >> 1), DC - 1) : c + (q4 >> 1)), w);
#pragma unroll
          for (int i = 0; i < 2 && c + i < DC; ++i) {
            const uint32_t y0 = Pairs::prepare(w[2 * i]), y1 = Pairs::prepare(w[2 * i + 1]);
            const uint32_t a0 = Pairs::template pair<0, 2>(y0), a1 = Pairs::template pair<1, 3>(y0),
                           a2 = Pairs::template pair<0, 2>(y1), a3 = Pairs::template pair<1, 3>(y1);
            mma16816_f16(st.o[c + i], a0, a1, a2, a3, hi[j], hi[j + 1]);
            if constexpr (kFine) mma16816_f16(st.o[c + i], a0, a1, a2, a3, lo[j], lo[j + 1]);
          }
        }
      }
    }
    if (!WHOLE && C::kHasNan) sm100::fence_proxy_async_smem();   // the zeros above, before a later copy into this memory
  }

  // The pair's sums of this lane: o in its own units and l over the head's four lanes; m in base-2 units.
  static __device__ __forceinline__ void finish(const Args&, State& st) {
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
    if (st.m != -INFINITY) st.m *= st.factor;
    st.scale_heads(st.ref * (1.f / kWeightTop), threadIdx.x & 31);
  }

  static __device__ __forceinline__ void store_part(const Args& a, const State& st, float* part, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (2 * t + r >= a.rows) break;
      float* p = part + (2 * t + r) * (D + 2) + 2 * g;
#pragma unroll
      for (int i = 0; i < DC; ++i) *reinterpret_cast<float2*>(p + i * 16) = make_float2(st.o[i][r], st.o[i][2 + r]);
    }
    if (t == 0 && g < a.rows) *reinterpret_cast<float2*>(part + g * (D + 2) + D) = make_float2(st.m, st.l);
  }

  static __device__ __forceinline__ void store_rows(const Args& a, State& st, int b, int h, int lane) {
    const int g = lane >> 2, t = lane & 3;
    st.scale_heads(st.l == 0.f ? 0.f : 1.f / st.l, lane);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int in = (h % a.QG) * 8 + 2 * t + r;
      if (2 * t + r >= a.rows || in >= a.G) break;
      T* o = reinterpret_cast<T*>(a.o) + ((int64_t)b * a.H + (h / a.QG) * a.G + in) * a.dim + 2 * g;
#pragma unroll
      for (int i = 0; i < DC; ++i) {
        if (i * 16 >= a.dim) break;
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint32_t*>(o + i * 16) = sm100::pack_bf16x2(st.o[i][r], st.o[i][2 + r]);
        else
          *reinterpret_cast<float2*>(o + i * 16) = make_float2(st.o[i][r], st.o[i][2 + r]);
      }
    }
  }
};

template <typename F>
int launch_mma_q8(const Q8AttnArgs& x, int Hkv, cudaStream_t st) {
  Q8MmaArgs a;
  a.pools[0] = static_cast<const char*>(x.k_pages);
  a.pools[1] = static_cast<const char*>(x.v_pages);
  a.page_bytes[0] = x.ks[0];
  a.page_bytes[1] = x.vs[0];
  a.head_bytes[0] = x.ks[1];
  a.head_bytes[1] = x.vs[1];
  a.scales[0] = x.k_scales;
  a.scales[1] = x.v_scales;
  for (int i = 0; i < 3; ++i) {
    a.ss[0][i] = (int)x.kss[i];
    a.ss[1][i] = (int)x.vss[i];
  }
  a.block = x.block;
  a.block_shift = (x.block & (x.block - 1)) == 0 ? __builtin_ctz((unsigned)x.block) : -1;
  return launch_mma<F>(a, x, Hkv, st);
}

// Calls f(pieces as a constant) for the widths of the flat form: all but 4 and 8 pieces.
template <typename G>
auto flat_pieces(int dim, G f) {
  switch (dim / 16) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    case 5: return f(std::integral_constant<int, 5>());
    case 6: return f(std::integral_constant<int, 6>());
    default: return f(std::integral_constant<int, 7>());
  }
}
template <typename C, typename T>
int launch_flat(const Q8AttnArgs& a, int Hkv, cudaStream_t st) {
  return flat_pieces(a.Dh, [&](auto n) { return launch_mma_q8<Q8Tile<n.value, true, C, T>>(a, Hkv, st); });
}
// (in files of their own, which build beside each other)
int launch_flat_int8(const Q8AttnArgs& a, int Hkv, bool f32, cudaStream_t st);
int launch_flat_e4m3(const Q8AttnArgs& a, int Hkv, bool f32, cudaStream_t st);

}  // namespace paged
}  // namespace engpt
