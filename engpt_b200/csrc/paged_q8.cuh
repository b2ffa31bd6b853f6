// The paged cache in 8 bits: codes and their scales.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math.h>

namespace engpt {
namespace paged {

// One cache: k (0) and v (1).
struct Q8Cache {
  void* codes[2];
  float* scales[2];
  int64_t cs[2][3];       // element strides of the codes: page, head, slot
  int64_t ss[2][3];       // of the scales: page, head, block
  int H, Dh;
  int ps, block;          // tokens of a page, and of a block (which divides it)
  int ps_shift, block_shift;   // their logarithms, or -1
  int64_t n_slots;        // num_pages * page_size

  __device__ __forceinline__ int page_of(int slot) const { return ps_shift >= 0 ? slot >> ps_shift : slot / ps; }
  __device__ __forceinline__ int block_of(int slot) const { return block_shift >= 0 ? slot >> block_shift : slot / block; }

  // codes of (slot, head) and scale of (slot, head), as offsets
  __device__ __forceinline__ int64_t code_at(int part, int slot, int h) const {
    const int page = page_of(slot), off = slot - page * ps;
    return page * cs[part][0] + h * cs[part][1] + off * cs[part][2];
  }
  __device__ __forceinline__ int64_t scale_at(int part, int slot, int h) const {
    const int page = page_of(slot), off = slot - page * ps;
    return page * ss[part][0] + h * ss[part][1] + block_of(off) * ss[part][2];
  }
};

// Codes.  kTop: the largest one.  encode: of a number that the scale has brought within +-kTop (up to rounding), to the
// nearest code, even ones in the middle; NaN gives some code.
struct Int8Code {
  static constexpr float kTop = 127.f;
  static constexpr bool kHasNan = false, kInteger = true;
  static __device__ __forceinline__ float decode(uint8_t c) { return (float)(int8_t)c; }
  static __device__ __forceinline__ uint8_t encode(float x) {
    int r;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(r) : "f"(x));
    return (uint8_t)r;
  }
  // The codes of four numbers times f: the sum of a product and 1.5 2^23, rounded once, has the rounded product in its
  // low bits.
  static __device__ __forceinline__ uint32_t encode4(const float* x, float f) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(fmaf(x[i], f, 12582912.f));
    return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
  }
  static __device__ __forceinline__ void decode4(uint32_t w, float* x) {
    // (with the sign bit flipped a code is c + 128)
    const uint32_t y = w ^ 0x80808080u;
    x[0] = __uint_as_float(__byte_perm(y, 0x4b000000u, 0x7440)) - 8388736.f;
    x[1] = __uint_as_float(__byte_perm(y, 0x4b000000u, 0x7441)) - 8388736.f;
    x[2] = __uint_as_float(__byte_perm(y, 0x4b000000u, 0x7442)) - 8388736.f;
    x[3] = __uint_as_float(__byte_perm(y, 0x4b000000u, 0x7443)) - 8388736.f;
  }
};

struct E4m3Code {
  static constexpr float kTop = 448.f;
  static constexpr bool kHasNan = true, kInteger = false;
  static __device__ __forceinline__ float decode(uint8_t c) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
    return __half2float(__half(h));
  }
  static __device__ __forceinline__ uint8_t encode(float x) {
    return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  }
  static __device__ __forceinline__ uint32_t encode4(const float* x, float f) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[1] * f), "f"(x[0] * f));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[3] * f), "f"(x[2] * f));
    return (uint32_t)lo | (uint32_t)hi << 16;
  }
  static __device__ __forceinline__ void decode4(uint32_t w, float* x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t y;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(y) : "h"((uint16_t)(w >> (16 * i))));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};

// The scale that a block needs for numbers of at most |x| = `amax`, given as bits (so that the largest of them in
// whole-number order is the largest magnitude, infinities and NaN above all): NaN if they are not finite, and never so
// small that its reciprocal is infinite.
constexpr float kLeastAmax = 7.888609052210118e-31f;   // 2^-100
template <typename Code>
__device__ __forceinline__ float needed_scale(uint32_t amax) {
  if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return __fdiv_rn(fmaxf(__uint_as_float(amax), kLeastAmax), Code::kTop);
}

// Scale of a block that held tokens with scale `old` before.  NaN stays.
__device__ __forceinline__ float raised_scale(float old, float need) {
  if (isnan(old) || isnan(need)) return __uint_as_float(0x7fc00000u);
  return fmaxf(old, need);
}

}  // namespace paged
}  // namespace engpt
