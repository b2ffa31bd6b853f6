// Writing the paged key-value cache in 8 bits (paged_q8.cu: finished rows; paged_q8_append.cu: the post-process).
//
// The tokens that one call puts into a block of the cache stand side by side
// in it, in slots that follow one another; such a run is quantised as a whole:
//
//   need  = max(max |x|, 2^-100) / top        (top: 127 for int8, 448 for e4m3)
//   scale = need if the run holds the block's first slot, else max(scale, need)
//   code  = round(x / scale)
//
// (x / scale as the product with the rounded reciprocal of the scale: an x within 2^-23 of the middle between two codes,
// such as half of the block's largest, may go to either)
// and where the scale of a block that is not started anew grows, its codes
// outside the run become round(code * (scale before / scale)): the values
// stay, as far as the coarser step allows.
//
// Tokens that go on in the same block but not in the next slot would be a second run of it, in a race with the first one:
// they are recorded and left out.
//
// All of it is a pass over the numbers with a maximum in between, bound by HBM.
#pragma once

#include "paged_q8.cuh"

#include <type_traits>

namespace engpt {
namespace paged {

struct StoreArgs {
  Q8Cache c;
  const int* slots;        // [n]
  int64_t n;
  // write: finished rows
  const void* x[2];        // k, v
  int64_t row[2], head[2]; // element strides
  // append: raw projection rows [n, 3, H, Dh] and their post-process
  const void* qkv;
  const float* rho;
  const float* cos_tab;
  const float* sin_tab;
  int rope_rows, rope_half;
  const float* qk_scale;
  float qk_mult, eps;
  const int* positions;
  void* q;                 // [n, H, Dh]
};

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(v);
  else return v;
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(v);
  else return v;
}

__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// A token's slot as given, or -1 for none; one outside the pool is recorded (by the lane that is told to).
__device__ __forceinline__ int checked_slot(const StoreArgs& a, int slot, bool record) {
  if (slot >= 0 && slot < a.c.n_slots) return slot;
  if (slot != -1 && record) record_device_error(ENGPT_ERR_ARG, 43);
  return -1;
}

// Is slot `before` in the block that begins with slot `first` (0 or more)?  Negative ones are in none.
__device__ __forceinline__ bool in_block(const StoreArgs& a, int before, int first) {
  return before >= first && before - first < a.c.block;
}

// Numbers of one (token, head) row, as they go into the cache before the quantisation.
template <typename T, bool APPEND>
struct Row {
  const StoreArgs& a;
  const T* src;
  int part;                  // 0: k, 1: v, 2: q
  const float *c, *s, *scl;  // rotary row and scales
  float mult;                // 1 / norm, or 1 / rho
  bool live;

  // By a whole warp.
  __device__ __forceinline__ Row(const StoreArgs& args, int64_t n, int h, int p, int lane) : a(args), part(p) {
    const int64_t Dh = a.c.Dh;
    live = true;
    if constexpr (!APPEND) {
      src = reinterpret_cast<const T*>(a.x[part]) + n * a.row[part] + h * a.head[part];
    } else {
      src = reinterpret_cast<const T*>(a.qkv) + ((n * 3 + (part + 1) % 3) * a.c.H + h) * Dh;
      const int pos = a.positions[n];
      live = pos >= 0 && pos < a.rope_rows;
      if (!live) return;
      c = a.cos_tab + (int64_t)pos * a.rope_half;
      s = a.sin_tab + (int64_t)pos * a.rope_half;
      scl = a.qk_scale + h * Dh;
      if (part == 1) {
        mult = __fdiv_rn(1.f, a.rho[n]);
        return;
      }
      float ss = 0.f;
      for (int e = lane; e < a.c.Dh; e += 32) {
        const float v = to_f32(src[e]);
        ss = fmaf(v, v, ss);
      }
      float den = sqrtf(warp_sum_xor<32>(ss));
      if (a.eps > 0.f) den = fmaxf(den, a.rho[n] * a.eps);
      mult = __fdiv_rn(1.f, den);
    }
  }

  __device__ __forceinline__ float at(int e) const {
    if constexpr (!APPEND) {
      return to_f32(src[e]);
    } else {
      float v = to_f32(src[e]);
      if (part == 1) return v * mult;
      const int p = e >> 1;
      if (p < a.rope_half) {
        const float o = to_f32(src[e ^ 1]);
        v = e & 1 ? o * s[p] + v * c[p] : v * c[p] - o * s[p];
      }
      return v * mult * (scl[e] * a.qk_mult);
    }
  }
};

// Any head_dim, strides and alignment: one warp per (token, head, k | v | q).  The warp of a run's first token does the
// run, in two passes over its numbers (the second one reads from cache); the warps of the others have nothing to do.
template <typename T, typename Code, bool APPEND>
__global__ void __launch_bounds__(256) store_generic_kernel(StoreArgs a) {
  const int lane = threadIdx.x & 31;
  const int parts = APPEND ? 3 : 2;
  const int64_t task = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5);
  if (task >= a.n * parts * a.c.H) return;
  const int h = (int)(task % a.c.H);
  const int64_t np = task / a.c.H;
  const int part = (int)(np % parts);
  const int64_t n = np / parts;
  const int Dh = a.c.Dh;
  if constexpr (APPEND) {
    if (part == 2) {
      const Row<T, APPEND> row(a, n, h, part, lane);
      if (!row.live && h == 0 && lane == 0) record_device_error(ENGPT_ERR_ARG, 42);
      T* q = reinterpret_cast<T*>(a.q) + (n * a.c.H + h) * (int64_t)Dh;
      for (int e = lane; e < Dh; e += 32) q[e] = from_f32<T>(row.live ? row.at(e) : 0.f);
      return;
    }
  }
  const int slot = checked_slot(a, a.slots[n], part == 0 && h == 0 && lane == 0);
  if (slot < 0) return;
  const int off = slot % a.c.block, first = slot - off;   // (the block size divides the page size)
  if (n > 0 && in_block(a, a.slots[n - 1], first)) {   // of an earlier token's run, or astray
    if (a.slots[n - 1] != slot - 1 && part == 0 && h == 0 && lane == 0) record_device_error(ENGPT_ERR_ARG, 43);
    return;
  }
  int run = 1;
  while (off + run < a.c.block && n + run < a.n && a.slots[n + run] == slot + run) ++run;

  uint32_t amax = 0;
  bool any = false;
  for (int i = 0; i < run; ++i) {
    const Row<T, APPEND> row(a, n + i, h, part, lane);
    if (!row.live) continue;
    any = true;
    for (int e = lane; e < Dh; e += 32) amax = max(amax, abs_bits(row.at(e)));
  }
  if (!any) return;
  amax = __reduce_max_sync(0xffffffffu, amax);
  const float need = needed_scale<Code>(amax);
  float* scale_p = a.c.scales[part] + a.c.scale_at(part, slot, h);
  const float old = off > 0 ? *scale_p : 0.f;
  const float scale = off > 0 ? raised_scale(old, need) : need;
  uint8_t* codes = reinterpret_cast<uint8_t*>(a.c.codes[part]);
  if (off > 0 && scale > old) {      // (not for NaN)
    const float ratio = __fdiv_rn(old, scale);
    for (int j = 0; j < a.c.block; ++j) {
      if (j >= off && j < off + run) continue;
      uint8_t* p = codes + a.c.code_at(part, first + j, h);
      for (int e = lane; e < Dh; e += 32) p[e] = Code::encode(Code::decode(p[e]) * ratio);
    }
  }
  const float inv = isnan(scale) ? 0.f : __fdiv_rn(1.f, scale);
  for (int i = 0; i < run; ++i) {
    const Row<T, APPEND> row(a, n + i, h, part, lane);
    if (!row.live) continue;
    uint8_t* p = codes + a.c.code_at(part, slot + i, h);
    for (int e = lane; e < Dh; e += 32) p[e] = isnan(scale) ? (uint8_t)0 : Code::encode(row.at(e) * inv);
  }
  __syncwarp();                      // every lane has read the scale
  if (lane == 0) *scale_p = scale;
}

// ------------------------------------------------------------------ store, 8 elements a lane
//
// head_dim a multiple of 8, aligned.  LPR lanes (a power of two) share a row, 8 elements each; a warp has 32 / LPR rows
// of a run beside each other and S such steps, of k and of v, all loads in flight before the first is used.  They stay in
// registers as they were loaded (those with four bf16 or two fp32 rows a lane spill 40 to 136 bytes of them); the
// post-processed k waits for its scale in shared memory, as fp32.  W warps share a run, so that it fits one team and its
// numbers are read once; a longer run is read twice.
//
// A team looks after the runs that begin in a window of `window` tokens, of one head: a block's worth in a long call,
// which is one run then, a single token in a short one or where requests add a token each.
//
// 32768 tokens of 16 heads of 64, 15 of 16 with a slot, bf16 to int8 (190 MB move): 42.6 us = 4.5 TB/s, bound by the
// latency of a run's chain (slots, rows, maximum, codes) at 28 warps per SM.  The append of 8188 tokens of 16 heads of 128
// in blocks of 64 (168 MB): 57 us = 3.0 TB/s, bound by the same latency at 16 warps per SM, a window's q ahead of its slots
// (29 M instructions, 46 % of the issue slots); 72 with 8 warps and 4 steps, 80 with the post-process applied twice in place of the shared memory, 66 with v
// loaded beside k.
// The largest of m >= 0 and the magnitudes of x and y; NaN if one is.
__device__ __forceinline__ float most3(float m, float x, float y) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float most8(float m, const float* x) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) m = most3(m, x[i], x[i + 1]);
  return m;
}

// Eight elements as loaded.
template <typename T>
struct Raw {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = ld_once(p + i * (16 / sizeof(T)));
  }
  __device__ __forceinline__ void get(float* x) const {
    if constexpr (sizeof(T) == 2) {
      unpack8(v[0], x);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[4 * i] = __uint_as_float(v[i].x);
        x[4 * i + 1] = __uint_as_float(v[i].y);
        x[4 * i + 2] = __uint_as_float(v[i].z);
        x[4 * i + 3] = __uint_as_float(v[i].w);
      }
    }
  }
  __device__ __forceinline__ float most() const {
    if constexpr (sizeof(T) == 2) {
      // (magnitudes of bf16 numbers, infinities and NaN above them, are in the order of their 15 bits)
      const uint32_t a = __vmaxu2(__vmaxu2(v[0].x & 0x7fff7fffu, v[0].y & 0x7fff7fffu),
                                  __vmaxu2(v[0].z & 0x7fff7fffu, v[0].w & 0x7fff7fffu));
      return __uint_as_float(max(a << 16, a & 0xffff0000u));
    } else {
      float x[8];
      get(x);
      return most8(0.f, x);
    }
  }
};

// The post-process of engpt_qkv_append of this lane's slice (elements from e0 on) of a q or k row.
template <typename T>
struct PostProcess {
  static constexpr bool kFast = sizeof(T) == 2;   // bf16 rows use the approximate reciprocals (2 ulp)
  const StoreArgs& a;
  int p0;                  // first rotary pair, a multiple of 4 like rope_half: 4 pairs rotate together or not at all
  float scl[8];
  __device__ __forceinline__ PostProcess(const StoreArgs& args, int h, int e0) : a(args), p0(e0 >> 1) {
    const float* scale = args.qk_scale + (int64_t)h * args.c.Dh + e0;
    const float4 s0 = __ldg(reinterpret_cast<const float4*>(scale)), s1 = __ldg(reinterpret_cast<const float4*>(scale + 4));
    const float v[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) scl[k] = v[k] * a.qk_mult;
  }

  static __device__ __forceinline__ float per_rho(float rho) { return kFast ? __fdividef(1.0f, rho) : 1.0f / rho; }

  // x: the raw slice, then the post-processed one; by a whole warp.  Bit for bit what engpt_qkv_append does.
  template <int LPR>
  __device__ __forceinline__ void apply(float* x, float rho, int pos) const {
    float c[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
    const bool rot = p0 < a.rope_half;
    if (rot && (unsigned)pos < (unsigned)a.rope_rows) {
      const int64_t at = (int64_t)pos * a.rope_half + p0;
      const float4 c4 = __ldg(reinterpret_cast<const float4*>(a.cos_tab + at));
      const float4 s4 = __ldg(reinterpret_cast<const float4*>(a.sin_tab + at));
      c[0] = c4.x; c[1] = c4.y; c[2] = c4.z; c[3] = c4.w;
      sn[0] = s4.x; sn[1] = s4.y; sn[2] = s4.z; sn[3] = s4.w;
    }
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fmaf(x[k], x[k], ss);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    float inv;
    if (kFast) {
      inv = rsqrtf(ss);
      if (a.eps > 0.f) inv = fminf(inv, __fdividef(1.0f, rho * a.eps));
    } else {
      float den = sqrtf(ss);
      if (a.eps > 0.f) den = fmaxf(den, rho * a.eps);
      inv = 1.0f / den;
    }
    if (rot) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float xe = x[2 * k], xo = x[2 * k + 1];
        x[2 * k] = ((xe * c[k] - xo * sn[k]) * inv) * scl[2 * k];
        x[2 * k + 1] = ((xe * sn[k] + xo * c[k]) * inv) * scl[2 * k + 1];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = (x[k] * inv) * scl[k];
    }
  }
};
struct NoPostProcess {
  __device__ __forceinline__ NoPostProcess(const StoreArgs&, int, int) {}
};

// This lane's slices of S rows of a run, k and v.
template <typename T, bool APPEND, int LPR, int S, int W>
struct Rows {
  static constexpr int kRows = W * (32 / LPR);   // rows of the team's step
  using Post = std::conditional_t<APPEND, PostProcess<T>, NoPostProcess>;
  Raw<T> v[S], k[APPEND ? 1 : S];
  float4* s_k;             // appending: this lane's part of the warp's shared memory, [S][2][32]
  float v_mult[APPEND ? S : 1];
  uint32_t live;           // bit s: the row of step s is there, and its position in range

  // Rows 0, kRows, ... from this lane's first one on, `left` of the run behind it; n: that one's token; k0, v0: this
  // lane's elements of it.
  __device__ __forceinline__ void load(const StoreArgs& a, const Post& post, const T* k0, const T* v0, int64_t n, int left,
                                       bool mine) {
    Raw<T> kr[S];
    float rho[APPEND ? S : 1];
    int pos[APPEND ? S : 1];
    const int* pos_p = a.positions + n;
    const float* rho_p = a.rho + n;
    live = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const bool in = s * kRows < left;
      kr[s].clear();
      v[s].clear();
      if (in && mine) {
        kr[s].load(k0);
        if (!APPEND) v[s].load(v0);
      }
      k0 += kRows * a.row[0];
      if (!APPEND) v0 += kRows * a.row[1];
      if constexpr (APPEND) {
        pos[s] = in ? pos_p[s * kRows] : -1;
        rho[s] = in ? rho_p[s * kRows] : 1.f;
        if ((unsigned)pos[s] < (unsigned)a.rope_rows) live |= 1u << s;
      } else {
        live |= in ? 1u << s : 0u;
        k[s] = kr[s];
      }
    }
    if constexpr (APPEND) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        float x[8];
        kr[s].get(x);
        post.template apply<LPR>(x, rho[s], pos[s]);
        const bool on = mine && ((live >> s) & 1u);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = on ? x[e] : 0.f;
        s_k[s * 64] = make_float4(x[0], x[1], x[2], x[3]);
        s_k[s * 64 + 32] = make_float4(x[4], x[5], x[6], x[7]);
        most_k = most8(s == 0 ? 0.f : most_k, x);
        // (a token that is left out has zeros for v, and any number for rho)
        v_mult[s] = (live >> s) & 1u ? PostProcess<T>::per_rho(rho[s]) : 0.f;
      }
      // (v follows when k has given its registers up: more warps instead of more loads in flight per warp)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (mine && ((live >> s) & 1u)) v[s].load(v0);
        v0 += kRows * a.row[1];
      }
    }
  }
  float most_k;
  __device__ __forceinline__ float largest(int p) const {
    float m = APPEND && p == 0 ? most_k : 0.f;
#pragma unroll
    for (int s = 0; s < S; s += 1) {
      if (APPEND && p == 0) break;
      // (a product with 1 / rho rounds in the order of the magnitudes: the largest one's is the largest)
      const float x = p == 0 ? k[APPEND ? 0 : s].most() : v[s].most() * (APPEND ? v_mult[APPEND ? s : 0] : 1.f);
      m = most3(m, x, 0.f);
    }
    return m;
  }
  // The codes of part p (0: k, 1: v) of step s, for 1 / scale.
  template <typename Code>
  __device__ __forceinline__ uint2 codes(int p, int s, float inv) const {
    float x[8];
    if (APPEND && p == 0) {
      const float4 a = s_k[s * 64], b = s_k[s * 64 + 32];
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else if (p == 0) {
      k[APPEND ? 0 : s].get(x);
    } else {
      v[s].get(x);
      if constexpr (APPEND) {
        // (one by one: the product of the two factors can be infinite where x / rho is 0, or next to nothing)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= v_mult[s];
      }
    }
    return make_uint2(Code::encode4(x, inv), Code::encode4(x + 4, inv));
  }
};

// q of a window of tokens (appending).
template <typename T, int LPR, int S, int W>
__device__ __forceinline__ void store_q(const StoreArgs& a, int h, int64_t w0, int64_t w1, int me, int lane) {
  constexpr int RPW = 32 / LPR, kRows = W * RPW;
  int e0 = (lane % LPR) * 8;
  const bool mine = e0 < a.c.Dh;
  if (!mine) e0 = 0;
  const PostProcess<T> post(a, h, e0);
  const int width = a.c.H * a.c.Dh;
  int64_t n = w0 + me * RPW + lane / LPR;
  for (int left = (int)(w1 - n); __any_sync(0xffffffffu, left > 0); left -= S * kRows, n += S * kRows) {
    const T* src = reinterpret_cast<const T*>(a.qkv) + n * 3 * width + (int64_t)h * a.c.Dh + e0;
    T* dst = reinterpret_cast<T*>(a.q) + n * width + (int64_t)h * a.c.Dh + e0;
    const int* pos_p = a.positions + n;
    const float* rho_p = a.rho + n;
    Raw<T> raw[S];
    int pos[S];
    float rho[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const bool in = s * kRows < left;
      raw[s].clear();
      if (in && mine) raw[s].load(src);
      src += (int64_t)(3 * kRows) * width;
      pos[s] = in ? pos_p[s * kRows] : -1;
      rho[s] = in ? rho_p[s * kRows] : 1.f;
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float x[8];
      raw[s].get(x);
      post.template apply<LPR>(x, rho[s], pos[s]);
      if (s * kRows < left && mine) {
        if ((unsigned)pos[s] >= (unsigned)a.rope_rows) {
          if (h == 0 && e0 == 0) record_device_error(ENGPT_ERR_ARG, 42);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = 0.f;
        }
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(dst) = pack8(x);
        } else {
          *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
      }
      dst += (int64_t)kRows * width;
    }
  }
}

// CTAs of four warps per SM that the registers leave room for.  The write above: 42.6 us with 7, 43.9 with 6, 51 with 4,
// 55 with 10 (more of them spill); the append: 56 with 4 in its 8-step form, 65 with 3, 74 with 5.
template <bool APPEND, int BYTES>
constexpr int kStoreCtas = BYTES > 8 ? 4 : APPEND ? 6 : 7;

template <typename T, typename Code, bool APPEND, int LPR, int S, int W>
__global__ void __launch_bounds__(128, kStoreCtas<APPEND, S * (int)sizeof(T)>)
store_runs_kernel(StoreArgs a, int window) {
  static_assert(W == 1 || W == 4, "a team is a warp or the CTA");
  constexpr int RPW = 32 / LPR, kRows = W * RPW;
  __shared__ uint32_t s_most[W > 1 ? W : 1][2];
  __shared__ float4 s_k[APPEND ? 4 : 1][APPEND ? S * 64 : 1];
  if constexpr (APPEND) {
    // started ahead of the end of what runs before (usually the projection), and so may be what follows
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int me = W > 1 ? warp : 0;                     // this warp of its team
  const int64_t item = W > 1 ? blockIdx.x : blockIdx.x * 4ll + warp;
  const int64_t windows = (a.n + window - 1) / window;
  constexpr bool kApart = APPEND && S == 1;            // q is an item of its own
  if (item >= windows * (kApart ? 2 : 1) * a.c.H) return;   // (of the last CTA of single warps only)
  const int64_t wp = item <= 0xffffffffLL ? (int64_t)((uint32_t)item / (uint32_t)a.c.H) : item / a.c.H;
  const int h = (int)(item - wp * a.c.H);
  const int64_t w0 = (kApart ? wp >> 1 : wp) * window, w1 = min(a.n, w0 + window);
  if constexpr (APPEND) {
    if (!kApart || (wp & 1)) store_q<T, LPR, S, W>(a, h, w0, w1, me, lane);
    if (kApart && (wp & 1)) return;
  }
  int e0 = (lane % LPR) * 8;
  const bool mine = e0 < a.c.Dh;
  if (!mine) e0 = 0;
  const typename Rows<T, APPEND, LPR, S, W>::Post post(a, h, e0);
  const T* const src_k = reinterpret_cast<const T*>(a.x[0]) + h * a.head[0] + e0;
  const T* const src_v = reinterpret_cast<const T*>(a.x[1]) + h * a.head[1] + e0;
  const int row0 = me * RPW + lane / LPR;              // this lane's first row of a run
  Rows<T, APPEND, LPR, S, W> rows;
  rows.s_k = &s_k[APPEND ? warp : 0][APPEND ? lane : 0];

  for (int64_t t0 = w0; t0 < w1; t0 += 32) {
    // the slots of 32 tokens, and which of them begin a run (of those in the window)
    const int64_t mine_n = t0 + lane;
    const int given = mine_n < a.n ? a.slots[mine_n] : -1;
    int before = __shfl_up_sync(0xffffffffu, given, 1);
    if (lane == 0) before = mine_n > 0 ? a.slots[mine_n - 1] : -1;
    const bool window_token = mine_n < w1;
    const int slot = checked_slot(a, given, window_token && h == 0 && me == 0);
    const int my_off = max(slot, 0) - a.c.block_of(max(slot, 0)) * a.c.block;   // (blocks divide pages)
    const bool goes_on = in_block(a, before, slot - my_off);   // an earlier token's run, or is astray
    uint32_t heads = __ballot_sync(0xffffffffu, window_token && slot >= 0 && !goes_on);
    if (h == 0 && window_token && slot >= 0 && goes_on && before != slot - 1) record_device_error(ENGPT_ERR_ARG, 43);
    while (heads) {
      const int i = __ffs(heads) - 1;
      heads &= heads - 1;
      const int first = __shfl_sync(0xffffffffu, slot, i), off = __shfl_sync(0xffffffffu, my_off, i);
      const int64_t n0 = t0 + i;
      const int room = a.c.block - off;                // slots up to the block's end
      // this run's tokens: those whose slots go on from the first one's
      const uint32_t on = __ballot_sync(0xffffffffu, lane >= i && lane - i < room && slot == first + (lane - i));
      int run = __ffs(~(on >> i)) - 1;                 // (on >> i has a 1 at the bottom; -1: all 32)
      if (run < 0) run = 32;
      if (i + run == 32) {                             // it may go on behind these 32 tokens
        while (run < room) {
          const int64_t n = n0 + run + lane;
          const bool more = run + lane < room && n < a.n && a.slots[n] == first + run + lane;
          const uint32_t m = __ballot_sync(0xffffffffu, more);
          const int k = m == 0xffffffffu ? 32 : __ffs(~m) - 1;
          run += k;
          if (k < 32) break;
        }
      }
      const int64_t n1 = n0 + row0;                    // this lane's first token
      const T *k = src_k + n1 * a.row[0], *v = src_v + n1 * a.row[1];
      rows.load(a, post, k, v, n1, run - row0, mine);
      const int page = a.c.page_of(first), in_page = first - page * a.c.ps, block = a.c.block_of(in_page);
      float* scale_p[2];
      float old[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        scale_p[p] = a.c.scales[p] + page * a.c.ss[p][0] + h * a.c.ss[p][1] + block * a.c.ss[p][2];
        old[p] = off > 0 ? *scale_p[p] : 0.f;
      }
      float largest[2] = {rows.largest(0), rows.largest(1)};
      uint32_t any = rows.live;
      for (int r0 = S * kRows; r0 < run; r0 += S * kRows) {
        rows.load(a, post, k + r0 * a.row[0], v + r0 * a.row[1], n1 + r0, run - row0 - r0, mine);
        largest[0] = most3(largest[0], rows.largest(0), 0.f);
        largest[1] = most3(largest[1], rows.largest(1), 0.f);
        any |= rows.live;
      }
      uint32_t most[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) most[p] = __reduce_max_sync(0xffffffffu, __float_as_uint(largest[p]));
      if (APPEND) any = __any_sync(0xffffffffu, any != 0);
      if constexpr (W > 1) {
        // (a magnitude's top bit is free: whether there is any number at all)
        if (lane < 2) s_most[warp][lane] = (lane == 0 ? most[0] : most[1]) | (any ? 0x80000000u : 0u);
        __syncthreads();
        const uint32_t m = s_most[lane % W][(lane / W) & 1];   // lanes 0 .. W - 1: k, the next W: v
        most[0] = __reduce_max_sync(0xffffffffu, lane < W ? m & 0x7fffffffu : 0u);
        most[1] = __reduce_max_sync(0xffffffffu, lane >= W && lane < 2 * W ? m & 0x7fffffffu : 0u);
        any = __any_sync(0xffffffffu, m >> 31);
        __syncthreads();                               // before the next run's maxima
      }
      if (APPEND && !any) continue;
      float inv[2];
      uint8_t* code_p[2];                              // this lane's codes of its first row
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int64_t row = a.c.cs[p][2];
        uint8_t* at = reinterpret_cast<uint8_t*>(a.c.codes[p]) + page * a.c.cs[p][0] + h * a.c.cs[p][1] +
                      (in_page - off + row0) * row + e0;       // row row0 of the block
        const float need = needed_scale<Code>(most[p]);
        const float scale = off > 0 ? raised_scale(old[p], need) : need;
        if (off > 0 && scale > old[p]) {               // (not for NaN)
          const float ratio = __fdiv_rn(old[p], scale);
          uint8_t* to = at;
          for (int j = row0; j < a.c.block; j += kRows, to += kRows * row) {
            if ((j >= off && j < off + run) || !mine) continue;
            uint2* c = reinterpret_cast<uint2*>(to);
            const uint2 w = *c;
            float y[8];
            Code::decode4(w.x, y);
            Code::decode4(w.y, y + 4);
            *c = make_uint2(Code::encode4(y, ratio), Code::encode4(y + 4, ratio));
          }
        }
        inv[p] = isnan(scale) ? 0.f : __fdiv_rn(1.f, scale);
        code_p[p] = at + off * row;
        if (lane == 0 && me == 0) *scale_p[p] = scale;
      }
      // (a run of one load is still there)
      for (int r0 = 0; r0 < run; r0 += S * kRows) {
        if (run > S * kRows) rows.load(a, post, k + r0 * a.row[0], v + r0 * a.row[1], n1 + r0, run - row0 - r0, mine);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const bool here = ((rows.live >> s) & 1u) && mine;
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            if (here) *reinterpret_cast<uint2*>(code_p[p]) = rows.template codes<Code>(p, s, inv[p]);
            code_p[p] += kRows * a.c.cs[p][2];
          }
        }
      }
    }
  }
}

// Checks of a cache's description, common to all entry points; fills `c`.
inline int fill_q8_cache(const char* what, Q8Cache& c, void* k_pages, void* v_pages, float* k_scales, float* v_scales,
                  const int64_t* page_strides, const int64_t* scale_strides, int code, int H, int Dh, int num_pages,
                  int page_size, int block) {
  ENGPT_REQUIRE(H > 0 && Dh > 0 && (int64_t)H * Dh <= 0x7fffffffLL, ENGPT_ERR_SHAPE, "%s: H=%d Dh=%d", what, H, Dh);
  ENGPT_REQUIRE(num_pages >= 0 && page_size > 0 && (int64_t)num_pages * page_size <= 0x7fffffffLL, ENGPT_ERR_SHAPE,
                "%s: num_pages=%d page_size=%d", what, num_pages, page_size);
  ENGPT_REQUIRE(block > 0 && page_size % block == 0, ENGPT_ERR_SHAPE, "%s: blocks of %d tokens in pages of %d", what,
                block, page_size);
  ENGPT_REQUIRE(code == ENGPT_CODE_INT8 || code == ENGPT_CODE_E4M3, ENGPT_ERR_DTYPE, "%s: code type %d", what, code);
  ENGPT_REQUIRE(page_strides && scale_strides, ENGPT_ERR_ARG, "%s: null pointer", what);
  ENGPT_REQUIRE((k_pages && v_pages && k_scales && v_scales) || num_pages == 0, ENGPT_ERR_ARG, "%s: null cache", what);
  c.codes[0] = k_pages;
  c.codes[1] = v_pages;
  c.scales[0] = k_scales;
  c.scales[1] = v_scales;
  for (int p = 0; p < 2; ++p)
    for (int i = 0; i < 3; ++i) {
      // the stride of an axis of one element is never used, and may be anything
      c.cs[p][i] = (i == 0 ? num_pages : i == 1 ? H : page_size) == 1 ? 0 : page_strides[3 * p + i];
      c.ss[p][i] = (i == 0 ? num_pages : i == 1 ? H : page_size / block) == 1 ? 0 : scale_strides[3 * p + i];
    }
  c.H = H;
  c.Dh = Dh;
  c.ps = page_size;
  c.block = block;
  c.ps_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1;
  c.block_shift = (block & (block - 1)) == 0 ? __builtin_ctz((unsigned)block) : -1;
  c.n_slots = (int64_t)num_pages * page_size;
  return ENGPT_OK;
}

template <typename T, typename Code, bool APPEND>
int launch_store_generic(const StoreArgs& a, const char* what, cudaStream_t st) {
  const int64_t tasks = a.n * (APPEND ? 3 : 2) * a.c.H, blocks = (tasks + 7) / 8;
  ENGPT_REQUIRE(blocks <= 0x7fffffffLL, ENGPT_ERR_SHAPE, "%s: too large", what);
  store_generic_kernel<T, Code, APPEND><<<(unsigned)blocks, 256, 0, st>>>(a);
  return check_launch(what);
}

template <typename T, typename Code, bool APPEND, int LPR, int S, int W>
int launch_store_runs(const StoreArgs& a, int window, const char* what, cudaStream_t st) {
  const int64_t items = (a.n + window - 1) / window * (APPEND && S == 1 ? 2 : 1) * a.c.H, blocks = W > 1 ? items : (items + 3) / 4;
  ENGPT_REQUIRE(blocks <= 0x7fffffffLL, ENGPT_ERR_SHAPE, "%s: too large", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = APPEND ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, store_runs_kernel<T, Code, APPEND, LPR, S, W>, a, window);
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

template <typename T, typename Code, bool APPEND, int LPR>
int launch_store_team(const StoreArgs& a, const char* what, cudaStream_t st) {
  constexpr int kHeld = 8 / sizeof(T), RPW = 32 / LPR;    // steps: 4 of bf16 rows, 2 of fp32 ones, or twice as many
  // A token per window while that makes no more warps than run at once some times over.  Appending, the calls that
  // matter add a token per request, and a window of a block's tokens would be as many runs one after the other: 999
  // requests, 16 heads of 64: 23 us so, 61 in windows of 16 (one prompt of 1100 tokens: 27 us so, 8 in windows); a write
  // is a prompt's (2047 tokens: 6.3 us in windows, 17 a token each).  The rule sees the number of tokens alone: a step of
  // more than 1184 requests with 16 heads goes in windows too (4096: 130 us).
  const bool single = a.n * (APPEND ? 2 : 1) * a.c.H <= (int64_t)num_sms() * (APPEND ? 256 : 64);
  if (single) return launch_store_runs<T, Code, APPEND, LPR, 1, 1>(a, 1, what, st);
  if (a.c.block > 2 * kHeld * RPW) return launch_store_runs<T, Code, APPEND, LPR, 2 * kHeld, 4>(a, a.c.block, what, st);
  if (a.c.block > kHeld * RPW) return launch_store_runs<T, Code, APPEND, LPR, 2 * kHeld, 1>(a, a.c.block, what, st);
  return launch_store_runs<T, Code, APPEND, LPR, kHeld, 1>(a, a.c.block, what, st);
}

template <typename T, typename Code, bool APPEND>
int launch_store_code(const StoreArgs& a, bool vec, const char* what, cudaStream_t st) {
  const int Dh = a.c.Dh;
  if (!vec) return launch_store_generic<T, Code, APPEND>(a, what, st);
  if (Dh <= 16) return launch_store_team<T, Code, APPEND, 2>(a, what, st);
  if (Dh <= 32) return launch_store_team<T, Code, APPEND, 4>(a, what, st);
  if (Dh <= 64) return launch_store_team<T, Code, APPEND, 8>(a, what, st);
  if (Dh <= 128) return launch_store_team<T, Code, APPEND, 16>(a, what, st);
  return launch_store_team<T, Code, APPEND, 32>(a, what, st);
}

template <typename T, bool APPEND>
int launch_store(const StoreArgs& a, int code, bool vec, const char* what, cudaStream_t st) {
  const int esz = sizeof(T);
  const Q8Cache& c = a.c;
  vec = vec && c.Dh % 8 == 0 && c.Dh <= 256 && aligned(c.codes[0], 8) && aligned(c.codes[1], 8);
  for (int p = 0; p < 2; ++p) {
    for (int i = 0; i < 3; ++i) vec = vec && c.cs[p][i] % 8 == 0;
    if (!APPEND) vec = vec && aligned(a.x[p], 16) && a.row[p] * esz % 16 == 0 && a.head[p] * esz % 16 == 0;
  }
  return code == ENGPT_CODE_INT8 ? launch_store_code<T, Int8Code, APPEND>(a, vec, what, st)
                                 : launch_store_code<T, E4m3Code, APPEND>(a, vec, what, st);
}

// (in a file of its own, which builds beside the others)
int launch_append_f32(const StoreArgs& a, int code, bool vec, cudaStream_t st);

}  // namespace paged
}  // namespace engpt
