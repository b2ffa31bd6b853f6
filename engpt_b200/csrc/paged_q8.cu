// Writing and reading the paged key-value cache in 8 bits.
//
// The tokens that one call puts into a block of the cache stand side by side
// in it, in the order of their slots; such a run is quantised as a whole:
//
//   need  = max(max |x|, 2^-100) / top        (top: 127 for int8, 448 for e4m3)
//   scale = need if the run holds the block's first slot, else max(scale, need)
//   code  = round(x / scale)
//
// and where the scale of a block that is not started anew grows, its codes
// outside the run become round(code * (scale before / scale)): the values
// stay, as far as the coarser step allows.
//
// All of it is a pass over the numbers with a maximum in between, bound by HBM.
#include "paged_q8.cuh"

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

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// A token's slot as given, or -1 for none; one outside the pool is recorded (by the lane that is told to).
__device__ __forceinline__ int checked_slot(const StoreArgs& a, int slot, bool record) {
  if (slot >= 0 && slot < a.c.n_slots) return slot;
  if (slot != -1 && record) record_device_error(ENGPT_ERR_ARG, 43);
  return -1;
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
  if (off > 0 && n > 0 && a.slots[n - 1] == slot - 1) return;
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
// of a run beside each other and kSteps such steps in registers, all their loads in flight before the first is used.  W
// warps share a run, so that it fits the registers of one team: its numbers are read once.  (A longer run is read twice.)
//
// A team looks after the runs that begin in a window of `window` tokens of one head and one of k, v (and, appending, q):
// a block's worth in a long call, which is one run then, a single token in a short one or where requests add a token
// each.
constexpr int kSteps = 4;

// Eight elements of a row: as loaded, where the numbers are those of the cache, or as computed.
template <typename T, bool APPEND>
struct Held {
  float x[8];
  __device__ __forceinline__ void get(float* y) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
  }
  __device__ __forceinline__ uint32_t most(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(x[i]));
    return m;
  }
};
template <>
struct Held<__nv_bfloat16, false> {
  uint4 v;
  __device__ __forceinline__ void get(float* y) const { unpack8(v, y); }
  __device__ __forceinline__ uint32_t most(uint32_t m) const {
    // (magnitudes of bf16 numbers are in the order of their 16 bits, like those of fp32)
    const uint32_t a = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    return max(m, max(a << 16, a & 0xffff0000u));
  }
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (sizeof(T) == 2) {
    unpack8(ld_once(p), x);
  } else {
    const uint4 a = ld_once(p), b = ld_once(p + 4);
    x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
    x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y); x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
  }
}

// What a lane needs for its slice of the rows of one head and part.
template <typename T, int LPR, bool APPEND>
struct Slice {
  const StoreArgs& a;
  const T* src;            // its first element in token 0
  int64_t row;             // elements from token to token
  int part, e0;            // 0: k, 1: v, 2: q; first element
  bool mine;               // e0 is within the row
  float scl[8];
  __device__ __forceinline__ Slice(const StoreArgs& args, int h, int p, int lane) : a(args), part(p) {
    e0 = (lane % LPR) * 8;
    mine = e0 < a.c.Dh;
    if (!mine) e0 = 0;
    if constexpr (APPEND) {
      row = (int64_t)3 * a.c.H * a.c.Dh;
      src = reinterpret_cast<const T*>(a.qkv) + ((int64_t)(p + 1) % 3 * a.c.H + h) * a.c.Dh + e0;
      const float* s = a.qk_scale + (int64_t)h * a.c.Dh + e0;
      const float4 s0 = __ldg(reinterpret_cast<const float4*>(s)), s1 = __ldg(reinterpret_cast<const float4*>(s + 4));
      const float v[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) scl[i] = v[i] * a.qk_mult;
    } else {
      row = a.row[p];
      src = reinterpret_cast<const T*>(a.x[p]) + h * a.head[p] + e0;
    }
  }

  // The slice of N tokens, token n[i] if in[i]; by a whole warp.  live: the numbers are there (its position is not
  // out of range).  The arithmetic of engpt_qkv_append, bit for bit.
  template <int N>
  __device__ __forceinline__ void load(const int64_t* n, const bool* in, Held<T, APPEND>* out, bool* live) const {
    if constexpr (!APPEND) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        live[i] = in[i] && mine;
        if constexpr (sizeof(T) == 2) {
          out[i].v = make_uint4(0u, 0u, 0u, 0u);
          if (live[i]) out[i].v = ld_once(src + n[i] * row);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) out[i].x[k] = 0.f;
          if (live[i]) load8(src + n[i] * row, out[i].x);
        }
      }
    } else {
      constexpr bool kFast = sizeof(T) == 2;
      float rho[N];
      float4 c4[N], s4[N];
      const int p0 = e0 >> 1;
      const bool rot = part != 1 && p0 < a.rope_half;   // rope_half is a multiple of 4: 4 pairs rotate together or not
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int pos = in[i] ? a.positions[n[i]] : -1;
        live[i] = (unsigned)pos < (unsigned)a.rope_rows;
        rho[i] = 1.f;
        c4[i] = make_float4(1.f, 1.f, 1.f, 1.f);
        s4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) out[i].x[k] = 0.f;
        if (in[i]) {
          rho[i] = a.rho[n[i]];
          if (mine) load8(src + n[i] * row, out[i].x);
        }
        if (rot && live[i]) {
          c4[i] = __ldg(reinterpret_cast<const float4*>(a.cos_tab + (int64_t)pos * a.rope_half + p0));
          s4[i] = __ldg(reinterpret_cast<const float4*>(a.sin_tab + (int64_t)pos * a.rope_half + p0));
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float* x = out[i].x;
        if (part == 1) {
          const float inv_rho = kFast ? __fdividef(1.0f, rho[i]) : 1.0f / rho[i];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] *= inv_rho;
        } else {
          float ss = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) ss = fmaf(x[k], x[k], ss);
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          float inv_den;
          if (kFast) {
            inv_den = rsqrtf(ss);
            if (a.eps > 0.f) inv_den = fminf(inv_den, __fdividef(1.0f, rho[i] * a.eps));
          } else {
            float den = sqrtf(ss);
            if (a.eps > 0.f) den = fmaxf(den, rho[i] * a.eps);
            inv_den = 1.0f / den;
          }
          if (rot) {
            const float c[4] = {c4[i].x, c4[i].y, c4[i].z, c4[i].w}, sn[4] = {s4[i].x, s4[i].y, s4[i].z, s4[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float xe = x[2 * k], xo = x[2 * k + 1];
              x[2 * k] = ((xe * c[k] - xo * sn[k]) * inv_den) * scl[2 * k];
              x[2 * k + 1] = ((xe * sn[k] + xo * c[k]) * inv_den) * scl[2 * k + 1];
            }
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = (x[k] * inv_den) * scl[k];
          }
        }
        if (!live[i] || !mine) {      // (a row of length 0 may have given NaN behind the head_dim)
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = 0.f;
        }
        live[i] = live[i] && mine;
      }
    }
  }
};

template <typename T, typename Code, bool APPEND, int LPR, int W>
__global__ void __launch_bounds__(W > 4 ? 32 * W : 128) store_runs_kernel(StoreArgs a, int window) {
  constexpr int RPW = 32 / LPR, kRows = W * RPW;       // rows of a warp's step, of the team's
  __shared__ uint32_t s_most[W > 1 ? W : 1];
  if constexpr (APPEND) {
    // started ahead of the end of what runs before (usually the projection), and so may be what follows
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int me = W > 1 ? warp : 0;                     // this warp of its team
  const int parts = APPEND ? 3 : 2;
  const int64_t item = W > 1 ? blockIdx.x : blockIdx.x * 4ll + warp;
  const int64_t windows = (a.n + window - 1) / window;
  if (item >= windows * parts * a.c.H) return;         // (of the last CTA of single warps only)
  const int h = (int)(item % a.c.H);
  const int64_t wp = item / a.c.H;
  const int part = (int)(wp % parts);
  const int64_t w0 = wp / parts * window, w1 = min(a.n, w0 + window);
  const Slice<T, LPR, APPEND> slice(a, h, part, lane);
  const int sub = lane / LPR;

  if constexpr (APPEND) {
    if (part == 2) {
      T* q = reinterpret_cast<T*>(a.q) + (int64_t)h * a.c.Dh + slice.e0;
      for (int64_t t = w0 + me * RPW; t < w1; t += kRows) {
        const int64_t n = t + sub;
        const bool in = n < w1;
        Held<T, APPEND> x;
        bool live;
        slice.template load<1>(&n, &in, &x, &live);
        if (!in || !slice.mine) continue;
        if (!live && h == 0 && lane % LPR == 0) record_device_error(ENGPT_ERR_ARG, 42);
        T* dst = q + n * a.c.H * a.c.Dh;
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(dst) = pack8(x.x);
        } else {
          *reinterpret_cast<float4*>(dst) = make_float4(x.x[0], x.x[1], x.x[2], x.x[3]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(x.x[4], x.x[5], x.x[6], x.x[7]);
        }
      }
      return;
    }
  }
  uint8_t* const codes = reinterpret_cast<uint8_t*>(a.c.codes[part]) + h * a.c.cs[part][1] + slice.e0;
  float* const scales = a.c.scales[part] + h * a.c.ss[part][1];

  for (int64_t t0 = w0; t0 < w1; t0 += 32) {
    // the slots of 32 tokens, and which of them begin a run (of those in the window)
    const int64_t mine_n = t0 + lane;
    const int raw = mine_n < a.n ? a.slots[mine_n] : -1;
    const int before = mine_n > 0 && mine_n <= a.n ? a.slots[mine_n - 1] : -1;
    const bool window_token = mine_n < w1;
    const int slot = checked_slot(a, raw, window_token && part == 0 && h == 0 && me == 0);
    const int my_off = (int)((uint32_t)max(slot, 0) % (uint32_t)a.c.block);
    uint32_t heads = __ballot_sync(0xffffffffu, window_token && slot >= 0 && !(my_off > 0 && before == slot - 1));
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
      const int page = first / a.c.ps, in_page = first - page * a.c.ps;
      float* const scale_p = scales + page * a.c.ss[part][0] + in_page / a.c.block * a.c.ss[part][2];
      const float old = off > 0 ? *scale_p : 0.f;
      uint8_t* const block_p = codes + page * a.c.cs[part][0] + (in_page - off) * a.c.cs[part][2];   // the block's first row

      // the largest magnitude, with the numbers of the last kSteps steps kept
      Held<T, APPEND> x[kSteps];
      bool live[kSteps];
      const bool all = run <= kSteps * kRows;          // kept whole
      uint32_t most = 0;
      bool any = false;
      for (int r0 = 0; r0 < run; r0 += kSteps * kRows) {
        int64_t n[kSteps];
        bool in[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const int r = r0 + (s * W + me) * RPW + sub;
          in[s] = r < run;
          n[s] = n0 + r;
        }
        slice.template load<kSteps>(n, in, x, live);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          most = x[s].most(most);
          any = any || live[s];
        }
      }
      most = __reduce_max_sync(0xffffffffu, most);
      if (APPEND) any = __any_sync(0xffffffffu, any);
      if constexpr (W > 1) {
        // (most is a magnitude: its top bit says whether there is any number at all)
        if (lane == 0) s_most[warp] = most | (any ? 0x80000000u : 0u);
        __syncthreads();
        uint32_t m = 0;
        any = false;
#pragma unroll
        for (int k = 0; k < W; ++k) {
          m = max(m, s_most[k] & 0x7fffffffu);
          any = any || (s_most[k] & 0x80000000u);
        }
        most = m;
        __syncthreads();                               // before the next run's maxima
      }
      if (APPEND && !any) continue;
      const float need = needed_scale<Code>(most);
      const float scale = off > 0 ? raised_scale(old, need) : need;
      if (off > 0 && scale > old) {                    // (not for NaN)
        const float ratio = __fdiv_rn(old, scale);
        for (int j = me * RPW + sub; j < a.c.block; j += kRows) {
          if ((j >= off && j < off + run) || !slice.mine) continue;
          uint2* p = reinterpret_cast<uint2*>(block_p + j * a.c.cs[part][2]);
          const uint2 w = *p;
          float y[8];
          Code::decode4(w.x, y);
          Code::decode4(w.y, y + 4);
          *p = make_uint2(Code::encode4(y, ratio), Code::encode4(y + 4, ratio));
        }
      }
      const float inv = isnan(scale) ? 0.f : __fdiv_rn(1.f, scale);
      for (int r0 = 0; r0 < run; r0 += kSteps * kRows) {
        if (!all) {
          int64_t n[kSteps];
          bool in[kSteps];
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const int r = r0 + (s * W + me) * RPW + sub;
            in[s] = r < run;
            n[s] = n0 + r;
          }
          slice.template load<kSteps>(n, in, x, live);
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          if (!live[s]) continue;
          const int r = r0 + (s * W + me) * RPW + sub;
          float y[8];
          x[s].get(y);
          *reinterpret_cast<uint2*>(block_p + (off + r) * a.c.cs[part][2]) =
              make_uint2(Code::encode4(y, inv), Code::encode4(y + 4, inv));
        }
      }
      if (lane == 0 && me == 0) *scale_p = scale;
    }
  }
}

// ------------------------------------------------------------------ read
struct ReadArgs {
  Q8Cache c;
  const int* slots;
  int64_t n;
  void* out[2];            // [n, H, Dh]
};

// One thread per element of k and v.
template <typename T, typename Code>
__global__ void __launch_bounds__(256) read_generic_kernel(ReadArgs a) {
  const int64_t row = (int64_t)a.c.H * a.c.Dh, total = a.n * row;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t n = i / row;
    const int rest = (int)(i - n * row), h = rest / a.c.Dh, e = rest - h * a.c.Dh;
    const int slot = a.slots[n];
    const bool live = slot >= 0 && slot < a.c.n_slots;
    if (!live && slot != -1 && rest == 0) record_device_error(ENGPT_ERR_ARG, 43);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      float x = 0.f;
      if (live)
        x = Code::decode(reinterpret_cast<const uint8_t*>(a.c.codes[part])[a.c.code_at(part, slot, h) + e]) *
            a.c.scales[part][a.c.scale_at(part, slot, h)];
      reinterpret_cast<T*>(a.out[part])[i] = from_f32<T>(x);
    }
  }
}

// Checks of a cache's description, common to all entry points; fills `c`.
int fill_q8_cache(const char* what, Q8Cache& c, void* k_pages, void* v_pages, float* k_scales, float* v_scales,
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

template <typename T, typename Code, bool APPEND, int LPR, int W>
int launch_store_runs(const StoreArgs& a, int window, const char* what, cudaStream_t st) {
  const int64_t items = (a.n + window - 1) / window * (APPEND ? 3 : 2) * a.c.H, blocks = W > 1 ? items : (items + 3) / 4;
  ENGPT_REQUIRE(blocks <= 0x7fffffffLL, ENGPT_ERR_SHAPE, "%s: too large", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(W > 4 ? 32 * W : 128);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = APPEND ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, store_runs_kernel<T, Code, APPEND, LPR, W>, a, window);
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

template <typename T, typename Code, bool APPEND, int LPR>
int launch_store_team(const StoreArgs& a, const char* what, cudaStream_t st) {
  const int rows = kSteps * 32 / LPR;                  // that a warp holds
  // a token per window while that makes no more warps than run at once some times over
  const bool single = a.n * (APPEND ? 3 : 2) * a.c.H <= (int64_t)num_sms() * 128;
  if (single) return launch_store_runs<T, Code, APPEND, LPR, 1>(a, 1, what, st);
  if (a.c.block <= rows) return launch_store_runs<T, Code, APPEND, LPR, 1>(a, a.c.block, what, st);
  if (a.c.block <= 4 * rows) return launch_store_runs<T, Code, APPEND, LPR, 4>(a, a.c.block, what, st);
  return launch_store_runs<T, Code, APPEND, LPR, 8>(a, a.c.block, what, st);
}

template <typename T, typename Code, bool APPEND>
int launch_store_code(const StoreArgs& a, bool vec, const char* what, cudaStream_t st) {
  const int Dh = a.c.Dh;
  if (!vec) return launch_store_generic<T, Code, APPEND>(a, what, st);
  if (Dh <= 8) return launch_store_team<T, Code, APPEND, 1>(a, what, st);
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

template <typename T>
int launch_read(const ReadArgs& a, int code, cudaStream_t st) {
  const int64_t want = (a.n * a.c.H * a.c.Dh + 255) / 256, cap = (int64_t)num_sms() * 8;
  const unsigned blocks = (unsigned)(want < cap ? want : cap);
  if (code == ENGPT_CODE_INT8) read_generic_kernel<T, Int8Code><<<blocks, 256, 0, st>>>(a);
  else read_generic_kernel<T, E4m3Code><<<blocks, 256, 0, st>>>(a);
  return check_launch("read_kv_pages_q8");
}

}  // namespace paged
}  // namespace engpt

using namespace engpt;
using namespace engpt::paged;

extern "C" int engpt_write_kv_pages_q8(const void* k, const void* v, const int64_t* kv_strides, int dtype, int64_t n,
                                       int H, int Dh, const int* slots, void* k_pages, void* v_pages, float* k_scales,
                                       float* v_scales, const int64_t* page_strides, const int64_t* scale_strides,
                                       int code, int num_pages, int page_size, int block, void* stream) {
  clear_error();
  ENGPT_REQUIRE(n >= 0 && n <= 0x7fffffffLL, ENGPT_ERR_SHAPE, "write_kv_pages_q8: n=%lld", (long long)n);
  ENGPT_REQUIRE(dtype == ENGPT_BF16 || dtype == ENGPT_F32, ENGPT_ERR_DTYPE, "write_kv_pages_q8: dtype %d", dtype);
  StoreArgs a = {};
  if (int rc = fill_q8_cache("write_kv_pages_q8", a.c, k_pages, v_pages, k_scales, v_scales, page_strides,
                             scale_strides, code, H, Dh, num_pages, page_size, block))
    return rc;
  if (n == 0) return ENGPT_OK;
  ENGPT_REQUIRE(k && v && kv_strides && slots, ENGPT_ERR_ARG, "write_kv_pages_q8: null pointer");
  a.slots = slots;
  a.n = n;
  a.x[0] = k;
  a.x[1] = v;
  for (int i = 0; i < 2; ++i) {
    a.row[i] = kv_strides[2 * i];
    a.head[i] = kv_strides[2 * i + 1];
  }
  return dtype == ENGPT_BF16 ? launch_store<__nv_bfloat16, false>(a, code, true, "write_kv_pages_q8", as_stream(stream))
                             : launch_store<float, false>(a, code, true, "write_kv_pages_q8", as_stream(stream));
}

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
                             : launch_store<float, true>(a, code, vec, "qkv_append_q8", as_stream(stream));
}

extern "C" int engpt_read_kv_pages_q8(const int* slots, int64_t n, const void* k_pages, const void* v_pages,
                                      const float* k_scales, const float* v_scales, const int64_t* page_strides,
                                      const int64_t* scale_strides, int code, int H, int Dh, int num_pages,
                                      int page_size, int block, void* k_out, void* v_out, int dtype, void* stream) {
  clear_error();
  ENGPT_REQUIRE(n >= 0 && n <= 0x7fffffffLL, ENGPT_ERR_SHAPE, "read_kv_pages_q8: n=%lld", (long long)n);
  ENGPT_REQUIRE(dtype == ENGPT_BF16 || dtype == ENGPT_F32, ENGPT_ERR_DTYPE, "read_kv_pages_q8: dtype %d", dtype);
  ReadArgs a = {};
  if (int rc = fill_q8_cache("read_kv_pages_q8", a.c, const_cast<void*>(k_pages), const_cast<void*>(v_pages),
                             const_cast<float*>(k_scales), const_cast<float*>(v_scales), page_strides, scale_strides,
                             code, H, Dh, num_pages, page_size, block))
    return rc;
  if (n == 0) return ENGPT_OK;
  ENGPT_REQUIRE(slots && k_out && v_out, ENGPT_ERR_ARG, "read_kv_pages_q8: null pointer");
  a.slots = slots;
  a.n = n;
  a.out[0] = k_out;
  a.out[1] = v_out;
  return dtype == ENGPT_BF16 ? launch_read<__nv_bfloat16>(a, code, as_stream(stream))
                             : launch_read<float>(a, code, as_stream(stream));
}
