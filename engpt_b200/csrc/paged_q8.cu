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

template <typename T, bool APPEND>
int launch_store(const StoreArgs& a, int code, const char* what, cudaStream_t st) {
  return code == ENGPT_CODE_INT8 ? launch_store_generic<T, Int8Code, APPEND>(a, what, st)
                                 : launch_store_generic<T, E4m3Code, APPEND>(a, what, st);
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
  return dtype == ENGPT_BF16 ? launch_store<__nv_bfloat16, false>(a, code, "write_kv_pages_q8", as_stream(stream))
                             : launch_store<float, false>(a, code, "write_kv_pages_q8", as_stream(stream));
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
  return dtype == ENGPT_BF16 ? launch_store<__nv_bfloat16, true>(a, code, "qkv_append_q8", as_stream(stream))
                             : launch_store<float, true>(a, code, "qkv_append_q8", as_stream(stream));
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
