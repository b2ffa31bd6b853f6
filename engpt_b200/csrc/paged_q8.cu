// write_kv_pages_q8 and read_kv_pages_q8: finished rows quantised into the paged cache, and its numbers read back.
#include "paged_q8_store.cuh"

namespace engpt {
namespace paged {

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

// Head_dim a multiple of N = 8 or 16, aligned.  A thread owns N codes of a row (k and v) and walks over tokens; a CTA
// takes several tokens beside each other where a row has fewer pieces than it has threads.  The slot of the next token
// is on its way while this one's numbers are.  16 x 2048 tokens, half of them with a slot, 16 heads of 64, int8 to bf16
// (168 MB move): 32.4 us = 5.2 TB/s with the registers held to 6 CTAs per SM; 33.9 with 5, 36.7 with 7, 39 with 3; 8 codes
// a thread 47.
constexpr int kReadCtas = 6;

template <typename T>
__device__ __forceinline__ void store_row(T* p, const float* x, int n) {
#pragma unroll
  for (int i = 0; i < n; i += 32 / (int)sizeof(T)) {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      w[k] = sizeof(T) == 2 ? pack_bf16(x[i + 2 * k], x[i + 2 * k + 1]) : __float_as_uint(x[i + k]);
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p + i), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  }
}

template <typename T, typename Code, int N>
__global__ void __launch_bounds__(256, kReadCtas) read_vec_kernel(ReadArgs a, int pieces) {
  const int row = a.c.H * pieces, tokens = row >= (int)blockDim.x ? 1 : blockDim.x / row;
  const int idx = blockIdx.y * blockDim.x + threadIdx.x, sub = tokens > 1 ? idx / row : 0, at = idx - sub * row;
  if (sub >= tokens || at >= row) return;
  const int h = at / pieces, e = (at - h * pieces) * N;
  const char* codes[2];
  const float* scales[2];
  T* out[2];
  const int64_t step = (int64_t)gridDim.x * tokens, n0 = (int64_t)blockIdx.x * tokens + sub, width = (int64_t)row * N;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    codes[p] = (const char*)a.c.codes[p] + h * a.c.cs[p][1] + e;
    scales[p] = a.c.scales[p] + h * a.c.ss[p][1];
    out[p] = reinterpret_cast<T*>(a.out[p]) + n0 * width + (int64_t)at * N;
  }
  int next = n0 < a.n ? a.slots[n0] : -1;
  for (int64_t n = n0; n < a.n; n += step) {
    int slot = next;
    if (n + step < a.n) next = a.slots[n + step];
    if ((uint32_t)slot >= (uint64_t)a.c.n_slots) {
      if (slot != -1 && at == 0) record_device_error(ENGPT_ERR_ARG, 43);
      slot = -1;
    }
    uint32_t w[2][N / 4];
    float scale[2];
    const int page = a.c.page_of(slot), off = slot - page * a.c.ps, block = a.c.block_of(off);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) w[p][i] = 0u;
      scale[p] = 0.f;
      if (slot >= 0) {
        const char* c = codes[p] + page * a.c.cs[p][0] + off * a.c.cs[p][2];
        if constexpr (N == 16) {
          const uint4 r = ld_once(c);
          w[p][0] = r.x; w[p][1] = r.y; w[p][2] = r.z; w[p][3] = r.w;
        } else {
          asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[p][0]), "=r"(w[p][1]) : "l"(c));
        }
        scale[p] = scales[p][page * a.c.ss[p][0] + block * a.c.ss[p][2]];
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      float x[N];
#pragma unroll
      for (int i = 0; i < N / 4; ++i) Code::decode4(w[p][i], x + 4 * i);
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] *= scale[p];   // (both are 0 without a slot)
      if constexpr (N == 16) {
        store_row<T>(out[p], x, N);
      } else if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(out[p]) = pack8(x);
      } else {
        *reinterpret_cast<float4*>(out[p]) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(out[p] + 4) = make_float4(x[4], x[5], x[6], x[7]);
      }
      out[p] += step * width;
    }
  }
}

template <typename T, typename Code>
int launch_read_code(const ReadArgs& a, cudaStream_t st) {
  bool vec = a.c.Dh % 8 == 0, wide = a.c.Dh % 16 == 0;
  for (int p = 0; p < 2; ++p) {
    vec = vec && aligned(a.c.codes[p], 8) && aligned(a.out[p], 16);
    wide = wide && aligned(a.c.codes[p], 16) && aligned(a.out[p], 32);
    for (int i = 0; i < 3; ++i) {
      vec = vec && a.c.cs[p][i] % 8 == 0;
      wide = wide && a.c.cs[p][i] % 16 == 0;
    }
  }
  const int64_t most = (int64_t)num_sms() * kReadCtas;
  if (!vec) {
    const int64_t want = (a.n * a.c.H * a.c.Dh + 255) / 256;
    read_generic_kernel<T, Code><<<(unsigned)(want < most ? want : most), 256, 0, st>>>(a);
    return check_launch("read_kv_pages_q8");
  }
  const int pieces = a.c.Dh / (wide ? 16 : 8), row = a.c.H * pieces, y = (row + 255) / 256;
  const int tokens = row >= 256 ? 1 : 256 / row;
  ENGPT_REQUIRE(y <= 65535, ENGPT_ERR_SHAPE, "read_kv_pages_q8: H=%d Dh=%d", a.c.H, a.c.Dh);
  const int64_t groups = (a.n + tokens - 1) / tokens, cap = most / y > 0 ? most / y : 1;
  const dim3 grid((unsigned)(groups < cap ? groups : cap), (unsigned)y);
  if (wide) read_vec_kernel<T, Code, 16><<<grid, 256, 0, st>>>(a, pieces);
  else read_vec_kernel<T, Code, 8><<<grid, 256, 0, st>>>(a, pieces);
  return check_launch("read_kv_pages_q8");
}

template <typename T>
int launch_read(const ReadArgs& a, int code, cudaStream_t st) {
  return code == ENGPT_CODE_INT8 ? launch_read_code<T, Int8Code>(a, st) : launch_read_code<T, E4m3Code>(a, st);
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
