// Attention of one new token per request over a paged key-value cache.
//
//   o[b, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),  m = max_j scale q.k_j
//
// Every key and value is read once and used for 4 Dh flops, so the operator
// is bound by HBM.  The keys of a row are split over CTAs; each keeps a
// running maximum m, the sum l of the p_j and the unnormalised o, and two
// such parts join as
//   m = max(m1, m2),  l = l1 e^(m1-m) + l2 e^(m2-m),  o likewise.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace engpt {
namespace paged {

struct AttnArgs {
  const void* q;
  int64_t q_row, q_head;
  const void* k_pages;
  const void* v_pages;
  int64_t ks[3], vs[3];   // element strides: page, head, slot
  int B, H, G, Dh;        // G = H / Hkv query heads share a kv head
  int P, ps;
  const int* table;
  int64_t table_stride;
  int W;
  const int* lengths;
  float scale_log2;       // scale * log2(e): the exponentials are taken to the base 2
  void* o;
  float* work;            // parts [B * H][splits][Dh + 2]: o, m, l
  int splits;
};

// Usable length of row b: negative counts as 0, more than the table row holds is recorded and cut.
__device__ __forceinline__ int row_length(const AttnArgs& a, int b) {
  const int len = a.lengths[b];
  if (len <= 0) return 0;
  const int64_t most = (int64_t)a.W * a.ps;
  if (len <= most) return len;
  record_device_error(ENGPT_ERR_ARG, 44);
  return (int)most;
}

template <typename T>
__device__ __forceinline__ void store1(T* p, float v);
template <>
__device__ __forceinline__ void store1<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void store1<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* x) {
  if constexpr (VEC == 8) {
    unpack8(ld_stream(p), x);
  } else if constexpr (VEC == 4) {
    const uint4 r = ld_stream(p);
    x[0] = __uint_as_float(r.x);
    x[1] = __uint_as_float(r.y);
    x[2] = __uint_as_float(r.z);
    x[3] = __uint_as_float(r.w);
  } else if constexpr (sizeof(T) == 2) {
    x[0] = __bfloat162float(*p);
  } else {
    x[0] = *p;
  }
}

constexpr int kThreads = 128;
constexpr int kGroups = kThreads / 8;

// m2 - m for the joining weights; a part without keys has m = -inf and weighs nothing.
__device__ __forceinline__ float join_weight(float m_part, float m) {
  return m_part == -INFINITY ? 0.f : sm100::ex2_approx(m_part - m);
}

// CUDA-core kernel: any head_dim up to 256, fp32 or bf16, any strides.  Eight lanes share a key (each owns NC
// pieces of VEC elements, VEC = 16 bytes where the addresses allow it); a lane group keeps its own m, l and o
// over every kGroups-th key of the CTA's range, and the groups join through shared memory at the end.
template <typename T, int VEC, int NC>
__global__ void __launch_bounds__(kThreads) decode_simt_kernel(AttnArgs a) {
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int sub = threadIdx.x & 7, grp = threadIdx.x >> 3;
  const int len = row_length(a, b);
  // this CTA's keys [j0, j1)
  const int64_t chunk = ((int64_t)len + a.splits - 1) / a.splits;
  const int j0 = (int)min((int64_t)len, split * chunk), j1 = (int)min((int64_t)len, j0 + chunk);

  const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_row + h * a.q_head;
  const int hk = h / a.G;
  const T* kp = reinterpret_cast<const T*>(a.k_pages) + hk * a.ks[1];
  const T* vp = reinterpret_cast<const T*>(a.v_pages) + hk * a.vs[1];
  const int* row = a.table + b * a.table_stride;

  float qf[NC * VEC], o[NC * VEC];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = (c * 8 + sub) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) qf[c * VEC + i] = o[c * VEC + i] = 0.f;
    if (e < a.Dh) {
      load_vec<T, VEC>(q + e, qf + c * VEC);
#pragma unroll
      for (int i = 0; i < VEC; ++i) qf[c * VEC + i] *= a.scale_log2;
    }
  }
  for (int jb = j0; jb < j1; jb += kGroups) {   // CTA-uniform trip count: the shuffles need whole warps
    const int j = jb + grp;
    bool live = j < j1;
    int page = 0, off = 0;
    if (live) {
      const int pj = j / a.ps;
      off = j - pj * a.ps;
      page = row[pj];
      if (page < 0 || page >= a.P) {
        record_device_error(ENGPT_ERR_ARG, 44);
        live = false;
      }
    }
    float kf[NC * VEC], vf[NC * VEC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int e = (c * 8 + sub) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) kf[c * VEC + i] = vf[c * VEC + i] = 0.f;
      if (live && e < a.Dh) {
        load_vec<T, VEC>(kp + page * a.ks[0] + off * a.ks[2] + e, kf + c * VEC);
        load_vec<T, VEC>(vp + page * a.vs[0] + off * a.vs[2] + e, vf + c * VEC);
      }
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NC * VEC; ++i) s = fmaf(qf[i], kf[i], s);
#pragma unroll
    for (int w = 4; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    if (live) {
      const float mn = fmaxf(m, s);
      const float ms = mn == -INFINITY ? 0.f : mn;
      const float corr = sm100::ex2_approx(m - ms), p = sm100::ex2_approx(s - ms);
      m = mn;
      l = fmaf(l, corr, p);
#pragma unroll
      for (int i = 0; i < NC * VEC; ++i) o[i] = fmaf(o[i], corr, p * vf[i]);
    }
  }
  // join the CTA's lane groups
  extern __shared__ float sm[];
  float* s_o = sm;                       // [kGroups][Dh]
  float* s_m = sm + kGroups * a.Dh;      // [kGroups]
  float* s_l = s_m + kGroups;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = (c * 8 + sub) * VEC;
    if (e < a.Dh) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) s_o[grp * a.Dh + e + i] = o[c * VEC + i];
    }
  }
  if (sub == 0) {
    s_m[grp] = m;
    s_l[grp] = l;
  }
  __syncthreads();
  float mx = -INFINITY;
  for (int g = 0; g < kGroups; ++g) mx = fmaxf(mx, s_m[g]);
  float lx = 0.f;
  for (int g = 0; g < kGroups; ++g) lx += s_l[g] * join_weight(s_m[g], mx);
  const int64_t bh = (int64_t)b * a.H + h;
  float* part = a.work + (bh * a.splits + split) * (a.Dh + 2);
  for (int e = threadIdx.x; e < a.Dh; e += kThreads) {
    float ox = 0.f;
    for (int g = 0; g < kGroups; ++g) ox = fmaf(s_o[g * a.Dh + e], join_weight(s_m[g], mx), ox);
    if (a.splits == 1)
      store1(reinterpret_cast<T*>(a.o) + bh * a.Dh + e, len == 0 || lx == 0.f ? 0.f : ox / lx);
    else
      part[e] = ox;
  }
  if (a.splits > 1 && threadIdx.x == 0) {
    part[a.Dh] = mx;
    part[a.Dh + 1] = lx;
  }
}

// Joins the parts of one (row, head) per CTA.
template <typename T>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(AttnArgs a) {
  const int64_t bh = blockIdx.x;
  const float* part = a.work + bh * a.splits * (a.Dh + 2);
  const int step = a.Dh + 2;
  float mx = -INFINITY;
  for (int s = 0; s < a.splits; ++s) mx = fmaxf(mx, part[s * step + a.Dh]);
  float lx = 0.f;
  for (int s = 0; s < a.splits; ++s) lx += part[s * step + a.Dh + 1] * join_weight(part[s * step + a.Dh], mx);
  for (int e = threadIdx.x; e < a.Dh; e += kThreads) {
    float ox = 0.f;
    for (int s = 0; s < a.splits; ++s) ox = fmaf(part[s * step + e], join_weight(part[s * step + a.Dh], mx), ox);
    store1(reinterpret_cast<T*>(a.o) + bh * a.Dh + e, lx == 0.f ? 0.f : ox / lx);
  }
}

// Key splits of a launch: about four CTAs per SM, at least 128 keys each at the longest length the table holds.
inline int simt_splits(int B, int H, int64_t most) {
  const int64_t rows = (int64_t)B * H;
  int64_t s = rows > 0 ? (4 * 148 + rows - 1) / rows : 1;
  const int64_t by_len = (most + 127) / 128;
  if (s > by_len) s = by_len;
  if (s > 256) s = 256;
  return s < 1 ? 1 : (int)s;
}

template <typename T, int VEC, int NC>
int launch_simt(const AttnArgs& a, cudaStream_t st) {
  const size_t smem = sizeof(float) * (size_t)(kGroups * (a.Dh + 2));
  decode_simt_kernel<T, VEC, NC><<<dim3(a.splits, a.H, a.B), kThreads, smem, st>>>(a);
  int rc = check_launch("paged_attention");
  if (rc || a.splits == 1) return rc;
  decode_join_kernel<T><<<(unsigned)((int64_t)a.B * a.H), kThreads, 0, st>>>(a);
  return check_launch("paged_attention (join)");
}

template <typename T>
int dispatch_simt(const AttnArgs& a, bool vec, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const int nc = vec ? (a.Dh + 8 * V - 1) / (8 * V) : (a.Dh + 7) / 8;
  if (vec) {
    if (nc <= 1) return launch_simt<T, V, 1>(a, st);
    if (nc <= 2) return launch_simt<T, V, 2>(a, st);
    if (nc <= 4) return launch_simt<T, V, 4>(a, st);
    if (sizeof(T) == 4) return launch_simt<T, V, 8>(a, st);
  }
  if (nc <= 8) return launch_simt<T, 1, 8>(a, st);
  return launch_simt<T, 1, 32>(a, st);
}

}  // namespace paged
}  // namespace engpt

using namespace engpt;
using namespace engpt::paged;

extern "C" int64_t engpt_paged_attention_floats(int dtype, int B, int H, int Hkv, int Dh, int table_width,
                                                int page_size) {
  (void)dtype;
  (void)Hkv;
  if (B <= 0 || H <= 0 || Dh <= 0 || table_width < 0 || page_size <= 0) return 0;
  const int splits = simt_splits(B, H, (int64_t)table_width * page_size);
  return splits > 1 ? (int64_t)B * H * splits * (Dh + 2) : 0;
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
  ENGPT_REQUIRE(table_width >= 0 && table_stride >= table_width && (int64_t)table_width * page_size <= 0x7fffffffLL,
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
  ENGPT_REQUIRE(a.splits == 1 || workspace, ENGPT_ERR_ARG, "paged_attention: null workspace");
  bool vec = aligned(q, 16) && aligned(k_pages, 16) && aligned(v_pages, 16) && Dh * esz % 16 == 0 &&
             a.q_row * esz % 16 == 0 && a.q_head * esz % 16 == 0;
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = page_strides[i];
    a.vs[i] = page_strides[3 + i];
    vec = vec && a.ks[i] * esz % 16 == 0 && a.vs[i] * esz % 16 == 0;
  }
  cudaStream_t st = as_stream(stream);
  return dtype == ENGPT_BF16 ? dispatch_simt<__nv_bfloat16>(a, vec, st) : dispatch_simt<float>(a, vec, st);
}
