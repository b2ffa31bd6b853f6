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

#include <cudaTypedefs.h>
#include <math.h>

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
  // (coherent loads: the kernel may have been started while an earlier one was still writing the pages)
  if constexpr (VEC == 8) {
    unpack8(ld_once(p), x);
  } else if constexpr (VEC == 4) {
    const uint4 r = ld_once(p);
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
constexpr int kSimtCluster = 8;
constexpr int64_t kMostKeys = 0x7fffffff - 4096;   // of a row: key indices are ints and run a tile or two past it

// m2 - m for the joining weights; a part without keys has m = -inf and weighs nothing.
__device__ __forceinline__ float join_weight(float m_part, float m) {
  return m_part == -INFINITY ? 0.f : sm100::ex2_approx(m_part - m);
}

// The splits' parts ([splits][Dh + 2]: o, m, l) of row and head bh, joined by one CTA into the output.
template <typename T>
__device__ __forceinline__ void join_parts(const AttnArgs& a, const float* part, int64_t bh) {
  const int step = a.Dh + 2;
  float mx = -INFINITY;
  for (int s = 0; s < a.splits; ++s) mx = fmaxf(mx, part[s * step + a.Dh]);
  float lx = 0.f;
  for (int s = 0; s < a.splits; ++s) lx = fmaf(part[s * step + a.Dh + 1], join_weight(part[s * step + a.Dh], mx), lx);
  for (int e = threadIdx.x; e < a.Dh; e += kThreads) {
    float ox = 0.f;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) ox = fmaf(part[s * step + e], join_weight(part[s * step + a.Dh], mx), ox);
    store1(reinterpret_cast<T*>(a.o) + bh * a.Dh + e, lx == 0.f ? 0.f : ox / lx);
  }
}

// CUDA-core kernel: any head_dim up to 256, fp32 or bf16, any strides.  Eight lanes share a key (each owns NC pieces
// of VEC elements, VEC = 16 bytes where the addresses allow it); a lane group keeps its own m, l and o of HG query
// heads of one kv head over every kGroups-th key of the CTA's range, U keys in flight at a time, and the groups join
// through shared memory.  The `splits` CTAs of a row and its heads are a cluster while there are at most 8 and join in
// the shared memory of the first; otherwise they leave parts in the workspace for decode_join_kernel.
template <typename T, int VEC, int NC, int U, int HG>
__global__ void __launch_bounds__(kThreads) decode_simt_kernel(AttnArgs a) {
  const int split = blockIdx.x, h0 = blockIdx.y * HG, b = blockIdx.z;
  const int sub = threadIdx.x & 7, grp = threadIdx.x >> 3;
  const bool cluster = a.splits > 1 && a.splits <= kSimtCluster;
  if (cluster) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");   // nothing of an earlier kernel has been touched before
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int len = row_length(a, b);
  // this CTA's keys [j0, j1)
  const int64_t chunk = ((int64_t)len + a.splits - 1) / a.splits;
  const int j0 = (int)min((int64_t)len, split * chunk), j1 = (int)min((int64_t)len, j0 + chunk);

  const int hk = h0 / a.G;
  const T* kp = reinterpret_cast<const T*>(a.k_pages) + hk * a.ks[1];
  const T* vp = reinterpret_cast<const T*>(a.v_pages) + hk * a.vs[1];
  const int* row = a.table + b * a.table_stride;

  float qf[HG][NC * VEC], o[HG][NC * VEC], m[HG], l[HG];
#pragma unroll
  for (int g = 0; g < HG; ++g) {
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_row + (h0 + g) * a.q_head;
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int e = (c * 8 + sub) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) qf[g][c * VEC + i] = o[g][c * VEC + i] = 0.f;
      if (e < a.Dh) {
        load_vec<T, VEC>(q + e, qf[g] + c * VEC);
#pragma unroll
        for (int i = 0; i < VEC; ++i) qf[g][c * VEC + i] *= a.scale_log2;
      }
    }
  }
  for (int jb = j0; jb < j1; jb += U * kGroups) {   // CTA-uniform trip count: the shuffles need whole warps
    int page[U], off[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = jb + u * kGroups + grp;
      const int pj = j / a.ps;
      off[u] = j - pj * a.ps;
      page[u] = j < j1 ? row[pj] : -1;
      if (j >= j1) off[u] = -1;                     // no key, as opposed to a bad page
    }
    float kf[U][NC * VEC], vf[U][NC * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool live = page[u] >= 0 && page[u] < a.P;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int e = (c * 8 + sub) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) kf[u][c * VEC + i] = vf[u][c * VEC + i] = 0.f;
        if (live && e < a.Dh) {
          load_vec<T, VEC>(kp + page[u] * a.ks[0] + off[u] * a.ks[2] + e, kf[u] + c * VEC);
          load_vec<T, VEC>(vp + page[u] * a.vs[0] + off[u] * a.vs[2] + e, vf[u] + c * VEC);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float s[HG];
#pragma unroll
      for (int g = 0; g < HG; ++g) {
        s[g] = 0.f;
#pragma unroll
        for (int i = 0; i < NC * VEC; ++i) s[g] = fmaf(qf[g][i], kf[u][i], s[g]);
      }
#pragma unroll
      for (int w = 4; w > 0; w >>= 1)
#pragma unroll
        for (int g = 0; g < HG; ++g) s[g] += __shfl_xor_sync(0xffffffffu, s[g], w);
      if (page[u] >= 0 && page[u] < a.P) {
#pragma unroll
        for (int g = 0; g < HG; ++g) {
          const float mn = fmaxf(m[g], s[g]);
          const float ms = mn == -INFINITY ? 0.f : mn;
          const float corr = sm100::ex2_approx(m[g] - ms), p = sm100::ex2_approx(s[g] - ms);
          m[g] = mn;
          l[g] = fmaf(l[g], corr, p);
#pragma unroll
          for (int i = 0; i < NC * VEC; ++i) o[g][i] = fmaf(o[g][i], corr, p * vf[u][i]);
        }
      } else if (off[u] >= 0) {
        record_device_error(ENGPT_ERR_ARG, 44);
      }
    }
  }
  // join the CTA's lane groups, head by head
  extern __shared__ float sm[];
  float* s_o = sm;                           // [kGroups][Dh]
  float* s_m = sm + kGroups * a.Dh;          // [HG][kGroups]
  float* s_l = s_m + HG * kGroups;
  float* s_cta = s_l + HG * kGroups;         // cluster: [HG][splits][Dh + 2] (first CTA)
  if (sub == 0) {
#pragma unroll
    for (int g = 0; g < HG; ++g) {
      s_m[g * kGroups + grp] = m[g];
      s_l[g * kGroups + grp] = l[g];
    }
  }
  if (cluster) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // every CTA has started
#pragma unroll
  for (int g = 0; g < HG; ++g) {
    if (g > 0) __syncthreads();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int e = (c * 8 + sub) * VEC;
      if (e < a.Dh) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) s_o[grp * a.Dh + e + i] = o[g][c * VEC + i];
      }
    }
    __syncthreads();
    float wgt[kGroups], mx = -INFINITY, lx = 0.f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) mx = fmaxf(mx, s_m[g * kGroups + k]);
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      wgt[k] = join_weight(s_m[g * kGroups + k], mx);
      lx = fmaf(s_l[g * kGroups + k], wgt[k], lx);
    }
    const int64_t bh = (int64_t)b * a.H + h0 + g;
    float* part = a.work + (bh * a.splits + split) * (a.Dh + 2);
    if (cluster)
      asm("mapa.u64 %0, %1, %2;" : "=l"(part) : "l"(s_cta + (g * a.splits + split) * (a.Dh + 2)), "r"(0));
    for (int e = threadIdx.x; e < a.Dh; e += kThreads) {
      float ox = 0.f;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) ox = fmaf(s_o[k * a.Dh + e], wgt[k], ox);
      if (a.splits == 1)
        store1(reinterpret_cast<T*>(a.o) + bh * a.Dh + e, lx == 0.f ? 0.f : ox / lx);
      else
        part[e] = ox;
    }
    if (a.splits > 1 && threadIdx.x == 0) {
      part[a.Dh] = mx;
      part[a.Dh + 1] = lx;
    }
  }
  if (cluster) {
    sm100::cluster_sync_all();
    if (split == 0)
      for (int g = 0; g < HG; ++g)
        join_parts<T>(a, s_cta + g * a.splits * (a.Dh + 2), (int64_t)b * a.H + h0 + g);
  }
}

// Joins the parts of one (row, head) per CTA.
template <typename T>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(AttnArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  join_parts<T>(a, a.work + (int64_t)blockIdx.x * a.splits * (a.Dh + 2), blockIdx.x);
}

// Key splits of a launch: about four CTAs per SM if every query head had one of its own (heads that share a reading of
// their kv head's keys leave a half or a quarter as many), at least 64 keys each at the longest length the table holds.
// One cluster rather than a second launch where that leaves a CTA no more than 256 keys.
inline int simt_splits(int B, int H, int64_t most) {
  const int64_t rows = (int64_t)B * H;
  int64_t s = rows > 0 ? (4 * (int64_t)num_sms() + rows - 1) / rows : 1;
  const int64_t by_len = (most + 63) / 64;
  if (s > by_len) s = by_len;
  if (s > kSimtCluster && most <= 256 * kSimtCluster) s = kSimtCluster;
  if (s > 256) s = 256;
  return s < 1 ? 1 : (int)s;
}

template <typename T, int VEC, int NC, int U, int HG>
int launch_simt(const AttnArgs& a, cudaStream_t st) {
  const bool cluster = a.splits > 1 && a.splits <= kSimtCluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.splits, a.H / HG, a.B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes =
      sizeof(float) * (size_t)(kGroups * (a.Dh + 2 * HG) + (cluster ? HG * a.splits * (a.Dh + 2) : 0));
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, decode_simt_kernel<T, VEC, NC, U, HG>, a);
  if (e == cudaSuccess && a.splits > kSimtCluster) {
    cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.H));
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, decode_join_kernel<T>, a);
  }
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "paged_attention: %s", cudaGetErrorString(e));
  return check_launch("paged_attention");
}

// Query heads that share a kv head and one reading of its keys: 4, 2 or 1 (8 fp32 rows of 1024 tokens, 32 heads on 4
// of 128: 28 us with four heads per reading, 41 with one).
template <typename T, int VEC, int NC, int U>
int launch_simt_heads(const AttnArgs& a, cudaStream_t st) {
  if (a.G % 4 == 0) return launch_simt<T, VEC, NC, U, 4>(a, st);
  if (a.G % 2 == 0) return launch_simt<T, VEC, NC, U, 2>(a, st);
  return launch_simt<T, VEC, NC, U, 1>(a, st);
}

template <typename T>
int dispatch_simt(const AttnArgs& a, bool vec, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const int nc = vec ? (a.Dh + 8 * V - 1) / (8 * V) : (a.Dh + 7) / 8;
  if (vec && sizeof(T) == 4) {
    if (nc <= 1) return launch_simt_heads<T, V, 1, 4>(a, st);
    if (nc <= 2) return launch_simt_heads<T, V, 2, 4>(a, st);
    if (nc <= 4) return launch_simt_heads<T, V, 4, 2>(a, st);
    return launch_simt<T, V, 8, 1, 1>(a, st);
  }
  if (vec) {   // bf16 comes here with a head_dim above 128, or pages of an odd size
    if (nc <= 2) return launch_simt<T, V, 2, 2, 1>(a, st);
    return launch_simt<T, V, 4, 1, 1>(a, st);
  }
  if (nc <= 8) return launch_simt<T, 1, 8, 2, 1>(a, st);
  return launch_simt<T, 1, 32, 1, 1>(a, st);
}

// ------------------------------------------------------------------ tensor-core kernel (bf16, head_dim up to 128)
//
// Built for a width D of 64 or 128; a smaller head_dim is padded with zeros by TMA, in shared memory only.
//
// A tile is KT keys of one kv head, kTileBytes of keys and as many of values.  The tiles of all (row, kv head) pairs
// form one list, cut into contiguous ranges of equal cost, one per warp ("worker") of a persistent grid, so the load is
// even whatever the lengths.  A warp fetches its own tiles, one at a time, into its own 16 KB of shared memory:
// TMA boxes of R rows (R divides the page size) at the page that the block table names, 128-byte swizzled, completing
// on the warp's mbarrier; no warp waits for another one until the end.
//
// Per tile, with up to 8 query heads of the kv head as rows 0-7 of the 16-row mma.sync operand:
//   S = Q K^T (rows 8-15 are zero), p = 2^(S scale - m), and O += P V with P's bf16 value in rows 0-7 and the
//   remainder p - bf16(p), again as bf16, in rows 8-15: adding the two halves of O at the end gives the product
//   with weights of 16 mantissa bits for the price of the otherwise idle half of the operand.
// The products do not bound anything here (64 mma.sync of 16x8x16 per 16 KB), which is why this is not built on
// tcgen05: its 128-row operand would be 1/128 to 1/16 full and P would take a trip through TMEM.
//
// A range that begins or ends inside a pair leaves a part (o, m, l) in shared memory.  After a CTA barrier the parts
// of a pair are joined by the warp that holds its first one; a pair that runs over CTAs leaves one part per CTA in
// the workspace, joined by decode_join_list_kernel.
//
// Warps and tiles are what 64 rows of up to 4096 tokens (16 heads of 64) run best with: eight warps, each of which idles
// while its 16 KB fly but has seven others beside it, 87 us; 10 or 12 such warps 90 and 89, six or four with two tiles
// in flight each 101 and 105, eight with two tiles of 8 KB 97.
constexpr int kWarps = 8;
constexpr int kPairWarps = 4;           // of the form with a cluster per pair: two CTAs per SM
constexpr size_t kPairSmem = 80 * 1024;
constexpr int kTileBytes = 8192;        // one of K, V
constexpr int kMaxListRows = 8192;      // of the list form: an int of shared memory each
template <int D>
struct Mma {
  static constexpr int KT = kTileBytes / (2 * D);
  static constexpr int NT = KT / 8;     // 8-key tiles
  static constexpr int KC = KT / 16;    // 16-key steps of P V
  static constexpr int DK = D / 16;     // 16-dim steps of Q K^T
  static constexpr int DN = D / 8;      // 8-dim tiles of O
};

struct MmaArgs {
  const __nv_bfloat16* q;
  int64_t q_row, q_head;
  int dim;                 // head_dim, at most D and a multiple of 8; TMA fills the columns behind it with zeros
  int B, H, G, HQ, QG;     // HQ: (kv head, group of up to 8 query heads) per row; QG: such groups per kv head
  int rows;                // query heads per group, min(G, 8)
  int P, ps, ps_shift;     // ps_shift: log2(page size), or -1
  int R, r_shift;          // R = 2^r_shift keys per box
  const int* table;
  int64_t table_stride;
  int W;
  const int* lengths;
  float scale_log2;        // |scale| log2(e)
  uint32_t q_flip;         // sign bits to flip in q for a negative scale
  __nv_bfloat16* o;
  float* work;             // [CTAs][2][rows][D + 2]
  int tile_units, end_units;   // list form: cost of a tile and of a pair's end
};

// Units of a pair of T tiles.
__device__ __forceinline__ int pair_units(const MmaArgs& a, int T) {
  return T > 0 ? T * a.tile_units + a.end_units : 0;
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
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

// Usable length of row b (a length beyond the table is recorded once, by the kernel's prologue).
__device__ __forceinline__ int clip_length(const MmaArgs& a, int len) {
  return (int)min((int64_t)max(len, 0), (int64_t)a.W * a.ps);
}

// Position in the list of tiles: tile t of T of (row b of length len, head group h of kv head hk), at unit u.
struct Cursor {
  int b, h, t, T, len, hk, u;
};

// A box of the tile to come: its page as the table has it (looked at only when the copy is issued, so that nothing
// waits for the look-up before) and first row in the page, -1 for a box past the length.
struct Box {
  int page, off;
};

template <int D>
struct Worker {
  using C = Mma<D>;
  const MmaArgs& a;
  const CUtensorMap *mk, *mv;
  uint32_t tile;            // this warp's tile in shared memory: keys, then values
  uint32_t bar;             // its mbarrier
  int lane;

  __device__ __forceinline__ void enter_row(Cursor& c) const {
    c.len = c.b < a.B ? clip_length(a, a.lengths[c.b]) : 0;
    c.T = (c.len + C::KT - 1) / C::KT;
  }

  __device__ __forceinline__ void advance(Cursor& c) const {
    c.u += a.tile_units;
    if (++c.t < c.T) return;
    c.u += a.end_units;
    c.t = 0;
    ++c.h;
    if (c.h < a.HQ) {
      c.hk = c.h / a.QG;
      return;
    }
    c.h = c.hk = 0;
    do {
      ++c.b;
      enter_row(c);
    } while (c.b < a.B && c.T == 0);
  }

  __device__ __forceinline__ Box find_box(const Cursor& c) const {
    const int key = c.t * C::KT + lane * a.R;
    if (lane * a.R >= C::KT || key >= c.len) return Box{0, -1};
    const int j = a.ps_shift >= 0 ? key >> a.ps_shift : key / a.ps;
    return Box{a.table[c.b * a.table_stride + j], key - j * a.ps};
  }

  // Start the copies of the cursor's tile; returns which of its boxes are copied.
  __device__ __forceinline__ uint32_t issue(const Cursor& c, const Box& x) const {
    const bool here = x.off >= 0 && (unsigned)x.page < (unsigned)a.P;
    const uint32_t mask = __ballot_sync(0xffffffffu, here);
    const uint32_t box = a.R * 128;
    if (lane == 0) sm100::mbar_expect_tx(bar, __popc(mask) * box * (D / 64) * 2);
    __syncwarp();
    if (here) {
      const uint32_t dst = tile + lane * box;
#pragma unroll
      for (int half = 0; half < D / 64; ++half) {
        sm100::tma_load_4d(dst + half * C::KT * 128, mk, half * 64, x.off, c.hk, x.page, bar);
        sm100::tma_load_4d(dst + half * C::KT * 128 + kTileBytes, mv, half * 64, x.off, c.hk, x.page, bar);
      }
    } else if (x.off >= 0) {   // a page outside the pool
      record_device_error(ENGPT_ERR_ARG, 44);
    }
    __syncwarp();
    return mask;
  }

  // A wait ran out: let the copies still in flight land (bounded) before the CTA's shared memory goes away.
  __device__ __forceinline__ void drain(uint32_t phase) const {
    const uint64_t t0 = globaltimer_ns();
    while (!sm100::mbar_try_wait_sleep(bar, phase, 100000u) && globaltimer_ns() - t0 < kWaitLimitNs) {
    }
  }
};

// The running state of one pair: rows 0-7 of S and O in the mma layout (row lane / 4, columns 2 (lane % 4) + {0, 1}
// of each 8-column tile).  m is in units of the raw product q.k.
template <int D>
struct State {
  float o[Mma<D>::DN][4];
  float m, l;
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < Mma<D>::DN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }
};

template <int D>
__device__ __forceinline__ void load_query(const MmaArgs& a, int b, int h, int lane, uint32_t (*qa)[2]) {
  const int g = lane >> 2, t = lane & 3;
  const int head = (h / a.QG) * a.G + (h % a.QG) * 8 + g;
  const bool live = g < a.rows && (h % a.QG) * 8 + g < a.G;
  const __nv_bfloat16* q = a.q + b * a.q_row + head * a.q_head + 2 * t;
#pragma unroll
  for (int k = 0; k < Mma<D>::DK; ++k) {
    qa[k][0] = live && k * 16 < a.dim ? *reinterpret_cast<const uint32_t*>(q + k * 16) ^ a.q_flip : 0u;
    qa[k][1] = live && k * 16 + 8 < a.dim ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8) ^ a.q_flip : 0u;
  }
}

// One tile: scores, softmax step, P V.  WHOLE: all its keys count.  Otherwise `live` keys from the tile's start are
// below the length, and boxes whose bit of `mask` is unset were not copied.
template <int D, bool WHOLE>
__device__ __forceinline__ void tile_step(const MmaArgs& a, uint32_t sk, const uint32_t (*qa)[2], State<D>& st,
                                          int live, uint32_t mask, int lane) {
  using C = Mma<D>;
  const uint32_t sv = sk + kTileBytes;
  const int r8 = lane & 7, q4 = lane >> 3, t = lane & 3;
  if (!WHOLE) {
    // absent values become 0: their weight 0 would not cancel a stale NaN or infinity
    for (int i = lane; i < C::KT * (D / 64) * 8; i += 32) {   // 16-byte pieces: half, key, piece
      const int key = (i >> 3) % C::KT;
      if (key >= live || !((mask >> (key >> a.r_shift)) & 1u))
        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(sv + i * 16), "r"(0u) : "memory");
    }
    __syncwarp();
  }
  float s[C::NT][4];
#pragma unroll
  for (int n = 0; n < C::NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
  for (int kp = 0; kp < C::DK / 2; ++kp) {
    uint32_t b[C::NT][4];
    const int c = kp * 4 + q4;
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
      ldsm4(sk + (c >> 3) * (C::KT * 128) + (n * 8 + r8) * 128 + (((c & 7) ^ r8) << 4), b[n]);
#pragma unroll
    for (int n = 0; n < C::NT; ++n) mma16816(s[n], qa[2 * kp][0], 0u, qa[2 * kp][1], 0u, b[n][0], b[n][1]);
#pragma unroll
    for (int n = 0; n < C::NT; ++n) mma16816(s[n], qa[2 * kp + 1][0], 0u, qa[2 * kp + 1][1], 0u, b[n][2], b[n][3]);
  }
  if (!WHOLE) {
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = n * 8 + 2 * t + i;
        if (key >= live || !((mask >> (key >> a.r_shift)) & 1u)) s[n][i] = -INFINITY;
      }
  }
  float mx = st.m;
#pragma unroll
  for (int n = 0; n < C::NT; ++n) mx = fmaxf(mx, fmaxf(s[n][0], s[n][1]));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const float ms = mx == -INFINITY ? 0.f : mx * a.scale_log2;
  if (__any_sync(0xffffffffu, mx > st.m)) {
    const float corr = st.m == -INFINITY ? 0.f : sm100::ex2_approx(st.m * a.scale_log2 - ms);
#pragma unroll
    for (int i = 0; i < C::DN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) st.o[i][j] *= corr;
    st.l *= corr;
    st.m = mx;
  }
  uint32_t hi[C::KC][2], lo[C::KC][2];
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < C::NT; ++n) {
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
  for (int j = 0; j < C::KC; ++j) {
    const int key = j * 16 + (q4 & 1) * 8 + r8;
    uint32_t b[C::DN / 2][4];
#pragma unroll
    for (int dp = 0; dp < C::DN / 2; ++dp) {
      const int c = 2 * dp + (q4 >> 1);
      ldsm4_t(sv + (c >> 3) * (C::KT * 128) + key * 128 + (((c & 7) ^ r8) << 4), b[dp]);
    }
#pragma unroll
    for (int dp = 0; dp < C::DN / 2; ++dp) {
      mma16816(st.o[2 * dp], hi[j][0], lo[j][0], hi[j][1], lo[j][1], b[dp][0], b[dp][1]);
      mma16816(st.o[2 * dp + 1], hi[j][0], lo[j][0], hi[j][1], lo[j][1], b[dp][2], b[dp][3]);
    }
  }
  if (!WHOLE) sm100::fence_proxy_async_smem();   // the zeros above, before a later copy into this memory
}

// The two halves of the operand added: (sum of bf16(p) v) + (sum of (p - bf16(p)) v).  Where a value is infinite the
// first half is the result; the second one, with weights of either sign or 0, would turn it into NaN.
__device__ __forceinline__ float add_halves(float hi, float lo) { return fabsf(hi) == INFINITY ? hi : hi + lo; }

// The pair's sums of this lane: o (both halves) and l over the row's four lanes; m in base-2 units.
template <int D>
__device__ __forceinline__ void finish_rows(const MmaArgs& a, State<D>& st) {
  st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
  st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
  if (st.m != -INFINITY) st.m *= a.scale_log2;
#pragma unroll
  for (int i = 0; i < Mma<D>::DN; ++i) {
    st.o[i][0] = add_halves(st.o[i][0], st.o[i][2]);
    st.o[i][1] = add_halves(st.o[i][1], st.o[i][3]);
  }
}

template <int D>
__device__ __forceinline__ void store_part(const MmaArgs& a, const State<D>& st, float* part, int lane) {
  const int g = lane >> 2, t = lane & 3;
  if (g >= a.rows) return;
  float* p = part + g * (D + 2);
#pragma unroll
  for (int i = 0; i < Mma<D>::DN; ++i) *reinterpret_cast<float2*>(p + i * 8 + 2 * t) = make_float2(st.o[i][0], st.o[i][1]);
  if (t == 0) *reinterpret_cast<float2*>(p + D) = make_float2(st.m, st.l);
}

template <int D>
__device__ __forceinline__ void store_rows(const MmaArgs& a, const State<D>& st, int b, int h, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const int in = (h % a.QG) * 8 + g;
  if (g >= a.rows || in >= a.G) return;
  __nv_bfloat16* o = a.o + ((int64_t)b * a.H + (h / a.QG) * a.G + in) * a.dim + 2 * t;
  const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
#pragma unroll
  for (int i = 0; i < Mma<D>::DN; ++i)
    if (i * 8 < a.dim) *reinterpret_cast<uint32_t*>(o + i * 8) = sm100::pack_bf16x2(st.o[i][0] * inv, st.o[i][1] * inv);
}

// Joins row r of n <= N parts (part(i): its rows) by one warp: into the output, or as one part at `to`.  Lane i holds
// part i's weight, and all loads are independent.
template <int D, int N, typename F>
__device__ __forceinline__ void join_row(const MmaArgs& a, int b, int h, int r, int n, F part, float* to, int lane) {
  constexpr int E = D / 32;
  if ((h % a.QG) * 8 + r >= a.G) return;
  float m = -INFINITY, l = 0.f;
  if (lane < n) {
    const float2 ml = *reinterpret_cast<const float2*>(part(lane) + r * (D + 2) + D);
    m = ml.x;
    l = ml.y;
  }
  float mx = m;
#pragma unroll
  for (int k = N / 2; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
  mx = __shfl_sync(0xffffffffu, mx, 0);
  const float w = join_weight(m, mx);
  l *= w;
#pragma unroll
  for (int k = N / 2; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
  l = __shfl_sync(0xffffffffu, l, 0);
  float x[N][E], o[E] = {};
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) x[k][e] = k < n ? part(k)[r * (D + 2) + lane + 32 * e] : 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float wk = __shfl_sync(0xffffffffu, w, k);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(x[k][e], wk, o[e]);
  }
  if (to) {
    to += r * (D + 2);
#pragma unroll
    for (int e = 0; e < E; ++e) to[lane + 32 * e] = o[e];
    if (lane == 0) {
      to[D] = mx;
      to[D + 1] = l;
    }
  } else {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    __nv_bfloat16* dst = a.o + ((int64_t)b * a.H + (h / a.QG) * a.G + (h % a.QG) * 8 + r) * a.dim;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < a.dim) dst[lane + 32 * e] = __float2bfloat16_rn(o[e] * inv);
  }
}

// Floats of shared memory for one part of each warp.
template <int D>
__host__ __device__ constexpr int part_floats(int rows) {
  return rows * (D + 2);
}

// First unit of every row, s_start[0 .. B] (exclusive prefix sums of a row's units times HQ), by a CTA of `threads`
// threads; returns their number.  For up to 32 rows every warp forms the same sums for itself (the warps write the
// same numbers) and keeps row `lane`'s length and first tile in `len` and `start`: no barrier before the first copy.
template <int KT>
__device__ __forceinline__ int list_starts(const MmaArgs& a, int* s_start, int* s_scan, int threads, bool record,
                                           int& len, int& start) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int carry = 0;
  for (int b0 = 0; b0 < a.B; b0 += threads) {
    const int b = b0 + (a.B <= 32 ? lane : tid);
    len = 0;
    if (b < a.B) {
      len = a.lengths[b];
      if (record && len > (int64_t)a.W * a.ps) record_device_error(ENGPT_ERR_ARG, 44);
      len = clip_length(a, len);
    }
    const int v = pair_units(a, (len + KT - 1) / KT) * a.HQ;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (a.B <= 32) {
      start = x - v;
      if (lane < a.B) s_start[lane] = start;
      carry = __shfl_sync(0xffffffffu, x, 31);
      if (lane == 0) s_start[a.B] = carry;
      __syncwarp();
      return carry;
    }
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    int before = carry, total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) before += s_scan[i];
      total += s_scan[i];
    }
    if (b < a.B) s_start[b] = before + x - v;
    carry += total;
    __syncthreads();
  }
  if (tid == 0) s_start[a.B] = carry;
  __syncthreads();
  return carry;
}

// Units of a worker; at least a tile's, so that no worker between two others of a pair is without one of its tiles.
__device__ __forceinline__ int worker_units(const MmaArgs& a, int total, int ctas) {
  const uint32_t workers = ctas * kWarps;
  return max(a.tile_units, (int)(((uint32_t)total + workers - 1) / workers));
}

// Last row whose first unit is <= f (rows without tiles share their successor's start).
// (A cut that gives every worker its exact share, i * total / workers, was slower: it cuts more pairs.)
__device__ __forceinline__ int list_row(const MmaArgs& a, const int* s_start, int f, int start) {
  const int lane = threadIdx.x & 31;
  if (a.B <= 32) return 31 - __clz(__ballot_sync(0xffffffffu, lane < a.B && start <= f));
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_start[mid] <= f) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The persistent form over the list of tiles.
template <int D>
__global__ void __launch_bounds__(kWarps * 32) decode_list_kernel(MmaArgs a, const __grid_constant__ CUtensorMap mk,
                                                                 const __grid_constant__ CUtensorMap mv) {
  using C = Mma<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (sm100::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* tiles = smem_raw + (base - sm100::smem_u32(smem_raw));           // one of each warp
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + kWarps * 2 * kTileBytes);   // [kWarps]
  const int pf = part_floats<D>(a.rows);
  float* s_part = reinterpret_cast<float*>(bars + kWarps);                  // [kWarps] first part of each warp
  int* s_start = reinterpret_cast<int*>(s_part + kWarps * pf);              // [B + 1] first unit of each row
  __shared__ int s_abort, s_scan[kWarps], s_head[kWarps], s_tail[kWarps], s_over[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  Worker<D> w{a, &mk, &mv, base + warp * 2 * kTileBytes, sm100::smem_u32(bars + warp), lane};
  if (lane == 0) {
    sm100::mbar_init(w.bar, 1);
    sm100::fence_mbar_init();
    s_abort = 0;         // (every warp: a wait may set it only seconds later)
    s_head[warp] = s_tail[warp] = -1;
  }
  if (tid == 0) {
    sm100::tma_prefetch_desc(&mk);
    sm100::tma_prefetch_desc(&mv);
  }
  __syncwarp();
  asm volatile("griddepcontrol.wait;" ::: "memory");   // nothing of an earlier kernel has been touched before

  // this worker's range [u0, u1) of the list's units and its first tile: the tiles that begin in the range are its own
  const int worker = blockIdx.x * kWarps + warp;
  int row_len = 0, row_start = 0;
  const int total = list_starts<C::KT>(a, s_start, s_scan, kWarps * 32, blockIdx.x == 0, row_len, row_start);
  const int per = worker_units(a, total, gridDim.x);
  const int u0 = (int)min((int64_t)total, (int64_t)worker * per), u1 = (int)min((int64_t)total, (int64_t)u0 + per);
  Cursor c;
  c.b = list_row(a, s_start, u0, row_start);
  if (a.B <= 32) {
    c.len = __shfl_sync(0xffffffffu, row_len, c.b);
    c.T = (c.len + C::KT - 1) / C::KT;
  } else {
    w.enter_row(c);
  }
  const uint32_t in = u0 - s_start[c.b], span = max(pair_units(a, c.T), 1);
  c.h = (int)(in / span);
  c.t = (int)((in - c.h * span + a.tile_units - 1) / (uint32_t)a.tile_units);   // the first tile that begins in the range
  c.hk = c.h / a.QG;
  c.u = s_start[c.b] + c.h * (int)span + c.t * a.tile_units;
  if (u0 >= u1) {
    c.u = u1;            // nothing to do
  } else if (c.t >= c.T) {
    c.t = c.T - 1;       // the range begins in the end of a pair: on to the next one
    c.u -= a.tile_units;
    w.advance(c);
  }

  // the first tile's copies; ci is the next tile to fetch, box its place
  Cursor ci = c;
  uint32_t mask = 0;
  Box box{0, -1};
  if (c.u < u1) {
    mask = w.issue(ci, w.find_box(ci));
    w.advance(ci);
    if (ci.u < u1) box = w.find_box(ci);
  }

  // the joining kernel may start: it reads nothing of this one before this one has ended
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // rows without keys
  for (int64_t i = blockIdx.x * (int64_t)(kWarps * 32) + tid; i < (int64_t)a.B * a.H;
       i += (int64_t)gridDim.x * kWarps * 32) {
    const int b = (int)(i / a.H);
    if (s_start[b + 1] == s_start[b])
      for (int e = 0; e < a.dim; e += 8) *reinterpret_cast<uint4*>(a.o + i * a.dim + e) = make_uint4(0u, 0u, 0u, 0u);
  }

  float* part = s_part + warp * pf;                                         // a pair that began before this range
  float* tail_part = reinterpret_cast<float*>(tiles + warp * 2 * kTileBytes);   // one that ends behind it (no tile left)
  State<D> st;
  st.reset();
  uint32_t qa[C::DK][2];
  uint32_t phase = 0;
  bool fresh = true;                // the next tile begins a segment
  int t0 = 0;
  while (c.u < u1) {
    if (fresh) {
      load_query<D>(a, c.b, c.h, lane, qa);
      t0 = c.t;
      fresh = false;
    }
    if (!__all_sync(0xffffffffu, sm100::mbar_wait(w.bar, phase, &s_abort, 45))) {
      w.drain(phase);
      break;   // (the pair keeps no part of this warp: its rows are wrong, and the status word says so)
    }
    phase ^= 1u;
    const int live = c.len - c.t * C::KT;
    if (live >= C::KT && mask == (1u << (C::KT >> a.r_shift)) - 1u)
      tile_step<D, true>(a, w.tile, qa, st, live, mask, lane);
    else
      tile_step<D, false>(a, w.tile, qa, st, live, mask, lane);
    __syncwarp();
    if (ci.u < u1) {
      mask = w.issue(ci, box);
      w.advance(ci);
      if (ci.u < u1) box = w.find_box(ci);
    }
    const bool pair_end = c.t + 1 == c.T;
    Cursor cn = c;
    w.advance(cn);
    if (pair_end || cn.u >= u1) {
      finish_rows<D>(a, st);
      if (t0 == 0 && pair_end) {
        store_rows<D>(a, st, c.b, c.h, lane);
      } else if (t0 == 0) {
        store_part<D>(a, st, tail_part, lane);   // the last tile of the range: nothing is being copied
        if (lane == 0) {
          s_tail[warp] = c.b * a.HQ + c.h;
          // does its last tile begin behind this CTA's units?
          s_over[warp] = (int64_t)c.u + (c.T - 1 - c.t) * a.tile_units >= (int64_t)(blockIdx.x + 1) * kWarps * per;
        }
      } else {
        store_part<D>(a, st, part, lane);
        if (lane == 0) s_head[warp] = c.b * a.HQ + c.h;
      }
      st.reset();
      fresh = true;
    }
    c = cn;
  }

  float* out = a.work + (int64_t)blockIdx.x * 2 * pf;
  __syncthreads();   // every worker's parts are written
  // Groups of parts of one pair: those that begin in warp g, and the one that comes in from an earlier CTA (g = -1:
  // warps 0, 1, ..).  With few rows a warp joins its own group (the last warp the incoming one too); with 8 all warps
  // share each group's rows.
  auto join_group = [&](int g, int r0, int step) {
    const int pair = g < 0 ? s_head[0] : s_tail[g];
    if (pair < 0) return;
    const int w0 = max(g, 0);
    int n = g < 0 ? 0 : 1;
    while (w0 + n < kWarps && s_head[w0 + n] == pair) ++n;
    const float* first = g < 0 ? s_part : reinterpret_cast<const float*>(tiles + g * 2 * kTileBytes);
    const float* rest = s_part + g * pf;
    float* to = g < 0 ? out : (s_over[g] ? out + pf : nullptr);   // at most one pair runs over the CTA's end
    const int b = pair / a.HQ, h = pair - b * a.HQ;
    for (int r = r0; r < a.rows; r += step)
      join_row<D, kWarps>(a, b, h, r, n, [=](int i) { return i == 0 ? first : (g < 0 ? first : rest) + i * pf; }, to, lane);
  };
  if (a.rows < kWarps) {
    join_group(warp, 0, 1);
    if (warp == kWarps - 1) join_group(-1, 0, 1);
  } else {
    for (int g = -1; g < kWarps; ++g) join_group(g, warp, kWarps);
  }
}

// One cluster of `cs` CTAs per pair: tile t goes to warp t mod (cs * kPairWarps) of the cluster, whose parts are joined
// through shared memory, then through the shared memory of the cluster's first CTA.  No prefix sums, no second
// launch, and the first page look-up does not wait for the length: the form for short rows and for few pairs.
template <int D>
__global__ void __launch_bounds__(kPairWarps * 32) decode_pair_kernel(MmaArgs a, const __grid_constant__ CUtensorMap mk,
                                                                  const __grid_constant__ CUtensorMap mv, int cs) {
  using C = Mma<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (sm100::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* tiles = smem_raw + (base - sm100::smem_u32(smem_raw));           // one of each warp
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + kPairWarps * 2 * kTileBytes);  // [kPairWarps]
  const int pf = part_floats<D>(a.rows);
  float* s_part = reinterpret_cast<float*>(bars + kPairWarps);              // [kPairWarps] the warps' parts
  float* s_cta = s_part + kPairWarps * pf;                                  // [cs] the CTAs' parts (rank 0)
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (cs > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  const int pair = blockIdx.x / cs, rank = blockIdx.x - pair * cs;
  const int me = rank * kPairWarps + warp, step = cs * kPairWarps;
  Worker<D> w{a, &mk, &mv, base + warp * 2 * kTileBytes, sm100::smem_u32(bars + warp), lane};
  Cursor c;
  c.b = pair / a.HQ;
  c.h = pair - c.b * a.HQ;
  c.hk = c.h / a.QG;
  c.t = me;
  if (lane == 0) {
    sm100::mbar_init(w.bar, 1);
    sm100::fence_mbar_init();
    s_abort = 0;                        // (every warp: a wait may set it only seconds later)
    if (warp == 0) {
      sm100::tma_prefetch_desc(&mk);
      sm100::tma_prefetch_desc(&mv);
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // nothing of an earlier kernel has been touched before
  const int len = a.lengths[c.b];
  c.len = c.T = a.W * a.ps;             // the look-up is bounded by the table row; the length cuts it below
  Box box = w.find_box(c);
  if (me == 0 && c.h == 0 && lane == 0 && len > (int64_t)a.W * a.ps) record_device_error(ENGPT_ERR_ARG, 44);
  uint32_t qa[C::DK][2];
  load_query<D>(a, c.b, c.h, lane, qa);
  __syncwarp();
  c.len = clip_length(a, len);
  c.T = (c.len + C::KT - 1) / C::KT;
  if (c.t * C::KT + lane * a.R >= c.len) box.off = -1;
  const int n = c.T > me ? (c.T - me + step - 1) / step : 0;   // this warp's tiles
  Cursor ci = c;
  uint32_t mask = 0;
  if (n > 0) {
    mask = w.issue(ci, box);
    ci.t += step;
    if (n > 1) box = w.find_box(ci);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  State<D> st;
  st.reset();
  uint32_t phase = 0;
  bool ok = true;
  for (int i = 0; i < n; ++i, c.t += step) {
    if (!__all_sync(0xffffffffu, sm100::mbar_wait(w.bar, phase, &s_abort, 46))) {
      w.drain(phase);
      ok = false;
      break;
    }
    phase ^= 1u;
    const int live = c.len - c.t * C::KT;
    if (live >= C::KT && mask == (1u << (C::KT >> a.r_shift)) - 1u)
      tile_step<D, true>(a, w.tile, qa, st, live, mask, lane);
    else
      tile_step<D, false>(a, w.tile, qa, st, live, mask, lane);
    __syncwarp();
    if (i + 1 < n) {
      mask = w.issue(ci, box);
      ci.t += step;
      if (i + 2 < n) box = w.find_box(ci);
    }
  }
  finish_rows<D>(a, st);

  if (c.T <= 1) {
    if (me == 0 && ok) store_rows<D>(a, st, c.b, c.h, lane);
    if (cs > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;
  }
  const int mine = min(max(c.T - rank * kPairWarps, 0), kPairWarps);   // this CTA's warps with tiles
  if (warp < mine && ok) store_part<D>(a, st, s_part + warp * pf, lane);
  __syncthreads();
  const float* parts = s_part;
  if (cs == 1) {
    for (int r = warp; r < a.rows; r += kPairWarps)
      join_row<D, kPairWarps>(a, c.b, c.h, r, mine, [=](int i) { return parts + i * pf; }, nullptr, lane);
    return;
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // every CTA of the cluster has started
  if (mine > 0) {
    float* to;
    asm("mapa.u64 %0, %1, %2;" : "=l"(to) : "l"(s_cta + rank * pf), "r"(0));
    for (int r = warp; r < a.rows; r += kPairWarps)
      join_row<D, kPairWarps>(a, c.b, c.h, r, mine, [=](int i) { return parts + i * pf; }, to, lane);
  }
  sm100::cluster_sync_all();
  if (rank == 0) {
    const float* ctas = s_cta;
    const int k = min(cs, (c.T + kPairWarps - 1) / kPairWarps);                 // CTAs with tiles
    for (int r = warp; r < a.rows; r += kPairWarps)
      join_row<D, 8>(a, c.b, c.h, r, k, [=](int i) { return ctas + i * pf; }, nullptr, lane);
  }
}

// Pairs that run over the end of a CTA of decode_list_kernel: a CTA per pair and row of its query heads, or per CTA
// end and row if there are more pairs than CTAs (of `ctas`); every warp takes a share of the parts.
// It starts while that kernel runs (whose CTAs have by then waited for all earlier work) and finds its pair from the
// lengths; only the parts have to wait.
template <int D>
__global__ void __launch_bounds__(kWarps * 32) decode_join_list_kernel(MmaArgs a, int ctas) {
  constexpr int E = D / 32;
  extern __shared__ int s_start[];
  __shared__ float s_o[kWarps][D];
  __shared__ float s_m[kWarps], s_l[kWarps];
  __shared__ int s_scan[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int row_len = 0, row_start = 0;
  const int total = list_starts<Mma<D>::KT>(a, s_start, s_scan, kWarps * 32, false, row_len, row_start);
  const int64_t per = (int64_t)kWarps * worker_units(a, total, ctas);   // of a CTA
  int first = 0, n = 0, b = 0, h = 0;
  if ((int)gridDim.x < ctas) {                        // pair blockIdx.x
    b = blockIdx.x / a.HQ;
    h = blockIdx.x - b * a.HQ;
    const int span = (s_start[b + 1] - s_start[b]) / a.HQ;
    const int64_t from = s_start[b] + (int64_t)h * span, to = from + span - a.end_units - a.tile_units;   // first, last tile
    if (span > 0 && from / per < to / per) {
      first = (int)(from / per);
      n = (int)(to / per) - first + 1;
    }
  } else {                                            // the pair that runs over the end of CTA blockIdx.x
    const int64_t end = (blockIdx.x + 1) * per;       // the first unit of the next CTA
    if (end < total) {
      b = list_row(a, s_start, (int)end, row_start);
      const int span = (s_start[b + 1] - s_start[b]) / a.HQ;
      h = ((int)end - s_start[b]) / span;
      const int64_t from = s_start[b] + (int64_t)h * span, to = from + span - a.end_units - a.tile_units;
      if (from < end && from >= end - per && to >= end) {   // it begins in this CTA
        first = blockIdx.x;
        n = (int)(to / per) - first + 1;
      }
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int pf = part_floats<D>(a.rows);
  const int r = blockIdx.y;
  if (n > 0 && (h % a.QG) * 8 + r < a.G) {
    float m = -INFINITY, l = 0.f, o[E] = {};
#pragma unroll 4
    for (int i = warp; i < n; i += kWarps) {
      const float* p = a.work + ((int64_t)(first + i) * 2 + (i == 0 ? 1 : 0)) * pf + r * (D + 2);
      const float2 ml = *reinterpret_cast<const float2*>(p + D);
      const float mx = fmaxf(m, ml.x);
      const float w0 = join_weight(m, mx), w1 = join_weight(ml.x, mx);
      l = l * w0 + ml.y * w1;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * w0 + p[lane + 32 * e] * w1;
      m = mx;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = o[e];
    if (lane == 0) {
      s_m[warp] = m;
      s_l[warp] = l;
    }
    __syncthreads();
    if (threadIdx.x < a.dim) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) mx = fmaxf(mx, s_m[i]);
      float lx = 0.f, ox = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float wgt = join_weight(s_m[i], mx);
        lx = fmaf(s_l[i], wgt, lx);
        ox = fmaf(s_o[i][threadIdx.x], wgt, ox);
      }
      a.o[((int64_t)b * a.H + (h / a.QG) * a.G + (h % a.QG) * 8 + r) * a.dim + threadIdx.x] =
          __float2bfloat16_rn(lx == 0.f ? 0.f : ox / lx);
    }
  }
}

static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

static int get_encode() {
  if (int rc = bind_thread_context()) return rc;
  if (g_encode) return ENGPT_OK;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult q;
  cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
  if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn)
    return set_error(ENGPT_ERR_LAUNCH, "paged_attention: cuTensorMapEncodeTiled unavailable");
  g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  return ENGPT_OK;
}

// [D, slots of a page, heads, pages] view of a bf16 page pool with element strides s (page, head, slot).
static int page_map(CUtensorMap* m, const void* base, int D, int ps, int heads, int P, const int64_t* s, int R) {
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)ps, (cuuint64_t)heads, (cuuint64_t)P};
  cuuint64_t strides[3] = {(cuuint64_t)s[2] * 2, (cuuint64_t)s[1] * 2, (cuuint64_t)s[0] * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)R, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = g_encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        s[2] == D ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(ENGPT_ERR_ALIGN, "paged_attention: tensor map encode failed (%d)", (int)r);
  return ENGPT_OK;
}

// Width of the tensor-core kernels for a head_dim, and keys of their tiles.
inline int mma_width(int dim) { return dim <= 64 ? 64 : 128; }
inline int tile_keys(int dim) { return kTileBytes / (2 * mma_width(dim)); }

inline int64_t most_tiles(int D, int table_width, int page_size) {
  return ((int64_t)table_width * page_size + tile_keys(D) - 1) / tile_keys(D);
}

// Does a launch of these sizes go to the tensor-core kernel (strides and alignment apart)?
inline bool mma_sizes(int dtype, int B, int H, int Hkv, int D, int table_width, int page_size) {
  return dtype == ENGPT_BF16 && D <= 128 && D % 8 == 0 && page_size % 8 == 0 && B <= kMaxListRows &&
         B * (int64_t)H * (2 * most_tiles(D, table_width, page_size) + 1) < (1ll << 31);
}

// CTAs per pair of the pair form, or 0 for the list form.
//
// The pair form starts and ends faster (an empty launch takes some 3 us, the list form's two 5.5) but does not balance
// rows of different length, so it has to be one wave of CTAs.  Its clusters are the widest that run at once: 8 CTAs up
// to one per SM in all (16 pairs of 32 tiles: 4.9 us with 8, 5.8 with 4, 8.3 with 2), 4 or 2 up to two per SM (64 pairs
// of 32 tiles: 10.6 us with 4, 12.1 with 2, 15.3 with 8 in three waves; list 13.1); narrower where a warp would be
// without a tile.  Its warps take their tiles one after the other, 2 us each, where the list form spreads them over all
// SMs at 16 KB / 6.2 TB/s = 1/380 us each: with t tiles per warp the pair form is taken while 2 (t - 1) <= 2 + pairs *
// tiles / 380 (16 pairs of 128 tiles: 12.3 against 13.0 us, 8 pairs of 128: 10.7 against 9.6, 16 pairs of 256: 19.2
// against 18.5), and, as the rows of a batch may differ and the longest one decides, with at most 4 tiles per warp if
// there are several rows (8 rows of 16 pairs of 32 tiles: 15.4 us against the list's 17.0 if all are that long).
inline int pair_ctas(int B, int H, int Hkv, int D, int table_width, int page_size) {
  const int64_t pairs = (int64_t)B * Hkv * ((H / Hkv + 7) / 8);
  const int64_t tiles = most_tiles(D, table_width, page_size);
  const int sms = num_sms();
  if (pairs > 2 * sms) return 0;
  int cs = pairs * 8 <= sms ? 8 : pairs * 4 <= 2 * sms ? 4 : pairs * 2 <= 2 * sms ? 2 : 1;
  while (cs > 1 && tiles <= kPairWarps * (cs / 2)) cs >>= 1;
  const int64_t per_warp = (tiles + kPairWarps * cs - 1) / (kPairWarps * cs);
  if (B > 1 && per_warp > 4) return 0;
  return 2 * (per_warp - 1) <= 2 + pairs * tiles / 380 ? cs : 0;
}

inline int64_t mma_floats(int H, int Hkv, int D) {
  const int rows = H / Hkv < 8 ? H / Hkv : 8;
  return (int64_t)num_sms() * 2 * rows * (mma_width(D) + 2);
}

template <int D>
size_t mma_smem(int rows, int warps, int parts) {
  return 1024 + (size_t)warps * (2 * kTileBytes + 8) + 4 * (size_t)parts * part_floats<D>(rows);
}

template <int D>
int launch_pair(const MmaArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int cs, cudaStream_t st) {
  auto kern = decode_pair_kernel<D>;
  // Two CTAs per SM and no third one, which would leave other SMs idle (one wave has at most two per SM; 128 pairs of 32
  // tiles: 15.2 us so, 16.5 if three fit).
  const size_t needed = mma_smem<D>(a.rows, kPairWarps, kPairWarps + cs), smem = needed > kPairSmem ? needed : kPairSmem;
  // (the attribute is the kernel's, not the launch's: every call sets it to the same, largest size, so that a call on
  // another host thread cannot lower it between here and the launch)
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)mma_smem<D>(8, kPairWarps, kPairWarps + 8));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.HQ * cs));
  cfg.blockDim = dim3(kPairWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cs;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cs > 1 ? 2 : 1;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kern, a, mk, mv, cs);
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "paged_attention: %s", cudaGetErrorString(e));
  return ENGPT_OK;
}

template <int D>
int launch_list(const MmaArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  auto kern = decode_list_kernel<D>;
  const size_t smem = mma_smem<D>(a.rows, kWarps, kWarps) + 4 * ((size_t)a.B + 1);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,   // as in launch_pair
                                       (int)(mma_smem<D>(8, kWarps, kWarps) + 4 * ((size_t)kMaxListRows + 1)));
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "paged_attention: %s", cudaGetErrorString(e));
  // both kernels may be started before what runs ahead of them has ended; they wait for it on the device
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)num_sms());
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, a, mk, mv);
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "paged_attention: %s", cudaGetErrorString(e));
  const int64_t pairs = (int64_t)a.B * a.HQ;
  cfg.gridDim = dim3((unsigned)(pairs < num_sms() ? pairs : num_sms()), a.rows);
  cfg.dynamicSmemBytes = 4 * ((size_t)a.B + 1);
  e = cudaLaunchKernelEx(&cfg, decode_join_list_kernel<D>, a, num_sms());
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "paged_attention (join): %s", cudaGetErrorString(e));
  return check_launch("paged_attention (join)");
}

template <int D>
int launch_mma(const AttnArgs& x, int Hkv, cudaStream_t st) {
  int rc = get_encode();
  if (rc) return rc;
  MmaArgs a;
  a.q = reinterpret_cast<const __nv_bfloat16*>(x.q);
  a.q_row = x.q_row;
  a.dim = x.Dh;
  a.q_head = x.q_head;
  a.B = x.B;
  a.H = x.H;
  a.G = x.G;
  a.QG = (x.G + 7) / 8;
  a.HQ = Hkv * a.QG;
  a.rows = x.G < 8 ? x.G : 8;
  a.P = x.P;
  a.ps = x.ps;
  a.ps_shift = (x.ps & (x.ps - 1)) == 0 ? __builtin_ctz((unsigned)x.ps) : -1;
  a.r_shift = 3;
  while (x.ps % (2 << a.r_shift) == 0 && (2 << a.r_shift) <= tile_keys(D)) ++a.r_shift;
  a.R = 1 << a.r_shift;
  a.table = x.table;
  a.table_stride = x.table_stride;
  a.W = x.W;
  a.lengths = x.lengths;
  a.scale_log2 = fabsf(x.scale_log2);
  a.q_flip = x.scale_log2 < 0.f ? 0x80008000u : 0u;
  a.o = reinterpret_cast<__nv_bfloat16*>(x.o);
  a.work = x.work;
  CUtensorMap mk, mv;
  if ((rc = page_map(&mk, x.k_pages, x.Dh, x.ps, Hkv, x.P, x.ks, a.R))) return rc;
  if ((rc = page_map(&mv, x.v_pages, x.Dh, x.ps, Hkv, x.P, x.vs, a.R))) return rc;
  const int cs = pair_ctas(x.B, x.H, Hkv, D, x.W, x.ps);
  // The end of a pair costs a worker about half a tile (its sums and stores, and tiles that are partly empty).  It is
  // counted once workers see such ends often (256 rows of 1 to 512 tokens: 51.8 us, 63.8 without); with few pairs the
  // ranges are whole tiles, which cuts fewer pairs (32 rows of 512 tokens, 16 heads: 16.9 us, 18.5 with).
  const bool ends = 2 * (int64_t)x.B * a.HQ > (int64_t)num_sms() * kWarps;
  a.tile_units = ends ? 2 : 1;
  a.end_units = ends ? 1 : 0;
  if (cs == 0) return launch_list<D>(a, mk, mv, st);
  return launch_pair<D>(a, mk, mv, cs, st);
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
  if (!mma_sizes(dtype, B, H, Hkv, Dh, table_width, page_size)) return simt;
  // strides and alignment decide at the call which of the two kernels runs
  const int64_t mma = pair_ctas(B, H, Hkv, Dh, table_width, page_size) == 0 ? mma_floats(H, Hkv, Dh) : 0;
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
  if (vec && positive && aligned(o, 16) && num_pages > 0 && mma_sizes(dtype, B, H, Hkv, Dh, table_width, page_size))
    return mma_width(Dh) == 64 ? launch_mma<64>(a, Hkv, st) : launch_mma<128>(a, Hkv, st);
  return dtype == ENGPT_BF16 ? dispatch_simt<__nv_bfloat16>(a, vec, st) : dispatch_simt<float>(a, vec, st);
}
