// Attention of one new token per request over a paged key-value cache: what does not depend on how the cache holds
// its numbers (paged_attn.cu: bf16 or fp32; paged_attn_q8.cu: 8 bits with scales).
//
//   o[b, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),  m = max_j scale q.k_j
//
// Every key and value is read once and used for 4 Dh flops, so the operator
// is bound by HBM.  The keys of a row are split over CTAs; each keeps a
// running maximum m, the sum l of the p_j and the unnormalised o, and two
// such parts join as
//   m = max(m1, m2),  l = l1 e^(m1-m) + l2 e^(m2-m),  o likewise.
#pragma once

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
  if constexpr (VEC == 8 && sizeof(T) == 4) {
    load_vec<T, 4>(p, x);
    load_vec<T, 4>(p + 4, x + 4);
  } else if constexpr (VEC == 8) {
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

// A cache of the type of q and o, for the CUDA-core kernel below.
template <typename Type>
struct PlainKv {
  using T = Type;                         // of q and o
  using Code = Type;                      // of the pools
  using Args = AttnArgs;
  static constexpr bool kScaled = false;
  template <int VEC>
  static __device__ __forceinline__ void load(const Code* p, float* x) { load_vec<T, VEC>(p, x); }
};

// CUDA-core kernel: any head_dim up to 256, fp32 or bf16, any strides.  Eight lanes share a key (each owns NC pieces
// of VEC elements, VEC = 16 bytes where the addresses allow it); a lane group keeps its own m, l and o of HG query
// heads of one kv head over every kGroups-th key of the CTA's range, U keys in flight at a time, and the groups join
// through shared memory.  The `splits` CTAs of a row and its heads are a cluster while there are at most 8 and join in
// the shared memory of the first; otherwise they leave parts in the workspace for decode_join_kernel.
template <typename KV, int VEC, int NC, int U, int HG>
__global__ void __launch_bounds__(kThreads) decode_simt_kernel(typename KV::Args a) {
  using T = typename KV::T;
  using Code = typename KV::Code;
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
  const Code* kp = reinterpret_cast<const Code*>(a.k_pages) + hk * a.ks[1];
  const Code* vp = reinterpret_cast<const Code*>(a.v_pages) + hk * a.vs[1];
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
    float kf[U][NC * VEC], vf[U][NC * VEC], ksc[U], vsc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool live = page[u] >= 0 && page[u] < a.P;
      if constexpr (KV::kScaled) {
        ksc[u] = live ? KV::key_scale(a, page[u], hk, off[u]) : 0.f;
        vsc[u] = live ? KV::value_scale(a, page[u], hk, off[u]) : 0.f;
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int e = (c * 8 + sub) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) kf[u][c * VEC + i] = vf[u][c * VEC + i] = 0.f;
        if (live && e < a.Dh) {
          KV::template load<VEC>(kp + page[u] * a.ks[0] + off[u] * a.ks[2] + e, kf[u] + c * VEC);
          KV::template load<VEC>(vp + page[u] * a.vs[0] + off[u] * a.vs[2] + e, vf[u] + c * VEC);
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
          if constexpr (KV::kScaled) s[g] *= ksc[u];
          const float mn = fmaxf(m[g], s[g]);
          const float ms = mn == -INFINITY ? 0.f : mn;
          const float corr = sm100::ex2_approx(m[g] - ms), p = sm100::ex2_approx(s[g] - ms);
          m[g] = mn;
          l[g] = fmaf(l[g], corr, p);
          float pv = p;
          if constexpr (KV::kScaled) pv *= vsc[u];
#pragma unroll
          for (int i = 0; i < NC * VEC; ++i) o[g][i] = fmaf(o[g][i], corr, pv * vf[u][i]);
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

template <typename KV, int VEC, int NC, int U, int HG>
int launch_simt(const typename KV::Args& a, cudaStream_t st) {
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
  cudaError_t e = cudaLaunchKernelEx(&cfg, decode_simt_kernel<KV, VEC, NC, U, HG>, a);
  if (e == cudaSuccess && a.splits > kSimtCluster) {
    cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.H));
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, decode_join_kernel<typename KV::T>, AttnArgs(a));
  }
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "paged_attention: %s", cudaGetErrorString(e));
  return check_launch("paged_attention");
}

// Query heads that share a kv head and one reading of its keys: 4, 2 or 1 (8 fp32 rows of 1024 tokens, 32 heads on 4
// of 128: 28 us with four heads per reading, 41 with one).
template <typename KV, int VEC, int NC, int U>
int launch_simt_heads(const typename KV::Args& a, cudaStream_t st) {
  if (a.G % 4 == 0) return launch_simt<KV, VEC, NC, U, 4>(a, st);
  if (a.G % 2 == 0) return launch_simt<KV, VEC, NC, U, 2>(a, st);
  return launch_simt<KV, VEC, NC, U, 1>(a, st);
}

// ------------------------------------------------------------------ tensor-core kernels
//
// A tile is KT keys of one kv head, kTile bytes of keys and as many of values.  The tiles of all (row, kv head) pairs
// form one list, cut into contiguous ranges of equal cost, one per warp ("worker") of a persistent grid, so the load is
// even whatever the lengths.  A warp fetches its own tiles, one at a time, into its own 2 kTile bytes of shared memory:
// TMA boxes of R rows (R divides the page size) at the page that the block table names, swizzled, completing
// on the warp's mbarrier; no warp waits for another one until the end.
//
// What a tile holds and how it is used is the business of a class F:
//   D, KT              width (a smaller head_dim is padded with zeros by TMA, in shared memory only), keys of a tile
//   kTile, kWarps, kPairWarps    bytes of a tile's keys, warps of a CTA of the list form and of the pair form
//   kPairPerSm, kTileUs, kPartsOver    of the pair form: CTAs per SM, time of a tile, parts that go where the tiles were
//   T, Args            type of q and o; kernel arguments (MmaArgs and what F adds)
//   kBoxes, kBoxRow    boxes of 64 columns of a group of R keys, bytes of a row of one
//   kFlat, rows_at     rows that are one behind the other in a page are copied as they are, in one piece
//   Spot, find         a look-up that is made a tile ahead of the tile's copies
//   Side, fetch        loads that start with the tile's copies
//   Query, load_query  a pair's query heads, up to 8, as rows 0-7 of the 16-row mma.sync operand
//   State, step, finish, store_part, store_rows    the running state of a pair and a tile's step on it
//
// The products do not bound anything here (64 mma.sync of 16x8x16 per 16 KB of bf16), which is why this is not built on
// tcgen05: its 128-row operand would be 1/128 to 1/16 full and P would take a trip through TMEM.
//
// A range that begins or ends inside a pair leaves a part (o, m, l) in shared memory.  After a CTA barrier the parts
// of a pair are joined by the warp that holds its first one; a pair that runs over CTAs leaves one part per CTA in
// the workspace, joined by decode_join_list_kernel.
constexpr size_t kPairSmem = 80 * 1024;  // of the form with a cluster per pair, at least: no more than two CTAs per SM
constexpr int kMaxListRows = 8192;      // of the list form: an int of shared memory each

struct MmaArgs {
  const void* q;
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
  bool negative;           // the scale is: q's sign is flipped
  void* o;
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

// Usable length of row b (a length beyond the table is recorded once, by the kernel's prologue).
__device__ __forceinline__ int clip_length(const MmaArgs& a, int len) {
  return (int)min((int64_t)max(len, 0), (int64_t)a.W * a.ps);
}

// Position in the list of tiles: tile t of T of (row b of length len, head group h of kv head hk), at unit u.
struct Cursor {
  int b, h, t, T, len, hk, u;
};

// A box of the tile to come: its page as the table has it (looked at only when the copy is issued, so that nothing
// waits for the look-up before) and first row in the page, -1 for a box past the length; and what else of a tile the
// cache has to look up.
template <typename F>
struct Box {
  int page, off;
  typename F::Spot spot;
};

template <typename F>
struct Worker {
  const typename F::Args& a;
  const CUtensorMap *mk, *mv;
  uint32_t tile;            // this warp's tile in shared memory: keys, then values
  uint32_t bar;             // its mbarrier
  int lane;

  __device__ __forceinline__ void enter_row(Cursor& c) const {
    c.len = c.b < a.B ? clip_length(a, a.lengths[c.b]) : 0;
    c.T = (c.len + F::KT - 1) / F::KT;
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

  __device__ __forceinline__ Box<F> find_box(const Cursor& c) const {
    const typename F::Spot spot = F::find(a, c, lane);
    const int key = c.t * F::KT + lane * a.R;
    if (lane * a.R >= F::KT || key >= c.len) return Box<F>{0, -1, spot};
    const int j = a.ps_shift >= 0 ? key >> a.ps_shift : key / a.ps;
    return Box<F>{a.table[c.b * a.table_stride + j], key - j * a.ps, spot};
  }

  // Start the copies of the cursor's tile and the loads of what else it needs; returns which of its boxes are copied.
  __device__ __forceinline__ uint32_t issue(const Cursor& c, const Box<F>& x, typename F::Side& side) const {
    const bool here = x.off >= 0 && (unsigned)x.page < (unsigned)a.P;
    const uint32_t mask = __ballot_sync(0xffffffffu, here);
    const uint32_t box = a.R * F::kBoxRow;
    if (lane == 0) sm100::mbar_expect_tx(bar, __popc(mask) * box * F::kBoxes * 2);
    __syncwarp();
    if (here) {
      const uint32_t dst = tile + lane * box;
      if constexpr (F::kFlat) {
        sm100::bulk_load(dst, F::rows_at(a, 0, x.page, c.hk, x.off), box, bar);
        sm100::bulk_load(dst + F::kTile, F::rows_at(a, 1, x.page, c.hk, x.off), box, bar);
      }
#pragma unroll
      for (int half = 0; !F::kFlat && half < F::kBoxes; ++half) {
        sm100::tma_load_4d(dst + half * F::KT * F::kBoxRow, mk, half * 64, x.off, c.hk, x.page, bar);
        sm100::tma_load_4d(dst + half * F::KT * F::kBoxRow + F::kTile, mv, half * 64, x.off, c.hk, x.page, bar);
      }
    } else if (x.off >= 0) {   // a page outside the pool
      record_device_error(ENGPT_ERR_ARG, 44);
    }
    F::fetch(a, c, x.spot, side);
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

// Joins row r of n <= N parts (part(i): its rows) by one warp: into the output, or as one part at `to`.  Lane i holds
// part i's weight, and all loads are independent.
template <typename F, int N, typename Part>
__device__ __forceinline__ void join_row(const MmaArgs& a, int b, int h, int r, int n, Part part, float* to, int lane) {
  constexpr int D = F::D, E = D / 32;
  constexpr int half = N > 16 ? 16 : N > 8 ? 8 : N > 4 ? 4 : N > 2 ? 2 : 1;   // of the lanes that hold a part
  if ((h % a.QG) * 8 + r >= a.G) return;
  float m = -INFINITY, l = 0.f;
  if (lane < n) {
    const float2 ml = *reinterpret_cast<const float2*>(part(lane) + r * (D + 2) + D);
    m = ml.x;
    l = ml.y;
  }
  float mx = m;
#pragma unroll
  for (int k = half; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
  mx = __shfl_sync(0xffffffffu, mx, 0);
  const float w = join_weight(m, mx);
  l *= w;
#pragma unroll
  for (int k = half; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
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
    typename F::T* dst = reinterpret_cast<typename F::T*>(a.o) + ((int64_t)b * a.H + (h / a.QG) * a.G + (h % a.QG) * 8 + r) * a.dim;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < a.dim) store1(dst + lane + 32 * e, o[e] * inv);
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
template <typename F>
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
    const int v = pair_units(a, (len + F::KT - 1) / F::KT) * a.HQ;
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
    for (int i = 0; i < F::kWarps; ++i) {
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
template <typename F>
__device__ __forceinline__ int worker_units(const MmaArgs& a, int total, int ctas) {
  const uint32_t workers = ctas * F::kWarps;
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
template <typename F>
__global__ void __launch_bounds__(F::kWarps * 32) decode_list_kernel(typename F::Args a,
                                                                 const __grid_constant__ CUtensorMap mk,
                                                                 const __grid_constant__ CUtensorMap mv) {
  constexpr int D = F::D;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (sm100::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* tiles = smem_raw + (base - sm100::smem_u32(smem_raw));           // one of each warp
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + F::kWarps * 2 * F::kTile);   // [F::kWarps]
  const int pf = part_floats<D>(a.rows);
  float* s_part = reinterpret_cast<float*>(bars + F::kWarps);                  // [F::kWarps] first part of each warp
  int* s_start = reinterpret_cast<int*>(s_part + F::kWarps * pf);              // [B + 1] first unit of each row
  __shared__ int s_abort, s_scan[F::kWarps], s_head[F::kWarps], s_tail[F::kWarps], s_over[F::kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  Worker<F> w{a, &mk, &mv, base + warp * 2 * F::kTile, sm100::smem_u32(bars + warp), lane};
  if (lane == 0) {
    sm100::mbar_init(w.bar, 1);
    sm100::fence_mbar_init();
    s_abort = 0;         // (every warp: a wait may set it only seconds later)
    s_head[warp] = s_tail[warp] = -1;
  }
  if (!F::kFlat && tid == 0) {
    sm100::tma_prefetch_desc(&mk);
    sm100::tma_prefetch_desc(&mv);
  }
  __syncwarp();
  asm volatile("griddepcontrol.wait;" ::: "memory");   // nothing of an earlier kernel has been touched before

  // this worker's range [u0, u1) of the list's units and its first tile: the tiles that begin in the range are its own
  const int worker = blockIdx.x * F::kWarps + warp;
  int row_len = 0, row_start = 0;
  const int total = list_starts<F>(a, s_start, s_scan, F::kWarps * 32, blockIdx.x == 0, row_len, row_start);
  const int per = worker_units<F>(a, total, gridDim.x);
  const int u0 = (int)min((int64_t)total, (int64_t)worker * per), u1 = (int)min((int64_t)total, (int64_t)u0 + per);
  Cursor c;
  c.b = list_row(a, s_start, u0, row_start);
  if (a.B <= 32) {
    c.len = __shfl_sync(0xffffffffu, row_len, c.b);
    c.T = (c.len + F::KT - 1) / F::KT;
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
  typename F::Side side;
  Box<F> box{0, -1, {}};
  if (c.u < u1) {
    mask = w.issue(ci, w.find_box(ci), side);
    w.advance(ci);
    if (ci.u < u1) box = w.find_box(ci);
  }

  // the joining kernel may start: it reads nothing of this one before this one has ended
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // rows without keys
  for (int64_t i = blockIdx.x * (int64_t)(F::kWarps * 32) + tid; i < (int64_t)a.B * a.H;
       i += (int64_t)gridDim.x * F::kWarps * 32) {
    const int b = (int)(i / a.H);
    if (s_start[b + 1] == s_start[b])
      for (int e = 0; e < a.dim; e += 16 / (int)sizeof(typename F::T))
        *reinterpret_cast<uint4*>(reinterpret_cast<typename F::T*>(a.o) + i * a.dim + e) = make_uint4(0u, 0u, 0u, 0u);
  }

  float* part = s_part + warp * pf;                                         // a pair that began before this range
  float* tail_part = reinterpret_cast<float*>(tiles + warp * 2 * F::kTile);   // one that ends behind it (no tile left)
  typename F::State st;
  st.reset();
  typename F::Query qa;
  uint32_t phase = 0;
  bool fresh = true;                // the next tile begins a segment
  int t0 = 0;
  while (c.u < u1) {
    if (fresh) {
      F::load_query(a, c.b, c.h, lane, qa);
      t0 = c.t;
      fresh = false;
    }
    if (!__all_sync(0xffffffffu, sm100::mbar_wait(w.bar, phase, &s_abort, 45))) {
      w.drain(phase);
      break;   // (the pair keeps no part of this warp: its rows are wrong, and the status word says so)
    }
    phase ^= 1u;
    const int live = c.len - c.t * F::KT;
    if (live >= F::KT && mask == (1u << (F::KT >> a.r_shift)) - 1u)
      F::template step<true>(a, w.tile, qa, side, st, live, mask, lane);
    else
      F::template step<false>(a, w.tile, qa, side, st, live, mask, lane);
    __syncwarp();
    if (ci.u < u1) {
      mask = w.issue(ci, box, side);
      w.advance(ci);
      if (ci.u < u1) box = w.find_box(ci);
    }
    const bool pair_end = c.t + 1 == c.T;
    Cursor cn = c;
    w.advance(cn);
    if (pair_end || cn.u >= u1) {
      F::finish(a, st);
      if (t0 == 0 && pair_end) {
        F::store_rows(a, st, c.b, c.h, lane);
      } else if (t0 == 0) {
        F::store_part(a, st, tail_part, lane);   // the last tile of the range: nothing is being copied
        if (lane == 0) {
          s_tail[warp] = c.b * a.HQ + c.h;
          // does its last tile begin behind this CTA's units?
          s_over[warp] = (int64_t)c.u + (c.T - 1 - c.t) * a.tile_units >= (int64_t)(blockIdx.x + 1) * F::kWarps * per;
        }
      } else {
        F::store_part(a, st, part, lane);
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
  // warps 0, 1, ..).  Eight warps with few rows join their own groups (the last warp the incoming one too), and share
  // each group's rows with 8; more warps share the rows of all groups.
  auto join_group = [&](int g, int r0, int step) {
    const int pair = g < 0 ? s_head[0] : s_tail[g];
    if (pair < 0) return;
    const int w0 = max(g, 0);
    int n = g < 0 ? 0 : 1;
    while (w0 + n < F::kWarps && s_head[w0 + n] == pair) ++n;
    const float* first = g < 0 ? s_part : reinterpret_cast<const float*>(tiles + g * 2 * F::kTile);
    const float* rest = s_part + g * pf;
    float* to = g < 0 ? out : (s_over[g] ? out + pf : nullptr);   // at most one pair runs over the CTA's end
    const int b = pair / a.HQ, h = pair - b * a.HQ;
    for (int r = r0; r < a.rows; r += step)
      join_row<F, F::kWarps>(a, b, h, r, n, [=](int i) { return i == 0 ? first : (g < 0 ? first : rest) + i * pf; }, to, lane);
  };
  if constexpr (F::kWarps > 8) {
    for (int i = warp; i < (F::kWarps + 1) * a.rows; i += F::kWarps) {
      const int g = i / a.rows;
      join_group(g - 1, i - g * a.rows, a.rows);
    }
  } else if (a.rows < F::kWarps) {
    join_group(warp, 0, 1);
    if (warp == F::kWarps - 1) join_group(-1, 0, 1);
  } else {
    for (int g = -1; g < F::kWarps; ++g) join_group(g, warp, F::kWarps);
  }
}

// One cluster of `cs` CTAs per pair: tile t goes to warp t mod (cs * F::kPairWarps) of the cluster, whose parts are joined
// through shared memory, then through the shared memory of the cluster's first CTA.  No prefix sums, no second
// launch, and the first page look-up does not wait for the length: the form for short rows and for few pairs.
template <typename F>
__global__ void __launch_bounds__(F::kPairWarps * 32) decode_pair_kernel(typename F::Args a,
                                                                     const __grid_constant__ CUtensorMap mk,
                                                                     const __grid_constant__ CUtensorMap mv, int cs) {
  constexpr int D = F::D;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (sm100::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* tiles = smem_raw + (base - sm100::smem_u32(smem_raw));           // one of each warp
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + F::kPairWarps * 2 * F::kTile);  // [F::kPairWarps]
  const int pf = part_floats<D>(a.rows);
  // the warps' parts: where their tiles were, or [F::kPairWarps] of their own; then [cs] the CTAs' parts (rank 0)
  constexpr bool over = F::kPartsOver;
  float* parts = over ? reinterpret_cast<float*>(tiles) : reinterpret_cast<float*>(bars + F::kPairWarps);
  const int per_warp = over ? 2 * F::kTile / 4 : pf;
  float* s_cta = reinterpret_cast<float*>(bars + F::kPairWarps) + (over ? 0 : F::kPairWarps * pf);
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (cs > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  const int pair = blockIdx.x / cs, rank = blockIdx.x - pair * cs;
  const int me = rank * F::kPairWarps + warp, step = cs * F::kPairWarps;
  Worker<F> w{a, &mk, &mv, base + warp * 2 * F::kTile, sm100::smem_u32(bars + warp), lane};
  Cursor c;
  c.b = pair / a.HQ;
  c.h = pair - c.b * a.HQ;
  c.hk = c.h / a.QG;
  c.t = me;
  if (lane == 0) {
    sm100::mbar_init(w.bar, 1);
    sm100::fence_mbar_init();
    s_abort = 0;                        // (every warp: a wait may set it only seconds later)
    if (!F::kFlat && warp == 0) {
      sm100::tma_prefetch_desc(&mk);
      sm100::tma_prefetch_desc(&mv);
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // nothing of an earlier kernel has been touched before
  const int len = a.lengths[c.b];
  c.len = c.T = a.W * a.ps;             // the look-up is bounded by the table row; the length cuts it below
  Box<F> box = w.find_box(c);
  if (me == 0 && c.h == 0 && lane == 0 && len > (int64_t)a.W * a.ps) record_device_error(ENGPT_ERR_ARG, 44);
  typename F::Query qa;
  F::load_query(a, c.b, c.h, lane, qa);
  __syncwarp();
  c.len = clip_length(a, len);
  c.T = (c.len + F::KT - 1) / F::KT;
  if (c.t * F::KT + lane * a.R >= c.len) box.off = -1;
  const int n = c.T > me ? (c.T - me + step - 1) / step : 0;   // this warp's tiles
  Cursor ci = c;
  uint32_t mask = 0;
  typename F::Side side;
  if (n > 0) {
    mask = w.issue(ci, box, side);
    ci.t += step;
    if (n > 1) box = w.find_box(ci);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  typename F::State st;
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
    const int live = c.len - c.t * F::KT;
    if (live >= F::KT && mask == (1u << (F::KT >> a.r_shift)) - 1u)
      F::template step<true>(a, w.tile, qa, side, st, live, mask, lane);
    else
      F::template step<false>(a, w.tile, qa, side, st, live, mask, lane);
    __syncwarp();
    if (i + 1 < n) {
      mask = w.issue(ci, box, side);
      ci.t += step;
      if (i + 2 < n) box = w.find_box(ci);
    }
  }
  F::finish(a, st);

  if (c.T <= 1) {
    if (me == 0 && ok) F::store_rows(a, st, c.b, c.h, lane);
    if (cs > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;
  }
  const int mine = min(max(c.T - rank * F::kPairWarps, 0), F::kPairWarps);   // this CTA's warps with tiles
  if (warp < mine && ok) F::store_part(a, st, parts + warp * per_warp, lane);   // (nothing is being copied any more)
  __syncthreads();
  if (cs == 1) {
    for (int r = warp; r < a.rows; r += F::kPairWarps)
      join_row<F, F::kPairWarps>(a, c.b, c.h, r, mine, [=](int i) { return parts + i * per_warp; }, nullptr, lane);
    return;
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // every CTA of the cluster has started
  if (mine > 0) {
    float* to;
    asm("mapa.u64 %0, %1, %2;" : "=l"(to) : "l"(s_cta + rank * pf), "r"(0));
    for (int r = warp; r < a.rows; r += F::kPairWarps)
      join_row<F, F::kPairWarps>(a, c.b, c.h, r, mine, [=](int i) { return parts + i * per_warp; }, to, lane);
  }
  sm100::cluster_sync_all();
  if (rank == 0) {
    const float* ctas = s_cta;
    const int k = min(cs, (c.T + F::kPairWarps - 1) / F::kPairWarps);                 // CTAs with tiles
    for (int r = warp; r < a.rows; r += F::kPairWarps)
      join_row<F, 8>(a, c.b, c.h, r, k, [=](int i) { return ctas + i * pf; }, nullptr, lane);
  }
}

// Pairs that run over the end of a CTA of decode_list_kernel: a CTA per pair and row of its query heads, or per CTA
// end and row if there are more pairs than CTAs (of `ctas`); every warp takes a share of the parts.
// It starts while that kernel runs (whose CTAs have by then waited for all earlier work) and finds its pair from the
// lengths; only the parts have to wait.
template <typename F>
__global__ void __launch_bounds__(F::kWarps * 32) decode_join_list_kernel(MmaArgs a, int ctas) {
  constexpr int D = F::D, E = D / 32;
  extern __shared__ int s_start[];
  __shared__ float s_o[F::kWarps][D];
  __shared__ float s_m[F::kWarps], s_l[F::kWarps];
  __shared__ int s_scan[F::kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int row_len = 0, row_start = 0;
  const int total = list_starts<F>(a, s_start, s_scan, F::kWarps * 32, false, row_len, row_start);
  const int64_t per = (int64_t)F::kWarps * worker_units<F>(a, total, ctas);   // of a CTA
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
    for (int i = warp; i < n; i += F::kWarps) {
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
      for (int i = 0; i < F::kWarps; ++i) mx = fmaxf(mx, s_m[i]);
      float lx = 0.f, ox = 0.f;
#pragma unroll
      for (int i = 0; i < F::kWarps; ++i) {
        const float wgt = join_weight(s_m[i], mx);
        lx = fmaf(s_l[i], wgt, lx);
        ox = fmaf(s_o[i][threadIdx.x], wgt, ox);
      }
      store1(reinterpret_cast<typename F::T*>(a.o) +
                 ((int64_t)b * a.H + (h / a.QG) * a.G + (h % a.QG) * 8 + r) * a.dim + threadIdx.x,
             lx == 0.f ? 0.f : ox / lx);
    }
  }
}

inline PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

inline int get_encode() {
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

// [D, slots of a page, heads, pages] view of a page pool of `type` (esz bytes each) with element strides s (page, head,
// slot), in boxes of R rows of `row` bytes.
inline int page_map(CUtensorMap* m, const void* base, CUtensorMapDataType type, int esz, int row, CUtensorMapSwizzle swizzle,
                    int D, int ps, int heads, int P, const int64_t* s, int R) {
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)ps, (cuuint64_t)heads, (cuuint64_t)P};
  cuuint64_t strides[3] = {(cuuint64_t)s[2] * esz, (cuuint64_t)s[1] * esz, (cuuint64_t)s[0] * esz};
  cuuint32_t box[4] = {(cuuint32_t)(row / esz), (cuuint32_t)R, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = g_encode(m, type, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle,
                        s[2] == D ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(ENGPT_ERR_ALIGN, "paged_attention: tensor map encode failed (%d)", (int)r);
  return ENGPT_OK;
}

// Width of the tensor-core kernels for a head_dim.
inline int mma_width(int dim) { return dim <= 64 ? 64 : 128; }

inline int64_t most_tiles(int KT, int table_width, int page_size) {
  return ((int64_t)table_width * page_size + KT - 1) / KT;
}

// Can the lists of tiles (of KT keys) of a launch be counted in 32 bits?
inline bool list_fits(int B, int H, int KT, int table_width, int page_size) {
  return B <= kMaxListRows && B * (int64_t)H * (2 * most_tiles(KT, table_width, page_size) + 1) < (1ll << 31);
}

// CTAs per pair of the pair form, or 0 for the list form.
//
// The pair form starts and ends faster (an empty launch takes some 3 us, the list form's two 5.5) but does not balance
// rows of different length, so it is meant to be one wave of CTAs (it is for kPairPerSm CTAs per SM, if F's registers
// leave room for as many).  Its clusters are the widest that run at once: 8 CTAs up
// to one per SM in all (16 pairs of 32 tiles: 4.9 us with 8, 5.8 with 4, 8.3 with 2), 4 or 2 up to two per SM (64 pairs
// of 32 tiles: 10.6 us with 4, 12.1 with 2, 15.3 with 8 in three waves; list 13.1); narrower where a warp would be
// without a tile.  Its warps take their tiles one after the other, 2 us each, where the list form spreads them over all
// SMs at 16 KB / 6.2 TB/s = 1/380 us each: with t tiles per warp the pair form is taken while 2 (t - 1) <= 2 + pairs *
// tiles / 380 (16 pairs of 128 tiles: 12.3 against 13.0 us, 8 pairs of 128: 10.7 against 9.6, 16 pairs of 256: 19.2
// against 18.5; an F gives the time of its own tiles in kTileUs), and, as the rows of a batch may differ and the longest one decides, with at most 4 tiles per warp if
// there are several rows (8 rows of 16 pairs of 32 tiles: 15.4 us against the list's 17.0 if all are that long).
template <typename F>
int pair_ctas(int B, int H, int Hkv, int table_width, int page_size) {
  const int64_t pairs = (int64_t)B * Hkv * ((H / Hkv + 7) / 8);
  const int64_t tiles = most_tiles(F::KT, table_width, page_size);
  const int sms = num_sms();
  const int slots = F::kPairPerSm * sms;
  if (pairs > slots) return 0;
  int cs = pairs * 8 <= sms ? 8 : pairs * 4 <= slots ? 4 : pairs * 2 <= slots ? 2 : 1;
  while (cs > 1 && tiles <= F::kPairWarps * (cs / 2)) cs >>= 1;
  const int64_t per_warp = (tiles + F::kPairWarps * cs - 1) / (F::kPairWarps * cs);
  if (B > 1 && per_warp > 4) return 0;
  return F::kTileUs * (per_warp - 1) <= 2 + pairs * tiles * (2 * F::kTile) / 6200000 ? cs : 0;
}

// Floats of workspace of the list form.
inline int64_t mma_floats(int H, int Hkv, int D) {
  const int rows = H / Hkv < 8 ? H / Hkv : 8;
  return (int64_t)num_sms() * 2 * rows * (mma_width(D) + 2);
}

template <typename F>
size_t mma_smem(int rows, int warps, int parts) {
  return 1024 + (size_t)warps * (2 * F::kTile + 8) + 4 * (size_t)parts * part_floats<F::D>(rows);
}

template <typename F>
int launch_pair(const typename F::Args& a, const CUtensorMap& mk, const CUtensorMap& mv, int cs, cudaStream_t st) {
  auto kern = decode_pair_kernel<F>;
  // Two CTAs per SM and no third one, which would leave other SMs idle (one wave has at most two per SM; 128 pairs of 32
  // tiles: 15.2 us so, 16.5 if three fit).
  constexpr size_t floor = kPairSmem;
  constexpr int own = F::kPartsOver ? 0 : F::kPairWarps;
  const size_t needed = mma_smem<F>(a.rows, F::kPairWarps, own + cs), smem = needed > floor ? needed : floor;
  // (the attribute is the kernel's, not the launch's: every call sets it to the same, largest size, so that a call on
  // another host thread cannot lower it between here and the launch)
  const size_t most = mma_smem<F>(8, F::kPairWarps, own + 8);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)(most > floor ? most : floor));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.HQ * cs));
  cfg.blockDim = dim3(F::kPairWarps * 32);
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

template <typename F>
int launch_list(const typename F::Args& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  auto kern = decode_list_kernel<F>;
  const size_t smem = mma_smem<F>(a.rows, F::kWarps, F::kWarps) + 4 * ((size_t)a.B + 1);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,   // as in launch_pair
                                       (int)(mma_smem<F>(8, F::kWarps, F::kWarps) + 4 * ((size_t)kMaxListRows + 1)));
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "paged_attention: %s", cudaGetErrorString(e));
  // both kernels may be started before what runs ahead of them has ended; they wait for it on the device
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)num_sms());
  cfg.blockDim = dim3(F::kWarps * 32);
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
  e = cudaLaunchKernelEx(&cfg, decode_join_list_kernel<F>, MmaArgs(a), num_sms());
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "paged_attention (join): %s", cudaGetErrorString(e));
  return check_launch("paged_attention (join)");
}

// Everything of a launch but what F adds to its arguments.
template <typename F>
int launch_mma(typename F::Args a, const AttnArgs& x, int Hkv, cudaStream_t st) {
  int rc = F::kFlat ? ENGPT_OK : get_encode();
  if (rc) return rc;
  a.q = x.q;
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
  while (x.ps % (2 << a.r_shift) == 0 && (2 << a.r_shift) <= F::KT) ++a.r_shift;
  a.R = 1 << a.r_shift;
  a.table = x.table;
  a.table_stride = x.table_stride;
  a.W = x.W;
  a.lengths = x.lengths;
  a.scale_log2 = fabsf(x.scale_log2);
  a.negative = x.scale_log2 < 0.f;
  a.o = x.o;
  a.work = x.work;
  CUtensorMap mk = {}, mv = {};
  if constexpr (!F::kFlat) {
    constexpr int esz = F::kCodeBytes;
    if ((rc = page_map(&mk, x.k_pages, F::kMapType, esz, F::kBoxRow, F::kSwizzle, x.Dh, x.ps, Hkv, x.P, x.ks, a.R)))
      return rc;
    if ((rc = page_map(&mv, x.v_pages, F::kMapType, esz, F::kBoxRow, F::kSwizzle, x.Dh, x.ps, Hkv, x.P, x.vs, a.R)))
      return rc;
  }
  const int cs = pair_ctas<F>(x.B, x.H, Hkv, x.W, x.ps);
  // The end of a pair costs a worker about half a tile (its sums and stores, and tiles that are partly empty).  It is
  // counted once workers see such ends often (256 rows of 1 to 512 tokens: 51.8 us, 63.8 without); with few pairs the
  // ranges are whole tiles, which cuts fewer pairs (32 rows of 512 tokens, 16 heads: 16.9 us, 18.5 with).
  const bool ends = 2 * (int64_t)x.B * a.HQ > (int64_t)num_sms() * F::kWarps;
  a.tile_units = ends ? 2 : 1;
  a.end_units = ends ? 1 : 0;
  if (cs == 0) return launch_list<F>(a, mk, mv, st);
  return launch_pair<F>(a, mk, mv, cs, st);
}

}  // namespace paged
}  // namespace engpt
