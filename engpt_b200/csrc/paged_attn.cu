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

// ------------------------------------------------------------------ tensor-core kernel (bf16, head_dim 64 or 128)
//
// A tile is KT keys of one kv head (KT * D = 4096: 8 KB of keys, 8 KB of values).  The tiles of all (row, kv head)
// pairs form one list, cut into equal contiguous ranges, one per warp ("worker") of a persistent grid, so the load
// is even whatever the lengths.  A warp fetches its own tiles through its own ring of STAGES tiles in shared memory:
// TMA boxes of R rows (R divides the page size) at the page that the block table names, 128-byte swizzled, one
// mbarrier per stage; no warp waits for another one until the end.
//
// Per tile, with up to 8 query heads of the kv head as rows 0-7 of the 16-row mma.sync operand:
//   S = Q K^T (rows 8-15 are zero), p = 2^(S scale - m), and O += P V with P's bf16 value in rows 0-7 and the
//   remainder p - bf16(p), again as bf16, in rows 8-15: adding the two halves of O at the end gives the product
//   with weights of 16 mantissa bits for the price of the otherwise idle half of the operand.
// The products are far from bounding anything here (64 mma.sync of 16x8x16 per 16 KB), which is why this is not
// built on tcgen05: its 128-row operand would be 1/128 to 1/16 full and would need TMEM round trips for P.
//
// A range that begins or ends inside a pair leaves a part (o, m, l).  Pairs within one CTA are joined by the warp
// that holds their beginning, after a CTA barrier; a pair that runs over CTAs by decode_join_mma_kernel.
template <int D>
struct Mma {
  static constexpr int KT = 4096 / D;
  static constexpr int NT = KT / 8;     // 8-key tiles
  static constexpr int KC = KT / 16;    // 16-key steps of P V
  static constexpr int DK = D / 16;     // 16-dim steps of Q K^T
  static constexpr int DN = D / 8;      // 8-dim tiles of O
};
constexpr int kTileBytes = 8192;        // one of K, V
constexpr int kWarps = 4;
constexpr int kStages = 3;

struct MmaArgs {
  const __nv_bfloat16* q;
  int64_t q_row, q_head;
  int B, H, G, HQ, QG;     // HQ: (kv head, group of up to 8 query heads) per row; QG: such groups per kv head
  int rows;                // query heads per group, min(G, 8)
  int P, ps, R, r_shift;   // R = 2^r_shift keys per box
  const int* table;
  int64_t table_stride;
  int W;
  const int* lengths;
  float scale_log2;
  __nv_bfloat16* o;
  float* work;             // [workers][2][rows][D + 2], then one Meta per CTA
  int stages;
};

struct Meta {
  int b, h, first, last;   // pair and its workers; first < 0: none
};

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
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// p as bf16 plus the bf16 of what that rounding left.
__device__ __forceinline__ void split_bf16x2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = sm100::pack_bf16x2(x, y);
  const float hx = __uint_as_float(hi << 16), hy = __uint_as_float(hi & 0xffff0000u);
  lo = sm100::pack_bf16x2(x - hx, y - hy);
}

// Usable length of row b without recording (the kernel's prologue records once).
__device__ __forceinline__ int clip_length(const MmaArgs& a, int b) {
  return (int)min((int64_t)max(a.lengths[b], 0), (int64_t)a.W * a.ps);
}

// Position in the list of tiles: tile t of T of (row b of length len, head group h).
struct Cursor {
  int b, h, t, T, len;
};

template <int D>
struct Worker {
  using C = Mma<D>;
  const MmaArgs& a;
  const CUtensorMap *mk, *mv;
  uint32_t ring;            // this warp's stages in shared memory
  uint32_t bars;            // its mbarriers
  int* masks;               // valid boxes of the tile in each stage
  volatile int* abort_flag;
  int lane;

  __device__ __forceinline__ void enter_row(Cursor& c) const {
    c.len = c.b < a.B ? clip_length(a, c.b) : 0;
    c.T = (c.len + C::KT - 1) / C::KT;
  }

  __device__ __forceinline__ void advance(Cursor& c) const {
    if (++c.t < c.T) return;
    c.t = 0;
    if (++c.h < a.HQ) return;
    c.h = 0;
    do {
      ++c.b;
      enter_row(c);
    } while (c.b < a.B && c.T == 0);
  }

  // Page of box `lane` of the cursor's tile: -1 past the length, -2 outside the pool.
  __device__ __forceinline__ int box_page(const Cursor& c) const {
    const int key = c.t * C::KT + lane * a.R;
    if (lane * a.R >= C::KT || key >= c.len) return -1;
    const int page = a.table[c.b * a.table_stride + key / a.ps];
    return page >= 0 && page < a.P ? page : -2;
  }

  // Start the copies of the cursor's tile into stage s.
  __device__ __forceinline__ void issue(const Cursor& c, int page, int s) const {
    const uint32_t mask = __ballot_sync(0xffffffffu, page >= 0);
    const uint32_t bar = bars + 8 * s;
    const uint32_t box = a.R * 128;
    if (lane == 0) {
      masks[s] = (int)mask;
      sm100::mbar_expect_tx(bar, __popc(mask) * box * (D / 64) * 2);
    }
    __syncwarp();
    if (page >= 0) {
      const int key = c.t * C::KT + lane * a.R;
      const int off = key % a.ps, hk = c.h / a.QG;
      const uint32_t dst = ring + s * 2 * kTileBytes + lane * box;
#pragma unroll
      for (int half = 0; half < D / 64; ++half) {
        sm100::tma_load_4d(dst + half * C::KT * 128, mk, half * 64, off, hk, page, bar);
        sm100::tma_load_4d(dst + half * C::KT * 128 + kTileBytes, mv, half * 64, off, hk, page, bar);
      }
    } else if (page == -2) {
      record_device_error(ENGPT_ERR_ARG, 44);
    }
  }

  // A wait ran out: let the copies still in flight land (bounded) before the CTA's shared memory goes away.
  __device__ __forceinline__ void drain(int next, int in_flight, uint32_t phases) const {
    for (int i = 0; i < in_flight; ++i) {
      const int s = (next + i) % a.stages;
      const uint64_t t0 = globaltimer_ns();
      while (!sm100::mbar_try_wait_sleep(bars + 8 * s, (phases >> s) & 1u, 100000u) &&
             globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    }
  }
};

// The running state of one pair: rows 0-7 of S and O in the mma layout (row lane / 4, columns 2 (lane % 4) + {0, 1}
// of each 8-column tile).
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
    qa[k][0] = live ? *reinterpret_cast<const uint32_t*>(q + k * 16) : 0u;
    qa[k][1] = live ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8) : 0u;
  }
}

// One tile: scores, softmax step, P V.  `live` keys from the tile's start are below the length; boxes whose bit of
// `mask` is unset were not copied.
template <int D>
__device__ __forceinline__ void tile_step(const MmaArgs& a, uint32_t sk, const uint32_t (*qa)[2], State<D>& st,
                                          int live, uint32_t mask, int lane) {
  using C = Mma<D>;
  const uint32_t sv = sk + kTileBytes;
  const int r8 = lane & 7, q4 = lane >> 3, t = lane & 3;
  const bool whole = live >= C::KT && mask == (1u << (C::KT >> a.r_shift)) - 1u;
  float s[C::NT][4];
#pragma unroll
  for (int n = 0; n < C::NT; ++n) {
    s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int kp = 0; kp < C::DK / 2; ++kp) {
      uint32_t b[4];
      const int c = kp * 4 + q4;
      ldsm4(sk + (c >> 3) * (C::KT * 128) + (n * 8 + r8) * 128 + (((c & 7) ^ r8) << 4), b);
      mma16816(s[n], qa[2 * kp][0], 0u, qa[2 * kp][1], 0u, b[0], b[1]);
      mma16816(s[n], qa[2 * kp + 1][0], 0u, qa[2 * kp + 1][1], 0u, b[2], b[3]);
    }
  }
  if (!whole) {
    // absent keys: score -inf (weight 0), and values 0, as the weight would not cancel a stale NaN or infinity
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = n * 8 + 2 * t + i;
        if (key >= live || !((mask >> (key >> a.r_shift)) & 1u)) s[n][i] = -INFINITY;
        else s[n][i] *= a.scale_log2;
      }
    for (int i = lane; i < C::KT * (D / 64) * 8; i += 32) {   // 16-byte pieces: half, key, piece
      const int key = (i >> 3) % C::KT;
      if (key >= live || !((mask >> (key >> a.r_shift)) & 1u))
        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(sv + i * 16), "r"(0u) : "memory");
    }
    __syncwarp();
  } else {
#pragma unroll
    for (int n = 0; n < C::NT; ++n) {
      s[n][0] *= a.scale_log2;
      s[n][1] *= a.scale_log2;
    }
  }
  float mx = st.m;
#pragma unroll
  for (int n = 0; n < C::NT; ++n) mx = fmaxf(mx, fmaxf(s[n][0], s[n][1]));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const float ms = mx == -INFINITY ? 0.f : mx;
  const float corr = sm100::ex2_approx(st.m - ms);
  if (__any_sync(0xffffffffu, mx > st.m)) {
#pragma unroll
    for (int i = 0; i < C::DN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) st.o[i][j] *= corr;
    st.l *= corr;
    st.m = mx;
  }
#pragma unroll
  for (int j = 0; j < C::KC; ++j) {
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = sm100::ex2_approx(s[2 * j + (i >> 1)][i & 1] - ms);
      st.l += p[i];
    }
    uint32_t h0, l0, h1, l1;
    split_bf16x2(p[0], p[1], h0, l0);
    split_bf16x2(p[2], p[3], h1, l1);
    const int key = j * 16 + (q4 & 1) * 8 + r8;
#pragma unroll
    for (int dp = 0; dp < C::DN / 2; ++dp) {
      uint32_t b[4];
      const int c = 2 * dp + (q4 >> 1);
      ldsm4_t(sv + (c >> 3) * (C::KT * 128) + key * 128 + (((c & 7) ^ r8) << 4), b);
      mma16816(st.o[2 * dp], h0, l0, h1, l1, b[0], b[1]);
      mma16816(st.o[2 * dp + 1], h0, l0, h1, l1, b[2], b[3]);
    }
  }
  if (!whole) sm100::fence_proxy_async_smem();   // the zeros above, before a later copy into this stage
}

// The pair's sums of this lane: o (both halves of the operand added) and l over the row's four lanes.
template <int D>
__device__ __forceinline__ void finish_rows(State<D>& st) {
  st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
  st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
#pragma unroll
  for (int i = 0; i < Mma<D>::DN; ++i) {
    st.o[i][0] += st.o[i][2];
    st.o[i][1] += st.o[i][3];
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
  __nv_bfloat16* o = a.o + ((int64_t)b * a.H + (h / a.QG) * a.G + in) * D + 2 * t;
  const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
#pragma unroll
  for (int i = 0; i < Mma<D>::DN; ++i)
    *reinterpret_cast<uint32_t*>(o + i * 8) = sm100::pack_bf16x2(st.o[i][0] * inv, st.o[i][1] * inv);
}

// Joins parts (one per index i < n, at part(i)) of a pair, one warp, and stores the rows.
template <int D, typename F>
__device__ __forceinline__ void join_rows(const MmaArgs& a, int b, int h, int n, F part, int lane) {
  constexpr int E = D / 32;
  for (int r = 0; r < a.rows && (h % a.QG) * 8 + r < a.G; ++r) {
    float mx = -INFINITY;
    for (int i = 0; i < n; ++i) mx = fmaxf(mx, part(i)[r * (D + 2) + D]);
    float o[E] = {}, l = 0.f;
    for (int i = 0; i < n; ++i) {
      const float* p = part(i) + r * (D + 2);
      const float w = join_weight(p[D], mx);
      l = fmaf(p[D + 1], w, l);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(p[lane + 32 * e], w, o[e]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    __nv_bfloat16* dst = a.o + ((int64_t)b * a.H + (h / a.QG) * a.G + (h % a.QG) * 8 + r) * D;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[lane + 32 * e] = __float2bfloat16_rn(o[e] * inv);
  }
}

// LIST: the persistent form over the list of tiles.  Otherwise one CTA per pair (its tiles dealt to the four warps
// in contiguous shares, joined in shared memory): no prefix sums, no second launch.
template <int D, bool LIST>
__global__ void __launch_bounds__(kWarps * 32) decode_mma_kernel(MmaArgs a, const __grid_constant__ CUtensorMap mk,
                                                                 const __grid_constant__ CUtensorMap mv) {
  using C = Mma<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (sm100::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* ring_ptr = smem_raw + (base - sm100::smem_u32(smem_raw));
  const int ring_bytes = a.stages * 2 * kTileBytes;
  uint8_t* tail = ring_ptr + kWarps * ring_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tail);                       // [kWarps][stages]
  int* masks = reinterpret_cast<int*>(bars + kWarps * a.stages);            // [kWarps][stages]
  int* s_abort = masks + kWarps * a.stages;
  int* s_scan = s_abort + 1;                                                // [kWarps]
  int* s_start = s_scan + kWarps;                                           // LIST: [B + 1] first tile of each row
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  Worker<D> w{a, &mk, &mv, base + warp * ring_bytes, sm100::smem_u32(bars + warp * a.stages), masks + warp * a.stages,
              s_abort, lane};
  if (lane == 0) {
    for (int s = 0; s < a.stages; ++s) sm100::mbar_init(w.bars + 8 * s, 1);
    sm100::fence_mbar_init();
    sm100::tma_prefetch_desc(&mk);
    sm100::tma_prefetch_desc(&mv);
  }
  if (tid == 0) *s_abort = 0;

  // this worker's range of the list [f0, f1) and its first tile
  const int worker = blockIdx.x * kWarps + warp;
  int f0, f1, per = 0;
  Cursor c;
  if (LIST) {
    // first tile of every row: exclusive prefix sums of tiles(b) * HQ
    int carry = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWarps * 32) {
      const int b = b0 + tid;
      int v = 0;
      if (b < a.B) {
        if (blockIdx.x == 0 && a.lengths[b] > (int64_t)a.W * a.ps) record_device_error(ENGPT_ERR_ARG, 44);
        v = (clip_length(a, b) + C::KT - 1) / C::KT * a.HQ;
      }
      int x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
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
    const int workers = gridDim.x * kWarps;
    per = (carry + workers - 1) / workers;
    f0 = (int)min((int64_t)carry, (int64_t)worker * per);
    f1 = min(carry, f0 + per);
    // last row whose first tile is <= f0 (rows without tiles share their successor's start)
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_start[mid] <= f0) lo = mid;
      else hi = mid;
    }
    c.b = lo;
    w.enter_row(c);
    const int in = f0 - s_start[lo], T = max(c.T, 1);
    c.h = in / T;
    c.t = in - c.h * T;
  } else {
    c.b = blockIdx.x / a.HQ;
    c.h = blockIdx.x - c.b * a.HQ;
    if (tid == 0 && c.h == 0 && a.lengths[c.b] > (int64_t)a.W * a.ps) record_device_error(ENGPT_ERR_ARG, 44);
    w.enter_row(c);
    per = (c.T + kWarps - 1) / kWarps;
    f0 = min(c.T, warp * per);
    f1 = min(c.T, f0 + per);
    c.t = f0;
    __syncthreads();   // *s_abort
  }

  // rows without keys
  if (LIST) {
    for (int64_t i = blockIdx.x * (int64_t)(kWarps * 32) + tid; i < (int64_t)a.B * a.H; i += (int64_t)gridDim.x * kWarps * 32) {
      const int b = (int)(i / a.H);
      if (s_start[b + 1] == s_start[b])
        for (int e = 0; e < D; e += 8) *reinterpret_cast<uint4*>(a.o + i * D + e) = make_uint4(0u, 0u, 0u, 0u);
    }
  }

  // fill the ring
  int n_issued = min(f1 - f0, a.stages);
  Cursor ci = c;
  int page = n_issued > 0 ? w.box_page(ci) : -1;
  for (int s = 0; s < n_issued; ++s) {
    Cursor cn = ci;
    w.advance(cn);
    const int pn = f0 + s + 1 < f1 ? w.box_page(cn) : -1;
    w.issue(ci, page, s);
    ci = cn;
    page = pn;
  }

  const int pair_tiles = c.T;   // one CTA per pair: its tiles
  State<D> st;
  st.reset();
  uint32_t qa[C::DK][2];
  uint32_t phases = 0;
  bool fresh = true;          // the next tile begins a segment
  bool ok = true, cut = false;
  int t0 = 0, my_last = 0;
  Cursor mine = c;            // the pair whose beginning this worker holds and whose end it does not
  int s = 0;
  for (int f = f0; f < f1; ++f) {
    if (fresh) {
      load_query<D>(a, c.b, c.h, lane, qa);
      t0 = c.t;
      fresh = false;
    }
    if (!__all_sync(0xffffffffu, sm100::mbar_wait(w.bars + 8 * s, (phases >> s) & 1u, s_abort, 45))) {
      w.drain(s, min(f1 - f, a.stages), phases);
      ok = false;
      break;
    }
    phases ^= 1u << s;
    tile_step<D>(a, w.ring + s * 2 * kTileBytes, qa, st, c.len - c.t * C::KT, (uint32_t)w.masks[s], lane);
    __syncwarp();
    if (f + a.stages < f1) {
      w.issue(ci, page, s);
      w.advance(ci);
      page = f + a.stages + 1 < f1 ? w.box_page(ci) : -1;
    }
    if (++s == a.stages) s = 0;
    const bool pair_end = c.t + 1 == c.T;
    if (pair_end || f + 1 == f1) {
      finish_rows<D>(st);
      if (LIST) {
        if (t0 == 0 && pair_end) {
          store_rows<D>(a, st, c.b, c.h, lane);
        } else {
          store_part<D>(a, st, a.work + ((int64_t)worker * 2 + (t0 == 0 ? 1 : 0)) * a.rows * (D + 2), lane);
          if (t0 == 0) {
            cut = true;
            mine = c;
            my_last = (s_start[c.b] + (c.h + 1) * c.T - 1) / per;
          }
        }
        st.reset();
        fresh = true;
      }
    }
    w.advance(c);
  }

  if (LIST) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ Meta s_meta;
    if (tid == 0) s_meta.first = -1;
    __syncthreads();   // every worker's parts are written
    if (cut && ok) {
      if (my_last / kWarps == (int)blockIdx.x) {
        const int first = worker, rows = a.rows;
        const float* work = a.work;
        join_rows<D>(a, mine.b, mine.h, my_last - first + 1,
                     [=](int i) { return work + ((int64_t)(first + i) * 2 + (i == 0 ? 1 : 0)) * rows * (D + 2); }, lane);
      } else if (lane == 0) {
        s_meta = Meta{mine.b, mine.h, worker, my_last};   // at most one pair runs over the CTA's end
      }
    }
    __syncthreads();
    if (tid == 0) {
      Meta* metas = reinterpret_cast<Meta*>(a.work + (int64_t)gridDim.x * kWarps * 2 * a.rows * (D + 2));
      metas[blockIdx.x] = s_meta;
    }
  } else {
    // parts in each warp's own (by now unused) ring memory
    float* part = reinterpret_cast<float*>(ring_ptr + warp * ring_bytes);
    if (f0 >= f1) finish_rows<D>(st);
    const int n = per > 0 ? (pair_tiles + per - 1) / per : 0;
    __syncwarp();
    if (n > 1 && ok) store_part<D>(a, st, part, lane);
    __syncthreads();
    const int b = blockIdx.x / a.HQ, h = blockIdx.x - b * a.HQ;
    if (warp == 0 && ok) {
      if (n <= 1)
        store_rows<D>(a, st, b, h, lane);
      else
        join_rows<D>(a, b, h, n, [=](int i) { return reinterpret_cast<const float*>(ring_ptr + i * ring_bytes); }, lane);
    }
  }
}

// Pairs that run over the end of a CTA of decode_mma_kernel: one CTA per such end, a warp's share of the parts each.
template <int D>
__global__ void __launch_bounds__(256) decode_join_mma_kernel(MmaArgs a, int ctas) {
  constexpr int E = D / 32, NW = 8;
  __shared__ float s_o[NW][D];
  __shared__ float s_m[NW], s_l[NW];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Meta mt = reinterpret_cast<const Meta*>(a.work + (int64_t)ctas * kWarps * 2 * a.rows * (D + 2))[blockIdx.x];
  if (mt.first < 0) return;
  const int n = mt.last - mt.first + 1;
  for (int r = 0; r < a.rows && (mt.h % a.QG) * 8 + r < a.G; ++r) {
    float m = -INFINITY, l = 0.f, o[E] = {};
    for (int i = warp; i < n; i += NW) {
      const float* p = a.work + (((int64_t)(mt.first + i) * 2 + (i == 0 ? 1 : 0)) * a.rows + r) * (D + 2);
      const float pm = p[D], mx = fmaxf(m, pm);
      const float w0 = join_weight(m, mx), w1 = join_weight(pm, mx);
      l = l * w0 + p[D + 1] * w1;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * w0 + p[lane + 32 * e] * w1;
      m = mx;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = o[e];
    if (lane == 0) {
      s_m[warp] = m;
      s_l[warp] = l;
    }
    __syncthreads();
    if (threadIdx.x < D) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NW; ++i) mx = fmaxf(mx, s_m[i]);
      float lx = 0.f, ox = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const float wgt = join_weight(s_m[i], mx);
        lx = fmaf(s_l[i], wgt, lx);
        ox = fmaf(s_o[i][threadIdx.x], wgt, ox);
      }
      a.o[((int64_t)mt.b * a.H + (mt.h / a.QG) * a.G + (mt.h % a.QG) * 8 + r) * D + threadIdx.x] =
          __float2bfloat16_rn(lx == 0.f ? 0.f : ox / lx);
    }
  }
}

static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

static int get_encode() {
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

inline int tile_keys(int D) { return 4096 / D; }

inline int64_t most_tiles(int D, int table_width, int page_size) {
  return ((int64_t)table_width * page_size + tile_keys(D) - 1) / tile_keys(D);
}

// Does a launch of these sizes go to the tensor-core kernel (strides and alignment apart)?
inline bool mma_sizes(int dtype, int B, int H, int Hkv, int D, int table_width, int page_size) {
  return dtype == ENGPT_BF16 && (D == 64 || D == 128) && page_size % 8 == 0 && B <= 8192 &&
         B * (int64_t)H * most_tiles(D, table_width, page_size) < (1ll << 31);
}

// One CTA per pair while the longest row that the table can hold has at most this many tiles per warp.
constexpr int kPairTiles = 2;

inline bool mma_list(int D, int table_width, int page_size) {
  return most_tiles(D, table_width, page_size) > kPairTiles * kWarps;
}

inline int64_t mma_floats(int H, int Hkv, int D) {
  const int rows = H / Hkv < 8 ? H / Hkv : 8;
  return (int64_t)num_sms() * (kWarps * 2 * (int64_t)rows * (D + 2) + 4);
}

template <int D, bool LIST>
int launch_mma_kernel(const MmaArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  auto kern = decode_mma_kernel<D, LIST>;
  const size_t smem = 1024 + (size_t)kWarps * a.stages * (2 * kTileBytes + 12) + 8 + 4 * kWarps +
                      (LIST ? 4 * ((size_t)a.B + 1) : 0);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "paged_attention: %s", cudaGetErrorString(e));
  const unsigned grid = LIST ? (unsigned)num_sms() : (unsigned)((int64_t)a.B * a.HQ);
  kern<<<grid, kWarps * 32, smem, st>>>(a, mk, mv);
  int rc = check_launch("paged_attention");
  if (rc || !LIST) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, decode_join_mma_kernel<D>, a, (int)grid);
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
  a.q_head = x.q_head;
  a.B = x.B;
  a.H = x.H;
  a.G = x.G;
  a.QG = (x.G + 7) / 8;
  a.HQ = Hkv * a.QG;
  a.rows = x.G < 8 ? x.G : 8;
  a.P = x.P;
  a.ps = x.ps;
  a.r_shift = 3;
  while (x.ps % (2 << a.r_shift) == 0 && (2 << a.r_shift) <= tile_keys(D)) ++a.r_shift;
  a.R = 1 << a.r_shift;
  a.table = x.table;
  a.table_stride = x.table_stride;
  a.W = x.W;
  a.lengths = x.lengths;
  a.scale_log2 = x.scale_log2;
  a.o = reinterpret_cast<__nv_bfloat16*>(x.o);
  a.work = x.work;
  CUtensorMap mk, mv;
  if ((rc = page_map(&mk, x.k_pages, D, x.ps, Hkv, x.P, x.ks, a.R))) return rc;
  if ((rc = page_map(&mv, x.v_pages, D, x.ps, Hkv, x.P, x.vs, a.R))) return rc;
  if (mma_list(D, x.W, x.ps)) {
    a.stages = kStages;
    return launch_mma_kernel<D, true>(a, mk, mv, st);
  }
  const int64_t per = (most_tiles(D, x.W, x.ps) + kWarps - 1) / kWarps;
  a.stages = per < 1 ? 1 : (per < kStages ? (int)per : kStages);
  return launch_mma_kernel<D, false>(a, mk, mv, st);
}

}  // namespace paged
}  // namespace engpt

using namespace engpt;
using namespace engpt::paged;

extern "C" int64_t engpt_paged_attention_floats(int dtype, int B, int H, int Hkv, int Dh, int table_width,
                                                int page_size) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || Dh <= 0 || table_width < 0 || page_size <= 0) return 0;
  const int splits = simt_splits(B, H, (int64_t)table_width * page_size);
  const int64_t simt = splits > 1 ? (int64_t)B * H * splits * (Dh + 2) : 0;
  if (!mma_sizes(dtype, B, H, Hkv, Dh, table_width, page_size)) return simt;
  // strides and alignment decide at the call which of the two kernels runs
  const int64_t mma = mma_list(Dh, table_width, page_size) ? mma_floats(H, Hkv, Dh) : 0;
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
  if (vec && positive && num_pages > 0 && mma_sizes(dtype, B, H, Hkv, Dh, table_width, page_size))
    return Dh == 64 ? launch_mma<64>(a, Hkv, st) : launch_mma<128>(a, Hkv, st);
  return dtype == ENGPT_BF16 ? dispatch_simt<__nv_bfloat16>(a, vec, st) : dispatch_simt<float>(a, vec, st);
}
