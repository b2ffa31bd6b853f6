// The paged key-value cache's bookkeeping and its plain write.
//
// advance_block_tables: with h_b the pages that a finished row holds and
// n_b = ceil((len_b + new_b) / ps) - ceil(len_b / ps) the pages that row b
// needs, the stack of free pages grows by the rows' pages at the exclusive
// prefix sums of h_b and shrinks from its top at the exclusive prefix sums of
// n_b; everything else is one table look-up per new token.
//
// write_kv_pages: a gathered copy, bound by HBM.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace engpt {
namespace paged {

constexpr int kMaxRows = 8192;      // five ints of shared memory per row
constexpr int kTableCluster = 8;    // CTAs of a large launch
constexpr int kPiece = 128;         // pages that a warp pushes at a time (four loads in flight per lane)

struct TableArgs {
  int* lengths;
  const int* new_tokens;
  const unsigned char* finished;
  int B;
  int* table;
  int64_t table_stride;
  int W;
  int* free_pages;
  int P;
  int* free_count;
  int ps;
  int max_new;
  int* slots;
  int* positions;
};

__device__ __forceinline__ int64_t warp_inclusive_sum(int64_t x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// One step of the allocator by one cluster (of one CTA for a small step).  Every CTA reads all rows and forms all
// prefix sums for itself; the cluster shares the copying of freed pages and, behind a barrier (everything that the
// step overwrites has been read), the new tokens, U consecutive ones of a row per thread.  Latency bound: two
// dependent trips to memory before the barrier, two behind it.
template <int U>
__global__ void __launch_bounds__(1024) advance_tables_kernel(TableArgs a, int ctas) {
  extern __shared__ int s_rows[];
  int* s_len = s_rows;               // length after the release
  int* s_new = s_rows + a.B;         // new tokens; -1: refused
  int* s_off = s_rows + 2 * a.B;     // pages taken by the rows before
  int* s_held = s_rows + 3 * a.B;    // pages to push
  int* s_push = s_rows + 4 * a.B;    // pages pushed by the rows before
  __shared__ int64_t s_warp[2][32];
  __shared__ int s_taken;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
  const int rank = blockIdx.x;       // the grid is one cluster
  const bool first = rank == 0;      // records what every CTA sees

  if (tid == 0) s_taken = 0;
  int n_free = *a.free_count;
  if (n_free < 0 || n_free > a.P) {
    if (first && tid == 0) record_device_error(ENGPT_ERR_ARG, 40);
    n_free = n_free < 0 ? 0 : a.P;
  }
  int64_t pushed = 0, needed = 0;
  for (int b0 = 0; b0 < a.B; b0 += threads) {
    const int b = b0 + tid;
    int held = 0, need = 0;
    if (b < a.B) {
      int len = max(a.lengths[b], 0), fresh = a.new_tokens[b];
      if (a.finished && a.finished[b]) {
        held = min((int)(((int64_t)len + a.ps - 1) / a.ps), a.W);
        len = 0;
      }
      const int64_t end = (int64_t)len + fresh;
      if (fresh < 0 || fresh > a.max_new || end > (int64_t)a.W * a.ps) {
        if (first) record_device_error(ENGPT_ERR_ARG, 40);
        fresh = -1;
      } else {
        need = (int)((uint32_t)(end + a.ps - 1) / (uint32_t)a.ps - ((uint32_t)len + a.ps - 1) / (uint32_t)a.ps);
      }
      s_len[b] = len;
      s_new[b] = fresh;
      s_held[b] = held;
    }
    const int64_t xh = warp_inclusive_sum(held, lane), xn = warp_inclusive_sum(need, lane);
    if (lane == 31) {
      s_warp[0][warp] = xh;
      s_warp[1][warp] = xn;
    }
    __syncthreads();
    if (warp < 2) {
      const int64_t v = lane < warps ? s_warp[warp][lane] : 0;
      s_warp[warp][lane] = warp_inclusive_sum(v, lane);
    }
    __syncthreads();
    if (b < a.B) {
      const int64_t most = 0x7fffffff;
      s_push[b] = (int)min(pushed + (warp ? s_warp[0][warp - 1] : 0) + xh - held, most);
      s_off[b] = (int)min(needed + (warp ? s_warp[1][warp - 1] : 0) + xn - need, most);
      // (whether the stack is deep enough for the row is known when everything has been pushed, below)
    }
    pushed += s_warp[0][31];
    needed += s_warp[1][31];
    __syncthreads();
  }
  // finished rows push their pages, a warp per piece of a row
  if (pushed > 0) {
    const int pieces = (a.W + kPiece - 1) / kPiece;
    const int64_t total = (int64_t)a.B * pieces;
    for (int64_t i = rank * warps + warp; i < total; i += (int64_t)ctas * warps) {
      const int b = total <= 0xffffffffLL ? (int)((uint32_t)i / (uint32_t)pieces) : (int)(i / pieces);
      const int j0 = (int)(i - (int64_t)b * pieces) * kPiece;
      const int held = s_held[b];
      if (j0 >= held) continue;
      const int* row = a.table + b * a.table_stride;
      int page[kPiece / 32];
#pragma unroll
      for (int k = 0; k < kPiece / 32; ++k) {
        const int j = j0 + k * 32 + lane;
        page[k] = j < held ? row[j] : 0;
      }
#pragma unroll
      for (int k = 0; k < kPiece / 32; ++k) {
        const int j = j0 + k * 32 + lane;
        const int64_t at = (int64_t)n_free + s_push[b] + j;
        if (j < held) {
          if (at < a.P) a.free_pages[at] = page[k];
          else record_device_error(ENGPT_ERR_ARG, 40);
        }
      }
    }
  }
  n_free = (int)min((int64_t)n_free + pushed, (int64_t)a.P);
  // rows that the stack is too short for.  The sums grow with the row, so the rows behind the first one that found
  // too few pages get none either, and the pages taken are those up to the last row that was served.
  for (int b = tid; b < a.B; b += threads) {
    const int len = s_len[b], fresh = s_new[b];
    if (fresh <= 0) continue;
    const int need = (int)(((uint32_t)len + fresh + a.ps - 1) / (uint32_t)a.ps - ((uint32_t)len + a.ps - 1) / (uint32_t)a.ps);
    if (need == 0) continue;
    if ((int64_t)s_off[b] + need > n_free) {
      if (first) record_device_error(ENGPT_ERR_ARG, 41);
      s_new[b] = -1;
    } else if (needed > n_free) {
      atomicMax(&s_taken, s_off[b] + need);
    }
  }
  if (ctas > 1) sm100::cluster_sync_all();
  else __syncthreads();
  // slots and positions; the first token of a page enters the page into the table
  const uint32_t per_row = (uint32_t)a.max_new / U;
  const uint32_t total = (uint32_t)a.B * per_row;
  for (uint32_t t = rank * threads + tid; t < total; t += ctas * threads) {
    const uint32_t b = per_row == 1 ? t : t / per_row;
    const int i0 = (int)(t - b * per_row) * U;
    const int fresh = s_new[b], len = s_len[b];
    int slot[U], pos[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      slot[u] = -1;
      pos[u] = 0;
    }
    if (i0 < fresh) {
      const int have = (int)(((uint32_t)len + a.ps - 1) / (uint32_t)a.ps);
      int j = (int)((uint32_t)(len + i0) / (uint32_t)a.ps), r = len + i0 - j * a.ps;
      int* entry = a.table + b * a.table_stride;
      const int* stack = a.free_pages + (n_free - 1 - s_off[b]);
      int page = j < have ? entry[j] : stack[have - j];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + u < fresh) {
          if (r == a.ps) {
            ++j;
            r = 0;
            page = stack[have - j];
          }
          if (r == 0) entry[j] = page;
          slot[u] = page * a.ps + r;
          pos[u] = len + i0 + u;
          ++r;
        }
      }
    }
    if constexpr (U == 4) {
      reinterpret_cast<int4*>(a.slots)[t] = make_int4(slot[0], slot[1], slot[2], slot[3]);
      reinterpret_cast<int4*>(a.positions)[t] = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
      a.slots[t] = slot[0];
      a.positions[t] = pos[0];
    }
  }
  if (first) {
    for (int b = tid; b < a.B; b += threads) a.lengths[b] = s_len[b] + max(s_new[b], 0);
    if (tid == 0) *a.free_count = n_free - (needed > n_free ? s_taken : (int)needed);
  }
}

// ------------------------------------------------------------------ write
struct WriteArgs {
  const void* k;
  const void* v;
  int64_t k_row, k_head, v_row, v_head;
  int64_t n;
  int H, Dh;
  const int* slots;
  void* k_pages;
  void* v_pages;
  int64_t ks[3], vs[3];
  int64_t n_slots;
  int ps, ps_shift;   // ps_shift: log2(page size), or -1
};

// 32768 tokens of 16 heads of 64 in bf16, 15 of 16 with a slot (252 MB move): 42.3 us = 5.95 TB/s with two pieces and
// 8 CTAs per SM; 46.7 with one piece, 46.1 with four, 45.4 with 32 CTAs.  All 32768 with one (268 MB): 44.2 us = 6.07 TB/s.
constexpr int kWriteUnroll = 2, kWriteCtas = 8;

// One thread per V-sized piece of a (token, head) row, for k and v, U pieces a grid apart at a time: all their slots,
// then all their loads are in flight before the first store.  V: uint4 (16 bytes), or the element itself.
template <typename V, int U>
__global__ void __launch_bounds__(256) write_pages_kernel(WriteArgs a, int pieces, int esz) {
  const uint32_t per_row = (uint32_t)a.H * pieces;
  const int64_t total = a.n * per_row, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i0 = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i0 < total; i0 += U * step) {
    int slot[U];
    int64_t row[U];
    int h[U], c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * step;
      row[u] = total <= 0xffffffffLL ? (uint32_t)i / per_row : i / per_row;
      const uint32_t rest = (uint32_t)(i - row[u] * per_row);
      h[u] = (int)(rest / (uint32_t)pieces);
      c[u] = (int)(rest - h[u] * (uint32_t)pieces);
      slot[u] = i < total ? a.slots[row[u]] : -1;
    }
    V kv[U], vv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (slot[u] >= 0 && slot[u] < a.n_slots) {
        const int64_t byte = (int64_t)c[u] * sizeof(V);
        kv[u] = *reinterpret_cast<const V*>((const char*)a.k + (row[u] * a.k_row + h[u] * a.k_head) * esz + byte);
        vv[u] = *reinterpret_cast<const V*>((const char*)a.v + (row[u] * a.v_row + h[u] * a.v_head) * esz + byte);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (slot[u] >= 0 && slot[u] < a.n_slots) {
        const int page = a.ps_shift >= 0 ? slot[u] >> a.ps_shift : slot[u] / a.ps;
        const int off = slot[u] - page * a.ps;
        const int64_t byte = (int64_t)c[u] * sizeof(V);
        *reinterpret_cast<V*>((char*)a.k_pages + (page * a.ks[0] + h[u] * a.ks[1] + off * a.ks[2]) * esz + byte) = kv[u];
        *reinterpret_cast<V*>((char*)a.v_pages + (page * a.vs[0] + h[u] * a.vs[1] + off * a.vs[2]) * esz + byte) = vv[u];
      } else if (slot[u] != -1) {
        record_device_error(ENGPT_ERR_ARG, 43);
      }
    }
  }
}

}  // namespace paged
}  // namespace engpt

using namespace engpt;
using namespace engpt::paged;

extern "C" int engpt_advance_block_tables(int* lengths, const int* new_tokens, const unsigned char* finished, int B,
                                          int* block_table, int64_t table_stride, int table_width, int* free_pages,
                                          int num_pages, int* free_count, int page_size, int max_new, int* slots,
                                          int* positions, void* stream) {
  clear_error();
  ENGPT_REQUIRE(B >= 0 && max_new >= 0 && table_width >= 0 && table_stride >= table_width, ENGPT_ERR_SHAPE,
                "advance_block_tables: B=%d max_new=%d table_width=%d", B, max_new, table_width);
  ENGPT_REQUIRE(num_pages >= 0 && page_size > 0 && (int64_t)num_pages * page_size <= 0x7fffffffLL, ENGPT_ERR_SHAPE,
                "advance_block_tables: num_pages=%d page_size=%d", num_pages, page_size);
  ENGPT_REQUIRE((int64_t)table_width * page_size <= 0x7fffffffLL, ENGPT_ERR_SHAPE,
                "advance_block_tables: table_width=%d page_size=%d", table_width, page_size);
  ENGPT_REQUIRE(B <= kMaxRows, ENGPT_ERR_UNSUPPORTED, "advance_block_tables: %d rows (at most %d)", B, kMaxRows);
  if (B == 0) return ENGPT_OK;
  ENGPT_REQUIRE(lengths && new_tokens && free_count && (block_table || table_width == 0) &&
                    (free_pages || num_pages == 0) && ((slots && positions) || max_new == 0),
                ENGPT_ERR_ARG, "advance_block_tables: null pointer");
  TableArgs a{lengths, new_tokens, finished, B, block_table, table_stride, table_width, free_pages, num_pages,
              free_count, page_size, max_new, slots, positions};
  ENGPT_REQUIRE((int64_t)B * max_new <= 0x7fffffffLL, ENGPT_ERR_SHAPE, "advance_block_tables: B=%d max_new=%d", B,
                max_new);
  const bool vec = max_new % 4 == 0 && aligned(slots, 16) && aligned(positions, 16);
  // A step of a few hundred rows is one small CTA (less to start); longer ones share the tokens and the freed pages
  // over a cluster.
  const bool small = B <= 256 && (int64_t)B * max_new <= 1024;
  const int ctas = small ? 1 : kTableCluster;
  const size_t smem = sizeof(int) * 5 * (size_t)B;
  auto kern = vec ? advance_tables_kernel<4> : advance_tables_kernel<1>;
  // (the attribute is the kernel's, not the launch's: every call that needs it sets the same, largest size, so that a
  // call on another host thread cannot lower it between here and the launch)
  cudaError_t e = cudaSuccess;
  if (smem > 40 * 1024)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(int) * 5 * kMaxRows);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(small ? 256 : 1024);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kern, a, ctas);
  if (e != cudaSuccess) return set_error(ENGPT_ERR_LAUNCH, "advance_block_tables: %s", cudaGetErrorString(e));
  return check_launch("advance_block_tables");
}

extern "C" int engpt_write_kv_pages(const void* k, const void* v, const int64_t* kv_strides, int dtype, int64_t n,
                                    int H, int Dh, const int* slots, void* k_pages, void* v_pages,
                                    const int64_t* page_strides, int num_pages, int page_size, void* stream) {
  clear_error();
  ENGPT_REQUIRE(n >= 0 && n <= 0x7fffffffLL && H > 0 && Dh > 0, ENGPT_ERR_SHAPE, "write_kv_pages: n=%lld H=%d Dh=%d",
                (long long)n, H, Dh);
  ENGPT_REQUIRE(num_pages >= 0 && page_size > 0 && (int64_t)num_pages * page_size <= 0x7fffffffLL, ENGPT_ERR_SHAPE,
                "write_kv_pages: num_pages=%d page_size=%d", num_pages, page_size);
  ENGPT_REQUIRE(dtype == ENGPT_BF16 || dtype == ENGPT_F32, ENGPT_ERR_DTYPE, "write_kv_pages: dtype %d", dtype);
  if (n == 0) return ENGPT_OK;
  ENGPT_REQUIRE(k && v && kv_strides && slots && k_pages && v_pages && page_strides, ENGPT_ERR_ARG,
                "write_kv_pages: null pointer");
  const int esz = dtype == ENGPT_BF16 ? 2 : 4;
  WriteArgs a;
  a.k = k;
  a.v = v;
  a.k_row = kv_strides[0];
  a.k_head = kv_strides[1];
  a.v_row = kv_strides[2];
  a.v_head = kv_strides[3];
  a.n = n;
  a.H = H;
  a.Dh = Dh;
  a.slots = slots;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.n_slots = (int64_t)num_pages * page_size;
  a.ps = page_size;
  a.ps_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1;
  bool vec = Dh * esz % 16 == 0 && aligned(k, 16) && aligned(v, 16) && aligned(k_pages, 16) && aligned(v_pages, 16);
  for (int i = 0; i < 4; ++i) vec = vec && kv_strides[i] * esz % 16 == 0;
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = page_strides[i];
    a.vs[i] = page_strides[3 + i];
    vec = vec && a.ks[i] * esz % 16 == 0 && a.vs[i] * esz % 16 == 0;
  }
  const int pieces = vec ? Dh * esz / 16 : Dh;
  const int64_t total = n * H * pieces;
  ENGPT_REQUIRE((int64_t)H * pieces <= 0x7fffffffLL, ENGPT_ERR_SHAPE, "write_kv_pages: H=%d Dh=%d", H, Dh);
  const int64_t want = (total + 255) / 256, cap = (int64_t)num_sms() * kWriteCtas;
  const unsigned blocks = (unsigned)(want < cap ? want : cap);
  cudaStream_t st = as_stream(stream);
  if (vec) write_pages_kernel<uint4, kWriteUnroll><<<blocks, 256, 0, st>>>(a, pieces, esz);
  else if (esz == 2) write_pages_kernel<unsigned short, 1><<<blocks, 256, 0, st>>>(a, pieces, esz);
  else write_pages_kernel<float, 1><<<blocks, 256, 0, st>>>(a, pieces, esz);
  return check_launch("write_kv_pages");
}
