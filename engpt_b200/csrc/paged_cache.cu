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

namespace engpt {
namespace paged {

constexpr int kTableThreads = 1024;
constexpr int kMaxRows = 8192;   // three ints of shared memory per row

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

// Exclusive prefix sum over the CTA's threads (thread order), with the total.
__device__ __forceinline__ int64_t block_exclusive_sum(int v, int64_t* s_warp, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int64_t w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  const int64_t before = warp ? s_warp[warp - 1] : 0;
  total = s_warp[31];
  __syncthreads();
  return before + x - v;
}

__global__ void __launch_bounds__(kTableThreads) advance_tables_kernel(TableArgs a) {
  extern __shared__ int s_rows[];
  int* s_len = s_rows;              // length after the release
  int* s_off = s_rows + a.B;        // pages pushed, then pages taken, by the rows before
  int* s_new = s_rows + 2 * a.B;    // new tokens; -1: refused
  __shared__ int64_t s_warp[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  int n_free = *a.free_count;
  if (n_free < 0 || n_free > a.P) {
    if (tid == 0) record_device_error(ENGPT_ERR_ARG, 40);
    n_free = n_free < 0 ? 0 : a.P;
  }
  // 1. finished rows push their pages
  int64_t pushed = 0;
  for (int b0 = 0; b0 < a.B; b0 += kTableThreads) {
    const int b = b0 + tid;
    int len = 0, held = 0;
    if (b < a.B) {
      len = max(a.lengths[b], 0);
      if (a.finished && a.finished[b]) held = min((int)(((int64_t)len + a.ps - 1) / a.ps), a.W);
    }
    int64_t total;
    const int64_t off = block_exclusive_sum(held, s_warp, total) + pushed;
    pushed += total;
    if (b < a.B) {
      s_len[b] = len;
      s_off[b] = (int)min(off, (int64_t)0x7fffffff);
    }
  }
  __syncthreads();
  if (a.finished) {
    for (int b = warp; b < a.B; b += kTableThreads / 32) {
      if (!a.finished[b]) continue;
      const int held = min((int)(((int64_t)s_len[b] + a.ps - 1) / a.ps), a.W);
      const int* row = a.table + b * a.table_stride;
      for (int j = lane; j < held; j += 32) {
        const int64_t at = (int64_t)n_free + s_off[b] + j;
        if (at < a.P) a.free_pages[at] = row[j];
        else record_device_error(ENGPT_ERR_ARG, 40);
      }
      __syncwarp();
      if (lane == 0) s_len[b] = 0;
    }
    __syncthreads();
  }
  n_free = (int)min((int64_t)n_free + pushed, (int64_t)a.P);
  // 2. pages for the new tokens
  int64_t need_before = 0;
  int taken = 0;
  for (int b0 = 0; b0 < a.B; b0 += kTableThreads) {
    const int b = b0 + tid;
    int need = 0, fresh = 0;
    if (b < a.B) {
      fresh = a.new_tokens[b];
      const int64_t len = s_len[b], end = len + fresh;
      if (fresh < 0 || fresh > a.max_new || end > (int64_t)a.W * a.ps) {
        record_device_error(ENGPT_ERR_ARG, 40);
        fresh = -1;
      } else {
        need = (int)((end + a.ps - 1) / a.ps - (len + a.ps - 1) / a.ps);
      }
    }
    int64_t total;
    const int64_t off = block_exclusive_sum(need, s_warp, total) + need_before;
    need_before += total;
    if (need > 0 && off + need > n_free) {   // off grows with b: once the stack is short it stays short
      record_device_error(ENGPT_ERR_ARG, 41);
      fresh = -1;
      need = 0;
    }
    int64_t got;
    block_exclusive_sum(need, s_warp, got);
    taken += (int)got;
    if (b < a.B) {
      s_off[b] = (int)min(off, (int64_t)0x7fffffff);
      s_new[b] = fresh;
    }
  }
  __syncthreads();
  // 3. slots and positions; the first token of a page enters the page into the table
  const int64_t tokens = (int64_t)a.B * a.max_new;
  for (int64_t t = tid; t < tokens; t += kTableThreads) {
    const int b = (int)(t / a.max_new), i = (int)(t - (int64_t)b * a.max_new);
    int slot = -1, pos = 0;
    if (i < s_new[b]) {
      const int len = s_len[b];
      pos = len + i;
      const int j = pos / a.ps, r = pos - j * a.ps;
      const int have = (int)(((int64_t)len + a.ps - 1) / a.ps);
      int* entry = a.table + b * a.table_stride + j;
      int page;
      if (j < have) {
        page = *entry;
      } else {
        page = a.free_pages[n_free - 1 - s_off[b] - (j - have)];
        if (r == 0) *entry = page;
      }
      slot = page * a.ps + r;
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
  for (int b = tid; b < a.B; b += kTableThreads) a.lengths[b] = s_len[b] + max(s_new[b], 0);
  if (tid == 0) *a.free_count = n_free - taken;
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
  int ps;
};

// One thread per V-sized piece of a (token, head) row, for k and v.  V: uint4 (16 bytes), or the element itself.
template <typename V>
__global__ void __launch_bounds__(256) write_pages_kernel(WriteArgs a, int pieces, int esz) {
  const int64_t per_row = (int64_t)a.H * pieces;
  const int64_t total = a.n * per_row;
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t row = i / per_row;
    const int rest = (int)(i - row * per_row);
    const int h = rest / pieces, c = rest - h * pieces;
    const int slot = a.slots[row];
    if (slot < 0 || slot >= a.n_slots) {
      if (slot != -1) record_device_error(ENGPT_ERR_ARG, 43);
      continue;
    }
    const int page = slot / a.ps, off = slot - page * a.ps;
    const int64_t byte = (int64_t)c * sizeof(V);
    const V kv = *reinterpret_cast<const V*>((const char*)a.k + (row * a.k_row + h * a.k_head) * esz + byte);
    const V vv = *reinterpret_cast<const V*>((const char*)a.v + (row * a.v_row + h * a.v_head) * esz + byte);
    *reinterpret_cast<V*>((char*)a.k_pages + (page * a.ks[0] + h * a.ks[1] + off * a.ks[2]) * esz + byte) = kv;
    *reinterpret_cast<V*>((char*)a.v_pages + (page * a.vs[0] + h * a.vs[1] + off * a.vs[2]) * esz + byte) = vv;
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
  const size_t smem = sizeof(int) * 3 * (size_t)B;
  if (smem > 48 * 1024)
    cudaFuncSetAttribute(advance_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  advance_tables_kernel<<<1, kTableThreads, smem, as_stream(stream)>>>(a);
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
  bool vec = Dh * esz % 16 == 0 && aligned(k, 16) && aligned(v, 16) && aligned(k_pages, 16) && aligned(v_pages, 16);
  for (int i = 0; i < 4; ++i) vec = vec && kv_strides[i] * esz % 16 == 0;
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = page_strides[i];
    a.vs[i] = page_strides[3 + i];
    vec = vec && a.ks[i] * esz % 16 == 0 && a.vs[i] * esz % 16 == 0;
  }
  const int pieces = vec ? Dh * esz / 16 : Dh;
  const int64_t total = n * H * pieces;
  const int64_t want = (total + 255) / 256, cap = (int64_t)num_sms() * 16;
  const unsigned blocks = (unsigned)(want < cap ? want : cap);
  cudaStream_t st = as_stream(stream);
  if (vec) write_pages_kernel<uint4><<<blocks, 256, 0, st>>>(a, pieces, esz);
  else if (esz == 2) write_pages_kernel<unsigned short><<<blocks, 256, 0, st>>>(a, pieces, esz);
  else write_pages_kernel<float><<<blocks, 256, 0, st>>>(a, pieces, esz);
  return check_launch("write_kv_pages");
}
