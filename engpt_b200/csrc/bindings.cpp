// Python module engpt_b200._native: the paged key-value cache operators on torch tensors.
//
// A decoding step makes these calls once per layer on a few microseconds of GPU work, so their argument checks,
// output allocation and stream look-up are here rather than in Python (a call costs about 5 us of host time instead
// of 20 to 30).  The work itself goes through the C ABI (include/engpt_b200.h) like every other call of the package.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/engpt_b200.h"

namespace py = pybind11;
using at::Tensor;

namespace {

void check_status(const char* name, int rc) {
  if (rc == ENGPT_OK) return;
  // engpt_b200._lib raises its own exception type
  py::module_::import("engpt_b200._lib").attr("raise_status")(name, rc, std::string(engpt_last_error()));
}

void require_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "engpt_b200 ops run on CUDA tensors only (no CPU fallback)");
}

void require_device(const Tensor& t, const c10::Device& dev) {
  require_cuda(t);
  TORCH_CHECK(t.device() == dev, "engpt_b200 ops: all tensors must be on the same device");
}

void forward_only(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->requires_grad(),
                                "engpt_b200 kernels are forward-only; call under torch.no_grad()");
}

// Tensors that a call has written through their addresses: counted as torch's own in-place operators are, so that
// autograd notices where it kept one of them.
void written(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

int dtype_code(const Tensor& t) {
  const auto dt = t.scalar_type();
  TORCH_CHECK_NOT_IMPLEMENTED(dt == at::kBFloat16 || dt == at::kFloat,
                              "engpt_b200 kernels support float32 and bfloat16, got ", dt);
  return dt == at::kBFloat16 ? ENGPT_BF16 : ENGPT_F32;
}

// A contiguous int32 tensor of the given shape on the cache's device.
void check_index(const Tensor& t, const char* name, at::IntArrayRef shape, const c10::Device& dev) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.sizes() == shape && t.is_contiguous(), name,
                    " must be a contiguous int32 tensor of shape ", shape, ", got ", t.scalar_type(), " ", t.sizes());
  require_device(t, dev);
}

void check_table(const Tensor& t, int64_t rows, const c10::Device& dev) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == rows &&
                        (t.size(1) <= 1 || t.stride(1) == 1),
                    "block_table must be int32 [batch, pages per request] with contiguous rows");
  require_device(t, dev);
}

int64_t table_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct Pools {
  int num_pages, heads, page_size, dim, code;
  int64_t strides[6];
};

// A cache in 8 bits: its codes and scales.
struct Q8Pools {
  int num_pages, heads, page_size, dim, block, code;
  int64_t strides[6], scale_strides[6];
};

int to_int(int64_t v, const char* what) {
  TORCH_CHECK_VALUE(v <= 0x7fffffffLL, what, " is too large: ", v);
  return (int)v;
}

Pools check_pools(const Tensor& k, const Tensor& v) {
  require_cuda(k);
  require_device(v, k.device());
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
                    "k_pages and v_pages must share a shape [num_pages, kv_heads, page_size, head_dim] and dtype");
  TORCH_CHECK_VALUE(k.size(3) <= 1 || (k.stride(3) == 1 && v.stride(3) == 1),
                    "k_pages and v_pages need a contiguous head_dim axis");
  Pools p;
  p.num_pages = to_int(k.size(0), "num_pages");
  p.heads = to_int(k.size(1), "kv_heads");
  p.page_size = to_int(k.size(2), "page_size");
  p.dim = to_int(k.size(3), "head_dim");
  p.code = dtype_code(k);
  for (int i = 0; i < 3; ++i) {
    p.strides[i] = k.stride(i);
    p.strides[3 + i] = v.stride(i);
  }
  return p;
}

Q8Pools check_q8_pools(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
  require_cuda(k);
  for (const Tensor* t : {&v, &ks, &vs}) require_device(*t, k.device());
  const auto dt = k.scalar_type();
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes() && v.scalar_type() == dt,
                    "k_pages and v_pages must share a shape [num_pages, kv_heads, page_size, head_dim] and dtype");
  TORCH_CHECK_NOT_IMPLEMENTED(dt == at::kChar || dt == at::kFloat8_e4m3fn,
                              "an 8-bit cache holds int8 or float8_e4m3fn, got ", dt);
  TORCH_CHECK_VALUE(k.size(3) <= 1 || (k.stride(3) == 1 && v.stride(3) == 1),
                    "k_pages and v_pages need a contiguous head_dim axis");
  TORCH_CHECK_VALUE(ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat && ks.dim() == 3 &&
                        ks.sizes() == vs.sizes() && ks.size(0) == k.size(0) && ks.size(1) == k.size(1) &&
                        ks.size(2) > 0 && k.size(2) > 0 && k.size(2) % ks.size(2) == 0,
                    "k_scales and v_scales must be float32 [num_pages, kv_heads, blocks per page], with a page_size that "
                    "is a multiple of the blocks");
  Q8Pools p;
  p.num_pages = to_int(k.size(0), "num_pages");
  p.heads = to_int(k.size(1), "kv_heads");
  p.page_size = to_int(k.size(2), "page_size");
  p.dim = to_int(k.size(3), "head_dim");
  p.block = (int)(k.size(2) / ks.size(2));
  p.code = dt == at::kChar ? ENGPT_CODE_INT8 : ENGPT_CODE_E4M3;
  for (int i = 0; i < 3; ++i) {
    p.strides[i] = k.stride(i);
    p.strides[3 + i] = v.stride(i);
    p.scale_strides[i] = ks.stride(i);
    p.scale_strides[3 + i] = vs.stride(i);
  }
  return p;
}

Tensor f32c(const Tensor& t) {
  return t.scalar_type() == at::kFloat && t.is_contiguous() ? t : t.to(at::kFloat).contiguous();
}

void* stream_of(const c10::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

py::tuple advance_block_tables(const Tensor& lengths, const Tensor& new_tokens, const Tensor& block_table,
                               const Tensor& free_pages, const Tensor& free_count, int64_t page_size, int64_t max_new,
                               const std::optional<Tensor>& finished) {
  require_cuda(lengths);
  const auto dev = lengths.device();
  TORCH_CHECK_VALUE(lengths.dim() == 1, "lengths must have shape [batch]");
  const int64_t b = lengths.size(0);
  check_index(lengths, "lengths", {b}, dev);
  check_index(new_tokens, "new_tokens", {b}, dev);
  check_table(block_table, b, dev);
  TORCH_CHECK_VALUE(free_pages.dim() == 1, "free_pages must have shape [num_pages]");
  check_index(free_pages, "free_pages", free_pages.sizes(), dev);
  check_index(free_count, "free_count", {1}, dev);
  if (finished) {
    TORCH_CHECK_VALUE((finished->scalar_type() == at::kBool || finished->scalar_type() == at::kByte) &&
                          finished->dim() == 1 && finished->size(0) == b && finished->is_contiguous(),
                      "finished must be a contiguous bool or uint8 tensor [batch]");
    require_device(*finished, dev);
  }
  TORCH_CHECK_VALUE(page_size >= 1 && max_new >= 0, "page_size must be positive and max_new not negative");
  c10::cuda::CUDAGuard guard(dev);
  Tensor slots = at::empty({b, max_new}, lengths.options()), positions = at::empty({b, max_new}, lengths.options());
  check_status("engpt_advance_block_tables",
               engpt_advance_block_tables(
                   (int*)lengths.data_ptr(), (const int*)new_tokens.data_ptr(),
                   finished ? (const unsigned char*)finished->data_ptr() : nullptr, to_int(b, "batch"),
                   (int*)block_table.data_ptr(), table_stride(block_table), to_int(block_table.size(1), "table width"),
                   (int*)free_pages.data_ptr(), to_int(free_pages.size(0), "num_pages"), (int*)free_count.data_ptr(),
                   to_int(page_size, "page_size"), to_int(max_new, "max_new"), (int*)slots.data_ptr(),
                   (int*)positions.data_ptr(), stream_of(dev)));
  written({&lengths, &block_table, &free_pages, &free_count});
  return py::make_tuple(slots, positions);
}

Tensor qkv_append(const Tensor& qkv_in, const Tensor& rho, const Tensor& cos, const Tensor& sin,
                  const Tensor& qk_scale, double norm_eps, const Tensor& positions, const Tensor& slots,
                  const Tensor& k_pages, const Tensor& v_pages, double qk_mult) {
  const Pools p = check_pools(k_pages, v_pages);
  const auto dev = k_pages.device();
  for (const Tensor* t : {&qkv_in, &rho, &cos, &sin, &qk_scale}) require_device(*t, dev);
  forward_only({&qkv_in, &rho, &cos, &sin, &qk_scale, &k_pages, &v_pages});
  const int64_t nd = qkv_in.dim();
  TORCH_CHECK_VALUE(nd >= 3 && qkv_in.size(nd - 3) == 3 && qkv_in.size(nd - 2) == p.heads &&
                        qkv_in.size(nd - 1) == p.dim && qkv_in.scalar_type() == k_pages.scalar_type(),
                    "qkv must have shape [..., 3, H, Dh] and the cache's heads, head_dim and dtype");
  const auto lead = qkv_in.sizes().slice(0, nd - 3);
  TORCH_CHECK_VALUE(rho.sizes() == lead, "rho must have qkv's leading shape");
  TORCH_CHECK_VALUE(qk_scale.dim() == 2 && qk_scale.size(0) == p.heads && qk_scale.size(1) == p.dim,
                    "qk_scale must have shape [n_head, head_dim]");
  const int half = p.dim / 2;
  TORCH_CHECK_VALUE(cos.dim() == 2 && cos.size(1) == half && sin.sizes() == cos.sizes(),
                    "cos/sin must have shape [T, head_dim // 2]");
  check_index(positions, "positions", lead, dev);
  check_index(slots, "slots", lead, dev);
  c10::cuda::CUDAGuard guard(dev);
  const Tensor qkv = qkv_in.contiguous(), r = f32c(rho), c = f32c(cos), s = f32c(sin), sc = f32c(qk_scale);
  at::DimVector shape(lead.begin(), lead.end());
  shape.push_back(p.heads);
  shape.push_back(p.dim);
  Tensor q = at::empty(shape, qkv.options());
  check_status("engpt_qkv_append",
               engpt_qkv_append(qkv.data_ptr(), p.code, (const float*)r.data_ptr(), (const float*)c.data_ptr(),
                                (const float*)s.data_ptr(), to_int(c.size(0), "rotary rows"), half,
                                (const float*)sc.data_ptr(), (float)qk_mult, (float)norm_eps, r.numel(), p.heads,
                                p.dim, (const int*)positions.data_ptr(), (const int*)slots.data_ptr(), q.data_ptr(),
                                k_pages.data_ptr(), v_pages.data_ptr(), p.strides, p.num_pages, p.page_size,
                                stream_of(dev)));
  written({&k_pages, &v_pages});
  return q;
}

// [..., H, Dh] as [n, H, Dh] rows with a contiguous last axis (a view where the strides allow it).
Tensor kv_rows(const Tensor& t) {
  Tensor r = t.dim() == 3 ? t : t.reshape({-1, t.size(-2), t.size(-1)});
  return r.size(2) <= 1 || r.stride(2) == 1 ? r : r.contiguous();
}

void write_kv_pages(const Tensor& k_in, const Tensor& v_in, const Tensor& slots, const Tensor& k_pages,
                    const Tensor& v_pages) {
  const Pools p = check_pools(k_pages, v_pages);
  const auto dev = k_pages.device();
  require_device(k_in, dev);
  require_device(v_in, dev);
  forward_only({&k_in, &v_in, &k_pages, &v_pages});
  const int64_t nd = k_in.dim();
  TORCH_CHECK_VALUE(nd >= 2 && k_in.sizes() == v_in.sizes() && k_in.size(nd - 2) == p.heads &&
                        k_in.size(nd - 1) == p.dim,
                    "k and v must share a shape [..., H, Dh] with the cache's heads and head_dim");
  TORCH_CHECK_VALUE(k_in.scalar_type() == k_pages.scalar_type() && v_in.scalar_type() == k_pages.scalar_type(),
                    "k and v must have the cache's dtype");
  check_index(slots, "slots", k_in.sizes().slice(0, nd - 2), dev);
  if (slots.numel() == 0) return;
  at::NoGradGuard no_grad;
  c10::cuda::CUDAGuard guard(dev);
  const Tensor k = kv_rows(k_in), v = kv_rows(v_in);
  const int64_t strides[4] = {k.stride(0), k.stride(1), v.stride(0), v.stride(1)};
  check_status("engpt_write_kv_pages",
               engpt_write_kv_pages(k.data_ptr(), v.data_ptr(), strides, p.code, k.size(0), p.heads, p.dim,
                                    (const int*)slots.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), p.strides,
                                    p.num_pages, p.page_size, stream_of(dev)));
  written({&k_pages, &v_pages});
}

Tensor paged_sdpa(const Tensor& q_in, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                  const Tensor& lengths, double scale) {
  const Pools p = check_pools(k_pages, v_pages);
  const auto dev = k_pages.device();
  require_device(q_in, dev);
  forward_only({&q_in, &k_pages, &v_pages});
  TORCH_CHECK_VALUE(q_in.dim() == 3 && q_in.size(2) == p.dim && q_in.scalar_type() == k_pages.scalar_type(),
                    "q must have shape [batch, n_head, head_dim] and the cache's head_dim and dtype");
  const int64_t b = q_in.size(0), h = q_in.size(1);
  TORCH_CHECK_VALUE(h > 0 && p.heads > 0 && h % p.heads == 0,
                    "the number of query heads must be a multiple of the cache's heads");
  check_index(lengths, "lengths", {b}, dev);
  check_table(block_table, b, dev);
  c10::cuda::CUDAGuard guard(dev);
  const Tensor q = p.dim <= 1 || q_in.stride(2) == 1 ? q_in : q_in.contiguous();
  Tensor o = at::empty({b, h, p.dim}, q.options());
  const int bi = to_int(b, "batch"), hi = to_int(h, "n_head"), width = to_int(block_table.size(1), "table width");
  const int64_t floats = engpt_paged_attention_floats(p.code, bi, hi, p.heads, p.dim, width, p.page_size);
  // scratch of this call alone: calls on other streams, and captured graphs, have their own
  Tensor work;
  if (floats > 0) work = at::empty({floats}, q.options().dtype(at::kFloat));
  const int64_t strides[2] = {q.stride(0), q.stride(1)};
  check_status("engpt_paged_attention",
               engpt_paged_attention(q.data_ptr(), strides, k_pages.data_ptr(), v_pages.data_ptr(), p.strides, p.code,
                                     bi, hi, p.heads, p.dim, p.num_pages, p.page_size,
                                     (const int*)block_table.data_ptr(), table_stride(block_table), width,
                                     (const int*)lengths.data_ptr(), (float)scale, o.data_ptr(),
                                     floats > 0 ? (float*)work.data_ptr() : nullptr, stream_of(dev)));
  return o;
}

void write_kv_pages_q8(const Tensor& k_in, const Tensor& v_in, const Tensor& slots, const Tensor& k_pages,
                       const Tensor& v_pages, const Tensor& k_scales, const Tensor& v_scales) {
  const Q8Pools p = check_q8_pools(k_pages, v_pages, k_scales, v_scales);
  const auto dev = k_pages.device();
  require_device(k_in, dev);
  require_device(v_in, dev);
  forward_only({&k_in, &v_in, &k_pages, &v_pages, &k_scales, &v_scales});
  const int64_t nd = k_in.dim();
  TORCH_CHECK_VALUE(nd >= 2 && k_in.sizes() == v_in.sizes() && k_in.scalar_type() == v_in.scalar_type() &&
                        k_in.size(nd - 2) == p.heads && k_in.size(nd - 1) == p.dim,
                    "k and v must share a dtype and a shape [..., H, Dh] with the cache's heads and head_dim");
  const int code = dtype_code(k_in);
  check_index(slots, "slots", k_in.sizes().slice(0, nd - 2), dev);
  if (slots.numel() == 0) return;
  at::NoGradGuard no_grad;
  c10::cuda::CUDAGuard guard(dev);
  const Tensor k = kv_rows(k_in), v = kv_rows(v_in);
  const int64_t strides[4] = {k.stride(0), k.stride(1), v.stride(0), v.stride(1)};
  check_status("engpt_write_kv_pages_q8",
               engpt_write_kv_pages_q8(k.data_ptr(), v.data_ptr(), strides, code, k.size(0), p.heads, p.dim,
                                       (const int*)slots.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                                       (float*)k_scales.data_ptr(), (float*)v_scales.data_ptr(), p.strides,
                                       p.scale_strides, p.code, p.num_pages, p.page_size, p.block, stream_of(dev)));
  written({&k_pages, &v_pages, &k_scales, &v_scales});
}

Tensor qkv_append_q8(const Tensor& qkv_in, const Tensor& rho, const Tensor& cos, const Tensor& sin,
                     const Tensor& qk_scale, double norm_eps, const Tensor& positions, const Tensor& slots,
                     const Tensor& k_pages, const Tensor& v_pages, const Tensor& k_scales, const Tensor& v_scales,
                     double qk_mult) {
  const Q8Pools p = check_q8_pools(k_pages, v_pages, k_scales, v_scales);
  const auto dev = k_pages.device();
  for (const Tensor* t : {&qkv_in, &rho, &cos, &sin, &qk_scale}) require_device(*t, dev);
  forward_only({&qkv_in, &rho, &cos, &sin, &qk_scale, &k_pages, &v_pages, &k_scales, &v_scales});
  const int64_t nd = qkv_in.dim();
  TORCH_CHECK_VALUE(nd >= 3 && qkv_in.size(nd - 3) == 3 && qkv_in.size(nd - 2) == p.heads &&
                        qkv_in.size(nd - 1) == p.dim,
                    "qkv must have shape [..., 3, H, Dh] and the cache's heads and head_dim");
  const int code = dtype_code(qkv_in);
  const auto lead = qkv_in.sizes().slice(0, nd - 3);
  TORCH_CHECK_VALUE(rho.sizes() == lead, "rho must have qkv's leading shape");
  TORCH_CHECK_VALUE(qk_scale.dim() == 2 && qk_scale.size(0) == p.heads && qk_scale.size(1) == p.dim,
                    "qk_scale must have shape [n_head, head_dim]");
  const int half = p.dim / 2;
  TORCH_CHECK_VALUE(cos.dim() == 2 && cos.size(1) == half && sin.sizes() == cos.sizes(),
                    "cos/sin must have shape [T, head_dim // 2]");
  check_index(positions, "positions", lead, dev);
  check_index(slots, "slots", lead, dev);
  c10::cuda::CUDAGuard guard(dev);
  const Tensor qkv = qkv_in.contiguous(), r = f32c(rho), c = f32c(cos), s = f32c(sin), sc = f32c(qk_scale);
  at::DimVector shape(lead.begin(), lead.end());
  shape.push_back(p.heads);
  shape.push_back(p.dim);
  Tensor q = at::empty(shape, qkv.options());
  check_status("engpt_qkv_append_q8",
               engpt_qkv_append_q8(qkv.data_ptr(), code, (const float*)r.data_ptr(), (const float*)c.data_ptr(),
                                   (const float*)s.data_ptr(), to_int(c.size(0), "rotary rows"), half,
                                   (const float*)sc.data_ptr(), (float)qk_mult, (float)norm_eps, r.numel(), p.heads,
                                   p.dim, (const int*)positions.data_ptr(), (const int*)slots.data_ptr(),
                                   q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), (float*)k_scales.data_ptr(),
                                   (float*)v_scales.data_ptr(), p.strides, p.scale_strides, p.code, p.num_pages,
                                   p.page_size, p.block, stream_of(dev)));
  written({&k_pages, &v_pages, &k_scales, &v_scales});
  return q;
}

py::tuple read_kv_pages_q8(const Tensor& slots, const Tensor& k_pages, const Tensor& v_pages, const Tensor& k_scales,
                           const Tensor& v_scales, at::ScalarType dtype) {
  const Q8Pools p = check_q8_pools(k_pages, v_pages, k_scales, v_scales);
  const auto dev = k_pages.device();
  forward_only({&k_pages, &v_pages, &k_scales, &v_scales});
  TORCH_CHECK_NOT_IMPLEMENTED(dtype == at::kBFloat16 || dtype == at::kFloat,
                              "engpt_b200 kernels support float32 and bfloat16, got ", dtype);
  check_index(slots, "slots", slots.sizes(), dev);
  c10::cuda::CUDAGuard guard(dev);
  at::DimVector shape(slots.sizes().begin(), slots.sizes().end());
  shape.push_back(p.heads);
  shape.push_back(p.dim);
  Tensor k = at::empty(shape, k_scales.options().dtype(dtype)), v = at::empty_like(k);
  check_status("engpt_read_kv_pages_q8",
               engpt_read_kv_pages_q8((const int*)slots.data_ptr(), slots.numel(), k_pages.data_ptr(),
                                      v_pages.data_ptr(), (const float*)k_scales.data_ptr(),
                                      (const float*)v_scales.data_ptr(), p.strides, p.scale_strides, p.code, p.heads,
                                      p.dim, p.num_pages, p.page_size, p.block, k.data_ptr(), v.data_ptr(),
                                      dtype == at::kBFloat16 ? ENGPT_BF16 : ENGPT_F32, stream_of(dev)));
  return py::make_tuple(k, v);
}

Tensor paged_sdpa_q8(const Tensor& q_in, const Tensor& k_pages, const Tensor& v_pages, const Tensor& k_scales,
                     const Tensor& v_scales, const Tensor& block_table, const Tensor& lengths, double scale) {
  const Q8Pools p = check_q8_pools(k_pages, v_pages, k_scales, v_scales);
  const auto dev = k_pages.device();
  require_device(q_in, dev);
  forward_only({&q_in, &k_pages, &v_pages, &k_scales, &v_scales});
  TORCH_CHECK_VALUE(q_in.dim() == 3 && q_in.size(2) == p.dim,
                    "q must have shape [batch, n_head, head_dim] and the cache's head_dim");
  const int code = dtype_code(q_in);
  const int64_t b = q_in.size(0), h = q_in.size(1);
  TORCH_CHECK_VALUE(h > 0 && p.heads > 0 && h % p.heads == 0,
                    "the number of query heads must be a multiple of the cache's heads");
  check_index(lengths, "lengths", {b}, dev);
  check_table(block_table, b, dev);
  c10::cuda::CUDAGuard guard(dev);
  const Tensor q = p.dim <= 1 || q_in.stride(2) == 1 ? q_in : q_in.contiguous();
  Tensor o = at::empty({b, h, p.dim}, q.options());
  const int bi = to_int(b, "batch"), hi = to_int(h, "n_head"), width = to_int(block_table.size(1), "table width");
  const int64_t floats = engpt_paged_attention_q8_floats(code, bi, hi, p.heads, p.dim, width, p.page_size, p.block);
  // scratch of this call alone: calls on other streams, and captured graphs, have their own
  Tensor work;
  if (floats > 0) work = at::empty({floats}, q.options().dtype(at::kFloat));
  const int64_t strides[2] = {q.stride(0), q.stride(1)};
  check_status("engpt_paged_attention_q8",
               engpt_paged_attention_q8(q.data_ptr(), strides, k_pages.data_ptr(), v_pages.data_ptr(),
                                        (const float*)k_scales.data_ptr(), (const float*)v_scales.data_ptr(),
                                        p.strides, p.scale_strides, code, p.code, bi, hi, p.heads, p.dim, p.num_pages,
                                        p.page_size, p.block, (const int*)block_table.data_ptr(),
                                        table_stride(block_table), width, (const int*)lengths.data_ptr(),
                                        (float)scale, o.data_ptr(), floats > 0 ? (float*)work.data_ptr() : nullptr,
                                        stream_of(dev)));
  return o;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("advance_block_tables", &advance_block_tables);
  m.def("qkv_append", &qkv_append);
  m.def("write_kv_pages", &write_kv_pages);
  m.def("paged_sdpa", &paged_sdpa);
  m.def("write_kv_pages_q8", &write_kv_pages_q8);
  m.def("qkv_append_q8", &qkv_append_q8);
  m.def("read_kv_pages_q8", [](const Tensor& slots, const Tensor& k_pages, const Tensor& v_pages,
                               const Tensor& k_scales, const Tensor& v_scales, const py::object& dtype) {
    TORCH_CHECK_TYPE(THPDtype_Check(dtype.ptr()), "dtype must be a torch.dtype");
    return read_kv_pages_q8(slots, k_pages, v_pages, k_scales, v_scales,
                            reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type);
  });
  m.def("paged_sdpa_q8", &paged_sdpa_q8);
}
