// Python binding of the paged cache's and the sampler's entry points: the argument checks, the
// output tensors and the launch in one call from Python.  These launches are shorter than their
// host side (a 2 us kernel behind 13 us of checks and allocations in Python, per layer and step
// of a server that does not record its step), which is why they have this binding beside the C
// ABI's; what it calls is the C ABI, on the tensors' device and its current stream, whichever
// device is the current one.
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <string>
#include <tuple>
#include <utility>

#include "ddtree_b200.h"

namespace py = pybind11;
using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

namespace {

[[noreturn]] void refuse(const std::string& why) { throw py::value_error(why); }

// A refusal of the library, as mdflash_b200._lib.check raises it.
void check(int rc, const char* what) {
  if (rc != DDT_OK) py::module_::import("mdflash_b200._lib").attr("check")(rc, what);
}

// All on one CUDA device: its index.
template <typename... T>
int device_of(const Tensor& first, const T&... others) {
  const int idx = first.get_device();
  if (idx < 0 || !(others.is_cuda() && ...)) refuse("ddtree_b200 kernels need CUDA tensors");
  if (!((others.get_device() == idx) && ...)) refuse("all tensors must be on the same device");
  return idx;
}

const char* name_of(at::ScalarType t) {
  return t == at::kInt ? "torch.int32" : t == at::kLong ? "torch.int64"
         : t == at::kFloat ? "torch.float32" : "torch.bfloat16";
}

void need(const Tensor& t, at::ScalarType dtype, at::IntArrayRef shape, const char* name) {
  if (t.scalar_type() == dtype && t.sizes() == shape && t.is_contiguous()) return;
  std::string s = std::string(name) + " must be contiguous " + name_of(dtype) + " [";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
  refuse(s + "]");
}

Tensor fresh(at::IntArrayRef shape, at::ScalarType dtype, int idx) {
  return at::empty(shape, at::TensorOptions().dtype(dtype).device(at::Device(at::kCUDA, idx)));
}

// n elements of `dtype` from element `first` (of that type) on of the storage of `of`: one
// allocation for several outputs, without a dispatched view for each (three times as long).
Tensor part(const Tensor& of, int64_t first, int64_t n, at::ScalarType dtype) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(of.storage()), of.key_set(),
                                                      c10::scalarTypeToTypeMeta(dtype));
  t.unsafeGetTensorImpl()->set_storage_offset(first);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

template <typename T = void>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <typename T>
T* ptr(const MaybeTensor& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// The status word is written by the kernel.
void need_status(const Tensor& first, const Tensor& status) {
  device_of(first, status);
  if (status.scalar_type() != at::kInt || status.numel() < 1) refuse("status must be an i32 word");
}

void* stream_of(int idx) { return c10::cuda::getCurrentCUDAStream(idx).stream(); }

// The recording that the current stream of a device takes part in, or 0.
uint64_t capture_id(int idx) {
  cudaStreamCaptureStatus status;
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(c10::cuda::getCurrentCUDAStream(idx).stream(), &status, &id));
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

// (row stride, columns) of a block table i32 [requests, max_pages]
std::pair<int64_t, int64_t> table_view(const Tensor& t, int64_t requests) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != requests || t.stride(1) != 1)
    refuse("block_table must be i32 [requests, max_pages] with unit stride");
  return {requests > 1 ? t.stride(0) : t.size(1), t.size(1)};
}

// A page pool: logical [pages, kv_heads, page_size, head_dim] bf16 with any strides but the last.
struct Pool {
  int64_t pages, heads, page, dim, page_stride, head_stride, row_stride;
  Pool(const Tensor& k, const Tensor& v) {
    if (k.dim() != 4 || k.sizes() != v.sizes() || k.strides() != v.strides() || k.stride(3) != 1)
      refuse("k_pages / v_pages must be [pages, kv_heads, page_size, head_dim] with the same "
             "strides and contiguous rows");
    if (k.scalar_type() != at::kBFloat16 || v.scalar_type() != at::kBFloat16)
      throw py::type_error("paged K/V are bf16");
    pages = k.size(0), heads = k.size(1), page = k.size(2), dim = k.size(3);
    page_stride = k.stride(0), head_stride = k.stride(1), row_stride = k.stride(2);
  }
};

using Step = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

Step page_tables(const Tensor& old_lens, const Tensor& new_lens, const Tensor& block_table,
                 const Tensor& free_pages, const Tensor& free_count, int64_t page_size,
                 int64_t max_tokens, const std::optional<Step>& out, const Tensor& status,
                 const Tensor& workspace) {
  const int idx = device_of(old_lens, new_lens, block_table, free_pages, free_count);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(idx));
  const int64_t R = old_lens.numel();
  need(old_lens, at::kInt, {R}, "old_lens");
  need(new_lens, at::kInt, {R}, "new_lens");
  need(free_count, at::kInt, {1}, "free_count");
  const auto [stride, cols] = table_view(block_table, R);
  if (free_pages.scalar_type() != at::kInt || free_pages.dim() != 1 || !free_pages.is_contiguous())
    refuse("free_pages must be a contiguous i32 vector");
  need_status(old_lens, status);
  if (max_tokens < 0) refuse("max_tokens must not be negative");
  Step o;
  if (out) {
    o = *out;
    const auto& [kv_lens, cu_new, slots, positions, count] = o;
    device_of(old_lens, kv_lens, cu_new, slots, positions, count);
    need(kv_lens, at::kInt, {R}, "out.kv_lens");
    need(cu_new, at::kInt, {R + 1}, "out.cu_new");
    need(slots, at::kLong, {max_tokens}, "out.slot_map");
    need(positions, at::kLong, {max_tokens}, "out.positions");
    need(count, at::kInt, {1}, "out.free_count");
  } else {
    const Tensor all = fresh({2 * max_tokens + R + 1}, at::kLong, idx);
    const int64_t lens = 4 * max_tokens;  // the 32-bit parts start here
    o = Step(part(all, lens, R, at::kInt), part(all, lens + R, R + 1, at::kInt),
             part(all, 0, max_tokens, at::kLong), part(all, max_tokens, max_tokens, at::kLong),
             part(all, lens + 2 * R + 1, 1, at::kInt));
  }
  const auto& [kv_lens, cu_new, slots, positions, count] = o;
  check(ddt_page_tables(ptr<int32_t>(old_lens), ptr<int32_t>(new_lens), R, ptr<int32_t>(block_table),
                        stride, cols, page_size, ptr<int32_t>(free_pages), free_pages.numel(),
                        ptr<int32_t>(free_count), ptr<int32_t>(kv_lens), ptr<int32_t>(cu_new),
                        ptr<int64_t>(slots), ptr<int64_t>(positions), max_tokens,
                        ptr<int32_t>(count), ptr(workspace), workspace.numel(),
                        ptr<int32_t>(status), stream_of(idx)),
        "ddt_page_tables");
  return o;
}

Tensor paged_qk_norm_rope(const Tensor& qkv, const Tensor& q_norm_w, const Tensor& k_norm_w,
                          const Tensor& rope_table, const Tensor& slot_map, const Tensor& k_pages,
                          const Tensor& v_pages, double eps, const MaybeTensor& out) {
  const int idx = device_of(qkv, q_norm_w, k_norm_w, rope_table, slot_map, k_pages, v_pages);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(idx));
  const Pool pool(k_pages, v_pages);
  const int64_t d = pool.dim;
  if (qkv.dim() != 2 || qkv.scalar_type() != at::kBFloat16 || qkv.stride(1) != 1 || d == 0 ||
      qkv.size(1) % d)
    refuse("qkv must be bf16 [tokens, heads * head_dim] with unit stride");
  const int64_t T = qkv.size(0), width = qkv.size(1), hq = width / d - 2 * pool.heads;
  if (hq <= 0) refuse("qkv holds no query heads beside the pool's KV heads");
  if (q_norm_w.scalar_type() != at::kBFloat16 || k_norm_w.scalar_type() != at::kBFloat16 ||
      q_norm_w.sizes() != at::IntArrayRef({d}) || k_norm_w.sizes() != at::IntArrayRef({d}) ||
      !q_norm_w.is_contiguous() || !k_norm_w.is_contiguous())
    refuse("norm weights must be bf16 [head_dim]");
  need(rope_table, at::kInt, {T, d / 2}, "rope_table");
  if (slot_map.scalar_type() != at::kLong || slot_map.dim() != 1 || slot_map.size(0) < T ||
      !slot_map.is_contiguous())
    refuse("slot_map must be contiguous i64 with a slot per token");
  Tensor o;
  if (out) {
    need(*out, at::kBFloat16, {T, hq, d}, "out");
    device_of(qkv, *out);
    o = *out;
  } else {
    o = fresh({T, hq, d}, at::kBFloat16, idx);
  }
  check(ddt_paged_qk_norm_rope(ptr(qkv), T > 1 ? qkv.stride(0) : width, T, hq, pool.heads, d,
                               ptr(q_norm_w), ptr(k_norm_w), static_cast<float>(eps),
                               ptr(rope_table), ptr<int64_t>(slot_map), ptr(o), ptr(k_pages),
                               ptr(v_pages), pool.pages, pool.page, pool.page_stride,
                               pool.head_stride, pool.row_stride, stream_of(idx)),
        "ddt_paged_qk_norm_rope");
  return o;
}

// With wait_check (first CTA without loads, limit of the waits in ns): ddt_paged_attn_wait_check.
using WaitCheck = std::optional<std::pair<int64_t, uint64_t>>;
Tensor paged_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                       const Tensor& block_table, const Tensor& cu_new, const Tensor& kv_lens,
                       int64_t max_new, std::optional<double> scale, const MaybeTensor& out,
                       const Tensor& status, const Tensor& workspace, const WaitCheck& wait_check) {
  const int idx = device_of(q, k_pages, v_pages, block_table, cu_new, kv_lens);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(idx));
  const Pool pool(k_pages, v_pages);
  if (q.dim() != 3 || q.scalar_type() != at::kBFloat16 || q.stride(2) != 1)
    refuse("q must be bf16 [tokens, q_heads, head_dim] with contiguous rows");
  const int64_t T = q.size(0), hq = q.size(1), d = q.size(2), R = kv_lens.numel();
  if (d != pool.dim) refuse("q and the pages differ in head_dim");
  need(kv_lens, at::kInt, {R}, "kv_lens");
  need(cu_new, at::kInt, {R + 1}, "cu_new");
  const std::pair<int64_t, int64_t> table = table_view(block_table, R);
  need_status(q, status);
  Tensor o;
  if (out) {
    if (out->sizes() != q.sizes() || out->scalar_type() != q.scalar_type() ||
        out->stride(2) != 1 || out->get_device() != idx)
      refuse("out must be like q");
    o = *out;
  } else {
    o = fresh({T, hq, d}, at::kBFloat16, idx);
  }
  const auto call = [&](auto entry, const char* name, auto... wait) {
    check(entry(ptr(q), q.stride(0), q.stride(1), ptr(k_pages), ptr(v_pages), pool.pages, pool.page,
                pool.page_stride, pool.head_stride, pool.row_stride, ptr<int32_t>(block_table),
                table.first, table.second, ptr<int32_t>(cu_new), ptr<int32_t>(kv_lens), R, T, max_new,
                hq, pool.heads, d,
                static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(d))), ptr(o),
                o.stride(0), o.stride(1), ptr(workspace), workspace.numel(), ptr<int32_t>(status),
                wait..., stream_of(idx)),
          name);
  };
  if (wait_check)
    call(ddt_paged_attn_wait_check, "ddt_paged_attn_wait_check", wait_check->first, wait_check->second);
  else
    call(ddt_paged_attn, "ddt_paged_attn");
  return o;
}

std::tuple<Tensor, Tensor> sample(const Tensor& logits, const Tensor& u, const Tensor& temperature,
                                  const MaybeTensor& top_k, const MaybeTensor& top_p,
                                  const MaybeTensor& min_p, const MaybeTensor& out,
                                  const MaybeTensor& logprobs) {
  const int idx = device_of(logits, u, temperature);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(idx));
  if (logits.dim() != 2 || logits.stride(1) != 1)
    refuse("logits must be [rows, vocab] with unit stride");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  auto per_row = [&](const Tensor& t, at::ScalarType dtype, const char* name) {
    device_of(logits, t);
    need(t, dtype, {rows}, name);
  };
  per_row(u, at::kFloat, "u");
  per_row(temperature, at::kFloat, "temperature");
  if (top_k) per_row(*top_k, at::kInt, "top_k");
  if (top_p) per_row(*top_p, at::kFloat, "top_p");
  if (min_p) per_row(*min_p, at::kFloat, "min_p");
  if (out) per_row(*out, at::kLong, "out");
  if (logprobs) per_row(*logprobs, at::kFloat, "logprobs");
  if (logits.scalar_type() != at::kBFloat16 && logits.scalar_type() != at::kFloat)
    throw py::type_error(std::string("unsupported dtype ") + c10::toString(logits.scalar_type()));
  const Tensor o = out ? *out : fresh({rows}, at::kLong, idx);
  const Tensor lp = logprobs ? *logprobs : fresh({rows}, at::kFloat, idx);
  check(ddt_sample(ptr(logits), logits.scalar_type() == at::kFloat ? DDT_F32 : DDT_BF16, rows, vocab,
                   rows > 1 ? logits.stride(0) : vocab, ptr<float>(u), ptr<float>(temperature),
                   ptr<int32_t>(top_k), ptr<float>(top_p), ptr<float>(min_p), ptr<int64_t>(o),
                   ptr<float>(lp), stream_of(idx)),
        "ddt_sample");
  return {o, lp};
}

}  // namespace

PYBIND11_MODULE(_bind, m) {
  m.def("capture_id", &capture_id);
  m.def("page_tables", &page_tables);
  m.def("paged_qk_norm_rope", &paged_qk_norm_rope);
  m.def("paged_attention", &paged_attention);
  m.def("sample", &sample);
}
