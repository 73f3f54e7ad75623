// The host side of retrievalattention_b200/paged.py: checks of the arguments, workspaces, and the calls into libri_b200.so.
//
// A decode step calls these once per layer and token.  Written in Python over ctypes, as the calls of the other modules are, the
// checks of a dozen tensors took 12 to 20 microseconds a call against 5 to 7 for the library's own part, and more than the
// kernels of a small batch take.  The library's functions are handed over by address, so nothing here links against it.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <climits>
#include <optional>
#include <string>

#include "ri_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

constexpr int64_t kDim = RI_HEAD_DIM;

struct Library {
  decltype(&ri_last_error) last_error = nullptr;
  decltype(&ri_rope_paged_append) append = nullptr;
  decltype(&ri_paged_decode_scratch_bytes) decode_bytes = nullptr;
  decltype(&ri_paged_decode) decode = nullptr;
  decltype(&ri_paged_observe_scratch_bytes) observe_bytes = nullptr;
  decltype(&ri_paged_observe) observe = nullptr;
  decltype(&ri_paged_evict_scratch_bytes) evict_bytes = nullptr;
  decltype(&ri_paged_evict) evict = nullptr;
  int32_t* status = nullptr;               // the process's status word
  py::object* first_use = nullptr;         // told of every GPU that a call runs on, once
  py::object* report = nullptr;            // raises what the status word says
  bool used[64] = {};
} lib;

[[noreturn]] void fail(const char* what, const std::string& message) { throw py::value_error(std::string(what) + ": " + message); }
void check(int64_t rc, const char* what) {
  if (rc < 0) throw std::runtime_error(std::string(what) + " failed (" + std::to_string(rc) + "): " + lib.last_error());
}

bool given(const OptTensor& x) { return x.has_value() && x->defined(); }
void* address(const OptTensor& x) { return given(x) ? x->data_ptr() : nullptr; }
bool dense(const Tensor& x, at::IntArrayRef sizes, at::ScalarType type, c10::Device device) {
  return x.scalar_type() == type && x.sizes() == sizes && x.device() == device && x.is_contiguous();
}
// Heads of 128 behind one another from dimension `first` on; the dimension in front may have any stride.
bool dense_rows(const Tensor& x, int64_t first) {
  int64_t step = 1;
  for (int64_t d = x.dim() - 1; d >= first; --d) {
    if (x.size(d) != 1 && x.stride(d) != step) return false;
    step *= x.size(d);
  }
  return true;
}
void touched(const Tensor& x) {
  if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}
void touched(const OptTensor& x) {
  if (given(x)) touched(*x);
}

int32_t type_code(const Tensor& x) {
  if (x.scalar_type() == at::kBFloat16) return RI_BF16;
  if (x.scalar_type() == at::kHalf) return RI_F16;
  throw py::type_error(std::string("only bfloat16 and float16 are supported, got ") + c10::toString(x.scalar_type()));
}

// The calls run on the tensors' GPU, on its current stream.
struct OnDevice {
  std::optional<c10::cuda::CUDAGuard> guard;
  explicit OnDevice(const Tensor& x) {
    if (x.device().index() != c10::cuda::current_device()) guard.emplace(x.device());
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream().stream(); }
};

int64_t page_stride(const char* what, const Tensor& pages, const char* name) {
  if (!dense_rows(pages, 1)) fail(what, std::string("every page of ") + name + " must be dense");
  return pages.size(0) > 1 ? pages.stride(0) : pages.size(1) * pages.size(2) * kDim;
}

ri_paged describe(const char* what, const Tensor& key_pages, const OptTensor& value_pages, const Tensor& page_table,
                  const Tensor& lengths, const OptTensor& weight, const OptTensor& token, int64_t group) {
  if (key_pages.dim() != 4 || key_pages.size(3) != kDim || !key_pages.is_cuda())
    fail(what, "expected key_pages [pages, kv_heads, page_size, 128] on a GPU");
  const int64_t pages = key_pages.size(0), heads = key_pages.size(1), page = key_pages.size(2);
  const auto device = key_pages.device();
  ri_paged p = {};
  p.dtype = type_code(key_pages);
  p.key_page_stride = page_stride(what, key_pages, "key_pages");
  if (given(value_pages)) {
    if (value_pages->sizes() != key_pages.sizes() || value_pages->scalar_type() != key_pages.scalar_type() || value_pages->device() != device)
      fail(what, "value_pages must be like key_pages");
    p.value_page_stride = page_stride(what, *value_pages, "value_pages");
  }
  if (key_pages.requires_grad() || (given(value_pages) && value_pages->requires_grad())) fail(what, "there are no gradients");
  if (page_table.dim() != 2 || page_table.scalar_type() != at::kInt || page_table.device() != device || !dense_rows(page_table, 1))
    fail(what, "expected an int32 page_table [batch, pages of a request] with dense rows on the pools' GPU");
  const int64_t batch = page_table.size(0), width = page_table.size(1), stride = batch > 1 ? page_table.stride(0) : width;
  if (stride < width) fail(what, "the rows of page_table overlap");
  if (!dense(lengths, {batch}, at::kInt, device)) fail(what, "expected dense int32 lengths [batch] on the pools' GPU");
  if (given(weight) && !dense(*weight, {pages, heads, page}, at::kFloat, device))
    fail(what, "expected dense fp32 weight [pages, kv_heads, page_size] on the pools' GPU");
  if (given(weight) && weight->requires_grad()) fail(what, "there are no gradients");
  if (given(token) && !dense(*token, {pages, heads, page}, at::kInt, device))
    fail(what, "expected dense int32 token [pages, kv_heads, page_size] on the pools' GPU");
  for (int64_t n : {batch, heads, group, page, pages, stride})
    if (n > INT_MAX) fail(what, "too large");
  p.batch = (int32_t)batch;
  p.kv_heads = (int32_t)heads;
  p.group_size = (int32_t)group;
  p.page_size = (int32_t)page;
  p.n_pages = (int32_t)pages;
  p.table_stride = (int32_t)stride;
  p.table_width = (int32_t)width;
  p.d_keys = key_pages.data_ptr();
  p.d_values = address(value_pages);
  p.d_weight = static_cast<float*>(address(weight));
  p.d_token = static_cast<int32_t*>(address(token));
  p.d_table = static_cast<const int32_t*>(page_table.data_ptr());
  p.d_lengths = static_cast<const int32_t*>(lengths.data_ptr());
  p.d_status = lib.status;
  return p;
}

// Behind a call's launches: what the status word says of it or of an earlier call.
void done(const Tensor& x) {
  const int device = x.device().index();
  if (device >= 64 || !lib.used[device]) {
    (*lib.first_use)(device);
    if (device < 64) lib.used[device] = true;
  }
  if (*static_cast<volatile int32_t*>(lib.status)) (*lib.report)();
}

Tensor workspace(int64_t bytes, const Tensor& like, const char* what) {
  check(bytes, what);
  return at::empty({bytes}, like.options().dtype(at::kByte));
}

void append(const Tensor& qkv, const Tensor& cos_sin, const Tensor& positions, const py::bytes& axis_of, const Tensor& q,
            const Tensor& key_pages, const OptTensor& value_pages, const Tensor& page_table, const Tensor& lengths,
            const OptTensor& row_start, const OptTensor& weight, const OptTensor& token, const OptTensor& seen, const OptTensor& keys,
            const OptTensor& values) {
  const char* what = "rope_paged_append";
  const int64_t heads = key_pages.dim() == 4 ? key_pages.size(1) : 0;
  if (qkv.dim() != 2 || q.dim() != 3 || heads < 1 || q.size(1) < heads || q.size(1) % heads)
    fail(what, "expected qkv [rows, (q_heads + 2 kv_heads) * 128] and q [rows, q_heads, 128], q_heads a multiple of kv_heads");
  const int64_t rows = qkv.size(0), q_heads = q.size(1);
  const auto device = qkv.device();
  if (qkv.size(1) != (q_heads + 2 * heads) * kDim || !dense_rows(qkv, 1))
    fail(what, "expected qkv [rows, (q_heads + 2 kv_heads) * 128] with dense rows");
  if (!given(value_pages)) fail(what, "value_pages is missing");
  const auto type = key_pages.scalar_type();
  if (qkv.scalar_type() != type || device != key_pages.device()) fail(what, "expected qkv and the pages of one type on one GPU");
  if (!dense(q, {rows, q_heads, kDim}, type, device)) fail(what, "expected dense q [rows, q_heads, 128] of the pages' type on their GPU");
  for (const OptTensor* x : {&keys, &values})
    if (given(*x) && !dense(**x, {rows, heads, kDim}, type, device))
      fail(what, "expected dense keys and values [rows, kv_heads, 128] of the pages' type on their GPU");
  if (qkv.requires_grad() || q.requires_grad() || (given(keys) && keys->requires_grad()) || (given(values) && values->requires_grad()))
    fail(what, "there are no gradients");
  if (cos_sin.dim() != 2 || !dense(cos_sin, {cos_sin.size(0), kDim}, at::kFloat, device)) fail(what, "expected dense fp32 cos_sin [positions, 128]");
  const int64_t axes = positions.dim() == 2 ? positions.size(0) : 1;
  if (positions.dim() < 1 || positions.dim() > 2 || positions.size(-1) != rows || positions.scalar_type() != at::kLong ||
      positions.device() != device || !positions.is_contiguous())
    fail(what, "expected dense int64 positions [axes, rows]");
  char* of = nullptr;
  Py_ssize_t n_of = 0;
  if (PyBytes_AsStringAndSize(axis_of.ptr(), &of, &n_of) != 0) throw py::error_already_set();
  if (n_of != kDim / 2) fail(what, "axis_of names an axis for each of the 64 frequencies");
  if (rows > INT_MAX || axes > INT_MAX) fail(what, "too large");
  const ri_paged p = describe(what, key_pages, value_pages, page_table, lengths, weight, token, q_heads / heads);
  if (given(row_start) && !dense(*row_start, {p.batch + 1}, at::kInt, device)) fail(what, "expected dense int32 row_start [batch + 1]");
  if (given(seen) && !dense(*seen, {p.batch}, at::kInt, device)) fail(what, "expected dense int32 seen [batch]");
  if (given(token) && !given(seen)) fail(what, "token numbers need `seen`");
  if (rows == 0) return;
  const OnDevice on(key_pages);
  check(lib.append(&p, qkv.data_ptr(), rows > 1 ? qkv.stride(0) : qkv.size(1), static_cast<const float*>(cos_sin.data_ptr()),
                   cos_sin.size(0), static_cast<const int64_t*>(positions.data_ptr()), reinterpret_cast<const uint8_t*>(of), (int32_t)axes,
                   (int32_t)rows, static_cast<const int32_t*>(address(row_start)), static_cast<const int32_t*>(address(seen)),
                   q.data_ptr(), address(keys), address(values), on.stream()), what);
  touched(q);
  touched(key_pages);
  for (const OptTensor* x : {&value_pages, &weight, &token, &keys, &values}) touched(*x);
  done(key_pages);
}

Tensor decode(const Tensor& q, const Tensor& key_pages, const OptTensor& value_pages, const Tensor& page_table, const Tensor& lengths,
              const OptTensor& given_out, const OptTensor& lse, const OptTensor& weight, double scale) {
  const char* what = "paged_decode";
  if (q.dim() != 4 || key_pages.dim() != 4 || page_table.dim() != 2 || !given(value_pages))
    fail(what, "expected q [batch, 1, q_heads, 128] and pages [pages, kv_heads, page_size, 128]");
  const int64_t batch = q.size(0), q_heads = q.size(2), heads = key_pages.size(1);
  if (q.size(1) != 1 || q.size(3) != kDim || heads < 1 || q_heads < heads || q_heads % heads || page_table.size(0) != batch)
    fail(what, "expected q [batch, 1, q_heads, 128], q_heads a multiple of kv_heads, one page table row per request");
  if (!dense_rows(q, 1)) fail(what, "the heads of a request must lie dense in q");
  if (q.scalar_type() != key_pages.scalar_type() || q.device() != key_pages.device() || q.requires_grad())
    fail(what, "expected q and the pages of one type on one GPU, without gradients");
  const ri_paged p = describe(what, key_pages, value_pages, page_table, lengths, weight, std::nullopt, q_heads / heads);
  if (given(given_out) && (!dense(*given_out, q.sizes(), q.scalar_type(), q.device()) || given_out->requires_grad()))
    fail(what, "expected dense out like q");
  if (given(lse) && (!dense(*lse, {batch, q_heads}, at::kFloat, q.device()) || lse->requires_grad()))
    fail(what, "expected dense fp32 lse [batch, q_heads]");
  const OnDevice on(key_pages);
  const Tensor out = given(given_out) ? *given_out : at::empty(q.sizes(), q.options());
  const Tensor scratch = workspace(lib.decode_bytes(&p), q, what);
  check(lib.decode(&p, q.data_ptr(), batch > 1 ? q.stride(0) : q_heads * kDim, out.data_ptr(), static_cast<float*>(address(lse)),
                   (float)scale, scratch.data_ptr(), on.stream()), what);
  touched(given_out);
  touched(lse);
  touched(weight);
  done(key_pages);
  return out;
}

void observe(const Tensor& q, const Tensor& key_pages, const Tensor& page_table, const Tensor& lengths, const OptTensor& weight,
             double scale) {
  const char* what = "paged_observe";
  if (q.dim() != 4 || key_pages.dim() != 4 || page_table.dim() != 2 || !given(weight))
    fail(what, "expected q [batch, window, q_heads, 128], pages [pages, kv_heads, page_size, 128] and weights");
  const int64_t window = q.size(1), q_heads = q.size(2), heads = key_pages.size(1);
  if (q.size(3) != kDim || window < 1 || heads < 1 || q_heads < heads || q_heads % heads || page_table.size(0) != q.size(0) ||
      !q.is_contiguous())
    fail(what, "expected dense q [batch, window, q_heads, 128], q_heads a multiple of kv_heads, one page table row per request");
  if (q.scalar_type() != key_pages.scalar_type() || q.device() != key_pages.device() || q.requires_grad())
    fail(what, "expected q and the pages of one type on one GPU, without gradients");
  if (window > INT_MAX) fail(what, "too large");
  const ri_paged p = describe(what, key_pages, std::nullopt, page_table, lengths, weight, std::nullopt, q_heads / heads);
  const OnDevice on(key_pages);
  const Tensor scratch = workspace(lib.observe_bytes(&p), q, what);
  check(lib.observe(&p, q.data_ptr(), (int32_t)window, (float)scale, scratch.data_ptr(), on.stream()), what);
  touched(weight);
  done(key_pages);
}

void evict(const Tensor& key_pages, const OptTensor& value_pages, const OptTensor& weight, const OptTensor& token,
           const Tensor& page_table, const Tensor& lengths, const Tensor& seen, int64_t keep, int64_t n_sink, int64_t n_recent) {
  const char* what = "paged_evict";
  if (!given(value_pages) || !given(weight) || !given(token)) fail(what, "keys, values, weights and token numbers move together: none may be missing");
  const ri_paged p = describe(what, key_pages, value_pages, page_table, lengths, weight, token, 1);
  if (!dense(seen, {p.batch}, at::kInt, key_pages.device())) fail(what, "expected dense int32 seen [batch]");
  for (int64_t n : {keep, n_sink, n_recent})
    if (n > INT_MAX || n < INT_MIN) fail(what, "too large");
  const OnDevice on(key_pages);
  const Tensor scratch = workspace(lib.evict_bytes(&p, (int32_t)keep), key_pages, what);
  check(lib.evict(&p, static_cast<const int32_t*>(seen.data_ptr()), (int32_t)keep, (int32_t)n_sink, (int32_t)n_recent,
                  scratch.data_ptr(), on.stream()), what);
  touched(key_pages);
  for (const OptTensor* x : {&value_pages, &weight, &token}) touched(*x);
  done(key_pages);
}

void connect(const py::dict& addresses, const py::object& first_use, const py::object& report) {
  auto take = [&](const char* name, auto& slot) {
    slot = reinterpret_cast<std::remove_reference_t<decltype(slot)>>(addresses[name].cast<uintptr_t>());
  };
  take("ri_last_error", lib.last_error);
  take("ri_rope_paged_append", lib.append);
  take("ri_paged_decode_scratch_bytes", lib.decode_bytes);
  take("ri_paged_decode", lib.decode);
  take("ri_paged_observe_scratch_bytes", lib.observe_bytes);
  take("ri_paged_observe", lib.observe);
  take("ri_paged_evict_scratch_bytes", lib.evict_bytes);
  take("ri_paged_evict", lib.evict);
  lib.status = addresses["status_word"].is_none() ? nullptr : reinterpret_cast<int32_t*>(addresses["status_word"].cast<uintptr_t>());
  lib.first_use = new py::object(first_use);             // for the life of the process
  lib.report = new py::object(report);
}

}  // namespace

PYBIND11_MODULE(_paged_binding, m) {
  m.def("connect", &connect);
  m.def("append", &append);
  m.def("decode", &decode);
  m.def("observe", &observe);
  m.def("evict", &evict);
}
