// The torch side of the router's training entries and of the 8-bit integer products: checks of tensors, outputs from
// torch's allocator, the tensors' device and its current stream, and the C ABI call (include/k3moe.h).  k3moe.py is its
// only caller.  A decode step makes such calls every few microseconds, and in Python the checks, the allocations and the
// argument conversion took longer than the kernels (8.9 us for a quantiser call, 18 us for the balance loss): here they
// take 1 to 3 us.
#include <ATen/Context.h>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/pybind.h>

#include <climits>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/k3moe.h"

namespace {

using at::ScalarType;
using at::Tensor;
using MaybeTensor = std::optional<Tensor>;
using Quantised = std::optional<std::tuple<Tensor, Tensor>>;

PyObject* g_error = nullptr;  // k3moe.K3MoeError

[[noreturn]] void refuse(const std::string& text) {
  PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, text.c_str());
  throw py::error_already_set();
}

int as_int(int64_t v, const char* name) {
  if (v < 0 || v > INT_MAX) refuse(std::string(name) + ": " + std::to_string(v) + " is out of range");
  return (int)v;
}

struct Types {
  ScalarType a, b;
  bool has(ScalarType t) const { return t == a || t == b; }
  std::string text() const { return std::string(c10::toString(a)) + (a == b ? "" : std::string(" or ") + c10::toString(b)); }
};
constexpr Types kI8{ScalarType::Char, ScalarType::Char}, kI32{ScalarType::Int, ScalarType::Int},
    kF32{ScalarType::Float, ScalarType::Float}, kBF16{ScalarType::BFloat16, ScalarType::BFloat16},
    kFloats{ScalarType::BFloat16, ScalarType::Float}, kFlags{ScalarType::Byte, ScalarType::Bool},
    kWords{ScalarType::Int, ScalarType::UInt32};

// A matrix argument: dtype, device, shape, rows that are runs of elements and share none; its row stride.  cols, n: -1
// for any.
int64_t rows_of(const Tensor& t, const char* name, Types types, const c10::Device* dev, int64_t cols = -1, int64_t n = -1) {
  const std::string at = std::string(name) + ": ";
  if (!t.defined() || t.layout() != c10::kStrided || !t.is_cuda()) refuse(at + "a CUDA tensor is needed");
  if (!types.has(t.scalar_type())) refuse(at + "dtype " + c10::toString(t.scalar_type()) + ", " + types.text() + " is needed");
  if (dev && t.device() != *dev) refuse(at + "on " + t.device().str() + ", the other tensors on " + dev->str());
  if (t.dim() != 2 || (cols >= 0 && t.size(1) != cols) || (n >= 0 && t.size(0) != n))
    refuse(at + "a matrix of " + (n >= 0 ? std::to_string(n) : "any") + " rows and " +
           (cols >= 0 ? std::to_string(cols) : "any") + " columns is needed");
  const int64_t r = t.size(0), c = t.size(1);
  // one row, or rows of one element, or none: their strides say nothing
  if ((t.stride(1) != 1 && c > 1) || (r > 1 && t.stride(0) < c)) refuse(at + "rows of consecutive elements are needed");
  return r > 1 ? t.stride(0) : c;
}

// An array argument of n elements (-1: any number), contiguous.
void array(const Tensor& t, const char* name, Types types, int64_t n, const c10::Device& dev) {
  if (t.defined() && t.layout() == c10::kStrided && types.has(t.scalar_type()) && t.device() == dev && t.is_contiguous() &&
      (n < 0 || t.numel() == n))
    return;
  refuse(std::string(name) + ": a contiguous tensor of " + (n >= 0 ? std::to_string(n) + " elements of " : "") +
         types.text() + " on " + dev.str() + " is needed");
}

// the tables' four words, which the kernels read by index
void meta_words(const Tensor& t, const c10::Device& dev) {
  array(t, "tables.meta", kI32, -1, dev);
  if (t.numel() < 4) refuse("tables.meta: " + std::to_string(t.numel()) + " elements, four are needed");
}

// rows_of an int8 operand: 16-byte aligned, its row stride a multiple of 16 (of a single row: rounded up)
int64_t int8_rows(const Tensor& t, const char* name, const c10::Device* dev, int64_t cols = -1, int64_t n = -1) {
  int64_t ld = rows_of(t, name, kI8, dev, cols, n);
  if (t.size(0) <= 1) ld = (ld + 15) / 16 * 16;
  if (ld % 16 || reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16)
    refuse(std::string(name) + ": 16-byte aligned rows are needed (quant_int8 pads them)");
  return ld;
}

int dtype_code(ScalarType t) {
  if (t == ScalarType::BFloat16) return K3MOE_BF16;
  if (t == ScalarType::Float) return K3MOE_F32;
  refuse(std::string("dtype ") + c10::toString(t) + ", bfloat16 or float32 is needed");
}

template <typename T = void>
T* ptr(const Tensor& t) {
  return reinterpret_cast<T*>(t.data_ptr());
}
template <typename T = void>
T* ptr(const MaybeTensor& t) {
  return t ? reinterpret_cast<T*>(t->data_ptr()) : nullptr;
}

// A call's outputs, straight from torch's CUDA allocator: its dispatcher would take another third of a microsecond each.
// It is asked where somebody listens: a dispatch mode is on, or new tensors are filled for determinism.
struct Outputs {
  c10::Device dev;
  bool dispatched;
  explicit Outputs(const c10::Device& d) : dev(d), dispatched(c10::impl::TorchDispatchModeTLS::any_modes_set()) {
    const auto& c = at::globalContext();
    dispatched = dispatched || (c.deterministicAlgorithms() && c.deterministicFillUninitializedMemory());
  }
  Tensor empty(at::IntArrayRef shape, ScalarType type) const {
    if (dispatched) return at::empty(shape, at::TensorOptions().dtype(type).device(dev));
    return at::detail::empty_cuda(shape, type, dev, std::nullopt);
  }
  Tensor empty_rows(int64_t rows, int64_t cols, int64_t ld, ScalarType type) const {
    if (ld == cols) return empty({rows, cols}, type);
    if (dispatched) return at::empty_strided({rows, cols}, {ld, 1}, at::TensorOptions().dtype(type).device(dev));
    return Tensor(at::detail::empty_strided_cuda({rows, cols}, {ld, 1}, type, dev));
  }
};

k3moe_stream_t stream_of(const c10::Device& dev) {
  return reinterpret_cast<k3moe_stream_t>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

void check(int rc, const char* what) {
  if (rc == K3MOE_OK) return;
  const char* why = rc == K3MOE_EINVAL    ? "invalid argument"
                    : rc == K3MOE_EDRIVER ? "CUDA driver tensor-map entry unavailable"
                    : rc == K3MOE_ETMAP   ? "tensor map could not be encoded (alignment / size)"
                    : rc == K3MOE_ELAUNCH ? "kernel launch failed"
                                          : "failed";
  refuse(std::string(what) + ": " + why + " (" + std::to_string(rc) + ")");
}

// ---------------------------------------------------------------- the router's training side
struct Router {
  c10::Device dev;
  int T, E, K, B, lds;
};
Router router(const Tensor& S, const Tensor& idx, const MaybeTensor& seq, const MaybeTensor& mask) {
  const int64_t ld = rows_of(S, "S", kF32, nullptr);
  Router r{S.device(), as_int(S.size(0), "S"), as_int(S.size(1), "S"), 0, 1, as_int(ld, "S's row stride")};
  array(idx, "idx", kI32, -1, r.dev);
  if (idx.dim() != 2 || idx.size(0) != r.T) refuse("idx: [" + std::to_string(r.T) + ", K] is needed");
  r.K = as_int(idx.size(1), "idx");
  if (seq) {
    array(*seq, "seq", kI32, -1, r.dev);
    if (seq->numel() < 2) refuse("seq: offsets [B + 1] are needed");
    r.B = as_int(seq->numel() - 1, "seq");
  }
  if (mask) array(*mask, "mask", kFlags, r.T, r.dev);
  return r;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> balance_loss(const Tensor& S, const Tensor& idx, double alpha,
                                                        const MaybeTensor& seq, const MaybeTensor& mask) {
  const Router r = router(S, idx, seq, mask);
  const c10::cuda::CUDAGuard guard(r.dev);
  const size_t bytes = k3moe_balance_scratch_bytes(r.T, r.E, r.B);
  if (bytes == 0) check(K3MOE_EINVAL, "balance_loss");
  const Outputs make(r.dev);
  const Tensor scratch = make.empty({(int64_t)bytes}, ScalarType::Byte);
  const Tensor loss = make.empty({1}, ScalarType::Float), rows = make.empty({r.B}, ScalarType::Int);
  const Tensor counts = make.empty({r.B, r.E}, ScalarType::Int), prob = make.empty({r.B, r.E}, ScalarType::Float);
  check(k3moe_balance_loss(ptr<float>(S), r.lds, ptr<int32_t>(idx), r.T, r.E, r.K, ptr<int32_t>(seq), r.B,
                           ptr<uint8_t>(mask), (float)alpha, ptr(scratch), ptr<int32_t>(counts), ptr<float>(prob),
                           ptr<int32_t>(rows), ptr<float>(loss), stream_of(r.dev)),
        "balance_loss");
  return {loss, counts, prob, rows};
}

Tensor route_backward(const Tensor& S, const Tensor& idx, double alpha, const MaybeTensor& counts, const MaybeTensor& rows,
                      const MaybeTensor& dloss, const MaybeTensor& dwts, const MaybeTensor& rs, const MaybeTensor& seq,
                      const MaybeTensor& mask, ScalarType dtype, const MaybeTensor& out) {
  const Router r = router(S, idx, seq, mask);
  if (counts.has_value() != rows.has_value()) refuse("counts and rows are given together");
  if (!counts && !dwts) refuse("counts and rows, or dwts and rs, are needed");
  if (counts) {
    array(*counts, "counts", kI32, (int64_t)r.B * r.E, r.dev);
    array(*rows, "rows", kI32, r.B, r.dev);
  }
  if (dloss) array(*dloss, "dloss", kF32, 1, r.dev);
  if (dwts) {
    array(*dwts, "dwts", kF32, (int64_t)r.T * r.K, r.dev);
    if (!rs) refuse("dwts needs rs");
    array(*rs, "rs", kBF16, 1, r.dev);
  }
  const int code = dtype_code(out ? out->scalar_type() : dtype);
  const int ldd = out ? as_int(rows_of(*out, "out", kFloats, &r.dev, r.E, r.T), "out's row stride") : r.E;
  const c10::cuda::CUDAGuard guard(r.dev);
  const Tensor dS = out ? *out : Outputs(r.dev).empty({r.T, r.E}, dtype);
  check(k3moe_route_backward(ptr<float>(S), r.lds, ptr<int32_t>(idx), r.T, r.E, r.K, ptr<int32_t>(seq), r.B,
                             ptr<uint8_t>(mask), (float)alpha, ptr<int32_t>(counts), ptr<int32_t>(rows), ptr<float>(dloss),
                             ptr<float>(dwts), ptr(rs), ptr(dS), ldd, code, stream_of(r.dev)),
        "route_backward");
  return dS;
}

// ---------------------------------------------------------------- products in 8-bit integers
struct Int8Out {
  Tensor q, scale;
  int64_t ld;
};
Int8Out int8_out(const Quantised& out, int64_t rows, int64_t cols, const c10::Device& dev) {
  if (out) {
    const auto& [q, scale] = *out;
    const int64_t ld = int8_rows(q, "out q", &dev, cols, rows);
    array(scale, "out scale", kF32, rows, dev);
    return {q, scale, ld};
  }
  const int64_t ld = (cols + 15) / 16 * 16;
  const Outputs make(dev);
  return {make.empty_rows(rows, cols, ld, ScalarType::Char), make.empty({rows}, ScalarType::Float), ld};
}

std::tuple<Tensor, Tensor> quant_int8(const Tensor& x, const Quantised& out) {
  const int64_t ldx = rows_of(x, "x", kFloats, nullptr);
  const c10::Device dev = x.device();
  const c10::cuda::CUDAGuard guard(dev);
  const Int8Out o = int8_out(out, x.size(0), x.size(1), dev);
  check(k3moe_quant_int8(ptr(x), dtype_code(x.scalar_type()), ldx, x.size(0), as_int(x.size(1), "x"), ptr<int8_t>(o.q), o.ld,
                         ptr<float>(o.scale), stream_of(dev)),
        "quant_int8");
  return {o.q, o.scale};
}

std::tuple<Tensor, Tensor> act_quant_int8(const Tensor& gu, int activation, const MaybeTensor& limit,
                                          const MaybeTensor& meta, int64_t max_ctas, const Quantised& out) {
  const int64_t ldg = rows_of(gu, "gu", kBF16, nullptr);
  const c10::Device dev = gu.device();
  if (gu.size(1) % 2) refuse("gu: " + std::to_string(gu.size(1)) + " columns, gate and up halves are needed");
  if (limit) {
    if (gu.size(0) > max_ctas * 128) refuse("gu: " + std::to_string(gu.size(0)) + " rows, more than the tables' tiles hold");
    array(*limit, "tables.cta_limit", kI32, max_ctas, dev);
    meta_words(meta.value(), dev);
  }
  const c10::cuda::CUDAGuard guard(dev);
  const Int8Out o = int8_out(out, gu.size(0), gu.size(1) / 2, dev);
  check(k3moe_act_quant_int8(ptr(gu), ldg, gu.size(0), as_int(gu.size(1) / 2, "gu"), activation, ptr<int32_t>(limit),
                             ptr<int32_t>(meta), as_int(max_ctas, "tables.max_ctas"), ptr<int8_t>(o.q), o.ld,
                             ptr<float>(o.scale), stream_of(dev)),
        "act_quant_int8");
  return {o.q, o.scale};
}

std::tuple<Tensor, Tensor> quant_int8_permute(const Tensor& x, const Tensor& exp2perm, const Tensor& meta, int64_t cap,
                                              const Quantised& out) {
  const int64_t ldx = rows_of(x, "x", kBF16, nullptr);
  const c10::Device dev = x.device();
  array(exp2perm, "tables.exp2perm", kI32, -1, dev);
  if (exp2perm.dim() != 2 || exp2perm.size(0) != x.size(0)) refuse("tables.exp2perm: a row for each of x is needed");
  meta_words(meta, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Int8Out o = int8_out(out, cap, x.size(1), dev);
  check(k3moe_quant_int8_permute(ptr(x), ldx, as_int(x.size(0), "x"), as_int(x.size(1), "x"), as_int(exp2perm.size(1), "K"),
                                 ptr<int32_t>(exp2perm), ptr<int32_t>(meta), ptr<int8_t>(o.q), o.ld, ptr<float>(o.scale),
                                 as_int(cap, "tables.cap_rows"), stream_of(dev)),
        "quant_int8_permute");
  return {o.q, o.scale};
}

struct Product {
  c10::Device dev;
  int64_t T, C, ldq, ldw;
};
Product product(const Tensor& q, const Tensor& sx, const Tensor& w, const Tensor& sw, const MaybeTensor& err) {
  const int64_t ldq = int8_rows(q, "q", nullptr);
  Product p{q.device(), q.size(0), q.size(1), ldq, 0};
  p.ldw = int8_rows(w, "w", &p.dev, p.C);
  array(sx, "sx", kF32, p.T, p.dev);
  array(sw, "sw", kF32, w.size(0), p.dev);
  if (err) {
    array(*err, "err", kWords, -1, p.dev);
    if (err->numel() < 2) refuse("err: two words are needed");
  }
  return p;
}
struct ProductOut {
  Tensor out;
  int64_t ld;
  int code;
};
ProductOut product_out(const Product& p, int64_t N, ScalarType dtype, const MaybeTensor& out) {
  if (out) return {*out, rows_of(*out, "out", kFloats, &p.dev, N, p.T), dtype_code(out->scalar_type())};
  const int code = dtype_code(dtype);
  return {Outputs(p.dev).empty({p.T, N}, dtype), N, code};
}

Tensor gemm_int8(const Tensor& q, const Tensor& sx, const Tensor& w, const Tensor& sw, ScalarType dtype,
                 const MaybeTensor& out, const MaybeTensor& err) {
  const Product p = product(q, sx, w, sw, err);
  const c10::cuda::CUDAGuard guard(p.dev);
  const ProductOut o = product_out(p, w.size(0), dtype, out);
  check(k3moe_gemm_int8(ptr<int8_t>(q), p.ldq, ptr<float>(sx), ptr<int8_t>(w), p.ldw, ptr<float>(sw), as_int(p.T, "q"),
                        as_int(w.size(0), "w"), as_int(p.C, "q"), ptr(o.out), o.ld, o.code, ptr<uint32_t>(err),
                        stream_of(p.dev)),
        "gemm_int8");
  return o.out;
}

Tensor grouped_gemm_int8(const Tensor& q, const Tensor& sx, const Tensor& w, const Tensor& sw, const Tensor& cta_batch,
                         const Tensor& cta_limit, const Tensor& meta, int64_t max_ctas, int64_t cap, int64_t n_experts,
                         ScalarType dtype, const MaybeTensor& out, const MaybeTensor& err) {
  const Product p = product(q, sx, w, sw, err);
  if (n_experts < 1 || w.size(0) % n_experts || p.T != cap)
    refuse("q of " + std::to_string(p.T) + " rows (capacity " + std::to_string(cap) + "), w of " +
           std::to_string(w.size(0)) + " rows for " + std::to_string(n_experts) + " experts");
  array(cta_batch, "tables.cta_batch", kI32, max_ctas, p.dev);
  array(cta_limit, "tables.cta_limit", kI32, max_ctas, p.dev);
  meta_words(meta, p.dev);
  const int64_t N = w.size(0) / n_experts;
  const c10::cuda::CUDAGuard guard(p.dev);
  const ProductOut o = product_out(p, N, dtype, out);
  check(k3moe_grouped_gemm_int8(ptr<int8_t>(q), p.ldq, ptr<float>(sx), ptr<int8_t>(w), p.ldw, ptr<float>(sw),
                                ptr<int32_t>(cta_batch), ptr<int32_t>(cta_limit), ptr<int32_t>(meta), as_int(N, "w"),
                                as_int(p.C, "q"), as_int(n_experts, "n_experts"), as_int(cap, "tables.cap_rows"),
                                as_int(max_ctas, "tables.max_ctas"), ptr(o.out), o.ld, o.code, ptr<uint32_t>(err),
                                stream_of(p.dev)),
        "grouped_gemm_int8");
  return o.out;
}

}  // namespace

// torch's own errors (out of memory among them) reach Python as its types
PYBIND11_MODULE(k3moe_torch, m) {
  m.def("set_error", [](py::object cls) { g_error = cls.release().ptr(); });
  m.def("balance_loss", torch::wrap_pybind_function(balance_loss));
  m.def("route_backward", torch::wrap_pybind_function(route_backward));
  m.def("quant_int8", torch::wrap_pybind_function(quant_int8));
  m.def("act_quant_int8", torch::wrap_pybind_function(act_quant_int8));
  m.def("quant_int8_permute", torch::wrap_pybind_function(quant_int8_permute));
  m.def("gemm_int8", torch::wrap_pybind_function(gemm_int8));
  m.def("grouped_gemm_int8", torch::wrap_pybind_function(grouped_gemm_int8));
}
