// torch binding of the grouped routing, norm and int8 entry points of
// libb200moe.so: checks the tensors, allocates the outputs and calls the C ABI
// on the current stream of their device. These calls are short on the device
// (3 to 9 us for a decode step's rows), and the same work through ctypes and
// torch.empty took 13 to 26 us of host time a call.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <sstream>
#include <string>

#include "b200moe.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

template <class... A>
[[noreturn]] void bad(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw py::value_error(s.str());
}
template <class... A>
void need(bool ok, const A&... a) {
  if (!ok) bad(a...);
}

// A library status as the exception that _lib.check raises for it.
void check(int rc, const char* what) {
  if (rc == B200MOE_OK) return;
  const std::string msg = std::string(what) + ": " + b200moe_last_error();
  if (rc == B200MOE_ERR_INVALID) throw py::value_error(msg);
  PyErr_SetString(rc == B200MOE_ERR_UNSUPPORTED ? PyExc_NotImplementedError : PyExc_RuntimeError, msg.c_str());
  throw py::error_already_set();
}

int on_cuda(const Tensor& t, const char* what) {
  need(t.is_cuda(), what, " must be a CUDA tensor (b200moe has no CPU path), got ", t.device());
  return t.get_device();
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// From the caching allocator directly (through the dispatcher a call with four
// outputs takes 1 us longer).
Tensor empty(c10::IntArrayRef shape, const Tensor& like, at::ScalarType type) {
  return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}

const void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

// The row stride of a 2D tensor with contiguous rows.
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// 0 / 1: the C calls' fp32 / bf16 switch.
int is_bf16(const Tensor& t, const char* what) {
  const at::ScalarType s = t.scalar_type();
  need(s == at::kFloat || s == at::kBFloat16, what, " must be float32 or bfloat16, got ", s);
  return s == at::kBFloat16;
}

void check_rows(const Tensor& t, int device, const char* what) {
  need(t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1 && t.is_cuda() && t.get_device() == device,
       what, " must be a 2D bfloat16 tensor with contiguous rows on cuda:", device, ", got ", t.scalar_type(), " ",
       t.sizes(), " on ", t.device());
}

void check_int32(const Tensor& t, int device, int64_t n, const char* what) {
  need(t.scalar_type() == at::kInt && t.is_contiguous() && t.is_cuda() && t.get_device() == device && t.numel() >= n,
       what, " must be contiguous int32 of ", n, " elements on cuda:", device, ", got ", t.scalar_type(), " ", t.sizes(),
       " on ", t.device());
}

int to_int(int64_t v, const char* what) {
  need(v >= 0 && v <= 0x7fffffff, what, " is out of range");
  return static_cast<int>(v);
}

template <class F>
int enqueue(F&& f) {
  py::gil_scoped_release free_gil;   // a full launch queue blocks
  return f();
}

// ------------------------------------------------------------ routing
py::tuple route_grouped(const Tensor& logits, const OptTensor& bias, int64_t top_k, int n_group, int topk_group,
                        int group_top, int scoring, bool normalize, float scale) {
  const int device = on_cuda(logits, "logits");
  const int bf16 = is_bf16(logits, "logits");
  need(logits.dim() == 2 && logits.stride(1) == 1, "logits must be a 2D tensor with contiguous rows");
  const int64_t T = logits.size(0), E = logits.size(1);
  if (bias)
    need(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == E && bias->is_contiguous() &&
             bias->is_cuda() && bias->get_device() == device,
         "bias must be contiguous float32 [", E, "] on ", logits.device());
  need(top_k >= 1 && top_k <= E, "top_k must be in [1, ", E, "], got ", top_k);
  Tensor scores = empty({T, top_k}, logits, at::kFloat);
  Tensor indices = empty({T, top_k}, logits, at::kLong);
  Tensor counts = empty({E}, logits, at::kInt);
  const int t = to_int(T, "tokens"), e = to_int(E, "experts");
  check(enqueue([&] {
          return b200moe_route_grouped(device, stream_of(device), logits.data_ptr(), bf16, row_stride(logits),
                                       static_cast<const float*>(ptr(bias)), t, e, static_cast<int>(top_k), n_group,
                                       topk_group, group_top, scoring, normalize, scale, scores.data_ptr<float>(),
                                       reinterpret_cast<long long*>(indices.data_ptr<int64_t>()),
                                       counts.data_ptr<int>());
        }),
        "route_grouped");
  return py::make_tuple(scores, indices, counts);
}

// ------------------------------------------------------------ 8-bit rows
struct QuantRows {
  Tensor q, scale;
  // this, if these are rows of the type and width on the device
  const QuantRows& checked(at::ScalarType type, int64_t k_pad, const at::Device& device) const {
    need(q.scalar_type() == type && q.dim() == 2 && q.size(1) == k_pad && q.is_contiguous(),
         "quantised rows must be contiguous ", type, " [rows, ", k_pad, "], got ", q.scalar_type(), " ", q.sizes());
    const int64_t groups = (k_pad + 127) / 128;
    need(scale.scalar_type() == at::kFloat && scale.is_contiguous() && scale.dim() == (type == at::kChar ? 1 : 2) &&
             scale.size(0) == q.size(0) && (type == at::kChar || scale.size(1) == groups),
         "row scales must be contiguous float32, one per ", type == at::kChar ? "row" : "row and 128 columns", ", got ",
         scale.scalar_type(), " ", scale.sizes());
    need(q.device() == device && scale.device() == device, "quantised rows must be on ", device);
    return *this;
  }
};

struct Range {   // places of a rank's experts only
  const int* offsets = nullptr;
  int lo = 0, hi = 0;
};
Range expert_range(const OptTensor& offsets, int lo, int hi, int device) {
  if (!offsets) return {};
  need(lo >= 0 && hi >= lo, "need 0 <= expert_lo <= expert_hi");
  check_int32(*offsets, device, int64_t(hi) + 1, "offsets");
  return {offsets->data_ptr<int>(), lo, hi};
}

QuantRows act_quant_int8(const Tensor& x, std::optional<int64_t> width, const OptTensor& inverse, int64_t copies,
                         const OptTensor& offsets, int expert_lo, int expert_hi) {
  const int device = on_cuda(x, "x");
  check_rows(x, device, "x");
  const int64_t rows = x.size(0), k = x.size(1), k_pad = width ? *width : (k + 127) / 128 * 128;
  int64_t out = rows;
  need(copies >= 1 && (inverse || copies == 1), "copies need inverse");
  if (inverse) {
    out = rows * copies;
    check_int32(*inverse, device, out, "inverse");
    need(inverse->numel() == out, "inverse must have rows * copies = ", out, " elements");
  }
  need(k_pad >= k, "k_pad must be at least ", k, ", got ", k_pad);
  const Range r = expert_range(offsets, expert_lo, expert_hi, device);
  const int n = to_int(rows, "rows"), m = to_int(out, "rows"), kv = to_int(k, "columns"), kp = to_int(k_pad, "k_pad");
  QuantRows q{empty({out, k_pad}, x, at::kChar), empty({out}, x, at::kFloat)};
  check(enqueue([&] {
          return b200moe_act_quant_int8(device, stream_of(device), x.data_ptr(), row_stride(x), n, kv, kp,
                                        static_cast<const int*>(ptr(inverse)), static_cast<int>(copies), m, r.offsets,
                                        r.lo, r.hi, q.q.data_ptr(), q.scale.data_ptr<float>());
        }),
        "act_quant_int8");
  return q;
}

QuantRows scatter_rows_8bit(const QuantRows& rows, const Tensor& inverse, int64_t copies, const OptTensor& offsets,
                            int expert_lo, int expert_hi) {
  const int device = on_cuda(rows.q, "rows");
  const at::ScalarType type = rows.q.scalar_type();
  need(type == at::kChar || type == at::kFloat8_e4m3fn, "rows must be int8 or float8_e4m3fn, got ", type);
  need(rows.q.dim() == 2, "rows must be 2D");
  rows.checked(type, rows.q.size(1), rows.q.device());
  const int64_t n = rows.q.size(0), width = rows.q.size(1), out = n * copies;
  need(copies >= 1, "copies must be at least 1");
  check_int32(inverse, device, out, "inverse");
  need(inverse.numel() == out, "inverse must have rows * copies = ", out, " elements");
  const int64_t groups = type == at::kChar ? 1 : rows.scale.size(1);
  const Range r = expert_range(offsets, expert_lo, expert_hi, device);
  const int nr = to_int(n, "rows"), m = to_int(out, "rows");
  QuantRows q{empty({out, width}, rows.q, type),
              type == at::kChar ? empty({out}, rows.q, at::kFloat) : empty({out, groups}, rows.q, at::kFloat)};
  check(enqueue([&] {
          return b200moe_scatter_rows_8bit(device, stream_of(device), rows.q.data_ptr(), static_cast<int>(width),
                                           rows.scale.data_ptr<float>(), static_cast<int>(groups), nr,
                                           inverse.data_ptr<int>(), static_cast<int>(copies), m, r.offsets, r.lo, r.hi,
                                           q.q.data_ptr(), q.scale.data_ptr<float>());
        }),
        "scatter_rows_8bit");
  return q;
}

// ------------------------------------------------------------ norm
py::tuple add_rmsnorm(const Tensor& x, const Tensor& weight, float eps, const OptTensor& residual,
                      const OptTensor& residual_out, int quant, std::optional<int64_t> width, bool normed) {
  const int device = on_cuda(x, "x");
  check_rows(x, device, "x");
  const int64_t T = x.size(0), H = x.size(1);
  need(weight.dim() == 1 && weight.size(0) == H && weight.is_contiguous() && weight.is_cuda() &&
           weight.get_device() == device,
       "weight must be contiguous [", H, "] on ", x.device(), ", got ", weight.sizes(), " on ", weight.device());
  const int f32 = 1 - is_bf16(weight, "weight");
  need(quant != B200MOE_QUANT_NONE || normed, "nothing to compute: no quantised rows and no bf16 output");
  need(residual || !residual_out, "residual_out needs a residual");
  OptTensor sum, out;
  if (residual) {
    check_rows(*residual, device, "residual");
    need(residual->sizes() == x.sizes(), "residual must have x's shape ", x.sizes(), ", got ", residual->sizes());
    if (residual_out) {
      check_rows(*residual_out, device, "residual_out");
      need(residual_out->sizes() == x.sizes(), "residual_out must have x's shape ", x.sizes(), ", got ",
           residual_out->sizes());
      sum = residual_out;
    } else {
      sum = empty({T, H}, x, at::kBFloat16);
    }
  }
  if (normed) out = empty({T, H}, x, at::kBFloat16);
  std::optional<QuantRows> rows;
  int64_t k_pad = 0;
  if (quant != B200MOE_QUANT_NONE) {
    const bool fp8 = quant == B200MOE_QUANT_FP8;
    const int64_t unit = fp8 ? 64 : 128;   // what the experts of that form take
    k_pad = width ? *width : (H + unit - 1) / unit * unit;
    need(k_pad >= H && k_pad <= 0x7fffffff, "k_pad must be at least ", H);
    rows = QuantRows{empty({T, k_pad}, x, fp8 ? at::kFloat8_e4m3fn : at::kChar),
                     fp8 ? empty({T, (k_pad + 127) / 128}, x, at::kFloat) : empty({T}, x, at::kFloat)};
  }
  const int t = to_int(T, "tokens"), h = to_int(H, "columns");
  check(enqueue([&] {
          return b200moe_add_rmsnorm(
              device, stream_of(device), x.data_ptr(), row_stride(x), ptr(residual), residual ? row_stride(*residual) : 0,
              const_cast<void*>(ptr(sum)), sum ? row_stride(*sum) : 0, weight.data_ptr(), f32, eps, t, h,
              const_cast<void*>(ptr(out)), H, quant, rows ? rows->q.data_ptr() : nullptr, static_cast<int>(k_pad),
              rows ? rows->scale.data_ptr<float>() : nullptr);
        }),
        "add_rmsnorm");
  return py::make_tuple(out, sum, rows);
}

// ------------------------------------------------------------ int8 products
struct Int8Matrix {
  int n_experts, planes;
  int64_t n_feat, k_valid, feat_pad, k_pad;
  Tensor weight, scale;
  OptTensor bias;
  int epilogue;
  float alpha, limit;

  Int8Matrix(int n_experts_, int planes_, int64_t n_feat_, int64_t k_valid_, int64_t feat_pad_, int64_t k_pad_,
             Tensor weight_, Tensor scale_, OptTensor bias_, int epilogue_, float alpha_, float limit_)
      : n_experts(n_experts_), planes(planes_), n_feat(n_feat_), k_valid(k_valid_), feat_pad(feat_pad_), k_pad(k_pad_),
        weight(std::move(weight_)), scale(std::move(scale_)), bias(std::move(bias_)), epilogue(epilogue_),
        alpha(alpha_), limit(limit_) {
    need(planes == 1 || planes == 2, "planes must be 1 or 2");
    need(n_experts >= 1 && n_feat >= 1 && n_feat <= feat_pad && k_valid >= 1 && k_valid <= k_pad &&
             feat_pad % 128 == 0 && k_pad % 128 == 0 && feat_pad <= 0x7fffffff && k_pad <= 0x7fffffff,
         "bad sizes of int8 weights");
    const int64_t rows = n_experts * (feat_pad / (planes == 2 ? 64 : 128)) * 128;
    need(weight.scalar_type() == at::kChar && weight.is_contiguous() && weight.numel() == rows * k_pad,
         "weight must be contiguous int8 tiles of ", rows * k_pad, " elements");
    for (const Tensor* t : {&scale, bias ? &*bias : nullptr})
      if (t)
        need(t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == rows &&
                 t->device() == weight.device(),
             "scale and bias must be contiguous float32 of ", rows, " elements on ", weight.device());
  }
};

struct Placement {   // where an int8 launch's rows are, and what scales them
  OptTensor offsets;
  int expert_begin;
  OptTensor row_weight, row_src;
  OptTensor out;
  int token_tile;
};

// The arguments of a launch over at most R rows (b_rows allocated); allocates
// the output where none is given.
b200moe_gemm_args gemm_args(const Int8Matrix& m, Placement& p, int device, int64_t R, int64_t b_rows) {
  b200moe_gemm_args a{};
  need(R >= 0, "max_rows must not be negative");
  if (!p.out) p.out = empty({R, m.planes == 2 ? m.feat_pad : m.n_feat}, m.weight, at::kBFloat16);
  check_rows(*p.out, device, "output");
  need(p.out->size(0) >= R && p.out->size(1) >= m.n_feat, "output must hold ", R, " rows of ", m.n_feat,
       " columns, got ", p.out->sizes());
  if (p.offsets) {
    need(p.expert_begin >= 0, "expert_begin must not be negative");
    check_int32(*p.offsets, device, int64_t(p.expert_begin) + m.n_experts + 1, "offsets");
    a.offsets = p.offsets->data_ptr<int>();
  }
  if (p.row_weight) {
    a.row_weight_bf16 = is_bf16(*p.row_weight, "row_weight");
    need(p.row_weight->is_contiguous() && p.row_weight->is_cuda() && p.row_weight->get_device() == device &&
             p.row_weight->numel() >= R,
         "row_weight must be contiguous, one per row, on ", m.weight.device());
    need(p.row_src.has_value(), "row_weight needs row_src");
    check_int32(*p.row_src, device, R, "row_src");
    a.row_weight = p.row_weight->data_ptr();
    a.row_src = p.row_src->data_ptr<int>();
  }
  a.expert_begin = p.expert_begin;
  a.n_experts = m.n_experts;
  a.max_rows = to_int(R, "rows");
  a.token_tile = p.token_tile;
  a.wfmt = B200MOE_W_INT8;
  a.planes = m.planes;
  a.feat_pad = static_cast<int>(m.feat_pad);
  a.n_feat = static_cast<int>(m.n_feat);
  a.k_pad = static_cast<int>(m.k_pad);
  a.weight = m.weight.data_ptr();
  a.b_rows = to_int(b_rows, "rows");
  a.b_div = 1;
  a.epilogue = m.epilogue;
  a.alpha = m.alpha;
  a.limit = m.limit;
  a.out = p.out->data_ptr();
  a.ldo = p.out->size(0) > 1 ? p.out->stride(0) : m.n_feat;
  return a;
}

Tensor int8_gemm(const Int8Matrix& m, const QuantRows& rows, const OptTensor& offsets, int expert_begin,
                 std::optional<int64_t> max_rows, const OptTensor& row_weight, const OptTensor& row_src,
                 const OptTensor& out, int token_tile) {
  const int device = on_cuda(m.weight, "weight");
  rows.checked(at::kChar, m.k_pad, m.weight.device());
  const int64_t n = rows.q.size(0), R = max_rows ? *max_rows : n;
  Placement p{offsets, expert_begin, row_weight, row_src, out, token_tile};
  const b200moe_gemm_args a = gemm_args(m, p, device, R, n);
  check(enqueue([&] {
          return b200moe_int8_gemm(device, stream_of(device), &a, rows.q.data_ptr(), rows.scale.data_ptr<float>(),
                                   m.scale.data_ptr<float>(), static_cast<const float*>(ptr(m.bias)));
        }),
        "int8_gemm");
  return *p.out;
}

Tensor int8_project(const Int8Matrix& m, const Tensor& x, const OptTensor& offsets, int expert_begin,
                    const OptTensor& inverse, int64_t copies, const OptTensor& row_weight, const OptTensor& row_src,
                    const OptTensor& out, int token_tile) {
  const int device = on_cuda(m.weight, "weight");
  check_rows(x, device, "x");
  need(x.size(1) >= m.k_valid, "x has ", x.size(1), " columns, the weights take ", m.k_valid);
  const int64_t rows = x.size(0);
  int64_t R = rows;
  need(copies >= 1 && (inverse || copies == 1), "copies need inverse");
  if (inverse) {
    R = rows * copies;
    check_int32(*inverse, device, R, "inverse");
    need(inverse->numel() == R, "inverse must have rows * copies = ", R, " elements");
  }
  Placement p{offsets, expert_begin, row_weight, row_src, out, token_tile};
  const b200moe_gemm_args a = gemm_args(m, p, device, R, R);
  const int n = to_int(rows, "rows");
  const size_t bytes = b200moe_int8_project_workspace(a.b_rows, a.k_pad);
  Tensor ws = empty({static_cast<int64_t>(bytes)}, m.weight, at::kByte);
  check(enqueue([&] {
          return b200moe_int8_project(device, stream_of(device), &a, x.data_ptr(),
                                      rows > 1 ? x.stride(0) : m.k_valid, n, static_cast<int>(m.k_valid),
                                      static_cast<const int*>(ptr(inverse)), static_cast<int>(copies),
                                      m.scale.data_ptr<float>(), static_cast<const float*>(ptr(m.bias)),
                                      ws.data_ptr(), bytes);
        }),
        "int8_project");
  return *p.out;
}

}  // namespace

PYBIND11_MODULE(_ext, mod) {
  mod.attr("built_for") = B200MOE_BUILT_FOR;   // the torch and Python of the build, by its command
  py::class_<QuantRows>(mod, "QuantRows",
                        "Rows in 8 bits with their scales: e4m3 ``q`` [rows, k_pad] with fp32\n``scale`` [rows, "
                        "ceil(k_pad / 128)] (W8A8 FP8 experts) or int8 ``q`` with\n``scale`` [rows] (int8 experts and "
                        "products).")
      .def(py::init([](Tensor q, Tensor s) { return QuantRows{std::move(q), std::move(s)}; }), py::arg("q"),
           py::arg("scale"))
      .def_readonly("q", &QuantRows::q)
      .def_readonly("scale", &QuantRows::scale)
      .def(
          "checked",
          [](py::object self, at::ScalarType type, int64_t k_pad, at::Device device) {
            self.cast<const QuantRows&>().checked(type, k_pad, device);
            return self;
          },
          "Self, if these are rows of the dtype and width on the device.")
      .def(py::pickle([](const QuantRows& r) { return py::make_tuple(r.q, r.scale); },
                      [](py::tuple t) { return QuantRows{t[0].cast<Tensor>(), t[1].cast<Tensor>()}; }));
  py::class_<Int8Matrix>(mod, "Int8Matrix",
                         "Int8 weights in tile layout (layout.int8_experts / int8_linear) with\nwhat the int8 GEMM has "
                         "to know of them; checked once, here.")
      .def(py::init<int, int, int64_t, int64_t, int64_t, int64_t, Tensor, Tensor, OptTensor, int, float, float>(),
           py::arg("n_experts"), py::arg("planes"), py::arg("n_feat"), py::arg("k_valid"), py::arg("feat_pad"),
           py::arg("k_pad"), py::arg("weight"), py::arg("scale"), py::arg("bias"), py::arg("epilogue"),
           py::arg("alpha") = 1.702f, py::arg("limit") = 7.0f)
      .def_readonly("n_experts", &Int8Matrix::n_experts)
      .def_readonly("planes", &Int8Matrix::planes)
      .def_readonly("n_feat", &Int8Matrix::n_feat)
      .def_readonly("k_valid", &Int8Matrix::k_valid)
      .def_readonly("feat_pad", &Int8Matrix::feat_pad)
      .def_readonly("k_pad", &Int8Matrix::k_pad)
      .def_readonly("weight", &Int8Matrix::weight)
      .def_readonly("scale", &Int8Matrix::scale)
      .def_readonly("bias", &Int8Matrix::bias)
      .def_readonly("epilogue", &Int8Matrix::epilogue)
      .def_readonly("alpha", &Int8Matrix::alpha)
      .def_readonly("limit", &Int8Matrix::limit)
      .def(py::pickle(
          [](const Int8Matrix& m) {
            return py::make_tuple(m.n_experts, m.planes, m.n_feat, m.k_valid, m.feat_pad, m.k_pad, m.weight, m.scale,
                                  m.bias, m.epilogue, m.alpha, m.limit);
          },
          [](py::tuple t) {
            return Int8Matrix(t[0].cast<int>(), t[1].cast<int>(), t[2].cast<int64_t>(), t[3].cast<int64_t>(),
                              t[4].cast<int64_t>(), t[5].cast<int64_t>(), t[6].cast<Tensor>(), t[7].cast<Tensor>(),
                              t[8].cast<OptTensor>(), t[9].cast<int>(), t[10].cast<float>(), t[11].cast<float>());
          }));
  mod.def("route_grouped", &route_grouped);
  mod.def("act_quant_int8", &act_quant_int8);
  mod.def("scatter_rows_8bit", &scatter_rows_8bit);
  mod.def("add_rmsnorm", &add_rmsnorm);
  mod.def("int8_gemm", &int8_gemm);
  mod.def("int8_project", &int8_project);
}
