// Python bindings of the expert-layer operators (ep/expert_ops.h): every
// argument is checked here, so a kernel never sees a shape, a stride or an
// alignment that it does not handle.

#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <numeric>
#include <vector>

#include "../ep/expert_ops.h"

namespace py = pybind11;

namespace uccl {

namespace {

using ep::Elem;
using ep::Mat;
using OptTensor = std::optional<at::Tensor>;

hipStream_t stream_of(at::Tensor const& t) {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device())
      .stream();
}

void check_launch(char const* what) {
  hipError_t const e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, "uccl_amd: ", what,
              " could not be launched: ", hipGetErrorString(e));
}

Elem elem_of(at::Tensor const& t, char const* name) {
  switch (t.scalar_type()) {
    case at::kFloat8_e4m3fn: return Elem::kF8;
    case at::kBFloat16: return Elem::kBF16;
    case at::kHalf: return Elem::kF16;
    case at::kFloat: return Elem::kF32;
    default:
      TORCH_CHECK(false, "uccl_amd: ", name, " has unsupported dtype ",
                  t.scalar_type());
  }
}

void check_on(at::Tensor const& t, at::Tensor const& first, char const* name) {
  TORCH_CHECK(t.device() == first.device(), "uccl_amd: ", name, " is on ",
              t.device(), ", the first operand on ", first.device());
}

// The last check: everything else about an operand can be refused wherever
// it lies.
void check_gpu(at::Tensor const& first, char const* name) {
  TORCH_CHECK(first.is_cuda(), "uccl_amd: ", name, " must be on GPU");
}

void check_shape(at::Tensor const& t, std::vector<int64_t> const& want,
                 char const* name) {
  TORCH_CHECK(t.sizes().vec() == want, "uccl_amd: ", name, " has shape ",
              t.sizes(), ", expected ", at::IntArrayRef(want));
}

void check_dense(at::Tensor const& t, char const* name) {
  TORCH_CHECK(t.is_contiguous(), "uccl_amd: ", name, " must be contiguous");
}

// Bytes from the first element on that `t` reaches into.
int64_t span_of(at::Tensor const& t) {
  if (t.numel() == 0) return 0;
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += t.stride(d) * (t.size(d) - 1);
  return (last + 1) * t.element_size();
}

// Whether no element of `a` shares memory with one of `b`, as far as their
// spans or the columns of a common pitch tell.
bool lie_apart(at::Tensor const& a, at::Tensor const& b) {
  if (a.numel() == 0 || b.numel() == 0) return true;
  auto const begin_a = reinterpret_cast<uintptr_t>(a.data_ptr());
  auto const begin_b = reinterpret_cast<uintptr_t>(b.data_ptr());
  if (begin_a + span_of(a) <= begin_b || begin_b + span_of(b) <= begin_a)
    return true;
  // Rows of contiguous elements, all of which start at multiples of `pitch`
  // bytes from the tensor's first.
  int64_t pitch = 0;
  auto row_of = [&](at::Tensor const& t) {
    int64_t row = 0;
    for (int64_t d = 0; d < t.dim(); ++d) {
      if (t.size(d) <= 1) continue;
      if (t.stride(d) == 1 && row == 0)
        row = t.size(d) * t.element_size();
      else
        pitch = std::gcd(pitch, t.stride(d) * t.element_size());
    }
    return row ? row : t.element_size();
  };
  int64_t const row_a = row_of(a), row_b = row_of(b);
  if (pitch == 0) return false;
  // where rows of b start behind those of a
  auto const ahead = static_cast<int64_t>(
      begin_b >= begin_a ? (begin_b - begin_a) % pitch
                         : (pitch - (begin_a - begin_b) % pitch) % pitch);
  return row_a <= ahead && ahead + row_b <= pitch;
}

// A result: no two elements share memory, and none shares it with an operand
// or with the counts.
void check_result(at::Tensor const& out, char const* name,
                  std::vector<at::Tensor> const& operands,
                  OptTensor const& counts = {}) {
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t d = 0; d < out.dim(); ++d)
    if (out.size(d) > 1) dims.emplace_back(out.stride(d), out.size(d));
  std::sort(dims.begin(), dims.end());
  int64_t extent = 1;
  for (auto const& [stride, size] : dims) {
    TORCH_CHECK(stride >= extent, "uccl_amd: elements of ", name,
                " share memory (strides ", out.strides(), ")");
    extent += stride * (size - 1);
  }
  for (auto const& t : operands)
    TORCH_CHECK(lie_apart(out, t), "uccl_amd: ", name, " overlaps an operand");
  TORCH_CHECK(!counts || lie_apart(out, *counts), "uccl_amd: ", name,
              " overlaps the counts");
}

// [experts, rows, cols] with contiguous columns whose rows start at 16-byte
// boundaries (or `align` bytes).
Mat mat_of(at::Tensor const& t, char const* name, int align = 16) {
  TORCH_CHECK(t.size(2) <= 1 || t.stride(2) == 1, "uccl_amd: the columns of ",
              name, " must be contiguous (strides ", t.strides(), ")");
  int64_t const es = t.element_size();
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % align == 0;
  ok &= t.size(0) <= 1 || t.stride(0) * es % align == 0;
  ok &= t.size(1) <= 1 || t.stride(1) * es % align == 0;
  TORCH_CHECK(ok, "uccl_amd: the rows of ", name, " must start at ", align,
              "-byte boundaries (strides ", t.strides(), " elements)");
  return Mat{t.data_ptr(), t.size(0) > 1 ? t.stride(0) : 0,
             t.size(1) > 1 ? t.stride(1) : 0};
}

ep::SlotRows rows_of(at::Tensor const& x, OptTensor const& counts) {
  int64_t const experts = x.size(0), slots = x.size(1);
  TORCH_CHECK(experts >= 1 && experts <= ep::kMaxSlotExperts,
              "uccl_amd: 1 to ", ep::kMaxSlotExperts, " experts, got ",
              experts);
  TORCH_CHECK(experts * slots < (int64_t(1) << 30),
              "uccl_amd: too many slots");
  int64_t sources = 1;
  if (counts) {
    check_on(*counts, x, "counts");
    TORCH_CHECK(counts->scalar_type() == at::kInt, "uccl_amd: counts must be "
                "int32, got ", counts->scalar_type());
    TORCH_CHECK(counts->dim() == 2 && counts->size(0) == experts &&
                    counts->size(1) >= 1,
                "uccl_amd: counts has shape ", counts->sizes(),
                ", expected [", experts, ", sources]");
    check_dense(*counts, "counts");
    sources = counts->size(1);
    TORCH_CHECK(experts * sources <= ep::kMaxSlotCells,
                "uccl_amd: at most ", ep::kMaxSlotCells,
                " counts, got ", experts * sources);
    TORCH_CHECK(slots % sources == 0, "uccl_amd: ", slots,
                " slots do not divide among ", sources, " sources");
  }
  return ep::SlotRows{counts ? counts->data_ptr<int>() : nullptr,
                      static_cast<int>(experts), static_cast<int>(sources),
                      static_cast<int>(slots / sources)};
}

void check_slots(at::Tensor const& t, char const* name) {
  TORCH_CHECK(t.dim() == 3, "uccl_amd: ", name,
              " must be [experts, slots, columns], got ", t.sizes());
}

void check_16bit(at::Tensor const& t, char const* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf,
              "uccl_amd: ", name, " must be bfloat16 or float16, got ",
              t.scalar_type());
}

// What the kernels count in 32 bits: rows and columns with a tile's behind
// them, bytes of a row, tiles, threads for 16 columns each.
void check_tiles(int64_t experts, int64_t a, int64_t b) {
  TORCH_CHECK(a < (int64_t(1) << 28) && b < (int64_t(1) << 30) &&
                  experts * ((a + 15) / 16) * ((b + 15) / 16) <
                      (int64_t(1) << 31),
              "uccl_amd: the product is too large");
}

// --- routing ---------------------------------------------------------------

ep::RouteArgs route_args(at::Tensor const& logits, int64_t topk,
                         std::string const& scoring, bool renormalize,
                         double scale) {
  TORCH_CHECK(logits.dim() == 2, "uccl_amd: logits must be [tokens, experts], "
              "got ", logits.sizes());
  TORCH_CHECK(scoring == "softmax" || scoring == "sigmoid",
              "uccl_amd: scoring is 'softmax' or 'sigmoid', got '", scoring,
              "'");
  int64_t const experts = logits.size(1);
  TORCH_CHECK(experts >= 1 && experts <= ep::kMaxRouteExperts,
              "uccl_amd: 1 to ", ep::kMaxRouteExperts, " experts, got ",
              experts);
  // 64 lanes a token, and less than 2^32 lanes of a launch
  TORCH_CHECK(logits.size(0) < (int64_t(1) << 25),
              "uccl_amd: too many tokens");
  TORCH_CHECK(topk >= 1 && topk <= std::min<int64_t>(experts,
                                                     ep::kMaxRouteTopk),
              "uccl_amd: topk is 1 to ",
              std::min<int64_t>(experts, ep::kMaxRouteTopk), ", got ", topk);
  TORCH_CHECK(experts == 1 || logits.stride(1) == 1,
              "uccl_amd: the columns of logits must be contiguous");
  ep::RouteArgs a{};
  a.logits = logits.data_ptr();
  a.stride = logits.size(0) > 1 ? logits.stride(0) : 0;
  a.elem = elem_of(logits, "logits");
  TORCH_CHECK(a.elem != Elem::kF8, "uccl_amd: logits has unsupported dtype ",
              logits.scalar_type());
  a.tokens = static_cast<int>(logits.size(0));
  a.experts = static_cast<int>(experts);
  a.topk = static_cast<int>(topk);
  a.sigmoid = scoring == "sigmoid";
  a.groups = a.topk_groups = 1;
  a.group_best = 2;
  a.renormalize = renormalize;
  a.scale = static_cast<float>(scale);
  return a;
}

void route(at::Tensor logits, OptTensor bias, std::string const& scoring,
           int64_t groups, int64_t topk_groups, int64_t group_best,
           bool renormalize, double scale, at::Tensor idx,
           at::Tensor weights) {
  TORCH_CHECK(idx.dim() == 2, "uccl_amd: topk_idx must be [tokens, topk]");
  auto a = route_args(logits, idx.size(1), scoring, renormalize, scale);
  TORCH_CHECK(groups >= 1 && groups <= ep::kMaxRouteGroups &&
                  a.experts % groups == 0,
              "uccl_amd: num_groups is 1 to ", ep::kMaxRouteGroups,
              " and divides ", a.experts, " experts, got ", groups);
  TORCH_CHECK(topk_groups >= 1 && topk_groups <= groups,
              "uccl_amd: topk_groups is 1 to num_groups, got ", topk_groups);
  TORCH_CHECK(a.topk <= topk_groups * (a.experts / groups),
              "uccl_amd: topk ", a.topk, " exceeds the experts of ",
              topk_groups, " groups");
  TORCH_CHECK(group_best == 1 || group_best == 2,
              "uccl_amd: group_best is 1 or 2, got ", group_best);
  a.groups = static_cast<int>(groups);
  a.topk_groups = static_cast<int>(topk_groups);
  a.group_best = static_cast<int>(group_best);
  if (bias) {
    check_on(*bias, logits, "bias");
    TORCH_CHECK(bias->scalar_type() == at::kFloat,
                "uccl_amd: bias must be float32, got ", bias->scalar_type());
    check_shape(*bias, {a.experts}, "bias");
    check_dense(*bias, "bias");
    a.bias = bias->data_ptr<float>();
  }
  for (auto const& [t, name] : {std::pair(idx, "topk_idx"),
                                std::pair(weights, "topk_weights")}) {
    check_on(t, logits, name);
    check_shape(t, {a.tokens, a.topk}, name);
    check_dense(t, name);
  }
  TORCH_CHECK(idx.scalar_type() == at::kLong &&
              weights.scalar_type() == at::kFloat);
  check_gpu(logits, "logits");
  if (a.tokens == 0) return;
  c10::DeviceGuard guard(logits.device());
  ep::launch_route(a, idx.data_ptr<int64_t>(), weights.data_ptr<float>(),
                   stream_of(logits));
  check_launch("route");
}

void route_grad(at::Tensor grad_weights, at::Tensor logits, at::Tensor idx,
                std::string const& scoring, bool renormalize, double scale,
                at::Tensor out) {
  TORCH_CHECK(idx.dim() == 2, "uccl_amd: topk_idx must be [tokens, topk]");
  auto const a =
      route_args(logits, idx.size(1), scoring, renormalize, scale);
  check_on(idx, logits, "topk_idx");
  check_on(grad_weights, logits, "grad_weights");
  check_on(out, logits, "out");
  TORCH_CHECK(idx.scalar_type() == at::kLong,
              "uccl_amd: topk_idx must be int64, got ", idx.scalar_type());
  TORCH_CHECK(grad_weights.scalar_type() == at::kFloat,
              "uccl_amd: grad_weights must be float32, got ",
              grad_weights.scalar_type());
  TORCH_CHECK(out.scalar_type() == logits.scalar_type(),
              "uccl_amd: out must have the dtype of logits");
  check_shape(idx, {a.tokens, a.topk}, "topk_idx");
  check_shape(grad_weights, {a.tokens, a.topk}, "grad_weights");
  check_shape(out, {a.tokens, a.experts}, "out");
  check_dense(idx, "topk_idx");
  check_dense(grad_weights, "grad_weights");
  check_dense(out, "out");
  check_result(out, "out", {logits, idx, grad_weights});
  check_gpu(logits, "logits");
  if (a.tokens == 0) return;
  c10::DeviceGuard guard(logits.device());
  ep::launch_route_grad(a, grad_weights.data_ptr<float>(),
                        idx.data_ptr<int64_t>(), out.data_ptr(),
                        stream_of(logits));
  check_launch("route_grad");
}

// --- products --------------------------------------------------------------

void expert_matmul(at::Tensor x, at::Tensor w, OptTensor counts,
                   OptTensor x_scales, OptTensor w_scales, at::Tensor out,
                   int64_t expected_rows, bool precise) {
  check_slots(x, "x");
  check_on(w, x, "w");
  check_on(out, x, "out");
  TORCH_CHECK(w.dim() == 3 && w.size(0) == x.size(0) &&
                  w.size(2) == x.size(2),
              "uccl_amd: w has shape ", w.sizes(), ", expected [", x.size(0),
              ", n, ", x.size(2), "]");
  TORCH_CHECK(w.scalar_type() == x.scalar_type(),
              "uccl_amd: x is ", x.scalar_type(), ", w is ", w.scalar_type());
  int64_t const experts = x.size(0), slots = x.size(1), k = x.size(2),
                n = w.size(1);
  TORCH_CHECK(n >= 1 && k >= 1, "uccl_amd: w has no rows or no columns");
  check_shape(out, {experts, slots, n}, "out");
  check_tiles(experts, n, slots);
  TORCH_CHECK(k < (int64_t(1) << 28), "uccl_amd: the product is too large");
  TORCH_CHECK(expected_rows >= 0, "uccl_amd: expected_rows is negative");

  ep::MatmulArgs a{};
  a.rows = rows_of(x, counts);
  a.n = static_cast<int>(n);
  a.k = static_cast<int>(k);
  a.elem = elem_of(x, "x");
  a.out_elem = elem_of(out, "out");
  TORCH_CHECK(a.elem != Elem::kF32, "uccl_amd: x has unsupported dtype ",
              x.scalar_type());
  TORCH_CHECK(a.out_elem != Elem::kF8, "uccl_amd: out has unsupported dtype ",
              out.scalar_type());
  std::vector<at::Tensor> operands{x, w};
  if (a.elem == Elem::kF8) {
    TORCH_CHECK(x_scales && w_scales,
                "uccl_amd: 8-bit operands need x_scales and w_scales");
    TORCH_CHECK(k % 128 == 0,
                "uccl_amd: 8-bit products need k % 128 == 0, got ", k);
    TORCH_CHECK(n == 1 || w.stride(1) < (int64_t(1) << 24),
                "uccl_amd: rows of 8-bit weights are less than 16 MiB apart");
    TORCH_CHECK(a.out_elem != Elem::kF32 || precise,
                "uccl_amd: 8-bit products give bfloat16 or float16: the 8-bit "
                "matrix unit does not keep the precision of float32 "
                "(precise=True does without it)");
    a.precise = precise;
    for (auto const& [t, name] : {std::pair(*x_scales, "x_scales"),
                                  std::pair(*w_scales, "w_scales")}) {
      check_on(t, x, name);
      TORCH_CHECK(t.scalar_type() == at::kFloat, "uccl_amd: ", name,
                  " must be float32, got ", t.scalar_type());
      operands.push_back(t);
    }
    check_shape(*x_scales, {experts, slots, k / 128}, "x_scales");
    check_shape(*w_scales, {experts, (n + 127) / 128, k / 128}, "w_scales");
    a.x_scales = mat_of(*x_scales, "x_scales", 4);
    a.w_scales = mat_of(*w_scales, "w_scales", 4);
  } else {
    TORCH_CHECK(!x_scales && !w_scales,
                "uccl_amd: scales belong to 8-bit operands");
    TORCH_CHECK(!precise, "uccl_amd: precise belongs to 8-bit operands; sums "
                "of 16-bit ones are held in 32 bits");
    TORCH_CHECK(k % 8 == 0,
                "uccl_amd: 16-bit products need k % 8 == 0, got ", k);
  }
  a.x = mat_of(x, "x");
  a.w_turned = w.stride(2) != 1 && w.stride(1) == 1;
  if (a.w_turned) {
    TORCH_CHECK(a.elem != Elem::kF8,
                "uccl_amd: 8-bit weights must be contiguous along k");
    TORCH_CHECK(n % 8 == 0,
                "uccl_amd: transposed weights need n % 8 == 0, got ", n);
    a.w = mat_of(w.transpose(1, 2), "w");
  } else {
    a.w = mat_of(w, "w");
  }
  a.out = mat_of(out, "out", out.element_size());
  check_result(out, "out", operands, counts);
  a.expected_rows =
      static_cast<int>(expected_rows ? std::min(expected_rows, slots) : slots);
  check_gpu(x, "x");
  if (slots == 0) return;
  c10::DeviceGuard guard(x.device());
  ep::launch_expert_matmul(a, stream_of(x));
  check_launch("expert_matmul");
}

void expert_weight_grad(at::Tensor grad, at::Tensor x, OptTensor counts,
                        at::Tensor out) {
  check_slots(grad, "grad_out");
  check_slots(x, "x");
  check_on(x, grad, "x");
  check_on(out, grad, "out");
  check_16bit(x, "x");
  TORCH_CHECK(grad.scalar_type() == x.scalar_type(), "uccl_amd: grad_out is ",
              grad.scalar_type(), ", x is ", x.scalar_type());
  int64_t const experts = x.size(0), n = grad.size(2), k = x.size(2);
  TORCH_CHECK(grad.size(0) == experts && grad.size(1) == x.size(1),
              "uccl_amd: grad_out has shape ", grad.sizes(), ", x ",
              x.sizes());
  TORCH_CHECK(n >= 8 && k >= 8 && n % 8 == 0 && k % 8 == 0,
              "uccl_amd: the weight gradient needs n and k to be multiples of "
              "8, got ", n, " and ", k);
  check_shape(out, {experts, n, k}, "out");
  check_tiles(experts, n, k);
  TORCH_CHECK(k < (int64_t(1) << 28), "uccl_amd: the product is too large");
  ep::WeightGradArgs a{};
  a.rows = rows_of(x, counts);
  a.grad = mat_of(grad, "grad_out");
  a.x = mat_of(x, "x");
  a.out = mat_of(out, "out", out.element_size());
  a.n = static_cast<int>(n);
  a.k = static_cast<int>(k);
  a.elem = elem_of(x, "x");
  a.out_elem = elem_of(out, "out");
  TORCH_CHECK(a.out_elem != Elem::kF8, "uccl_amd: out has unsupported dtype ",
              out.scalar_type());
  check_result(out, "out", {grad, x}, counts);
  check_gpu(x, "x");
  c10::DeviceGuard guard(x.device());
  ep::launch_expert_weight_grad(a, stream_of(x));
  check_launch("expert_weight_grad");
}

// --- activation ------------------------------------------------------------

void expert_swiglu(at::Tensor h, OptTensor counts, at::Tensor out,
                   OptTensor scales) {
  check_slots(h, "h");
  check_on(out, h, "out");
  check_16bit(h, "h");
  int64_t const cols = h.size(2) / 2;
  TORCH_CHECK(cols >= 8 && h.size(2) % 16 == 0,
              "uccl_amd: h has two halves of a multiple of 8 columns, got ",
              h.size(2));
  check_shape(out, {h.size(0), h.size(1), cols}, "out");
  ep::SwigluArgs a{};
  a.rows = rows_of(h, counts);
  a.h = mat_of(h, "h");
  a.cols = static_cast<int>(cols);
  TORCH_CHECK(h.size(2) < (int64_t(1) << 24), "uccl_amd: too many columns");
  a.elem = elem_of(h, "h");
  a.quantize = scales.has_value();
  std::vector<at::Tensor> operands{h};
  if (a.quantize) {
    TORCH_CHECK(out.scalar_type() == at::kFloat8_e4m3fn,
                "uccl_amd: out must be float8_e4m3fn, got ",
                out.scalar_type());
    TORCH_CHECK(cols % 128 == 0, "uccl_amd: 8-bit results need a multiple of "
                "128 columns, got ", cols);
    check_on(*scales, h, "out_scales");
    TORCH_CHECK(scales->scalar_type() == at::kFloat,
                "uccl_amd: out_scales must be float32, got ",
                scales->scalar_type());
    check_shape(*scales, {h.size(0), h.size(1), cols / 128}, "out_scales");
    a.scales = mat_of(*scales, "out_scales", 4);
    check_result(*scales, "out_scales", {h, out}, counts);
  } else {
    TORCH_CHECK(out.scalar_type() == h.scalar_type(),
                "uccl_amd: out must have the dtype of h, got ",
                out.scalar_type());
  }
  a.out = mat_of(out, "out");
  check_result(out, "out", operands, counts);
  check_gpu(h, "h");
  if (h.size(1) == 0) return;
  c10::DeviceGuard guard(h.device());
  ep::launch_expert_swiglu(a, stream_of(h));
  check_launch("expert_swiglu");
}

void expert_swiglu_grad(at::Tensor grad, at::Tensor h, OptTensor counts,
                        at::Tensor out) {
  check_slots(h, "h");
  check_on(grad, h, "grad_out");
  check_on(out, h, "out");
  check_16bit(h, "h");
  int64_t const cols = h.size(2) / 2;
  TORCH_CHECK(cols >= 8 && h.size(2) % 16 == 0,
              "uccl_amd: h has two halves of a multiple of 8 columns, got ",
              h.size(2));
  TORCH_CHECK(h.size(2) < (int64_t(1) << 24), "uccl_amd: too many columns");
  TORCH_CHECK(grad.scalar_type() == h.scalar_type() &&
                  out.scalar_type() == h.scalar_type(),
              "uccl_amd: grad_out and out must have the dtype of h");
  check_shape(grad, {h.size(0), h.size(1), cols}, "grad_out");
  check_shape(out, h.sizes().vec(), "out");
  ep::SwigluArgs a{};
  a.rows = rows_of(h, counts);
  a.h = mat_of(h, "h");
  a.grad_out = mat_of(grad, "grad_out");
  a.out = mat_of(out, "out");
  a.cols = static_cast<int>(cols);
  a.elem = elem_of(h, "h");
  check_result(out, "out", {h, grad}, counts);
  check_gpu(h, "h");
  if (h.size(1) == 0) return;
  c10::DeviceGuard guard(h.device());
  ep::launch_expert_swiglu_grad(a, stream_of(h));
  check_launch("expert_swiglu_grad");
}

}  // namespace

void register_expert_ops(py::module_& m) {
  m.def("ep_route", &route);
  m.def("ep_route_grad", &route_grad);
  m.def("ep_expert_matmul", &expert_matmul);
  m.def("ep_expert_weight_grad", &expert_weight_grad);
  m.def("ep_expert_swiglu", &expert_swiglu);
  m.def("ep_expert_swiglu_grad", &expert_swiglu_grad);
}

}  // namespace uccl
