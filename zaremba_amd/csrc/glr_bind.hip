// Host entry points of the gated linear recurrence (glr.hip): argument
// checks, outputs and launches on the current stream of the gates' device.
#include <torch/extension.h>

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <limits>
#include <tuple>
#include <utility>

#include "bind.h"
#include "kernels.h"

namespace zamd {

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

GlrType glr_type(const Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return GlrType::F32;
    case torch::kFloat16: return GlrType::F16;
    case torch::kBFloat16: return GlrType::BF16;
    default:
      TORCH_CHECK(false, op, ": gates must be float32, float16 or bfloat16, "
                  "got ", t.scalar_type());
  }
}

// The kernels hand no tangent on.
void check_no_tangent(const Tensor& x, const char* op, const char* name) {
  TORCH_CHECK(!x._fw_grad(0).defined(), op, ": ", name, " has a tangent; "
              "there is no forward-mode derivative");
}

void check_gates(const Tensor& gates, int64_t dims, const char* op,
                 bool back = false) {
  TORCH_CHECK(gates.is_cuda(), op, ": gates must be on the GPU");
  TORCH_CHECK(gates.dim() == dims, op, ": gates must be ",
              dims == 3 ? "[T, B, 4H]" : "[B, 4H]", ", got ", gates.sizes());
  TORCH_CHECK(gates.size(-1) % 4 == 0, op,
              ": the last axis of gates holds the 4 gates, got ",
              gates.size(-1), " values");
  check_no_tangent(gates, op, "gates");
  const int64_t B = gates.size(-2), H = gates.size(-1) / 4;
  TORCH_CHECK(B * H < std::numeric_limits<int>::max() - 64 &&
              (dims == 2 ||
               (gates.size(0) < std::numeric_limits<int>::max() &&
                glr_threads(gates.size(0), B, H, back) < (int64_t)1 << 32)),
              op, ": sizes ", gates.sizes(), " are too large");
}

// A dense f32 [B, H] beside the gates.
Tensor state_like(const Tensor& c, const Tensor& gates, const char* op,
                  const char* name) {
  const int64_t B = gates.size(-2), H = gates.size(-1) / 4;
  TORCH_CHECK(c.scalar_type() == torch::kFloat32, op, ": ", name,
              " must be float32, got ", c.scalar_type());
  TORCH_CHECK(c.device() == gates.device(), op, ": ", name, " is on ",
              c.device(), " and gates on ", gates.device());
  TORCH_CHECK(c.dim() == 2 && c.size(0) == B && c.size(1) == H, op, ": ",
              name, " must be [", B, ", ", H, "], got ", c.sizes());
  check_no_tangent(c, op, name);
  return c.contiguous();
}

void set_lengths(GlrArgs& a, const OptTensor& lengths, Tensor& keep,
                 const Tensor& gates, const char* op) {
  if (!lengths) return;
  TORCH_CHECK(lengths->scalar_type() == torch::kInt32 ||
              lengths->scalar_type() == torch::kInt64,
              op, ": lengths must be int32 or int64, got ",
              lengths->scalar_type());
  TORCH_CHECK(lengths->device() == gates.device(), op, ": lengths is on ",
              lengths->device(), " and gates on ", gates.device());
  TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == gates.size(1), op,
              ": lengths must be [", gates.size(1), "], got ",
              lengths->sizes());
  keep = lengths->contiguous();
  a.lengths = keep.data_ptr();
  a.lengths_64 = keep.scalar_type() == torch::kInt64;
}

// Whether two tensors' ranges of addresses meet.
bool overlap(const Tensor& a, const Tensor& b) {
  auto range = [](const Tensor& t) {
    const char* at = static_cast<const char*>(t.data_ptr());
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d)
      last += (t.size(d) - 1) * t.stride(d);
    return std::make_pair(at, at + (last + 1) * t.element_size());
  };
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto x = range(a), y = range(b);
  return x.first < y.second && y.first < x.second;
}

// What is read while `out` is written.
void check_apart(const Tensor& out, const Tensor& x, const char* name,
                 const char* op) {
  TORCH_CHECK(!x.defined() || !overlap(out, x), op,
              ": out shares memory with ", name);
}

void check_out(const Tensor& out, const Tensor& gates, int64_t width,
               const char* op) {
  TORCH_CHECK(out.scalar_type() == gates.scalar_type() &&
              out.device() == gates.device() && out.dim() == 3 &&
              out.size(0) == gates.size(0) && out.size(1) == gates.size(1) &&
              out.size(2) == width && out.is_contiguous(),
              op, ": out must be a contiguous [", gates.size(0), ", ",
              gates.size(1), ", ", width, "] of the gates' type and device");
  TORCH_CHECK(!at::GradMode::is_enabled() || !out.requires_grad(), op,
              ": out requires a gradient, which this call does not record");
  check_apart(out, gates, "gates", op);
}

Tensor dense_rows(const Tensor& t) {
  return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous();
}

// [T, B, width], stored batch first where `like` is.
Tensor empty_as(const Tensor& like, int64_t width) {
  const int64_t T = like.size(0), B = like.size(1);
  if (T > 1 && B > 1 && like.stride(1) > like.stride(0))
    return torch::empty({B, T, width}, like.options()).transpose(0, 1);
  return torch::empty({T, B, width}, like.options());
}

void set_sizes(GlrArgs& a, const Tensor& gates) {
  a.T = (int)gates.size(0);
  a.B = (int)gates.size(1);
  a.H = (int)(gates.size(2) / 4);
  a.gates = gates.data_ptr();
  a.gates_t = gates.stride(0);
  a.gates_b = gates.stride(1);
}

int g_polls = GLR_POLLS;

// For tests: how often a block looks for a state before it gives up.
void set_glr_polls(int n) {
  TORCH_CHECK(n >= 0, "set_glr_polls: must not be negative, got ", n);
  g_polls = n;
}

void set_waits(GlrArgs& a, const OptTensor& gave_up, const Tensor& gates,
               const char* op) {
  a.polls = g_polls;
  if (!gave_up) return;
  TORCH_CHECK(gave_up->scalar_type() == torch::kInt32 &&
              gave_up->numel() == 1 && gave_up->device() == gates.device(),
              op, ": gave_up must be one int32 on the gates' device");
  a.gave_up = reinterpret_cast<unsigned*>(gave_up->data_ptr<int>());
}

int64_t mark_count(int64_t T) { return (T + GLR_MARK - 1) / GLR_MARK; }

// A workspace of this call alone: the caching allocator keeps those of other
// streams and of captured graphs apart.
Tensor workspace(GlrArgs& a, bool back, const Tensor& gates) {
  const int64_t words = glr_work_words(a, back, (int)gates.element_size());
  if (!words) return Tensor();
  Tensor work = torch::empty({words}, gates.options().dtype(torch::kInt64));
  a.work = reinterpret_cast<uint64_t*>(work.data_ptr<int64_t>());
  return work;
}

std::tuple<Tensor, Tensor, OptTensor> glr_forward(
    const Tensor& gates_in, const OptTensor& c0_in, const OptTensor& lengths,
    bool training, const OptTensor& out, const OptTensor& gave_up) {
  const char* op = "glr_forward";
  check_gates(gates_in, 3, op);
  const GlrType type = glr_type(gates_in, op);
  c10::DeviceGuard guard(gates_in.device());
  const Tensor gates = dense_rows(gates_in);
  GlrArgs a;
  set_sizes(a, gates);
  set_waits(a, gave_up, gates, op);
  Tensor keep, c0;
  set_lengths(a, lengths, keep, gates, op);
  if (c0_in) {
    c0 = state_like(*c0_in, gates, op, "c0");
    a.c0 = c0.data_ptr<float>();
  }
  Tensor h;
  if (out) {
    h = *out;
    check_out(h, gates, a.H, op);
    check_apart(h, c0, "c0", op);
    check_apart(h, keep, "lengths", op);
    h.unsafeGetTensorImpl()->bump_version();
  } else {
    h = empty_as(gates, a.H);
  }
  const auto f32 = gates.options().dtype(torch::kFloat32);
  Tensor cT = torch::empty({a.B, a.H}, f32);
  OptTensor marks;
  if (training) marks = torch::empty({mark_count(a.T), a.B, a.H}, f32);
  if (a.T == 0) {
    if (a.c0) cT.copy_(c0); else cT.zero_();
    return {h, cT, marks};
  }
  if (cT.numel() == 0) return {h, cT, marks};
  a.h = h.data_ptr();
  a.h_t = h.stride(0);
  a.h_b = h.stride(1);
  a.cT = cT.data_ptr<float>();
  if (marks) a.marks = marks->data_ptr<float>();
  Tensor work = workspace(a, false, gates);
  launch_glr_fwd(a, type, current_stream());
  HIP_CHECK(hipGetLastError());
  return {h, cT, marks};
}

std::tuple<Tensor, Tensor> glr_backward(
    const OptTensor& dh_in, const OptTensor& dcT_in, const Tensor& gates_in,
    const OptTensor& c0_in, const Tensor& marks, const OptTensor& lengths,
    const OptTensor& out, const OptTensor& gave_up) {
  const char* op = "glr_backward";
  check_gates(gates_in, 3, op, true);
  const GlrType type = glr_type(gates_in, op);
  c10::DeviceGuard guard(gates_in.device());
  const Tensor gates = dense_rows(gates_in);
  GlrArgs a;
  set_sizes(a, gates);
  set_waits(a, gave_up, gates, op);
  Tensor keep, c0, dcT, dh;
  set_lengths(a, lengths, keep, gates, op);
  if (c0_in) {
    c0 = state_like(*c0_in, gates, op, "c0");
    a.c0 = c0.data_ptr<float>();
  }
  if (dcT_in) {
    dcT = state_like(*dcT_in, gates, op, "dcT");
    a.dcT = dcT.data_ptr<float>();
  }
  TORCH_CHECK(marks.scalar_type() == torch::kFloat32 &&
              marks.device() == gates.device() && marks.is_contiguous() &&
              marks.dim() == 3 && marks.size(0) == mark_count(a.T) &&
              marks.size(1) == a.B && marks.size(2) == a.H,
              op, ": marks must be what glr_forward(training=True) returned "
              "for these gates");
  if (dh_in) {
    TORCH_CHECK(dh_in->scalar_type() == gates.scalar_type(), op,
                ": dh must be of the gates' type ", gates.scalar_type(),
                ", got ", dh_in->scalar_type());
    TORCH_CHECK(dh_in->device() == gates.device(), op, ": dh is on ",
                dh_in->device(), " and gates on ", gates.device());
    TORCH_CHECK(dh_in->dim() == 3 && dh_in->size(0) == a.T &&
                dh_in->size(1) == a.B && dh_in->size(2) == a.H,
                op, ": dh must be [", a.T, ", ", a.B, ", ", a.H, "], got ",
                dh_in->sizes());
    check_no_tangent(*dh_in, op, "dh");
    dh = dense_rows(*dh_in);
  } else {
    dh = torch::zeros({1, 1, a.H}, gates.options()).expand({a.T, a.B, a.H});
  }
  Tensor dgates;
  if (out) {
    dgates = *out;
    check_out(dgates, gates, 4 * (int64_t)a.H, op);
    check_apart(dgates, dh, "dh", op);
    check_apart(dgates, dcT, "dcT", op);
    check_apart(dgates, marks, "marks", op);
    check_apart(dgates, keep, "lengths", op);
    dgates.unsafeGetTensorImpl()->bump_version();
  } else {
    dgates = empty_as(gates, 4 * (int64_t)a.H);
  }
  Tensor dc0 = torch::empty({a.B, a.H},
                            gates.options().dtype(torch::kFloat32));
  if (a.T == 0) {
    if (a.dcT) dc0.copy_(dcT); else dc0.zero_();
    return {dgates, dc0};
  }
  if (dc0.numel() == 0) return {dgates, dc0};
  a.dh = dh.data_ptr();
  a.dh_t = dh.stride(0);
  a.dh_b = dh.stride(1);
  a.dgates = dgates.data_ptr();
  a.dgates_t = dgates.stride(0);
  a.dgates_b = dgates.stride(1);
  a.marks = marks.data_ptr<float>();
  a.dc0 = dc0.data_ptr<float>();
  Tensor work = workspace(a, true, gates);
  launch_glr_bwd(a, type, current_stream());
  HIP_CHECK(hipGetLastError());
  return {dgates, dc0};
}

Tensor glr_step(const Tensor& gates_in, const Tensor& c) {
  const char* op = "glr_step";
  TORCH_CHECK(!at::GradMode::is_enabled() ||
              !(gates_in.requires_grad() || c.requires_grad()),
              op, ": has no backward pass; call it under torch.no_grad(), or "
              "use glr()");
  check_gates(gates_in, 2, op);
  const GlrType type = glr_type(gates_in, op);
  c10::DeviceGuard guard(gates_in.device());
  const Tensor gates = dense_rows(gates_in);
  GlrArgs a;
  a.T = 1;
  a.B = (int)gates.size(0);
  a.H = (int)(gates.size(1) / 4);
  TORCH_CHECK(c.scalar_type() == torch::kFloat32, op,
              ": c must be float32, got ", c.scalar_type());
  TORCH_CHECK(c.device() == gates.device(), op, ": c is on ", c.device(),
              " and gates on ", gates.device());
  TORCH_CHECK(c.dim() == 2 && c.size(0) == a.B && c.size(1) == a.H, op,
              ": c must be [", a.B, ", ", a.H, "], got ", c.sizes());
  TORCH_CHECK((a.H <= 1 || c.stride(1) == 1) &&
              (a.B <= 1 || c.stride(0) >= a.H),
              op, ": the rows of c must be dense and apart, got strides ",
              c.strides());
  check_no_tangent(c, op, "c");
  TORCH_CHECK(!overlap(c, gates), op, ": c shares memory with gates");
  Tensor h = torch::empty({a.B, a.H}, gates.options());
  if (h.numel() == 0) return h;
  c.unsafeGetTensorImpl()->bump_version();
  a.gates = gates.data_ptr();
  a.gates_b = gates.stride(0);
  a.h = h.data_ptr();
  a.h_b = a.H;
  a.cT = c.data_ptr<float>();
  a.c_b = c.stride(0);
  launch_glr_step(a, type, current_stream());
  HIP_CHECK(hipGetLastError());
  return h;
}

}  // namespace

void bind_glr(py::module_& m) {
  m.def("glr_forward", &glr_forward, py::arg("gates"), py::arg("c0"),
        py::arg("lengths"), py::arg("training"), py::arg("out"),
        py::arg("gave_up") = py::none());
  m.def("glr_backward", &glr_backward, py::arg("dh"), py::arg("dcT"),
        py::arg("gates"), py::arg("c0"), py::arg("marks"),
        py::arg("lengths"), py::arg("out"),
        py::arg("gave_up") = py::none());
  m.def("set_glr_polls", &set_glr_polls);
  m.def("glr_step", &glr_step, py::arg("gates"), py::arg("c"));
}

}  // namespace zamd
