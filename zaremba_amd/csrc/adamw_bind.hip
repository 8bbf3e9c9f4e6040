// Host entry point of the AdamW step (adamw.hip): argument checks and
// launches on the current stream of the parameters' device.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

#include "bind.h"
#include "kernels.h"

namespace zamd {

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using Tensors = std::vector<Tensor>;

void check_one(const Tensor& x, const Tensor& p, const char* name, size_t k,
               int64_t n) {
  TORCH_CHECK(x.device() == p.device(), "adamw_step_: ", name, "[", k,
              "] is on ", x.device(), " and params[0] on ", p.device());
  TORCH_CHECK(x.numel() == n, "adamw_step_: ", name, "[", k, "] has ",
              x.numel(), " values, expected ", n);
  TORCH_CHECK(x.is_contiguous(), "adamw_step_: ", name, "[", k,
              "] must be contiguous");
}

OptTensor adamw_step_(const Tensors& params, const Tensors& grads,
                   const Tensors& ms, const Tensors& vs, const Tensor& step,
                   double lr, double beta1, double beta2, double eps,
                   double weight_decay, c10::optional<double> max_norm,
                   double grad_scale, const c10::optional<Tensors>& m_scales,
                   const c10::optional<Tensors>& v_scales,
                   const c10::optional<std::vector<OptTensor>>& shadows) {
  const size_t count = params.size();
  TORCH_CHECK(count > 0, "adamw_step_: no parameters");
  TORCH_CHECK(grads.size() == count && ms.size() == count &&
              vs.size() == count && (!shadows || shadows->size() == count),
              "adamw_step_: the lists differ in length: ", count, " params, ",
              grads.size(), " grads, ", ms.size(), " exp_avgs, ", vs.size(),
              " exp_avg_sqs",
              shadows ? ", " + std::to_string(shadows->size()) + " shadows"
                      : std::string());
  const Tensor& first = params[0];
  TORCH_CHECK(first.is_cuda(), "adamw_step_: params must be on the GPU");
  c10::DeviceGuard guard(first.device());
  const auto state = ms[0].scalar_type();
  const bool bits8 = state == torch::kFloat8_e4m3fn;
  TORCH_CHECK(bits8 || state == torch::kFloat32,
              "adamw_step_: states must be float32 or float8_e4m3fn, got ",
              state);
  TORCH_CHECK(bits8 == (bool)m_scales && bits8 == (bool)v_scales,
              "adamw_step_: states in 8 bits need exp_avg_scales and "
              "exp_avg_sq_scales, states in 32 bits have none");
  if (bits8)
    TORCH_CHECK(m_scales->size() == count && v_scales->size() == count,
                "adamw_step_: ", count, " params, ", m_scales->size(),
                " exp_avg_scales and ", v_scales->size(),
                " exp_avg_sq_scales");
  const auto grad = grads[0].scalar_type();
  TORCH_CHECK(grad == torch::kFloat32 || grad == torch::kBFloat16,
              "adamw_step_: grads must be float32 or bfloat16, got ", grad);
  TORCH_CHECK(step.scalar_type() == torch::kInt64 && step.numel() == 1 &&
              step.device() == first.device(),
              "adamw_step_: step must be one int64 on the params' device");

  // what is written, as ranges of addresses
  std::vector<std::pair<const char*, const char*>> written;
  written.reserve(6 * count);
  std::vector<const Tensor*> to_bump;
  to_bump.reserve(6 * count + 1);
  auto writes = [&](const Tensor& x) {
    to_bump.push_back(&x);
    const char* at = static_cast<const char*>(x.data_ptr());
    if (x.numel()) written.emplace_back(at, at + x.nbytes());
  };
  writes(step);
  std::vector<AdamwTensor> all;
  all.reserve(count);
  for (size_t k = 0; k < count; ++k) {
    const Tensor& p = params[k];
    const int64_t n = p.numel();
    TORCH_CHECK(p.scalar_type() == torch::kFloat32,
                "adamw_step_: params must be float32, got ", p.scalar_type());
    TORCH_CHECK(grads[k].scalar_type() == grad &&
                ms[k].scalar_type() == state && vs[k].scalar_type() == state,
                "adamw_step_: all grads must be of one type, and all states, "
                "got others at ", k);
    check_one(p, first, "params", k, n);
    check_one(grads[k], first, "grads", k, n);
    check_one(ms[k], first, "exp_avgs", k, n);
    check_one(vs[k], first, "exp_avg_sqs", k, n);
    AdamwTensor t = {};
    if (bits8) {
      const int64_t blocks = (n + 255) / 256;
      for (const Tensors* l : {&*m_scales, &*v_scales}) {
        check_one((*l)[k], first, "scales", k, blocks);
        TORCH_CHECK((*l)[k].scalar_type() == torch::kFloat32,
                    "adamw_step_: scales must be float32, got ",
                    (*l)[k].scalar_type());
      }
      writes((*m_scales)[k]);
      writes((*v_scales)[k]);
      t.m_scale = (*m_scales)[k].data_ptr<float>();
      t.v_scale = (*v_scales)[k].data_ptr<float>();
    }
    if (shadows && (*shadows)[k]) {
      const Tensor& sh = *(*shadows)[k];
      check_one(sh, first, "shadows", k, n);
      TORCH_CHECK(sh.scalar_type() == torch::kBFloat16,
                  "adamw_step_: shadows must be bfloat16, got ",
                  sh.scalar_type());
      writes(sh);
      t.shadow = reinterpret_cast<bf16*>(sh.data_ptr());
    }
    if (n == 0) continue;
    t.p = p.data_ptr<float>();
    t.g = grads[k].data_ptr();
    t.m = ms[k].data_ptr();
    t.v = vs[k].data_ptr();
    t.n = n;
    writes(p);
    writes(ms[k]);
    writes(vs[k]);
    all.push_back(t);
  }
  std::sort(written.begin(), written.end());
  for (size_t k = 1; k < written.size(); ++k)
    TORCH_CHECK(written[k - 1].second <= written[k].first,
                "adamw_step_: parameters, states or shadows share memory");
  // other blocks read a gradient while these are written
  for (size_t k = 0; k < count; ++k) {
    const char* at = static_cast<const char*>(grads[k].data_ptr());
    const auto next = std::upper_bound(
        written.begin(), written.end(), at,
        [](const char* x, const auto& range) { return x < range.second; });
    TORCH_CHECK(next == written.end() ||
                next->first >= at + grads[k].nbytes(),
                "adamw_step_: grads[", k, "] shares memory with what the "
                "step writes");
  }

  int64_t total = 0;
  for (const auto& t : all) total += t.n;
  // a grid has fewer than 2^32 threads, 256 a block
  TORCH_CHECK(total / ADAMW_CHUNK + (int64_t)count < 1 << 24,
              "adamw_step_: too many values");
  AdamwScalars s = {};
  s.step = step.data_ptr<int64_t>();
  s.lr = lr;
  s.beta1 = beta1;
  s.beta2 = beta2;
  s.clip = max_norm.has_value();
  s.max_norm = max_norm.value_or(0);
  s.grad_scale = grad_scale;
  s.b1 = (float)beta1;
  s.c1 = (float)(1 - beta1);
  s.b2 = (float)beta2;
  s.c2 = (float)(1 - beta2);
  s.eps = (float)eps;
  s.keep = (float)(1 - lr * weight_decay);

  std::vector<AdamwTensors> launches;
  for (size_t k = 0; k < all.size(); k += ADAMW_TENSORS) {
    AdamwTensors a = {};
    a.count = (int)std::min<size_t>(ADAMW_TENSORS, all.size() - k);
    for (int i = 0; i < a.count; ++i) {
      a.t[i] = all[k + i];
      const int64_t n = a.t[i].n;
      a.begin[i + 1] = a.begin[i] + (int)((n + ADAMW_CHUNK - 1) / ADAMW_CHUNK);
      a.norm_begin[i + 1] =
          a.norm_begin[i] +
          (int)((n + ADAMW_NORM_CHUNK - 1) / ADAMW_NORM_CHUNK);
    }
    launches.push_back(a);
  }
  if (launches.empty()) launches.push_back(AdamwTensors{});  // step alone

  // One workspace a call: the caching allocator keeps those of captured
  // graphs apart.
  int partials = 0;
  for (const auto& a : launches)
    partials += adamw_norm_blocks(a, (int)launches.size());
  Tensor room = torch::empty({partials + 3}, first.options().dtype(
                                                 torch::kFloat64));
  Tensor norm;
  AdamwWork w;
  w.values = reinterpret_cast<AdamwValues*>(room.data_ptr<double>());
  w.partials = room.data_ptr<double>() + 2;
  w.count = s.clip ? partials : 0;
  w.norm = nullptr;
  if (s.clip) {
    norm = all.empty() ? torch::zeros({}, first.options())
                       : torch::empty({}, first.options());
    w.norm = norm.data_ptr<float>();
  }
  for (const Tensor* x : to_bump) x->unsafeGetTensorImpl()->bump_version();
  const auto stream = current_stream();
  int done = 0;
  for (const auto& a : launches) {
    if (done && !s.clip) break;
    const int blocks = adamw_norm_blocks(a, (int)launches.size());
    launch_adamw_norm(a, s, grad == torch::kBFloat16, done, blocks, w, stream);
    HIP_CHECK(hipGetLastError());
    done += blocks;
  }
  for (const auto& a : launches) {
    if (a.count == 0) continue;
    launch_adamw_update(a, s, grad == torch::kBFloat16, bits8,
                        &a == &launches[0], w, stream);
    HIP_CHECK(hipGetLastError());
  }
  return s.clip ? OptTensor(norm) : OptTensor();
}

}  // namespace

void bind_adamw(py::module_& m) {
  m.def("adamw_step_", &adamw_step_, py::arg("params"), py::arg("grads"),
        py::arg("exp_avgs"), py::arg("exp_avg_sqs"), py::arg("step"),
        py::arg("lr"), py::arg("beta1"), py::arg("beta2"), py::arg("eps"),
        py::arg("weight_decay"), py::arg("max_norm"), py::arg("grad_scale"),
        py::arg("exp_avg_scales"), py::arg("exp_avg_sq_scales"),
        py::arg("shadows"));
}

}  // namespace zamd
