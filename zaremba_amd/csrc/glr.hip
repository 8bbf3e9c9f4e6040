// Gated linear recurrence over [T, B, 4H] pre-activations, gate order
// (i, f, o, n) as in the LSTM cell, whose recurrent product it leaves out:
//
//   c_t = s(f_t) c_{t-1} + s(i_t) tanh(n_t)        s: the logistic function
//   h_t = s(o_t) tanh(c_t)
//
// With g_t = dL/dc_t and dh_t = dL/dh_t its backward pass is
//
//   g_t = dh_t s(o_t) (1 - tanh(c_t)^2) + s(f_{t+1}) g_{t+1}
//   di = g n i (1 - i)   df = g c_{t-1} f (1 - f)
//   do = dh tanh(c) o (1 - o)   dn = g i (1 - n^2)   dc0 = s(f_0) g_0
//
// From lengths[b] on, row b keeps its state, and its h and gate gradients
// are zero whatever stands there.
//
// One thread per channel walks the time axis. The forward pass keeps the
// state before every GLR_MARK-th step, and the backward pass walks those
// tiles from the last to the first and computes the states between again.
#include "common.h"
#include "kernels.h"

namespace zamd {

namespace {

DEV_INLINE float sigmoid_f(float x) {
  return __builtin_amdgcn_rcpf(1.f +
                               __builtin_amdgcn_exp2f(x * -1.44269504089f));
}

DEV_INLINE float tanh_f(float x) {
  const float e =
      __builtin_amdgcn_exp2f(__builtin_fabsf(x) * -2.88539008178f);
  return __builtin_copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
}

DEV_INLINE int row_length(const GlrArgs& a, int b) {
  if (!a.lengths) return a.T;
  const int64_t n =
      a.lengths_64 ? static_cast<const int64_t*>(a.lengths)[b]
                   : (int64_t)static_cast<const int*>(a.lengths)[b];
  return (int)(n < 0 ? 0 : n > a.T ? a.T : n);
}

template <typename E>
__global__ void glr_fwd_kernel(GlrArgs a) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (id >= (int64_t)a.B * a.H) return;
  const int b = (int)(id / a.H), j = (int)(id % a.H), H = a.H;
  const int n_live = row_length(a, b);
  const E* g = static_cast<const E*>(a.gates) + b * a.gates_b + j;
  E* h = static_cast<E*>(a.h) + b * a.h_b + j;
  float c = a.c0 ? a.c0[id] : 0.f;
  for (int t = 0; t < a.T; ++t, g += a.gates_t, h += a.h_t) {
    if (a.marks && t % GLR_MARK == 0)
      a.marks[(int64_t)(t / GLR_MARK) * a.B * a.H + id] = c;
    if (t < n_live) {
      c = sigmoid_f((float)g[H]) * c +
          sigmoid_f((float)g[0]) * tanh_f((float)g[3 * H]);
      *h = (E)(sigmoid_f((float)g[2 * H]) * tanh_f(c));
    } else {
      *h = (E)0.f;
    }
  }
  a.cT[id] = c;
}

template <typename E>
__global__ void glr_bwd_kernel(GlrArgs a) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (id >= (int64_t)a.B * a.H) return;
  const int b = (int)(id / a.H), j = (int)(id % a.H), H = a.H;
  const int n_live = row_length(a, b);
  const E* g0 = static_cast<const E*>(a.gates) + b * a.gates_b + j;
  const E* dh0 = static_cast<const E*>(a.dh) + b * a.dh_b + j;
  E* d0 = static_cast<E*>(a.dgates) + b * a.dgates_b + j;
  float carry = a.dcT ? a.dcT[id] : 0.f;
  float before[GLR_MARK];
  for (int tile = (a.T - 1) / GLR_MARK; tile >= 0; --tile) {
    float c = a.marks[(int64_t)tile * a.B * a.H + id];
    const int t0 = tile * GLR_MARK;
    const int n = min(GLR_MARK, a.T - t0);
    for (int k = 0; k < n; ++k) {
      const E* g = g0 + (t0 + k) * a.gates_t;
      before[k] = c;
      if (t0 + k < n_live)
        c = sigmoid_f((float)g[H]) * c +
            sigmoid_f((float)g[0]) * tanh_f((float)g[3 * H]);
    }
    for (int k = n - 1; k >= 0; --k) {
      const E* g = g0 + (t0 + k) * a.gates_t;
      E* d = d0 + (t0 + k) * a.dgates_t;
      if (t0 + k >= n_live) {
        d[0] = d[H] = d[2 * H] = d[3 * H] = (E)0.f;
        continue;
      }
      const float i = sigmoid_f((float)g[0]), f = sigmoid_f((float)g[H]);
      const float o = sigmoid_f((float)g[2 * H]), m = tanh_f((float)g[3 * H]);
      const float tc = tanh_f(f * before[k] + i * m);
      const float dh = (float)dh0[(t0 + k) * a.dh_t];
      const float dc = dh * o * (1.f - tc * tc) + carry;
      d[0] = (E)(dc * m * i * (1.f - i));
      d[H] = (E)(dc * before[k] * f * (1.f - f));
      d[2 * H] = (E)(dh * tc * o * (1.f - o));
      d[3 * H] = (E)(dc * i * (1.f - m * m));
      carry = f * dc;
    }
  }
  if (a.dc0) a.dc0[id] = carry;
}

template <typename E>
__global__ void glr_step_kernel(GlrArgs a) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (id >= (int64_t)a.B * a.H) return;
  const int b = (int)(id / a.H), j = (int)(id % a.H), H = a.H;
  const E* g = static_cast<const E*>(a.gates) + b * a.gates_b + j;
  float* cp = a.cT + b * a.c_b + j;
  const float c = sigmoid_f((float)g[H]) * *cp +
                  sigmoid_f((float)g[0]) * tanh_f((float)g[3 * H]);
  *cp = c;
  static_cast<E*>(a.h)[b * a.h_b + j] =
      (E)(sigmoid_f((float)g[2 * H]) * tanh_f(c));
}

template <typename F>
void by_type(GlrType type, F f) {
  switch (type) {
    case GlrType::F32: f(float{}); break;
    case GlrType::F16: f(_Float16{}); break;
    case GlrType::BF16: f(__bf16{}); break;
  }
}

}  // namespace

void launch_glr_fwd(const GlrArgs& a, GlrType type, hipStream_t stream) {
  const int grid = cdiv((int64_t)a.B * a.H, 64);
  by_type(type, [&](auto e) {
    hipLaunchKernelGGL(glr_fwd_kernel<decltype(e)>, dim3(grid), dim3(64), 0,
                       stream, a);
  });
}

void launch_glr_bwd(const GlrArgs& a, GlrType type, hipStream_t stream) {
  const int grid = cdiv((int64_t)a.B * a.H, 64);
  by_type(type, [&](auto e) {
    hipLaunchKernelGGL(glr_bwd_kernel<decltype(e)>, dim3(grid), dim3(64), 0,
                       stream, a);
  });
}

void launch_glr_step(const GlrArgs& a, GlrType type, hipStream_t stream) {
  const int grid = cdiv((int64_t)a.B * a.H, 256);
  by_type(type, [&](auto e) {
    hipLaunchKernelGGL(glr_step_kernel<decltype(e)>, dim3(grid), dim3(256), 0,
                       stream, a);
  });
}

}  // namespace zamd
