// AdamW over many tensors, with the global gradient norm clipped:
//
//   g = grad * scale * min(1, max_norm / (|grad| * scale + 1e-6))
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// m and v are f32, or blocks of 256 e4m3 codes with one f32 scale each, of m
// and of r = sqrt(v). The codes of m are the nearest ones. Those of r are one
// of the two neighbours, drawn so that v is right in the mean: with b2 =
// 0.999 an average moves by 0.05 % a step where codes are 6 to 12 % apart,
// and rounding to the nearest would hold it where it is. The draw is a hash
// of the step and the element's place in its tensor. A root that is not zero
// is never rounded to zero, so that no update divides by eps alone.
//
// Sums and the arithmetic of an update are in the order of the formulas, each
// product and sum rounded (no contraction), and the norm is summed in 64 bits
// over fixed chunks: the same inputs give the same bits.
#include "common.h"
#include "kernels.h"

#pragma clang fp contract(off)

namespace zamd {

namespace {

constexpr int THREADS = 256;
constexpr int QBLOCK = 256;  // elements that share a scale
constexpr float E4M3_MAX = 448.f;
constexpr float TINY = 0x1p-100f;

template <typename G>
__global__ __launch_bounds__(THREADS) void adamw_norm_kernel(
    AdamwTensors a, AdamwScalars s, int first, AdamwWork w) {
  __shared__ double part[THREADS / 64];
  if (first + blockIdx.x == 0 && threadIdx.x == 0) {
    const int64_t t = *s.step + 1;
    *s.step = t;
    double p1 = 1, p2 = 1, x1 = s.beta1, x2 = s.beta2;
    for (int64_t k = t; k > 0; k >>= 1) {
      if (k & 1) { p1 *= x1; p2 *= x2; }
      x1 *= x1;
      x2 *= x2;
    }
    w.values->rate = (float)(s.lr / (1 - p1));
    w.values->root = (float)(1 / __builtin_sqrt(1 - p2));
    w.values->step = (unsigned)t;
  }
  if (!s.clip) return;
  int k = 0;
  while (k + 1 < a.count && a.norm_begin[k + 1] <= (int)blockIdx.x) ++k;
  const int64_t at =
      (int64_t)((int)blockIdx.x - a.norm_begin[k]) * ADAMW_NORM_CHUNK;
  const int n = (int)min((int64_t)ADAMW_NORM_CHUNK, a.t[k].n - at);
  const G* g = static_cast<const G*>(a.t[k].g) + at;
  double sum = 0;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const double x = (double)(float)g[i];
    sum += x * x;
  }
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_down(sum, off, 64);
  if (lane_id() == 0) part[wave_id()] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    w.partials[first + blockIdx.x] =
        (part[0] + part[1]) + (part[2] + part[3]);
}

// What the gradients are multiplied by: in every block the same sum, in the
// same order.
DEV_INLINE float clip_scale(const AdamwScalars& s, const AdamwWork& w,
                            bool tell) {
  __shared__ double part[THREADS / 64];
  if (!s.clip) return (float)s.grad_scale;
  double sum = 0;
  for (int i = threadIdx.x; i < w.count; i += THREADS) sum += w.partials[i];
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_down(sum, off, 64);
  if (lane_id() == 0) part[wave_id()] = sum;
  __syncthreads();
  sum = (part[0] + part[1]) + (part[2] + part[3]);
  const double norm = __builtin_sqrt(sum) * s.grad_scale;
  if (tell && threadIdx.x == 0) *w.norm = (float)norm;
  double coef = s.max_norm / (norm + 1e-6);
  if (coef > 1) coef = 1;  // a norm that is NaN stays one
  return (float)(coef * s.grad_scale);
}

DEV_INLINE float hash_uniform(unsigned index, unsigned step) {
  unsigned x = index * 0x9E3779B1u + step * 0x85EBCA77u;
  x = (x ^ (x >> 16)) * 0x7FEB352Du;
  x = (x ^ (x >> 15)) * 0x846CA68Bu;
  return (float)((x ^ (x >> 16)) >> 8) * 0x1p-24f;
}

DEV_INLINE float from_e4m3(unsigned code) {
  return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
}

DEV_INLINE unsigned to_e4m3(float x) {
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xff;
}

// One of the two codes beside x (0 <= x), so that x^2 is right in the mean.
DEV_INLINE unsigned draw_e4m3(float x, unsigned index, unsigned step) {
  x = x > E4M3_MAX ? E4M3_MAX : x;
  const unsigned low =
      x < 0x1p-6f ? (unsigned)(x * 512.f)
                  : (__builtin_bit_cast(unsigned, x) >> 20) - 960u;
  if (low == 0) return x > 0 ? 1 : 0;
  if (low >= 126) return 126;
  const float a = from_e4m3(low), b = from_e4m3(low + 1);
  const float aa = a * a;
  return hash_uniform(index, step) * (b * b - aa) < x * x - aa ? low + 1
                                                               : low;
}

// The largest magnitude of a wave; a NaN is the largest of all.
DEV_INLINE float wave_amax(float x) {
  unsigned u = __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const unsigned o = __shfl_xor(u, off, 64);
    u = u > o ? u : o;
  }
  return __builtin_bit_cast(float, u);
}

template <typename G, bool BITS8>
__global__ __launch_bounds__(THREADS) void adamw_update_kernel(
    AdamwTensors a, AdamwScalars s, bool tell, AdamwWork w) {
  const float coef = clip_scale(s, w, tell && blockIdx.x == 0);
  const float rate = w.values->rate, root = w.values->root;
  const unsigned step = w.values->step;
  int k = 0;
  while (k + 1 < a.count && a.begin[k + 1] <= (int)blockIdx.x) ++k;
  const AdamwTensor& x = a.t[k];
  const int64_t at = (int64_t)((int)blockIdx.x - a.begin[k]) * ADAMW_CHUNK;
  const int64_t end = min(at + (int64_t)ADAMW_CHUNK, x.n);
  const G* gp = static_cast<const G*>(x.g);
  for (int64_t q = at + wave_id() * QBLOCK; q < end;
       q += THREADS / 64 * QBLOCK) {
    float m[4], r[4];
    const int64_t i0 = q + lane_id() * 4;
    float ms = 0, vs = 0;
    if (BITS8) {
      ms = x.m_scale[q / QBLOCK];
      vs = x.v_scale[q / QBLOCK];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t i = i0 + e;
      m[e] = r[e] = 0;
      if (i >= end) continue;
      const float g = (float)gp[i] * coef;
      float m0, v0;
      if (BITS8) {
        m0 = from_e4m3(static_cast<uint8_t*>(x.m)[i]) * ms;
        const float r0 = from_e4m3(static_cast<uint8_t*>(x.v)[i]) * vs;
        v0 = r0 * r0;
      } else {
        m0 = static_cast<float*>(x.m)[i];
        v0 = static_cast<float*>(x.v)[i];
      }
      m[e] = m0 * s.b1 + g * s.c1;
      const float v = v0 * s.b2 + g * g * s.c2;
      r[e] = __builtin_sqrtf(v);
      const float p =
          x.p[i] * s.keep - rate * (m[e] / (r[e] * root + s.eps));
      x.p[i] = p;
      if (x.shadow) x.shadow[i] = (bf16)p;
      if (!BITS8) {
        static_cast<float*>(x.m)[i] = m[e];
        static_cast<float*>(x.v)[i] = v;
      }
    }
    if (BITS8) {
      float am = m[0], ar = r[0];
      {
        unsigned um = 0, ur = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          um = max(um, __builtin_bit_cast(unsigned, m[e]) & 0x7fffffffu);
          ur = max(ur, __builtin_bit_cast(unsigned, r[e]) & 0x7fffffffu);
        }
        am = wave_amax(__builtin_bit_cast(float, um));
        ar = wave_amax(__builtin_bit_cast(float, ur));
      }
      const float im = am < TINY ? 0.f : 1.f / am * E4M3_MAX;
      const float ir = ar < TINY ? 0.f : 1.f / ar * E4M3_MAX;
      if (lane_id() == 0) {
        x.m_scale[q / QBLOCK] = am < TINY ? 0.f : am * (1.f / E4M3_MAX);
        x.v_scale[q / QBLOCK] = ar < TINY ? 0.f : ar * (1.f / E4M3_MAX);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t i = i0 + e;
        if (i >= end) continue;
        static_cast<uint8_t*>(x.m)[i] = (uint8_t)to_e4m3(m[e] * im);
        static_cast<uint8_t*>(x.v)[i] =
            (uint8_t)draw_e4m3(r[e] * ir, (unsigned)i, step);
      }
    }
  }
}

}  // namespace

void launch_adamw_norm(const AdamwTensors& a, const AdamwScalars& s,
                       bool bf16_grads, int first, const AdamwWork& w,
                       hipStream_t stream) {
  const int blocks = s.clip ? a.norm_begin[a.count] : 1;
  if (bf16_grads)
    hipLaunchKernelGGL(adamw_norm_kernel<bf16>, dim3(blocks), dim3(THREADS),
                       0, stream, a, s, first, w);
  else
    hipLaunchKernelGGL(adamw_norm_kernel<float>, dim3(blocks), dim3(THREADS),
                       0, stream, a, s, first, w);
}

void launch_adamw_update(const AdamwTensors& a, const AdamwScalars& s,
                         bool bf16_grads, bool bits8, bool tell,
                         const AdamwWork& w, hipStream_t stream) {
  auto kernel = bf16_grads ? (bits8 ? adamw_update_kernel<bf16, true>
                                    : adamw_update_kernel<bf16, false>)
                           : (bits8 ? adamw_update_kernel<float, true>
                                    : adamw_update_kernel<float, false>);
  hipLaunchKernelGGL(kernel, dim3(a.begin[a.count]), dim3(THREADS), 0, stream,
                     a, s, tell, w);
}

}  // namespace zamd
