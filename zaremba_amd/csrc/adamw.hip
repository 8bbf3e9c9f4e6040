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
// Two launches: the sum of squares (the norm is of all gradients, so they are
// read twice), and the update, in which a wave of each block first adds up the
// partial sums while all of the block's loads are in flight. At 66.0M
// parameters with bf16 shadows they take 418 us in 32 bits (2.25 GB with the
// second reading, 5.4 TB/s, more than the 5.2 of a copy as a cache holds some of
// it), and 272 us in 8 bits (1.46 GB, 5.4 TB/s; some 62 vector instructions a
// value).
//
// Sums and the arithmetic of an update are in the order of the formulas, each
// product and sum rounded (no contraction), and the norm is summed in 64 bits
// over fixed chunks: the same inputs give the same bits.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"

#pragma clang fp contract(off)

namespace zamd {

namespace {

constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;
constexpr int QBLOCK = 256;  // elements that share a scale: 4 a lane
constexpr float E4M3_MAX = 448.f;
constexpr float TINY = 0x1p-100f;

// Four neighbours at any alignment of the element.
template <typename T>
struct Quad {
  T v[4];
};

template <typename T>
DEV_INLINE Quad<T> load4(const T* p) {
  Quad<T> x;
  __builtin_memcpy(&x, p, sizeof x);
  return x;
}

template <typename T>
DEV_INLINE void store4(T* p, const Quad<T>& x) {
  __builtin_memcpy(p, &x, sizeof x);
}

// Of the first `n` of them; the others read as zeros and are not written.
template <typename T>
DEV_INLINE Quad<T> load_some(const T* p, int n) {
  Quad<T> x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x.v[e] = e < n ? p[e] : T(0);
  return x;
}

template <typename T>
DEV_INLINE void store_some(T* p, const Quad<T>& x, int n) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) p[e] = x.v[e];
}

// The tensor that chunk `c` of a launch belongs to: a lane for each, so that
// it costs one round trip to the arguments.
DEV_INLINE int tensor_of(const int* begin, int count, int c) {
  static_assert(ADAMW_TENSORS <= 64);
  const int lane = lane_id();
  const int b = begin[lane < count ? lane : 0];
  return __popcll(__ballot(lane < count && b <= c)) - 1;
}

// How many of a tensor's n values chunk number `c` has. The comparison is in 32
// bits: of a minimum in 64 bits of values that a block shares the compiler
// has selected the wrong one (s_cselect after a v_cmp that leaves scc alone).
DEV_INLINE int chunk_length(int64_t n, int c, int chunk) {
  const int64_t left = n - (int64_t)c * chunk;  // at least 1
  const unsigned low = (unsigned)left;
  return (left >> 32) != 0 || low > (unsigned)chunk ? chunk : (int)low;
}

DEV_INLINE double block_sum(double x, double* lds) {
  for (int off = 32; off > 0; off >>= 1) x += __shfl_down(x, off, 64);
  if (lane_id() == 0) lds[wave_id()] = x;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <typename G>
__global__ __launch_bounds__(THREADS) void adamw_norm_kernel(
    AdamwTensors a, AdamwScalars s, int first, int blocks, AdamwWork w) {
  __shared__ double lds[WAVES];
  if ((int)blockIdx.x == blocks) {
    // one block more, in the first launch, for the step's own values
    if (threadIdx.x) return;
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
    return;
  }
  double sum = 0;
  for (int c = blockIdx.x; c < a.norm_begin[a.count]; c += blocks) {
    const int k = tensor_of(a.norm_begin, a.count, c);
    const int rel = c - a.norm_begin[k];
    const int n = chunk_length(a.t[k].n, rel, ADAMW_NORM_CHUNK);
    const G* g =
        static_cast<const G*>(a.t[k].g) + (int64_t)rel * ADAMW_NORM_CHUNK;
    // A chunk that ends early reads its last four again, and leaves them out.
    constexpr int R = ADAMW_NORM_CHUNK / THREADS / 4;
    const int quads = n / 4;
    if (quads > 0) {
      Quad<G> x[R];
#pragma unroll
      for (int r = 0; r < R; ++r)
        x[r] = load4(g + min(r * THREADS + (int)threadIdx.x, quads - 1) * 4);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool in = r * THREADS + (int)threadIdx.x < quads;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const double y = in ? (double)(float)x[r].v[e] : 0.;
          sum = __builtin_fma(y, y, sum);  // y * y is exact
        }
      }
    }
    if ((int)threadIdx.x < n % 4) {
      const double y = (double)(float)g[quads * 4 + threadIdx.x];
      sum = __builtin_fma(y, y, sum);
    }
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) w.partials[first + blockIdx.x] = sum;
}

// What the gradients are multiplied by: in every block the same sum, in the
// same order, by one wave, as the root and the quotient in 64 bits cost as
// much as some 100 values.
DEV_INLINE float clip_scale(const AdamwScalars& s, const AdamwWork& w,
                            bool tell) {
  __shared__ float scale;
  if (!s.clip) return (float)s.grad_scale;
  if (wave_id() == 0) {
    constexpr int R = 8;  // loads in flight
    double sum = 0;
    for (int i = lane_id(); i < w.count; i += 64 * R) {
      double x[R];
#pragma unroll
      for (int r = 0; r < R; ++r)
        x[r] = w.partials[min(i + 64 * r, w.count - 1)];
#pragma unroll
      for (int r = 0; r < R; ++r) sum += i + 64 * r < w.count ? x[r] : 0.;
    }
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    const double norm = __builtin_sqrt(sum) * s.grad_scale;
    if (tell && threadIdx.x == 0) *w.norm = (float)norm;
    double coef = s.max_norm / (norm + 1e-6);
    if (coef > 1) coef = 1;  // a norm that is NaN stays one
    scale = (float)(coef * s.grad_scale);
  }
  __syncthreads();
  return scale;
}

// A published 32-bit mixer (C. Wellons, "Prospecting for Hash Functions",
// 2018), fed with multiples of two primes (the first two of Y. Collet's 32-bit
// xxHash).
constexpr unsigned HASH_INDEX = 0x9E3779B1u, HASH_STEP = 0x85EBCA77u;

DEV_INLINE float hash_uniform(unsigned x) {
  x = (x ^ (x >> 16)) * 0x7FEB352Du;
  x = (x ^ (x >> 15)) * 0x846CA68Bu;
  return (float)((x ^ (x >> 16)) >> 8) * 0x1p-24f;
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

// sqrt(x) of x >= 0, rounded to the nearest: the hardware's root is within
// one unit, and a root s is the nearest where x lies between s times its two
// neighbours (Tuckerman's test). The library's own form scales x < 2^-96
// first; here such a root may be a unit off, beside one that is never under
// eps. As bits, 0 and infinity have neighbours that are NaN, or too small to
// change the test.
DEV_INLINE float sqrt_f(float x) {
  const float s = __builtin_amdgcn_sqrtf(x);
  const unsigned u = __builtin_bit_cast(unsigned, s);
  const float down = __builtin_bit_cast(float, u - 1);
  const float up = __builtin_bit_cast(float, u + 1);
  const float r = __builtin_fmaf(-down, s, x) <= 0.f ? down : s;
  return __builtin_fmaf(-up, s, x) > 0.f ? up : r;
}

// Of y's nearest code and one of its neighbours, those on either side of y:
// the one below, or, as a draw has it, the one above, so that y^2 is right in
// the mean. hashed: step * C2 + index * C1 of the element.
DEV_INLINE unsigned draw_e4m3(float y, unsigned nearest, float value,
                              unsigned hashed) {
  unsigned low = nearest - (value > y);
  const f32x2 ab =
      __builtin_amdgcn_cvt_pk_f32_fp8((int)(low * 257u + 256u), false);
  const float aa = ab.x * ab.x;
  // above 126 is a NaN, and no number less than one
  low += hash_uniform(hashed) * (ab.y * ab.y - aa) < y * y - aa;
  return low;
}

// The codes of four x >= 0. Less than the least code is drawn as the least
// code; 0 stays 0.
DEV_INLINE unsigned draw4_e4m3(const float (&x)[4], unsigned hashed) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    y[e] = __builtin_fminf(__builtin_fmaxf(x[e], 0x1p-9f), E4M3_MAX);
  int near = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  near = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], near, true);
  unsigned codes =
      draw_e4m3(y[0], near & 255, __builtin_amdgcn_cvt_f32_fp8(near, 0),
                hashed) |
      draw_e4m3(y[1], near >> 8 & 255, __builtin_amdgcn_cvt_f32_fp8(near, 1),
                hashed + HASH_INDEX) << 8 |
      draw_e4m3(y[2], near >> 16 & 255, __builtin_amdgcn_cvt_f32_fp8(near, 2),
                hashed + 2 * HASH_INDEX) << 16 |
      draw_e4m3(y[3], (unsigned)near >> 24,
                __builtin_amdgcn_cvt_f32_fp8(near, 3),
                hashed + 3 * HASH_INDEX) << 24;
  const float least =
      __builtin_fminf(__builtin_fminf(x[0], x[1]), __builtin_fminf(x[2], x[3]));
  if (!(least > 0.f))
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(x[e] > 0.f)) codes &= ~(255u << 8 * e);
  return codes;
}

// The largest of a wave, in every lane.
DEV_INLINE unsigned wave_max(unsigned u) {
#define ZAMD_MAX_DPP(ctrl)                                                  \
  {                                                                         \
    const unsigned o =                                                      \
        (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, ctrl, 0xf, 0xf,    \
                                              false);                       \
    u = u > o ? u : o;                                                      \
  }
  ZAMD_MAX_DPP(0x111)  // row_shr:1
  ZAMD_MAX_DPP(0x112)  // row_shr:2
  ZAMD_MAX_DPP(0x114)  // row_shr:4
  ZAMD_MAX_DPP(0x118)  // row_shr:8
  ZAMD_MAX_DPP(0x142)  // row_bcast:15
  ZAMD_MAX_DPP(0x143)  // row_bcast:31
#undef ZAMD_MAX_DPP
  return (unsigned)__builtin_amdgcn_readlane((int)u, 63);
}

DEV_INLINE float from_lane(float x, int lane) {
  return __builtin_bit_cast(
      float,
      __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}

// As bits a NaN is larger than any number.
DEV_INLINE unsigned magnitude(float x) {
  return __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
}

// Where a block's chunk of a tensor begins: uniform, so that a lane needs a
// 32-bit offset only.
template <typename G, typename S>
struct Chunk {
  float* p;
  const G* g;
  S* m;
  S* v;
  float* ms;
  float* vs;
  bf16* shadow;
  unsigned hashed;  // of the chunk's first element

  DEV_INLINE Chunk(const AdamwTensor& x, int64_t at)
      : p(x.p + at), g(static_cast<const G*>(x.g) + at),
        m(static_cast<S*>(x.m) + at), v(static_cast<S*>(x.v) + at),
        ms(x.m_scale + at / QBLOCK), vs(x.v_scale + at / QBLOCK),
        shadow(x.shadow ? x.shadow + at : nullptr),
        hashed((unsigned)at * HASH_INDEX) {}
};

// 256 elements of a chunk, 4 a lane.
template <typename G, bool BITS8>
struct Block {
  using S = typename std::conditional<BITS8, uint8_t, float>::type;
  Quad<float> p;
  Quad<G> g;
  Quad<S> m, v;
  float ms, vs;

  // q: the block's first element. n: those left from this lane's on; 4 or
  // more throughout where WHOLE.
  template <bool WHOLE>
  DEV_INLINE void load(const Chunk<G, S>& x, int q, int n) {
    const unsigned i = q + lane_id() * 4;
    if (WHOLE) {
      g = load4(x.g + i);
      p = load4(x.p + i);
      m = load4(x.m + i);
      v = load4(x.v + i);
    } else {
      g = load_some(x.g + i, n);
      p = load_some(x.p + i, n);
      m = load_some(x.m + i, n);
      v = load_some(x.v + i, n);
    }
    if (BITS8) {
      ms = x.ms[q / QBLOCK];
      vs = x.vs[q / QBLOCK];
    }
  }

  template <bool WHOLE>
  DEV_INLINE void update(const Chunk<G, S>& x, int q, int n,
                         const AdamwScalars& s, float coef, float rate,
                         float root) {
    const unsigned i = q + lane_id() * 4;
    Quad<float> m1, r1;
    Quad<bf16> sh;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float gr = (float)g.v[e] * coef;
      float m0, v0;
      if constexpr (BITS8) {
        const float r0 = unpack(v, e) * vs;
        m0 = unpack(m, e) * ms;
        v0 = r0 * r0;
      } else {
        m0 = m.v[e];
        v0 = v.v[e];
      }
      m1.v[e] = m0 * s.b1 + gr * s.c1;
      const float v1 = v0 * s.b2 + gr * gr * s.c2;
      // In 8 bits the arithmetic takes over half of the time: one reciprocal,
      // off by one unit of 2^-23, in place of a division's dozen of steps.
      r1.v[e] = BITS8 ? sqrt_f(v1) : __builtin_sqrtf(v1);
      const float d = r1.v[e] * root + s.eps;
      const float move = BITS8 ? m1.v[e] * __builtin_amdgcn_rcpf(d)
                               : m1.v[e] / d;
      p.v[e] = p.v[e] * s.keep - rate * move;
      sh.v[e] = (bf16)p.v[e];
      if constexpr (!BITS8) {
        m.v[e] = m1.v[e];
        v.v[e] = v1;
      }
    }
    if constexpr (BITS8) {
      unsigned um = 0, ur = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        um = max(um, magnitude(m1.v[e]));
        ur = max(ur, __builtin_bit_cast(unsigned, r1.v[e]));
      }
      // half the wave divides for m, half for r
      const unsigned am = wave_max(um), ar = wave_max(ur);
      const float most =
          __builtin_bit_cast(float, lane_id() < 32 ? am : ar);
      const bool empty = most < TINY;
      const float inv = empty ? 0.f : 1.f / most * E4M3_MAX;
      const float scale = empty ? 0.f : most * (1.f / E4M3_MAX);
      if ((lane_id() & 31) == 0)
        (lane_id() ? x.vs : x.ms)[q / QBLOCK] = scale;
      const float im = from_lane(inv, 0), ir = from_lane(inv, 32);
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(m1.v[0] * im, m1.v[1] * im, 0,
                                              false);
      c = __builtin_amdgcn_cvt_pk_fp8_f32(m1.v[2] * im, m1.v[3] * im, c,
                                          true);
      __builtin_memcpy(&m, &c, 4);
      const unsigned hashed = x.hashed + i * HASH_INDEX;
      const float x4[4] = {r1.v[0] * ir, r1.v[1] * ir, r1.v[2] * ir,
                           r1.v[3] * ir};
      const unsigned codes = draw4_e4m3(x4, hashed);
      __builtin_memcpy(&v, &codes, 4);
    }
    if (WHOLE) {
      store4(x.p + i, p);
      store4(x.m + i, m);
      store4(x.v + i, v);
      if (x.shadow) store4(x.shadow + i, sh);
    } else {
      store_some(x.p + i, p, n);
      store_some(x.m + i, m, n);
      store_some(x.v + i, v, n);
      if (x.shadow) store_some(x.shadow + i, sh, n);
    }
  }

  static DEV_INLINE float unpack(const Quad<uint8_t>& q, int e) {
    int c;
    __builtin_memcpy(&c, &q, 4);
    const f32x2 x = e < 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(c, false)
                          : __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
    return e & 1 ? x.y : x.x;
  }
};

template <typename G, bool BITS8>
__global__ __launch_bounds__(THREADS) void adamw_update_kernel(
    AdamwTensors a, AdamwScalars s, bool tell, AdamwWork w) {
  constexpr int STRIDE = WAVES * QBLOCK;
  constexpr int EACH = ADAMW_CHUNK / STRIDE;  // blocks of 256 of a wave
  // From the last chunk to the first: the gradients that the norm read last
  // are those that a cache may still hold.
  const int c = a.begin[a.count] - 1 - (int)blockIdx.x;
  const int k = tensor_of(a.begin, a.count, c);
  const int rel = c - a.begin[k];
  const int n = chunk_length(a.t[k].n, rel, ADAMW_CHUNK);
  Chunk<G, typename Block<G, BITS8>::S> x(a.t[k], (int64_t)rel * ADAMW_CHUNK);
  const int whole = n / QBLOCK * QBLOCK;
  const int wave = __builtin_amdgcn_readfirstlane(wave_id());

  Block<G, BITS8> b[EACH];
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    const int q = wave * QBLOCK + r * STRIDE;
    if (q < whole) b[r].template load<true>(x, q, 4);
  }
  const float coef = clip_scale(s, w, tell && blockIdx.x == 0);
  const float rate = w.values->rate, root = w.values->root;
  x.hashed += w.values->step * HASH_STEP;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    const int q = wave * QBLOCK + r * STRIDE;
    if (q < whole)
      b[r].template update<true>(x, q, 4, s, coef, rate, root);
  }
  // what is left of the tensor behind its last whole 256
  if (whole < n && wave == whole / QBLOCK % WAVES) {
    const int left = n - whole - lane_id() * 4;
    Block<G, BITS8> last;
    last.template load<false>(x, whole, left);
    last.template update<false>(x, whole, left, s, coef, rate, root);
  }
}

}  // namespace

// Every block of the update reads the partial sums of all of these: at 66M
// parameters in 8 bits 512 take 285 us, 1024 290 and 256 286.
int adamw_norm_blocks(const AdamwTensors& a, int launches) {
  return std::max(1, std::min(a.norm_begin[a.count], 512 / launches));
}

void launch_adamw_norm(const AdamwTensors& a, const AdamwScalars& s,
                       bool bf16_grads, int first, int blocks,
                       const AdamwWork& w, hipStream_t stream) {
  auto kernel =
      bf16_grads ? adamw_norm_kernel<bf16> : adamw_norm_kernel<float>;
  if (!s.clip) blocks = 0;
  hipLaunchKernelGGL(kernel, dim3(blocks + (first == 0)), dim3(THREADS), 0,
                     stream, a, s, first, blocks, w);
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
