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
// are zero whatever stands there: such a step is (x, y) = (1, 0) by selects.
//
// Steps compose: c -> A c + C with A = prod x and C the state that the steps
// reach from zero. A block takes 64 channels and a tile of W * K steps, wave w
// holding K of them in registers: each wave finds its (A, C), the waves
// exchange them through LDS, and each then runs its own steps from the state
// that the waves before it leave. Data is read once, 4 K loads of a wave are
// in flight together, and a step waits for no other but through one exchange
// (two in the backward pass). Longer windows are many such blocks (see below).
//
// A lane has one channel, so that rows may have any length and alignment. Two
// channels a lane, with loads twice as wide, measured 264 to 290 us against
// 260 forward and 521 to 576 against 545 backward at 65536 x 1 x 1500 bf16:
// the registers of twice the steps leave half the waves.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "common.h"
#include "kernels.h"

namespace zamd {

namespace {

constexpr float LOG2E = 1.44269504089f;

DEV_INLINE float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }
DEV_INLINE float rcp_f(float x) { return __builtin_amdgcn_rcpf(x); }

// exp and 1 / x are one instruction each, off by one unit of 2^-23. An
// infinite exp(-x) gives rcp(inf) = 0, and exp(-inf) = 0 gives 1: closed and
// open gates are exact.
DEV_INLINE float sigmoid_f(float x) { return rcp_f(1.f + exp2_f(x * -LOG2E)); }

// 1 - exp(-2|x|) cancels for small x: its error is 2^-24 of 1. A value under
// SMALL is therefore taken from the series x - x^3 / 3 + 2 x^5 / 15, whose next
// term is under 2^-22 of it, and tanh is off by at most 16 * 2^-24 of itself.
// Where gates and h have 16 bits x itself does, a third of whose square is
// under 2^-17, and the bound is 330 * 2^-24, a twelfth of half a step of f16:
// at 65536 x 1 x 1500 bf16 this costs 249 -> 254 us forward, the series 279.
template <typename E>
constexpr float SMALL = sizeof(E) == 4 ? 0.125f : 0x1p-8f;

template <typename E>
DEV_INLINE float small_tanh(float a) {  // of a >= 0
  if (sizeof(E) < 4) return a;
  const float s = a * a;
  return a * __builtin_fmaf(__builtin_fmaf(s, 2.f / 15.f, -1.f / 3.f), s, 1.f);
}

// From exp(-2|x|) <= 1, which cannot overflow.
template <typename E>
DEV_INLINE float tanh_f(float x) {
  const float a = __builtin_fabsf(x);
  const float e = exp2_f(a * (-2.f * LOG2E));
  const float t = (1.f - e) * rcp_f(1.f + e);
  return __builtin_copysignf(a < SMALL<E> ? small_tanh<E>(a) : t, x);
}

// s(x) tanh(y) with one reciprocal.
template <typename E>
DEV_INLINE float sigmoid_tanh(float x, float y) {
  const float a = __builtin_fabsf(y);
  const float e = exp2_f(a * (-2.f * LOG2E));
  const float d = 1.f + e;
  const float r = rcp_f(__builtin_fmaf(exp2_f(x * -LOG2E), d, d));
  const float top = a < SMALL<E> ? small_tanh<E>(a) * d : 1.f - e;
  return __builtin_copysignf(top * r, y);
}

// A uniform base and a lane's 32-bit byte offset.
template <typename E>
DEV_INLINE const E& at(const E* base, unsigned offset) {
  return *reinterpret_cast<const E*>(reinterpret_cast<const char*>(base) +
                                     offset);
}
template <typename E>
DEV_INLINE E& at(E* base, unsigned offset) {
  return *reinterpret_cast<E*>(reinterpret_cast<char*>(base) + offset);
}

// One of a block's 64 channels: the b-th row of the launch, its j-th channel.
struct Channel {
  int first;      // row of the block's first lane
  int row;        // this lane's row, less `first`
  int j;
  int n_live;     // steps of the row
  int most;       // steps of the block's longest row
  int64_t state;  // place in a [B, H]

  DEV_INLINE Channel(const GlrArgs& a, int group) {
    const int id0 = group * 64, id = id0 + lane_id();
    // a lane behind the last channel repeats the block's first, with its stores
    const int b0 = id0 / a.H, r = (id < a.rows * a.H ? id : id0) - b0 * a.H;
    first = a.row0 + b0;
    row = a.H >= 64 ? r >= a.H : r / a.H;
    j = r - row * a.H;
    state = (int64_t)(first + row) * a.H + j;
    n_live = most = a.T;
    if (a.lengths) {
      const int64_t n = a.lengths_64
                            ? static_cast<const int64_t*>(a.lengths)[first + row]
                            : static_cast<const int*>(a.lengths)[first + row];
      n_live = (int)(n < 0 ? 0 : n > a.T ? a.T : n);
      int m = n_live;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) m = max(m, __shfl_xor(m, d));
      most = __builtin_amdgcn_readfirstlane(m);
    }
  }

  // Rows of a block lie less than 4 GB apart (rows_per_launch sees to it).
  template <typename E>
  DEV_INLINE unsigned offset(int64_t row_stride) const {
    return (unsigned)((row * row_stride + j) * sizeof(E));
  }
};

template <typename E, int K>
struct Gates {
  E i[K], f[K], o[K], n[K];

  // Steps [t0, t0 + K); those past `last` read it instead.
  DEV_INLINE void load(const GlrArgs& a, const E* base, unsigned offset,
                       int t0, int last) {
    const E* p = base + (int64_t)min(t0, last) * a.gates_t;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      i[k] = at(p, offset);
      f[k] = at(p + a.H, offset);
      o[k] = at(p + 2 * (int64_t)a.H, offset);
      n[k] = at(p + 3 * (int64_t)a.H, offset);
      p += t0 + k < last ? a.gates_t : 0;
    }
  }

  // Makes the steps from `stop` on stand for (x, y) = (1, 0).
  DEV_INLINE void mask(int t0, int stop) {
    if (__all(t0 + K <= stop)) return;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool on = t0 + k < stop;
      i[k] = on ? i[k] : (E)-INFINITY;
      f[k] = on ? f[k] : (E)INFINITY;
      n[k] = on ? n[k] : (E)0.f;
    }
  }
};

// (A, C) of each wave of a block, for each channel.
struct alignas(8) Pair {
  float A, C;
};

// c through the pairs of the waves [from, to).
DEV_INLINE float compose(float c, const Pair (*pairs)[64], int from, int to) {
  for (int q = from; q < to; ++q) {
    const Pair p = pairs[q][lane_id()];
    c = p.A * c + p.C;
  }
  return c;
}

// A window of more than one tile is a block for each tile, all in flight at
// once, that hand the state on: a scan in one pass with decoupled look-back
// (D. Merrill and M. Garland, 2016). Slot r, the r-th tile in the order of the
// scan, has a word for each channel. It first publishes its (A, C) there and,
// once it knows the state before it, the state behind it instead, marked by
// A = -1. A wave looks back over the slots before its own, DEPTH of them at a
// time, keeps up to SEEN pairs until it meets a state, and then composes them
// from that state on: the same roundings in the same order whichever state it
// was, so that results do not depend on when a block runs. A word says by
// itself whether it is there (all ones: not yet; no word that is written is),
// so that no order between stores is needed, and words go past the L2s, which
// do not see each other's writes. Looking at 1 or 4 words at a time, or
// keeping 16, measured the same within 2 %; keeping 4 takes 5 % longer at
// 16384 x 1 x 1000.
//
// A tile behind the last step of each of its rows writes zeros and ends; the
// chain ends, or in the backward pass begins, with the tile before. Rows of
// random lengths, forward / backward in tiles of 8 waves: 133 / 243 us against
// 155 / 279 with such tiles in the chain at 512 x 80 x 1500, 28 / 55 against
// 35 / 59 at 1001 x 17 x 651. Their reads are half of all; an XCD whose rows
// are short then waits for the others, and dealing groups out in smaller pieces
// costs as much in lines that two XCDs read.
//
// Blocks take their slots from counters as they start. A block therefore
// waits only for blocks that run already, and these only for earlier ones:
// every wait ends, whatever the number of blocks that fit the chip. Polls are
// bounded all the same; behind a bound that is reached the state is NaN, and
// a flag says so.
//
// From SHARED_FROM groups of 64 channels on each of the 8 XCDs has a counter
// and a share of the groups, neighbours side by side: rows of 64 values are
// seldom whole cache lines, and the other halves are then met in the same L2.
// (Blocks go round the XCDs in turn; no result depends on it.) Windows of one
// tile have the same shares: in us, against groups in the blocks' order, 35 x
// 20 x 1500 bf16 6.6 / 7.3 against 6.6 / 9.3 forward / backward, 100 x 20 x
// 1500 9.3 / 17.4 against 12.0 / 21.5, 35 x 128 x 1500 17 / 33 against 22 / 45,
// rows of whole lines (64 x 64 x 1024) the same. In a chain with fewer groups
// each has a counter of its own, as the blocks of one would queue at one
// address (14 ns a slot) and an XCD would have 3 groups or less.
// Measured in us, forward / backward in tiles of 8 waves, bf16, H = 1500: with
// a counter a group against shares, 23.4 groups x 65536 steps 250 / 537 against
// 276 / 578 (one counter for all: 260 / 545), 15.6 x 16384 (H = 1000) 53 / 90
// against 52 / 99, but 94 x 4096 69 / 141 against 65 / 120 and 375 x 1024 70 /
// 146 against 62 / 113.
//
// At T = 65536, B = 1, H = 1500, bf16 this takes 255 us forward (983 MB, 3.9
// TB/s of the 5.2 that a copy reaches) and 518 backward (1770 MB, 3.4 TB/s);
// with rows of whole lines, H = 1472, 209 (4.6 TB/s) and 353 (4.9). At H = 1500
// two XCDs read the same lines, 1.4 and 1.75 times the bytes to be read. That
// is not what bounds the backward pass: shares for XCDs take a quarter of its
// read bytes away and no time. What does is not known. Vector instructions
// take half of either. Before, finding the (A, C) of long chunks
// in a launch of its own, which reads three gates twice, took 360 and 680, and
// a block that loops over its tiles 2380 and 4500.
constexpr unsigned ABSENT = 0xffffffffu;
constexpr int XCDS = 8;
constexpr int SHARED_FROM = 32;    // groups: a counter for each XCD
constexpr int COUNTER_APART = 16;  // words: 128 bytes
constexpr int COUNTER_WORDS = COUNTER_APART * SHARED_FROM;  // go first
constexpr int DEPTH = 2, SEEN = 8;

DEV_INLINE unsigned to_bits(float x) {  // any NaN but ABSENT
  return x == x ? __builtin_bit_cast(unsigned, x) : 0x7fc00000u;
}

// A block's place in the time order, and its 64 channels.
struct Slot {
  int order, group;
};

// The groups of XCD x.
struct Share {
  int first, count;

  DEV_INLINE Share(const GlrArgs& a, int x)
      : first(a.groups * x / XCDS),
        count(a.groups * (x + 1) / XCDS - first) {}
};

// Of a window of one tile. The grid fits the largest share.
DEV_INLINE Slot one_tile(const GlrArgs& a) {
  const Share s(a, blockIdx.x % XCDS);
  const int k = blockIdx.x / XCDS;
  return {k < s.count ? 0 : 1, s.first + k};
}

struct Chain {
  uint64_t* words;  // [chunks, B * H]: A above C
  int64_t BH;
  int most_polls;
  unsigned* gave_up;

  DEV_INLINE Chain(const GlrArgs& a)
      : words(a.work + COUNTER_WORDS), BH((int64_t)a.B * a.H),
        most_polls(a.polls), gave_up(a.gave_up) {}

  // A counter deals out the slots of its groups in order. It gets at least as
  // many blocks as slots: order a.chunks is none.
  static DEV_INLINE Slot take_slot(const GlrArgs& a, int* lds) {
    const bool shared = a.groups >= SHARED_FROM;
    const int x = shared ? blockIdx.x % XCDS : blockIdx.x / XCDS % a.groups;
    if (threadIdx.x == 0)
      *lds = (int)__hip_atomic_fetch_add(
          reinterpret_cast<unsigned*>(a.work + x * COUNTER_APART), 1u,
          __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const Share share(a, shared ? x : 0);
    __syncthreads();
    const int k = __builtin_amdgcn_readfirstlane(*lds);
    if (!shared) return {min(k, a.chunks), x};
    return {min(k / share.count, a.chunks), share.first + k % share.count};
  }

  DEV_INLINE void publish(int slot, const Channel& ch, float A,
                          float C) const {
    __hip_atomic_store(words + slot * BH + ch.state,
                       (uint64_t)to_bits(A) << 32 | to_bits(C),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }

  // The state before `slot`, found by one wave.
  DEV_INLINE float look_back(int slot, const Channel& ch, float start,
                             Pair (*seen)[64]) const {
    const uint64_t* own = words + (int64_t)slot * BH + ch.state;
    float c = start;
    int n = 0;  // slots before this one whose words are kept in `seen`
    for (int polls = 0; n < slot;) {
      if (polls == most_polls) {
        c = __builtin_nanf("");
        if (gave_up && lane_id() == 0)
          __hip_atomic_store(gave_up, 1u, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
        break;
      }
      uint64_t p[DEPTH];
#pragma unroll
      for (int q = 0; q < DEPTH; ++q)
        p[q] = __hip_atomic_load(own - min(n + 1 + q, slot) * BH,
                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      bool met = false, more = true;
#pragma unroll
      for (int q = 0; q < DEPTH; ++q) {
        const unsigned bits = (unsigned)(p[q] >> 32);
        const Pair r = {__builtin_bit_cast(float, bits),
                        __builtin_bit_cast(float, (unsigned)p[q])};
        if (!more || n == slot) continue;
        if (__all(r.A < 0.f)) {
          c = r.C;
          met = true;
          more = false;
        } else if (n < SEEN && __all(bits != ABSENT)) {
          seen[n++][lane_id()] = r;
        } else {
          more = false;
        }
      }
      if (met) break;
      if (!more) {
        ++polls;
        __builtin_amdgcn_s_sleep(1);
      }
    }
    while (n > 0) {
      const Pair r = seen[--n][lane_id()];
      c = r.A < 0.f ? r.C : __builtin_fmaf(r.A, c, r.C);
    }
    return c;
  }

  // The state before `slot`, to all waves; the one behind it through `last`.
  DEV_INLINE float hand_on(int slot, const Channel& ch, float A, float C,
                           const float* start, float* lds, Pair (*seen)[64],
                           float* last, int w) const {
    if (w == 0) {
      publish(slot, ch, A, C);
      const float c = look_back(slot, ch, start ? start[ch.state] : 0.f, seen);
      lds[lane_id()] = c;
      const float behind = __builtin_fmaf(A, c, C);  // as look_back has it
      publish(slot, ch, -1.f, behind);
      if (last) last[ch.state] = behind;
    }
    __syncthreads();
    return lds[lane_id()];
  }
};

// Nothing is there yet, and no slot taken.
__global__ void glr_reset_kernel(uint4* work, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n)
    work[i] = i < COUNTER_WORDS / 2 ? uint4{0, 0, 0, 0}
                                    : uint4{ABSENT, ABSENT, ABSENT, ABSENT};
}

// W: waves of a block, in a chain; at most, where one tile is the window.
template <typename E, int K, int W, bool CHAIN>
__global__ __launch_bounds__(64 * W) void glr_fwd_kernel(GlrArgs a) {
  static_assert(GLR_MARK % K == 0);  // a mark is the start of a wave's steps
  __shared__ Pair lds[W][64];
  __shared__ float handed[64];
  __shared__ int taken;
  __shared__ Pair seen[CHAIN ? SEEN : 1][64];
  const int waves = CHAIN ? W : blockDim.x / 64, lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(wave_id());
  const Slot slot =
      CHAIN ? Chain::take_slot(a, &taken) : one_tile(a);
  if (slot.order >= (CHAIN ? a.chunks : 1)) return;
  const Channel ch(a, slot.group);
  const E* g0 = static_cast<const E*>(a.gates) + ch.first * a.gates_b;
  E* h0 = static_cast<E*>(a.h) + ch.first * a.h_b;
  const unsigned h_off = ch.offset<E>(a.h_b);
  const int t0 = (slot.order * waves + w) * K;
  const int tiles = max(1, cdiv_const(ch.most, W * K));
  if (CHAIN && slot.order >= tiles) {
    E* h = h0 + (int64_t)t0 * a.h_t;
    for (int t = t0; t < min(t0 + K, a.T); ++t, h += a.h_t)
      at(h, h_off) = (E)0.f;
    if (a.marks && t0 % GLR_MARK == 0 && t0 < a.T)
      a.marks[(int64_t)(t0 / GLR_MARK) * a.B * a.H + ch.state] = 0.f;
    return;
  }

  Gates<E, K> g;
  g.load(a, g0, ch.offset<E>(a.gates_b), t0, max(ch.most, 1) - 1);
  g.mask(t0, ch.n_live);
  float x[K], y[K], A = 1.f, C = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    x[k] = sigmoid_f((float)g.f[k]);
    y[k] = sigmoid_tanh<E>((float)g.i[k], (float)g.n[k]);
    C = x[k] * C + y[k];
    A *= x[k];
  }
  lds[w][lane] = {A, C};
  __syncthreads();
  float c;
  if (CHAIN) {
    if (w == 0)
#pragma unroll
      for (int q = 1; q < W; ++q) {
        const Pair p = lds[q][lane];
        C = p.A * C + p.C;
        A *= p.A;
      }
    c = Chain(a).hand_on(slot.order, ch, A, C, a.c0, handed, seen,
                         slot.order == tiles - 1 ? a.cT : nullptr, w);
  } else {
    c = a.c0 ? a.c0[ch.state] : 0.f;
  }
  c = compose(c, lds, 0, w);
  if (a.marks && t0 % GLR_MARK == 0 && t0 < a.T)
    a.marks[(int64_t)(t0 / GLR_MARK) * a.B * a.H + ch.state] = c;
  E* to = h0 + (int64_t)t0 * a.h_t;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int t = t0 + k;
    c = x[k] * c + y[k];
    const float h = sigmoid_tanh<E>((float)g.o[k], c);
    if (t < a.T) at(to, h_off) = t < ch.n_live ? (E)h : (E)0.f;
    to += a.h_t;
  }
  // steps past T keep the state
  if (!CHAIN && w == waves - 1) a.cT[ch.state] = c;
}

// Tiles begin at marks; in a chain the first slot has the last of them.
template <typename E, int K, int W, bool CHAIN>
__global__ __launch_bounds__(64 * W) void glr_bwd_kernel(GlrArgs a) {
  static_assert(K * W % GLR_MARK == 0);
  __shared__ Pair lds[W][64];   // (A, C) of the states
  __shared__ Pair back[W][64];  // (A, D) of their gradients, last wave first
  __shared__ float handed[64];
  __shared__ int taken;
  __shared__ Pair seen[CHAIN ? SEEN : 1][64];
  const int waves = CHAIN ? W : blockDim.x / 64, lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(wave_id());
  const int rw = waves - 1 - w;
  const Slot slot =
      CHAIN ? Chain::take_slot(a, &taken) : one_tile(a);
  if (slot.order >= (CHAIN ? a.chunks : 1)) return;
  const Channel ch(a, slot.group);
  const E* g0 = static_cast<const E*>(a.gates) + ch.first * a.gates_b;
  const E* dh0 = static_cast<const E*>(a.dh) + ch.first * a.dh_b;
  const unsigned dh_off = ch.offset<E>(a.dh_b);
  E* d0 = static_cast<E*>(a.dgates) + ch.first * a.dgates_b;
  const unsigned d_off = ch.offset<E>(a.dgates_b);
  const int tile = CHAIN ? a.chunks - 1 - slot.order : 0;
  const int begin = tile * W * K;
  const int t0 = begin + w * K, stop = ch.n_live;
  const int tiles = max(1, cdiv_const(ch.most, W * K));
  if (CHAIN && tile >= tiles) {
    E* d = d0 + (int64_t)t0 * a.dgates_t;
    for (int t = t0; t < min(t0 + K, a.T); ++t, d += a.dgates_t)
#pragma unroll
      for (int q = 0; q < 4; ++q) at(d + q * (int64_t)a.H, d_off) = (E)0.f;
    return;
  }

  const int last = max(ch.most, 1) - 1;
  Gates<E, K> g;
  g.load(a, g0, ch.offset<E>(a.gates_b), t0, last);
  E dh[K];
  const E* from = dh0 + (int64_t)min(t0, last) * a.dh_t;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    dh[k] = at(from, dh_off);
    from += t0 + k < last ? a.dh_t : 0;
  }
  float c = a.marks[(int64_t)(begin / GLR_MARK) * a.B * a.H + ch.state];
  g.mask(t0, stop);
  if (!__all(t0 + K <= stop)) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      g.o[k] = t0 + k < stop ? g.o[k] : (E)0.f;
      dh[k] = t0 + k < stop ? dh[k] : (E)0.f;
    }
  }
  float i[K], f[K], n[K], A = 1.f, C = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    i[k] = sigmoid_f((float)g.i[k]);
    f[k] = sigmoid_f((float)g.f[k]);
    n[k] = tanh_f<E>((float)g.n[k]);
    C = f[k] * C + i[k] * n[k];
    A *= f[k];
  }
  lds[w][lane] = {A, C};
  __syncthreads();
  c = compose(c, lds, 0, w);
  // Forward again through the own steps; u is what a step adds to g, and D
  // what the steps hand back from a gradient of zero behind them. The output
  // gate's gradient needs no more and is written at once.
  float before[K], u[K], D = 0.f;
  E* d = d0 + (int64_t)t0 * a.dgates_t;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int t = t0 + k;
    before[k] = c;
    c = f[k] * c + i[k] * n[k];
    const float tc = tanh_f<E>(c);
    const float o = sigmoid_f((float)g.o[k]);
    const float od = o * (float)dh[k];
    u[k] = od * (1.f - tc * tc);
    if (t < a.T)
      at(d + 2 * (int64_t)a.H, d_off) =
          t < stop ? (E)(od * tc * (1.f - o)) : (E)0.f;
    d += a.dgates_t;
  }
#pragma unroll
  for (int k = K - 1; k >= 0; --k) D = f[k] * (D + u[k]);
  back[rw][lane] = {A, D};
  __syncthreads();
  float carry;
  if (CHAIN) {
    float whole = 1.f, sum = 0.f;
    if (w == 0)
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const Pair p = back[q][lane];
        sum = p.A * sum + p.C;
        whole *= p.A;
      }
    carry = Chain(a).hand_on(tiles - 1 - tile, ch, whole, sum, a.dcT, handed,
                             seen, begin == 0 ? a.dc0 : nullptr, w);
  } else {
    carry = a.dcT ? a.dcT[ch.state] : 0.f;
  }
  carry = compose(carry, back, 0, rw);
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
    const int t = t0 + k;
    const float dc = carry + u[k], dci = dc * i[k], dcf = dc * f[k];
    carry = dcf;
    d -= a.dgates_t;
    if (t < a.T) {
      const bool on = t < stop;
      at(d, d_off) = on ? (E)(dci * n[k] * (1.f - i[k])) : (E)0.f;
      at(d + a.H, d_off) = on ? (E)(dcf * before[k] * (1.f - f[k])) : (E)0.f;
      at(d + 3 * (int64_t)a.H, d_off) =
          on ? (E)(dci * (1.f - n[k] * n[k])) : (E)0.f;
    }
  }
  if (!CHAIN && w == 0) a.dc0[ch.state] = carry;
}

template <typename E>
__global__ void glr_step_kernel(GlrArgs a) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (id >= (int64_t)a.B * a.H) return;
  const int b = (int)(id / a.H), j = (int)(id % a.H), H = a.H;
  const E* g = static_cast<const E*>(a.gates) + b * a.gates_b + j;
  float* cp = a.cT + b * a.c_b + j;
  const float c = sigmoid_f((float)g[H]) * *cp +
                  sigmoid_tanh<E>((float)g[0], (float)g[3 * H]);
  *cp = c;
  static_cast<E*>(a.h)[b * a.h_b + j] =
      (E)sigmoid_tanh<E>((float)g[2 * H], c);
}

template <typename F>
void by_type(GlrType type, F f) {
  switch (type) {
    case GlrType::F32: f(float{}); break;
    case GlrType::F16: f(_Float16{}); break;
    case GlrType::BF16: f(__bf16{}); break;
  }
}

// Steps of a wave, and waves of a block. Up to 128 steps are one tile of waves
// with 8 steps each, backward up to 64 of waves with 4: more waves to hide the
// one round of loads. 35 x 20 x 1500 bf16 takes 7.3 us with 4 against 8.3, 16 x
// 64 x 1500 8.1 against 9.5, but 64 x 128 x 650 23 against 21; forward 4
// measure 6.6 against 6.4, 17 against 16 at 35 x 128 x 1500, 14.5 against 12.6
// at 64 x 128 x 650. From 65 steps on a chain would take 13 / 18 us at 65 x 20
// x 1500 against 7.2 / 11.4, and 58 / 116 against 57 / 125 at 128 x 128 x 1500:
// there alone, backward with many channels, the one threshold is not the best.
//
// A chain's tiles are 128 steps forward, 64 backward, of 8 waves. 16 waves with
// 8 steps measured 218 us against 200 forward at 65536 x 1 x 1472, 4 waves with
// 16 566 against 545 backward at 65536 x 1 x 1500. Forward with MANY_GROUPS, a
// group for each CU, tiles are 64 steps of 4 waves: blocks end sooner, and more
// of them wait while others load. 300 x 64 x 650 takes 34 us against 39, 512 x
// 80 x 1500 135 against 147 and with random lengths 110 against 127, 1024 x 16
// x 1500 56 against 60, but 256 x 20 x 1500 21.8 against 21.3; with fewer
// groups 65536 x 1 x 1500 273 against 256, 8192 x 2 x 1024 f32 73 against 70.
// Backward the same costs 3 to 15 %. (All before the selects of small_tanh, up
// to 2 % on either side.) Blocks that loop over tiles, which need no chain,
// measured from 256 steps on up to four times a chain's time where channels are
// few (23 groups, 512 steps: 20 / 33 us against 10 / 14) and 1.1 to 1.4 times
// where they are many (1875 groups, 512 steps: 161 / 401 against 153 / 292).
constexpr int TILE_STEPS = 8, SHORT_STEPS = 4, TILE_WAVES = 16;
constexpr int FWD_STEPS = 16, BWD_STEPS = 8, CHAIN_WAVES = 8;
constexpr int MANY_GROUPS = 256, MANY_WAVES = 4;

// Rows of one launch: all, unless rows lie so far apart that those of a block
// do not fit a lane's 32-bit offset; then one.
int rows_per_launch(const GlrArgs& a, int size) {
  const int64_t most =
      std::max(std::max(std::abs(a.gates_b), std::abs(a.h_b)),
               std::max(std::abs(a.dh_b), std::abs(a.dgates_b)));
  const int64_t apart = 63 / a.H + 1;  // rows from a block's first to last
  return (apart * most + 4 * (int64_t)a.H) * size < (int64_t)1 << 32 ? a.B : 1;
}

int chain_waves(int64_t groups, bool back) {
  return back || groups < MANY_GROUPS ? CHAIN_WAVES : MANY_WAVES;
}

// Tiles of a chain; 0 where one tile is the window.
int chunks_of(int64_t T, int64_t groups, bool back) {
  return T > TILE_STEPS * TILE_WAVES
             ? cdiv(T, (back ? BWD_STEPS : FWD_STEPS) *
                           chain_waves(groups, back))
             : 0;
}

GlrArgs planned(GlrArgs a, bool back, int size) {
  a.rows = rows_per_launch(a, size);
  a.groups = cdiv((int64_t)a.rows * a.H, 64);
  a.chunks = chunks_of(a.T, a.groups, back);
  return a;
}

// Steps of a wave where one tile is the window.
int tile_steps(int64_t T, bool back) {
  return back && T <= SHORT_STEPS * TILE_WAVES ? SHORT_STEPS : TILE_STEPS;
}

// At least as many for each counter as it has slots, for each share as it has
// groups.
int64_t blocks_of(int64_t groups, int64_t chunks) {
  return chunks && groups < SHARED_FROM
             ? (int64_t)XCDS * cdiv(chunks, XCDS) * groups
             : (int64_t)XCDS * cdiv(groups, XCDS) *
                   std::max<int64_t>(chunks, 1);
}

template <bool BACK, typename E>
void launch(const GlrArgs& args, hipStream_t stream) {
  GlrArgs a = planned(args, BACK, sizeof(E));
  const int64_t blocks = blocks_of(a.groups, a.chunks);
  for (a.row0 = 0; a.row0 < a.B; a.row0 += a.rows) {
    if (a.chunks) {
      const int64_t n = glr_work_words(args, BACK, sizeof(E)) / 2;
      hipLaunchKernelGGL(glr_reset_kernel, dim3(cdiv(n, 256)), dim3(256), 0,
                         stream, reinterpret_cast<uint4*>(a.work), n);
      const int waves = chain_waves(a.groups, BACK);
      auto kernel = BACK ? glr_bwd_kernel<E, BWD_STEPS, CHAIN_WAVES, true>
                    : waves == CHAIN_WAVES
                        ? glr_fwd_kernel<E, FWD_STEPS, CHAIN_WAVES, true>
                        : glr_fwd_kernel<E, FWD_STEPS, MANY_WAVES, true>;
      hipLaunchKernelGGL(kernel, dim3(blocks),
                         dim3(64 * waves), 0, stream, a);
    } else {
      const int steps = tile_steps(a.T, BACK);
      auto kernel = glr_fwd_kernel<E, TILE_STEPS, TILE_WAVES, false>;
      if constexpr (BACK)
        kernel = steps == TILE_STEPS
                     ? glr_bwd_kernel<E, TILE_STEPS, TILE_WAVES, false>
                     : glr_bwd_kernel<E, SHORT_STEPS, TILE_WAVES, false>;
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * cdiv(a.T, steps)), 0,
                         stream, a);
    }
  }
}

}  // namespace

int64_t glr_work_words(const GlrArgs& args, bool back, int size) {
  const GlrArgs a = planned(args, back, size);
  if (!a.chunks) return 0;
  const int64_t n = COUNTER_WORDS + (int64_t)a.chunks * a.B * a.H;
  return n + (n & 1);
}

int64_t glr_threads(int64_t T, int64_t B, int64_t H, bool back) {
  const int64_t groups = cdiv(B * H, 64), chunks = chunks_of(T, groups, back);
  return blocks_of(groups, chunks) * 64 *
         (chunks ? chain_waves(groups, back) : cdiv(T, tile_steps(T, back)));
}

void launch_glr_fwd(const GlrArgs& a, GlrType type, hipStream_t stream) {
  by_type(type, [&](auto e) { launch<false, decltype(e)>(a, stream); });
}

void launch_glr_bwd(const GlrArgs& a, GlrType type, hipStream_t stream) {
  by_type(type, [&](auto e) { launch<true, decltype(e)>(a, stream); });
}

void launch_glr_step(const GlrArgs& a, GlrType type, hipStream_t stream) {
  const int grid = cdiv((int64_t)a.B * a.H, 256);
  by_type(type, [&](auto e) {
    hipLaunchKernelGGL(glr_step_kernel<decltype(e)>, dim3(grid), dim3(256), 0,
                       stream, a);
  });
}

}  // namespace zamd
