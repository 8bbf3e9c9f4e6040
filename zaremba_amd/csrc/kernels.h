// Host-side launcher prototypes for the gfx950 kernel library.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace zamd {

using bf16 = __bf16;

// gemm.hip — C[M,N] = A' @ B' (+bias); TRANS_A: A is [K,M]; TRANS_B: B is
// [K,N] (otherwise the NT weight layout B[N,K]).
template <bool TA, bool TB, typename OutT>
void launch_gemm_t(const bf16* A, const bf16* B, OutT* C, const float* bias,
                   int M, int N, int K, int lda, int ldb, int ldc,
                   hipStream_t stream);

// N-way split-K NT GEMM: one launch, grid.z = nz (returned), partials in
// C (with bias) and nz-1 stacked slices of C2 (without); K must be a
// BK(=64) multiple with >= 2 tiles.
template <typename OutT>
int launch_gemm_splitk_t(const bf16* A, const bf16* B, OutT* C, OutT* C2,
                         const float* bias, int M, int N, int K, int lda,
                         int ldb, int ldc, hipStream_t stream);

// lstm.hip (fragment-packed operands; see lstm.hip header comment)
void launch_pack_gated_w(const bf16* W, bf16* out, int rows, int ngates,
                         int K, hipStream_t stream);
void launch_pack_a(const bf16* A, bf16* out, int B, int K,
                   hipStream_t stream);
void launch_lstm_cell_fwd(const bf16* h_pack, const float* c_prev,
                          const bf16* gx, const bf16* W_pack, bf16* h_out,
                          bf16* h_pack_out, float* c_out, bf16* gates_out,
                          bf16* rec, int B, int H, int HSp,
                          hipStream_t stream);
void launch_lstm_cell_bwd_elt(const bf16* dy, const float* dh_rec,
                              const float* dh_rec2, float* dc,
                              const bf16* rec, bf16* dG, bf16* dG_pack,
                              int B, int H, int HSp, hipStream_t stream);
void launch_smallm_packed_nt(const bf16* A_pack, const bf16* W_pack,
                             float* C, float* C2, int M, int N, int K,
                             hipStream_t stream);
void launch_smallm_fused_bwd2(const bf16* A_pack, const bf16* W_pack,
                              float* P, const bf16* dY, float* dc,
                              const bf16* rec, bf16* dG, bf16* pack_mid,
                              bf16* pack_out, unsigned int* flags,
                              unsigned int* pstate,
                              unsigned int* abort_flag, int M, int N, int K,
                              int HSp, int t, unsigned int step1,
                              unsigned int gen, int64_t rstep, int nthreads,
                              hipStream_t stream);
void launch_smallm_fused_bwd(const bf16* A_pack, const bf16* W_pack,
                             float* P, const bf16* dy, float* dc,
                             const bf16* rec, bf16* dG, bf16* dG_pack_out,
                             unsigned int* flags, unsigned int* abort_flag,
                             int M, int N, int K, int HSp, unsigned int step,
                             int nsplit, int nthreads, hipStream_t stream);

// lstm_persistent.hip — one launch for a whole layer unroll
int persistent_hs(int H);
void set_fwd_threads_impl(int v);
size_t persistent_fwd_lds(int B, int H);
void launch_lstm_persistent_fwd(const bf16* gx, const bf16* W_h, bf16* h_all,
                                float* c_all, bf16* rec,
                                unsigned int* pstate,
                                unsigned int* abort_flag, int T, int B,
                                int H, hipStream_t stream);
size_t persistent_bwd_lds(int B, int H);
void launch_lstm_persistent_bwd(const bf16* dY, const bf16* rec,
                                const bf16* W_h_T, bf16* dG, bf16* dG_packT,
                                unsigned int* pstate,
                                unsigned int* abort_flag, int T, int B,
                                int H, hipStream_t stream);

// glr.hip — gated linear recurrence. Strides are in elements; the last axis
// is dense. c0, cT, dcT, dc0 and marks are f32 [.., B, H] and dense, but for
// the state of launch_glr_step (cT, read and written), whose rows are c_b
// apart.
constexpr int GLR_MARK = 32;  // steps between two kept states
constexpr int GLR_POLLS = 1 << 22;  // looks at a state that is not there yet
enum class GlrType { F32, F16, BF16 };
struct GlrArgs {
  const void* gates = nullptr;  // [T, B, 4H]
  int64_t gates_t = 0, gates_b = 0;
  void* h = nullptr;            // [T, B, H]
  int64_t h_t = 0, h_b = 0;
  const void* dh = nullptr;     // [T, B, H]
  int64_t dh_t = 0, dh_b = 0;
  void* dgates = nullptr;       // [T, B, 4H]
  int64_t dgates_t = 0, dgates_b = 0;
  const float* c0 = nullptr;    // null: zeros
  float* cT = nullptr;
  int64_t c_b = 0;
  const float* dcT = nullptr;   // null: zeros
  float* dc0 = nullptr;         // not null
  float* marks = nullptr;       // [ceil(T / GLR_MARK), B, H]; null: not kept
  const void* lengths = nullptr;  // [B] int32 or int64; null: all T
  bool lengths_64 = false;
  int T = 0, B = 0, H = 0;
  uint64_t* work = nullptr;  // glr_work_words of them, this call's own
  // set by the launchers: the rows of a launch, its blocks of 64 channels
  // and chunks of time
  int row0 = 0, rows = 0, groups = 0, chunks = 0;
  // A block whose state has not come after so many looks goes on with NaN and
  // sets *gave_up to 1, unless that is null. (Last: ahead of the sizes they
  // cost a short window 0.2 us, as the sizes then lie in another line.)
  int polls = GLR_POLLS;
  unsigned* gave_up = nullptr;
};
// Words of 64 bits that a call needs for itself; size: of a gate in bytes.
int64_t glr_work_words(const GlrArgs& a, bool back, int size);
// Threads of the largest launch for these sizes: a grid has fewer than 2^32.
int64_t glr_threads(int64_t T, int64_t B, int64_t H, bool back);
void launch_glr_fwd(const GlrArgs& a, GlrType type, hipStream_t stream);
void launch_glr_bwd(const GlrArgs& a, GlrType type, hipStream_t stream);
void launch_glr_step(const GlrArgs& a, GlrType type, hipStream_t stream);

// adamw.hip — AdamW over many tensors. The tensors of a launch travel in its
// arguments (4 KB at most), so that no call copies a table to the device.
constexpr int ADAMW_TENSORS = 48;
constexpr int ADAMW_NORM_CHUNK = 8192;  // values of a tensor at a time
// Values of a block of the update, of one tensor. At 66M parameters 1024, 2048
// and 4096 take 408, 416 and 422 us in 32 bits and 299, 279 and 285 in 8; at
// 4.7M 31, 29.6 and 29.6.
constexpr int ADAMW_CHUNK = 2048;
struct AdamwTensor {
  float* p;
  const void* g;       // f32 or bf16
  void* m;             // f32, or e4m3 codes
  void* v;             // f32, or e4m3 codes of its root
  float* m_scale;      // of 256 codes each
  float* v_scale;
  bf16* shadow;        // may be null
  int64_t n;
};
struct AdamwTensors {
  int count;
  int begin[ADAMW_TENSORS + 1];       // first chunk of each tensor, and the end
  int norm_begin[ADAMW_TENSORS + 1];  // the same in chunks of the norm
  AdamwTensor t[ADAMW_TENSORS];
};
struct AdamwScalars {
  int64_t* step;       // steps done; the norm's launch advances it
  double lr, beta1, beta2, max_norm, grad_scale;
  float b1, c1, b2, c2, eps, keep;  // c: 1 - b; keep: 1 - lr * decay
  bool clip;
};
struct AdamwValues {  // of this step, left by the norm's launch
  float rate, root;
  unsigned step;
};
struct AdamwWork {
  double* partials;    // [count] sums of squares
  int count;
  AdamwValues* values;
  float* norm;
};
int adamw_norm_blocks(const AdamwTensors& a, int launches);
void launch_adamw_norm(const AdamwTensors& a, const AdamwScalars& s,
                       bool bf16_grads, int first, int blocks,
                       const AdamwWork& w, hipStream_t stream);
void launch_adamw_update(const AdamwTensors& a, const AdamwScalars& s,
                         bool bf16_grads, bool bits8, bool tell,
                         const AdamwWork& w, hipStream_t stream);

// elementwise.hip
void launch_embedding_fwd(const bf16* W, const int64_t* idx, bf16* out,
                          int N, int H, hipStream_t stream);
void launch_embedding_bwd_det(const bf16* dY, const int64_t* idx, float* dW,
                              int N, int H, int V, hipStream_t stream);
void launch_embedding_bwd(const bf16* dY, const int64_t* idx, float* dW,
                          int N, int H, hipStream_t stream);
void launch_dropout_fwd(const bf16* x, bf16* y, float p, uint64_t seed,
                        uint64_t offset, int64_t n, hipStream_t stream);
void launch_dropout_bwd(const bf16* dy, bf16* dx, float p, uint64_t seed,
                        uint64_t offset, int64_t n, hipStream_t stream);
void launch_lsm_nll_fwd(const float* scores, const int64_t* y, float* lse,
                        float* loss_accum, int N, int V, hipStream_t stream);
void launch_lsm_nll_bwd(const float* scores, const float* lse,
                        const int64_t* y, const float* upstream, float scale,
                        float* dscores, int N, int V, hipStream_t stream);
void launch_norm2_accum(const float* g, int64_t n, float* accum,
                        hipStream_t stream);
void launch_norm2_mt(const int64_t* desc, int nchunk, float* accum,
                     hipStream_t stream);
void launch_sgd_mt(const int64_t* desc, int nchunk, const float* norm2,
                   float max_norm, float lr, float grad_scale,
                   hipStream_t stream);
void launch_sgd_update(float* master, const float* grad, bf16* shadow,
                       const float* norm2, float max_norm, float lr,
                       float grad_scale, int64_t n, hipStream_t stream);
void launch_transpose_bf16(const bf16* src, bf16* dst, int R, int C,
                           int ldd, hipStream_t stream);
void launch_add2_f32_bf16(const float* a, const float* b, bf16* out,
                          int64_t n, hipStream_t stream);
void launch_addn_f32_bf16(const float* a, const float* extra, int nextra,
                          bf16* out, int64_t n, hipStream_t stream);
void launch_colsum_bf16(const bf16* in, float* out, int R, int C,
                        hipStream_t stream);
void launch_colsum_f32(const float* in, float* out, int R, int C,
                       hipStream_t stream);
void launch_softmax_acc(const float* scores, float* acc, int N, int V,
                        hipStream_t stream);

}  // namespace zamd
