// Host-callable launchers of every dlvk_b200 CUDA kernel.  All pointers are
// device pointers; every launcher enqueues on the given stream and never
// synchronises.  Scratch buffers, where needed, are supplied by the caller.
#pragma once
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cstdint>

#include "dlvk/common.h"

namespace dlvk {

// ---- elementwise -----------------------------------------------------------
enum UnaryOp : int {
  UN_RELU = 0, UN_SIGMOID = 1, UN_TANH = 2, UN_SCALE = 3, UN_CLAMP = 4, UN_SQRT = 5, UN_COPY = 6,
  UN_SQUARE = 7, UN_ADD_SCALAR = 8, UN_ABS = 9, UN_EXP = 10, UN_LOG = 11, UN_GELU = 12,
};
enum BinaryOp : int {
  BIN_ADD = 0, BIN_SUB = 1, BIN_MUL = 2, BIN_DIV = 3, BIN_MAX = 4, BIN_MIN = 5,
  BIN_RELU_BWD = 6, BIN_SIGMOID_BWD = 7, BIN_TANH_BWD = 8, BIN_GELU_BWD = 9,
};
void unary(DType dt_in, DType dt_out, const void* x, void* y, int64_t n, int op, float a, float b, cudaStream_t s);
void binary(DType dt, const void* x, const void* y, void* z, int64_t n, int op, cudaStream_t s);
void bias_act(DType dt, DType dt_bias, const void* x, const void* bias, void* out, int64_t rows, int64_t cols, int act,
              cudaStream_t s);

// ---- reductions / layout ---------------------------------------------------
enum ReduceOp : int { RED_SUM = 0, RED_MAX = 1, RED_MIN = 2, RED_SUMSQ = 3, RED_ABSMAX = 4 };
int reduce_scratch_floats();
void reduce(DType dt, const void* x, int64_t n, int op, float scale, float* out, float* scratch, cudaStream_t s);
// out[c] = scale * sum_k partial[k * cols + c] (+ out[c]); fp32, fixed order.
void colsum_partials(const float* partial, int64_t chunks, int64_t cols, float scale, float* out, bool accumulate,
                     cudaStream_t s);
// scratch: colsum_scratch_floats(rows, cols) floats (may be null: single pass)
int64_t colsum_scratch_floats(int64_t rows, int64_t cols);
void colsum(DType dt, DType dt_out, const void* x, int64_t rows, int64_t cols, float scale, void* out, bool accumulate,
            float* scratch, cudaStream_t s);
void rowsum(DType dt, const void* x, int64_t rows, int64_t cols, float scale, float* out, cudaStream_t s);
void transpose2d(DType dt, const void* x, void* y, int64_t batch, int64_t rows, int64_t cols, cudaStream_t s);
void permute4(DType dt, const void* x, void* y, const int* in_dims, const int* perm, cudaStream_t s);

// ---- softmax / losses --------------------------------------------------------
enum LossKind : int { LOSS_MSE = 0, LOSS_BCE = 1 };
void softmax(DType dt, const void* x, void* y, int64_t rows, int64_t cols, bool log_out, cudaStream_t s);
void softmax_bwd(DType dt, const void* y, const void* dy, void* dx, int64_t rows, int64_t cols, cudaStream_t s);
void softmax_cross_entropy(DType dt, const void* logits, const int* labels, const float* probs, float* loss_rows,
                           void* dlogits, int64_t rows, int64_t cols, float grad_scale, cudaStream_t s);
int pointwise_loss_blocks(int64_t n);
void pointwise_loss(DType dt, int kind, const void* p, const float* t, int64_t n, float loss_scale, float grad_scale,
                    void* grad, float* out, float* scratch, cudaStream_t s);
void sum_rows_to_scalar(const float* rows_vals, int64_t n, float scale, float* out, cudaStream_t s);

// ---- GEMM -------------------------------------------------------------------
enum Act : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2 };
// C[b](m, n) = act(alpha * sum_k A[b](m, k) * B[b](k, n) + beta * C[b](m, n) + bias[n] + R[b](m, n))
// A(m,k) = A[m*sam + k*sak]; B(k,n) = B[k*sbk + n*sbn]; C(m,n) = C[m*ldc + n].
// Batches are two-level: b = (bo, bi), bo < batch, bi < batch2, with
// independent strides per level (e.g. (batch, head) of an attention tensor).
struct GemmArgs {
  const void* A = nullptr;
  const void* B = nullptr;
  void* C = nullptr;
  int64_t M = 0, N = 0, K = 0;
  int64_t sam = 0, sak = 0, sbk = 0, sbn = 0, ldc = 0;
  int64_t batch = 1, batch_stride_a = 0, batch_stride_b = 0, batch_stride_c = 0;
  int64_t batch2 = 1, batch2_stride_a = 0, batch2_stride_b = 0, batch2_stride_c = 0;
  float alpha = 1.f, beta = 0.f;
  const void* bias = nullptr;
  int bias_dtype = 0;
  int act = ACT_NONE;
  const void* residual = nullptr;  // same dtype as C, added before act
  int64_t ldr = 0, batch_stride_r = 0, batch2_stride_r = 0;
  bool residual_f32 = false;  // the residual is fp32 beside a bf16 C (tensor-core path, 2-D, beta 0)
  // Optional mask source (same dtype and shape as C): the output is zeroed
  // where mask <= 0.  Fuses the backward of a preceding ReLU into dX = dY W^T.
  const void* relu_mask = nullptr;
  int64_t ldm = 0, batch_stride_m = 0, batch2_stride_m = 0;
  // Optional column sums of the output (before its rounding to C's dtype):
  // per 32-row block, colsum[(m / 32) * N + n].  Needs gemm_tc_colsum_ok();
  // colsum_partials() then adds the ceil(M / 32) rows.  Fuses a bias
  // gradient db = sum_rows(dY) into the GEMM that produces dY.
  float* colsum = nullptr;
  // Optional fp32 bias per output row (added with the column bias, before
  // the activation): the per-channel bias of a convolution whose output
  // rows are channels (1x1 convolution in NCHW as a batched GEMM).  Tensor-
  // core path only.
  const float* row_bias = nullptr;
  // Optional ReLU bitmask, one bit per output element: bit n % 32 of word
  // [m * ldbits + n / 32].  relu_bits_out is written by a forward GEMM (bit
  // set where the output, after the activation, is > 0); relu_bits zeroes
  // the output where the bit is clear -- the backward of that ReLU, reading
  // 1/16 of the bytes of a bf16 mask.  2-D GEMMs only.
  uint32_t* relu_bits_out = nullptr;
  const uint32_t* relu_bits = nullptr;
  int64_t ldbits = 0;
  // Sum split-K partials in a fixed order (through the workspace) instead of
  // adding them into an fp32 C as they come.
  bool ordered = false;
  const float* alpha_ptr = nullptr;  // optional device factor of alpha (tensor-core path)
  // bf16 operands that hold an fp32 matrix in three parts side by side along
  // their contiguous dimension, pitch_a / pitch_b (multiples of 64) elements
  // apart (split_parts): C = the fp32 product, as six bf16 ones.  The padding
  // of K is zero.  Tensor-core path; gemm_tc_workspace_floats() says what room
  // its split-K takes, without which the sums are unsplit.  K is at most
  // GEMM_PARTS_K; a longer product is a sum of such ones (beta = 1), whose
  // pointers are k_done elements of K further on.
  bool parts = false;
  int64_t pitch_a = 0, pitch_b = 0, k_done = 0;
};
// The accumulators lose up to 2^-23 of themselves with every addition, always
// towards zero (plain fp32 rounds, and errs to both sides), so that a product
// in parts is as good as fp32 only while one accumulator sums few elements of K;
// the rest is summed by the split-K reduction, of at most 32 splits.
constexpr int64_t GEMM_PARTS_ACC = 1280, GEMM_PARTS_K = 32 * GEMM_PARTS_ACC;
// SIMT GEMM.  With a workspace of gemm_simt_workspace_floats(a) floats, a
// small 2-D GEMM with a plain epilogue splits K across blocks (fp32 partials,
// then a finish kernel; deterministic).
int64_t gemm_simt_workspace_floats(const GemmArgs& a);
void gemm_simt(DType in_dt, DType out_dt, const GemmArgs& a, cudaStream_t s, float* ws = nullptr,
               int64_t ws_floats = 0);
bool gemm_tc_supported(const GemmArgs& a);
// bf16 inputs, bf16 or f32 output, tcgen05 tensor cores.  `err` is the
// device error word; `max_ctas` caps the persistent grid (0 = #SMs).
// Split-K: when the tile grid underfills the GPU, partial sums go to an fp32
// `workspace` of gemm_tc_workspace_floats() floats (0 = none needed) and a
// reduce kernel applies the epilogue.  With a null/small workspace the GEMM
// runs unsplit.  An fp32 C with a linear epilogue (alpha, beta 0 or 1) needs
// no workspace: the partials are added into C by TMA reduces.
int64_t gemm_tc_workspace_floats(const GemmArgs& a, int max_ctas = 0, DType out_dt = DType::BF16,
                                 bool tf32 = false);
// CTA-pair (tcgen05 cta_group::2, 256 x 256 tiles) variant for unsplit bf16
// GEMMs with M >= 256; on by default (DLVK_GEMM_PAIR=0 turns it off).
bool gemm_tc_pair_enabled();
void gemm_tc_set_pair(bool on);
// 256 x 512 CTA-pair tile (two N = 256 MMAs per k-step, one TMEM buffer) for
// long-K GEMMs with few tiles.  Mode 0 never, 1 when the tiling model picks
// it (default; DLVK_GEMM_WIDE sets the initial mode), 2 whenever it applies.
void gemm_tc_set_wide(int mode);
// Forces the tile N (128 / 256 / 512), split-K factor and CTA-pair use of
// later GEMMs (0 / 0 / -1 restore the tiling model); for measurements.
void gemm_tc_set_tiling(int bn, int splits, int pair);
// The tiling the model picks for these operands: tile N (128/256/512), the
// split-K factor, and whether the CTA-pair kernel runs.
void gemm_tc_plan(DType out_dt, const GemmArgs& a, int max_ctas, int* bn, int* splits, int* pair);
bool gemm_tc_colsum_ok(DType out_dt, const GemmArgs& a);
void gemm_tc(DType out_dt, const GemmArgs& a, cudaStream_t s, uint32_t* err, int max_ctas = 0,
             float* workspace = nullptr, int64_t workspace_floats = 0);
// fp32 operands on the tensor cores (tcgen05 kind::tf32: each product uses
// the operands' top 19 bits, fp32 accumulation), single-CTA tiles; A / B
// K-major or M/N-major like gemm_tc, row strides multiples of 4 elements.
bool gemm_tf32_tc_supported(const GemmArgs& a);
void gemm_tf32_tc(DType out_dt, const GemmArgs& a, cudaStream_t s, uint32_t* err, int max_ctas = 0,
                  float* workspace = nullptr, int64_t workspace_floats = 0);
// Splits fp32 x into hi = x rounded to tf32 and lo = x - hi, so that
// A B ~= Ahi Bhi + Ahi Blo + Alo Bhi with every product exact in tf32 up to
// the lo terms' own rounding (relative error ~2^-21): the 3xTF32 scheme.
void tf32_split(const float* x, float* hi, float* lo, int64_t n, cudaStream_t s);

// ---- int8 ----------------------------------------------------------------------
// q[r, :] = round(x[r, :] / s[r]), s[r] = max|x[r, :]| / 127 (symmetric, per row).
void quantize_rows_int8(DType dt, const void* x, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq,
                        float* scale, cudaStream_t s);
bool gemm_i8_tc_supported(const void* A, const void* Bt, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb);
// C = act(sum_k A[m,k] Bt[n,k] * sa[m] * sb[n] + bias[n]); A [M,K], Bt [N,K] int8.
void gemm_i8_tc(const int8_t* A, const int8_t* Bt, const float* sa, const float* sb, const float* bias, int act,
                void* C, DType out_dt, int64_t ldc, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                cudaStream_t s, uint32_t* err);
void gemm_i8_simt(const int8_t* A, const int8_t* Bt, const float* sa, const float* sb, const float* bias, int act,
                  void* C, DType out_dt, int64_t ldc, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                  cudaStream_t s);

// ---- optimizers --------------------------------------------------------------
enum OptKind : int { OPT_SGD = 0, OPT_ADAM = 1, OPT_RMSPROP = 2 };
// Device-resident optimizer hyper-parameters (one per optimizer instance).
struct OptimHyper {
  float lr;
  float beta1, beta2, eps;
  float weight_decay;
  float momentum;
  float alpha;          // RMSprop smoothing
  float grad_scale;     // multiplies every gradient (e.g. 1/world, 1/loss_scale)
  float bc1, bc2;       // bias corrections, maintained by optim_advance
  int step;
  int bias_correction;  // 1: Adam with 1/(1-beta^t) corrections
  int decoupled_wd;     // 1: AdamW-style decay
  int pad_;
  const float* clip_coef_ptr;  // optional device scalar multiplying the grads
  const int* skip_flag_ptr;    // optional device flag: skip the update when set
};
void optim_advance(OptimHyper* h_dev, cudaStream_t s);
// max_ctas > 0 caps the grid (an update overlapped with other kernels).
void optim_update(int kind, const OptimHyper* h_dev, float* p, const void* g, DType g_dt, float* m, float* v,
                  __nv_bfloat16* p_bf16, int64_t n, float extra_scale, cudaStream_t s, int max_ctas = 0);
int grad_stats_scratch_floats();
void grad_stats(const void* g, DType g_dt, int64_t n, float scale, float max_norm, float* sumsq_out, int* flag,
                float* clip_out, bool accumulate, float* scratch, cudaStream_t s, const float* scale_ptr = nullptr);
// x[i] *= *s (s on the device: a loss scale that a captured graph re-reads).
void scale_by_device_scalar(DType dt, void* x, int64_t n, const float* s, cudaStream_t st);
// Fused L1/L2 regularisation over [n) flat parameters:
//   g += k * (l1 * sign(w) + l2 * w);  *loss_out += ll1 * |w| + 0.5 * ll2 * w^2 (if loss_out),
// with k = *gscale (a loss scale still applied to g) or 1.  The loss
// coefficients differ from the gradient ones for weight decay, which has a
// gradient term and no loss term.
void regularize(const float* w, void* g, DType g_dt, int64_t n, float l1, float l2, float ll1, float ll2,
                float* loss_out, cudaStream_t s, const float* gscale = nullptr);
void scaler_update(float* scale, int* good_steps, const int* found_inf, float growth, float backoff, int interval,
                   float smin, float smax, float* inv_scale, cudaStream_t s);

// ---- global gradient norm over a list of tensors (grad_norm.cu) -------------
constexpr int NORM_LIST_MAX = 1024;  // dense tensors per launch
// kind: bit 0 = bf16 input, bit 1 = bf16 output (else fp32).
struct DenseItem {
  const void* in;
  void* out;
  int64_t n;
  uint8_t kind;
};
// A tensor with gaps or of another element order than its output: sizes and
// strides (elements) over at most four dimensions, leading ones of size 1.
struct StridedItem {
  const void* in;
  void* out;
  int64_t n;
  int64_t size[4], in_stride[4], out_stride[4];
  uint8_t kind;
};
// Number of fp64 partial sums that grad_norm() writes for these items.
int grad_norm_parts(const DenseItem* dense, int n_dense, const StridedItem* strided, int n_strided);
// *norm = sqrt(sum of squares of all inputs); with `scale` also
// out = in * min(1, max_norm / (norm + 1e-6)), or 1 for a norm that is not
// finite.  `in == out` scales in place; otherwise inputs and outputs are disjoint.
void grad_norm(const DenseItem* dense, int n_dense, const StridedItem* strided, int n_strided, bool scale,
               float max_norm, float* norm, double* partial, cudaStream_t s);

// ---- convolution / pooling ---------------------------------------------------
struct ConvDesc {
  int N, Cin, H, W, Cout, KH, KW, stride, pad, Ho, Wo;
};
void conv2d_fwd(DType dt, const void* x, const void* w, const float* bias, void* y, const ConvDesc& d, bool relu,
                cudaStream_t s);
// relu_src (optional): the forward input of the preceding ReLU (or its output);
// dx is zeroed where relu_src <= 0, fusing that activation's backward.
void conv2d_dgrad(DType dt, const void* g, const void* w, void* dx, const void* relu_src, const ConvDesc& d,
                  cudaStream_t s);
// Implicit-GEMM tcgen05 convolution (conv_tc.cu), bf16 with channel counts
// that are multiples of 8.  Activations are gathered from NHWC copies; the
// outputs (y, dx) are written NCHW.
bool conv2d_tc_supported(DType dt, const ConvDesc& d);
void conv_tc_set_mode(int mode);  // 0 auto (large convolutions), 1 whenever supported, 2 never
int conv_tc_get_mode();
int64_t conv_pack_cols(int64_t k);  // packed weight row length for K = KH*KW*channels
// [OC][C][KH][KW] -> bf16 [OC][conv_pack_cols(KH*KW*C)] (forward) or
// [C][conv_pack_cols(KH*KW*OC)] (dgrad), taps outer and channels inner.
void conv_pack_weights(DType wdt, const void* w, __nv_bfloat16* out, const ConvDesc& d, bool dgrad, cudaStream_t s);
// forward: src = X (NHWC), out = Y (NCHW); dgrad: src = dY (NHWC), out = dX
// (NCHW), `mask` zeroes dX where the preceding ReLU was inactive.
void conv2d_igemm(const __nv_bfloat16* src_nhwc, const __nv_bfloat16* wpack, const ConvDesc& d, bool dgrad,
                  const float* bias, bool relu, const void* mask, void* out, bool out_f32, cudaStream_t s);
int64_t conv2d_wgrad_tc_ws_floats(const ConvDesc& d);
void conv2d_wgrad_tc(const __nv_bfloat16* x_nhwc, const __nv_bfloat16* dy_nhwc, const ConvDesc& d, float* ws,
                     float* dw, bool accumulate, cudaStream_t s);
int conv2d_wgrad_chunks(const ConvDesc& d);
int64_t conv2d_wgrad_scratch_floats(const ConvDesc& d);
void conv2d_wgrad(DType dt, const void* x, const void* g, float* dw, float* db, bool accumulate, const ConvDesc& d,
                  float* scratch, cudaStream_t s);
void maxpool2d_fwd(DType dt, const void* x, void* y, int32_t* idx, int64_t planes, int H, int W, int k, int stride,
                   cudaStream_t s);
void maxpool2d_bwd(DType dt, const void* g, const int32_t* idx, void* dx, int64_t planes, int H, int W, int k,
                   int stride, cudaStream_t s);
void avgpool2d_fwd(DType dt, const void* x, void* y, int64_t planes, int H, int W, int k, int stride, int pad,
                   cudaStream_t s);
void avgpool2d_bwd(DType dt, const void* g, void* dx, int64_t planes, int H, int W, int k, int stride, int pad,
                   cudaStream_t s);

// ---- normalisation / dropout / embedding -------------------------------------
// Philox dropout stream: key = seed, counter = {element/4, stream, step}.
struct DropoutDesc {
  float p = 0.f;                  // drop probability (0 = disabled)
  uint32_t stream = 0;            // distinct per dropout site
  uint64_t seed = 0;
  uint32_t step = 0;              // used when step_ptr is null
  const int64_t* step_ptr = nullptr;  // device step counter (graph replays)
};
// scratch (both passes): batchnorm_scratch_floats(N, C, S) floats.
int64_t batchnorm_scratch_floats(int N, int C, int S);
void batchnorm_fwd(DType dt, const void* x, const float* gamma, const float* beta, void* y, float* mean, float* rstd,
                   float* run_mean, float* run_var, int N, int C, int S, float momentum, float eps, bool training,
                   bool relu, const DropoutDesc& dd, float* scratch, cudaStream_t s);
void batchnorm_bwd(DType dt, const void* x, const void* dy, const float* mean, const float* rstd, const float* gamma,
                   const float* beta, void* dx, float* dgamma, float* dbeta, bool accumulate, int N, int C, int S,
                   bool relu, const DropoutDesc& dd, float* scratch, cudaStream_t s);
void layernorm_fwd(DType dt, const void* x, const float* gamma, const float* beta, void* y, float* mean, float* rstd,
                   int64_t rows, int D, float eps, cudaStream_t s);
int layernorm_bwd_blocks(int64_t rows);
int64_t layernorm_bwd_scratch_floats(int64_t rows, int D);
// dres (optional, same dtype/shape as dx): a residual-branch gradient added
// to dx, fusing the sum of the two gradients of a pre-norm block input.
// dres_colsum (optional, fp32 [D]): receives (or, with its accumulate flag,
// adds) the column sums of dres -- the bias gradient of the biased GEMM whose
// output gradient dres is.
void layernorm_bwd(DType dt, const void* x, const float* gamma, const float* mean, const float* rstd, const void* dy,
                   void* dx, float* dgamma, float* dbeta, bool accumulate, int64_t rows, int D, float* scratch,
                   cudaStream_t s, const void* dres = nullptr, float* dres_colsum = nullptr,
                   bool dres_colsum_accumulate = false);
void dropout(DType dt, const void* x, void* y, int64_t n, const DropoutDesc& dd, cudaStream_t s);
void embedding_fwd(DType dt, const int32_t* ids, const void* table, void* out, int64_t n, int64_t V, int D,
                   cudaStream_t s);
// dtable must be zeroed (or hold the gradient to accumulate into).
void embedding_bwd(DType dt, const int32_t* ids, const void* dy, float* dtable, int64_t n, int64_t V, int D,
                   cudaStream_t s);

// ---- softmax cross entropy of a projection, without keeping its logits --------
// z = x W + bias, x [rows, width], W [width, classes]; loss_i = log sum exp(z_i)
// - z_i[label_i].  A label outside [0, classes) or equal to `ignore` does not
// count.  Tensor-core passes (gemm_tc.cu): bf16 operands, the logits stay in
// the accumulators.
struct CeProjection {
  const __nv_bfloat16* x = nullptr;  // row stride ldx
  const __nv_bfloat16* w = nullptr;  // w_k: W^T, row (class) stride ldw; else W, row (width) stride ldw
  int64_t rows = 0, width = 0, classes = 0, ldx = 0, ldw = 0;
  bool w_k = false;
  const float* bias = nullptr;       // fp32 [classes]
  const void* labels = nullptr;
  bool labels64 = false;
  int64_t ignore = -1;
  float2* stats = nullptr;           // [ce_tc_stat_cols][rows] (maximum, sum of exp(z - maximum))
  float* zlabel = nullptr;           // [rows], written for rows that count
  const float2* norm = nullptr;      // [rows] maximum and 1 / sum, for the gradient
  const float* gscale = nullptr;     // device scalar: factor of ce_grad_tc's column sums
  // fp32 operands in three parts (GemmArgs::parts); ldx and ldw are then the
  // distances of whole rows of parts
  bool parts = false;
  int64_t pitch_x = 0, pitch_w = 0;
  unsigned* done = nullptr;          // set to 0 with the statistics (or null)
};
bool ce_tc_supported(const CeProjection& c);
// The statistics have one column per ce_tc_stat_width() classes.
int ce_tc_stat_width(int64_t rows, int64_t classes);
int ce_tc_stat_cols(int64_t rows, int64_t classes, bool parts);
void ce_stats_tc(const CeProjection& c, cudaStream_t s, uint32_t* err);
// The statistics, and e = 2^15 exp(z - the maximum of its statistics column),
// fp16 [rows, classes], row stride lde.
void ce_exp_tc(const CeProjection& c, void* e, int64_t lde, cudaStream_t s, uint32_t* err);
// dl [rows, classes] = softmax - onehot, bf16, row stride ldd; colsum (or
// null): gscale times its fp32 column sums per 32 rows [ceil(rows / 32)][classes],
// for colsum_partials.
void ce_grad_tc(const CeProjection& c, __nv_bfloat16* dl, int64_t ldd, float* colsum, cudaStream_t s, uint32_t* err);
// The passes around them, and the same statistics / gradient from logits in
// memory (vocab_loss.cu).
struct CeRows {
  int64_t rows = 0, classes = 0, ignore = -1;
  const void* labels = nullptr;
  bool labels64 = false;
};
// *gscale = (mean: 1 / counted rows, else 1) * (*grad_scale or 1); *done = 0.
void ce_count(const CeRows& r, bool mean, const float* grad_scale, float* gscale, unsigned* done, cudaStream_t s);
// Joins the statistics of one block of rows: rows_loss (0 where a row does
// not count) and norm; x_clean, when given, becomes a copy of x whose
// uncounted rows are 0.  The last of all `total_groups` groups of 32 rows (of
// every block of rows; this one's are first_group onwards) adds up the
// losses: *loss = sum (mean: / counted rows), and, when set_gscale, *gscale as
// ce_count's; where given, *loss_sum += the sum, *counted += the rows that
// count, *correct += those whose class has the largest logit.
// partial: 3 doubles per group.  `done` was set to 0 before the first block.
struct CeFinish {
  const float2* stats;
  int stat_cols;
  const float* zlabel;
  float* rows_loss;
  float2* norm;
  bool mean, set_gscale;
  const float* grad_scale;
  float *loss, *gscale;
  float* loss_sum;
  unsigned long long *counted, *correct;
  double* partial;
  unsigned* done;
  int first_group, total_groups;
  const void* x;
  int64_t ldx, width;
  void* x_clean;
  int64_t ldc;
};
void ce_finish(const CeRows& r, const CeFinish& f, DType dt, cudaStream_t s);
// e (ce_exp_tc's, fp16) becomes softmax - onehot in place, bf16; stat_width
// classes to a statistics column.  After ce_finish, or with `join` instead of
// it (bf16 x with x_clean), for as few statistics as ce_rescale_joins() says:
// every 2048 classes of a group read them all again (up to 8 MB, from L2).
bool ce_rescale_joins(int64_t rows, int64_t classes, int stat_cols);
void ce_rescale(const CeRows& r, const CeFinish& f, int stat_width, bool join, void* e, int64_t lde, cudaStream_t s);
// Statistics (ce_memory_stat_cols columns) and gradient of logits z [rows, classes] fp32, row
// stride ldz: z becomes (softmax - onehot) * gscale (not when keep_z is off);
// dl, when given, that
// rounded to bf16 (pitch 0, row stride ldz), or softmax - onehot in three
// parts (pitch of a part, row stride 3 pitch, zeros in the padding).
int ce_memory_stat_cols(int64_t rows, int64_t classes);
void ce_memory_stats(const CeRows& r, const float* z, int64_t ldz, float2* stats, float* zlabel, unsigned* done,
                     cudaStream_t s);
void ce_memory_grad(const CeRows& r, float* z, int64_t ldz, const float2* norm, const float* gscale, __nv_bfloat16* dl,
                    int64_t pitch, bool keep_z, cudaStream_t s);
// dst [rows, 3 pitch] bf16: src (fp32 [rows, cols], row stride ld) = the sum of
// its three parts to 2^-24; zeros in the padding, and with `mask` in the rows
// that do not count.
void split_parts(const float* src, int64_t ld, int64_t rows, int64_t cols, __nv_bfloat16* dst, int64_t pitch,
                 const CeRows* mask, cudaStream_t s);
// dst [rows, cols] (row stride ldd) = src (strides rs, cs), or += (accumulate);
// columns [cols, pad_to) become 0.  fp32 or bf16 each.
void copy_matrix(DType dst_dt, DType src_dt, const void* src, int64_t rs, int64_t cs, void* dst, int64_t ldd,
                 int64_t rows, int64_t cols, int64_t pad_to, bool accumulate, cudaStream_t s);

// ---- fp32 products with few rows (few_rows.cu) ---------------------------------
constexpr int FEW_ROWS = 16;
constexpr int64_t FEW_ROWS_K = 65535LL * 1024;  // longest K: a turned product has a block row for each 1024 of it
// out [rows, cols] = A [rows, K] B (+ bias per column), rows <= FEW_ROWS; B is
// [K, cols] with contiguous rows ldb apart, or (turned) its transpose is.
// scratch: few_rows_scratch_floats() floats.
int64_t few_rows_scratch_floats(int64_t rows, int64_t K, int64_t cols, bool turned);
void few_rows_product(const float* A, int64_t lda, const float* B, int64_t ldb, bool turned, const float* bias,
                      float* out, int64_t ldo, int64_t rows, int64_t K, int64_t cols, float* scratch, cudaStream_t s);
// out [A, cols] (or +=) = P^T Q, P [rows, A], Q [rows, cols], rows <= FEW_ROWS.
void few_rows_outer(const float* P, int64_t ldp, const float* Q, int64_t ldq, float* out, int64_t ldo, int64_t rows,
                    int64_t A, int64_t cols, bool accumulate, cudaStream_t s);

// ---- embedding lookup with scale, gradient by sorted tokens (embedding.cu) ---
// ids: int32 or int64 (ids64).  Rows of table / dy are ld elements apart.
// out[i, :] = scale * table[ids[i], :], zeros for ids outside [0, V).
void embedding_lookup(DType dt, bool ids64, const void* ids, const void* table, void* out, int64_t n, int64_t V, int D,
                      int64_t ld, float scale, cudaStream_t s);
// dtable[v, :] (fp32 [V, D]) = (or, accumulate, +=) scale * sum of dy[i, :] over
// ids[i] == v, in a fixed order; ids outside [0, V) and `padding` (-1: none)
// have no gradient.  Scratch: start embedding_grad_start_ints(V) ints, order and word n ints each,
// part embedding_grad_part_floats(n, D) floats.
// Fewer tokens and words than these: the places of the last block's chunks, up to
// 256 of 64 places past the end, are ints, and so are those of the words in the
// sort, of which each of up to 2^21 blocks may have one without a word.
constexpr int64_t EMBEDDING_GRAD_TOKENS = (1LL << 31) - 32768, EMBEDDING_GRAD_WORDS = (1LL << 31) - (1LL << 22);
int64_t embedding_grad_start_ints(int64_t V);
int64_t embedding_grad_part_floats(int64_t n, int D);
void embedding_grad(DType dt, bool ids64, const void* ids, const void* dy, int64_t ld, float* dtable, int64_t n,
                    int64_t V, int D, float scale, int64_t padding, bool accumulate, int* start, int* order, int* word,
                    float* part, cudaStream_t s);

// ---- operators over sequences with a state (short_conv.cu, state_scan.cu) ------
// Elements [B, T, D]: channels contiguous, tokens and sequences any number of
// elements apart.  p null: not there.
struct SeqRef {
  void* p = nullptr;
  int64_t batch = 0, token = 0;
};

// Causal depthwise convolution over `taps` tokens (2 to 4), with or without SiLU:
//   y[t] = act(bias + sum_j weight[:, j] x[t - taps + 1 + j])
// x before the first token is `state` [B, taps - 1, D], or zeros.  lengths
// (int32 [B], null: all T): positions past a sequence's length are neither read
// nor counted, and y is 0 there.
struct ShortConv {
  DType dt = DType::F32;
  int64_t B = 0, T = 0;
  int D = 0, taps = 0;
  bool silu = false;
  SeqRef x, state;
  const float* weight = nullptr;  // [D, taps]
  const float* bias = nullptr;    // [D]
  const int32_t* lengths = nullptr;
};
// out_state [B, taps - 1, D] (may be `state`): the last taps - 1 tokens that count.
void short_conv_fwd(const ShortConv& a, SeqRef y, SeqRef out_state, cudaStream_t s);
// dx, dweight [D, taps] and dbias [D] (either may be null), written or added to
// (accumulate).  part: short_conv_part_floats() floats.
int64_t short_conv_part_floats(const ShortConv& a);
void short_conv_bwd(const ShortConv& a, SeqRef dy, SeqRef dx, float* dweight, float* dbias, bool accumulate, float* part,
                    cudaStream_t s);

// Selective state space scan, for each channel d of its group's b and c:
//   s = softplus(dt + dt_bias)   h[t] = exp(-s exp(a_log)) h[t-1] + s u b[t]
//   y = (sum_n c h + skip u) silu(z)          (no gate where z is not there)
// h before the first token is `state`, or zeros.  lengths as above: a position
// past a sequence's length changes no state and its y is 0.
constexpr int STATE_SCAN_STATES = 64;  // most states of a channel
constexpr int STATE_SCAN_SPAN = 16;    // tokens between two kept states
struct StateScan {
  DType type = DType::F32;
  int64_t B = 0, T = 0;
  int D = 0, N = 0, G = 1;
  SeqRef u, dt, z;                  // [B, T, D]
  SeqRef b, c;                      // [B, T, G, N], groups and states contiguous
  const float* a_log = nullptr;     // [D, N]
  const float* skip = nullptr;      // [D]
  const float* dt_bias = nullptr;   // [D]
  const float* state = nullptr;     // [B, D, N]
  const int32_t* lengths = nullptr;
};
// out_state [B, D, N] (may be `state`): h after the last token that counts.
// saved [B, ceil(T / STATE_SCAN_SPAN), D, N]: h before every span's first token, for the backward pass.
// scratch: state_scan_fwd_scratch_floats() floats.
int64_t state_scan_fwd_scratch_floats(const StateScan& a);
void state_scan_fwd(const StateScan& a, SeqRef y, float* out_state, float* saved, float* scratch, cudaStream_t s);
struct StateScanGrads {
  SeqRef du, ddt, dz, db, dc;                                      // all written; dz where there is z
  float *da_log = nullptr, *dskip = nullptr, *ddt_bias = nullptr;  // written or (accumulate) added to; null: not wanted
  bool accumulate = false;
};
// scratch: state_scan_bwd_scratch_floats() floats.
int64_t state_scan_bwd_scratch_floats(const StateScan& a);
void state_scan_bwd(const StateScan& a, const float* saved, SeqRef dy, const StateScanGrads& g, float* scratch,
                    cudaStream_t s);

// ---- choice of the next word (sampling.cu) ---------------------------------------
// A setting: one value, or one for each row where the pointer is given.
template <typename T, typename One>
struct RowSetting {
  const T* rows = nullptr;
  One one = 0;
};
struct Sampling {
  DType dt = DType::F32;
  const void* logits = nullptr;  // [rows, words], rows ld elements apart
  int64_t rows = 0, words = 0, ld = 0;
  const float* uniform = nullptr;  // [rows]
  RowSetting<float, double> temperature, top_p, min_p;
  RowSetting<int32_t, int64_t> top_k;
};
constexpr int64_t SAMPLING_WORDS = 1 << 18;  // most words: sums of that many weights of 2^44 fit 64 bits
void sample_tokens(const Sampling& a, int32_t* tokens, cudaStream_t s);

// ---- device error word -------------------------------------------------------
uint32_t* device_error_word();     // per current device, zero-initialised
uint32_t read_device_error(bool clear);
void counter_add(int64_t* c, int64_t delta, cudaStream_t s);

// Per-step training metrics on the device: *loss_sum += *loss * loss_weight and
// *correct += #rows whose logits argmax equals the label (labels: int ids, or
// probs: target rows whose argmax is the class).  Either may be null.
void step_metrics(DType dt, const void* logits, int64_t rows, int cols, const int* labels, const float* probs,
                  const float* loss, float* loss_sum, unsigned long long* correct, float loss_weight, cudaStream_t s);

// ---- fused attention on tcgen05 (attention_tc.cu): head dim 64, S % 128 == 0 --
// qkv: [B, S, 3, H, 64] bf16; out: [B, S, H*64] bf16; lse: [B, H, S] fp32 (log2 units).
bool flash_attention_supported(int64_t B, int64_t S, int64_t H, int64_t D, const void* qkv);
void flash_attention_fwd(const __nv_bfloat16* qkv, __nv_bfloat16* out, float* lse, int B, int S, int H, float scale,
                         cudaStream_t s, uint32_t* err, int max_ctas = 0);
// dqkv: [B, S, 3, H, 64] bf16 (fully written); delta: [B, H, S] and dq_acc:
// [B*S, H*64] fp32 scratch.
void flash_attention_bwd(const __nv_bfloat16* qkv, const __nv_bfloat16* out, const __nv_bfloat16* dout,
                         const float* lse, float* delta, float* dq_acc, __nv_bfloat16* dqkv, int B, int S, int H,
                         float scale, cudaStream_t s, uint32_t* err, int max_ctas = 0);

// ---- recurrent cells (rnn.cu); kind 0 RNN-tanh, 1 LSTM, 2 GRU ---------------
// Every pointer addresses B rows with its own row stride (elements).
struct RnnCellFwd {
  int kind = 0;
  int64_t B = 0;
  int H = 0;
  const void* a = nullptr; int64_t lda = 0;        // pre-activations (GRU: input side) [B, G*H]
  const void* hg = nullptr; int64_t ldhg = 0;      // GRU hidden side h W_hh^T + b_hh [B, 3H]
  const void* h_prev = nullptr; int64_t ldhp = 0;  // GRU h_{t-1}
  const float* c_prev = nullptr; int64_t ldcp = 0; // LSTM c_{t-1} (null = 0)
  void* h_out = nullptr; int64_t ldo = 0;
  void* h_copy = nullptr; int64_t ldcopy = 0;      // optional second copy of h_t
  float* c_out = nullptr; int64_t ldco = 0;        // LSTM c_t
  float* saved = nullptr; int64_t lds = 0;         // LSTM (i,f,g,o) / GRU (r,z,n,hn) [B, 4H]
};
struct RnnCellBwd {
  int kind = 0;
  int64_t B = 0;
  int H = 0;
  const void* dh = nullptr; int64_t lddh = 0;
  const float* dc_next = nullptr; int64_t lddcn = 0;
  const void* h_t = nullptr; int64_t ldht = 0;
  const void* h_prev = nullptr; int64_t ldhp = 0;
  const float* c_t = nullptr; int64_t ldct = 0;
  const float* c_prev = nullptr; int64_t ldcp = 0;
  const float* saved = nullptr; int64_t lds = 0;
  void* dA = nullptr; int64_t ldda = 0;
  void* dAh = nullptr; int64_t lddah = 0;
  float* dc_prev = nullptr; int64_t lddcp = 0;
  const void* dy_prev = nullptr; int64_t lddyp = 0;
  void* resid = nullptr; int64_t ldres = 0;
};
void rnn_cell_fwd(const RnnCellFwd& p, DType dt, cudaStream_t s);
void rnn_cell_bwd(const RnnCellBwd& p, DType dt, cudaStream_t s);

// ---- batched image transforms (augment.cu), fp32 [N, C, H, W] ---------------
// theta: [N, 6] output->input maps (sx = t0*x + t1*y + t2, sy = t3*x + t4*y + t5);
// mode 0 nearest-floor, 1 nearest-round, 2 bilinear.
void image_affine_sample(const float* x, float* y, int N, int C, int H, int W, int OH, int OW, const float* theta,
                         int mode, float fill, cudaStream_t s);
// kind 0 contrast (params [N,2]: factor, -), 1 standardise, 2 min-max (params [N,2]: lo, hi).
void image_per_sample_stats(const float* x, float* y, int64_t N, int64_t len, int kind, const float* params,
                            bool clamp01, cudaStream_t s);
void image_channel_affine(const float* x, float* y, int64_t N, int C, int64_t HW, const float* mean,
                          const float* inv_std, const float* sample_add, bool clamp01, cudaStream_t s);
void image_gaussian_noise(const float* x, float* y, int64_t n, float sigma, uint64_t seed, uint32_t stream,
                          cudaStream_t s);

}  // namespace dlvk
