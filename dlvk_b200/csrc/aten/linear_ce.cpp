// ATen-level softmax cross entropy of a vocabulary projection: loss and
// gradients from x [rows, width] and W [width, classes] without an array of
// logits (gemm_tc.cu EPI 3 / 4, vocab_loss.cu).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>

#include "dlvk/aten_ops.h"
#include "dlvk/kernels.h"

namespace dlvk {
namespace aten {
namespace {

int64_t round_up(int64_t n, int64_t a) { return (n + a - 1) / a * a; }
int64_t ceil_div(int64_t n, int64_t a) { return (n + a - 1) / a; }

// Rows of one launch: every pass covers at least 32 of them with one of the
// 65535 blocks of a grid's second dimension.
constexpr int64_t GRID_ROWS = 1LL << 20;

// A matrix whose rows (one of its two strides is 1) can be read 16 bytes at
// a time; otherwise a copy that can, in the same orientation.
at::Tensor rows_of_16(const at::Tensor& t) {
  const int64_t step = 16 / t.element_size();
  const bool rows = t.stride(1) == 1 || t.size(1) == 1, cols = t.stride(0) == 1 || t.size(0) == 1;
  const bool aligned = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  if (aligned && rows && t.stride(1) == 1 && t.stride(0) % step == 0 && t.stride(0) >= t.size(1)) return t;
  if (aligned && cols && t.stride(0) == 1 && t.stride(1) % step == 0 && t.stride(1) >= t.size(0)) return t;
  const bool turn = !rows && cols;
  const at::Tensor v = turn ? t.t() : t;
  const int64_t ld = round_up(v.size(1), step);
  at::Tensor c = at::empty({v.size(0), ld}, t.options());
  copy_matrix(to_dtype(t), to_dtype(t), v.data_ptr(), v.stride(0), v.stride(1), c.data_ptr(), ld, v.size(0), v.size(1),
              ld, false, stream());
  const at::Tensor n = c.narrow(1, 0, v.size(1));
  return turn ? n.t() : n;
}

// An operand of the products: a matrix with one unit stride, as it is or
// (fp32 on the tensor cores) in three bf16 parts `pitch` apart.
struct Operand {
  const char* p;
  int64_t rows, cols, rs, cs;
  int64_t pitch = 0;
  at::ScalarType type;
  int64_t done = 0;  // of its columns (or, on the right, rows) before p
  Operand t() const { return {p, cols, rows, cs, rs, pitch, type, done}; }
};
// Rows [r0, r0 + n) of a row-major matrix with rows ld apart.
Operand rows_operand(const at::Tensor& t, int64_t r0, int64_t n, int64_t cols, int64_t ld) {
  return {static_cast<const char*>(t.data_ptr()) + r0 * ld * t.element_size(), n, cols, ld, 1, 0, t.scalar_type()};
}
Operand operand(const at::Tensor& t) {
  return {static_cast<const char*>(t.data_ptr()), t.size(0), t.size(1), t.stride(0), t.stride(1), 0, t.scalar_type()};
}
// Rows [r0, r0 + n) of the parts [.., 3 pitch] of a matrix.
Operand parts_operand(const at::Tensor& parts, int64_t r0, int64_t n, int64_t cols) {
  const int64_t pitch = parts.size(1) / 3;
  return {static_cast<const char*>(parts.data_ptr()) + r0 * 6 * pitch, n, cols, 3 * pitch, 1, pitch, at::kBFloat16};
}
// A row-major output, rows ld apart.
struct Out {
  char* p;
  int64_t rows, cols, ld;
  at::ScalarType type;
};
Out rows_out(const at::Tensor& t, int64_t r0, int64_t n, int64_t cols, int64_t ld) {
  return {static_cast<char*>(t.data_ptr()) + r0 * ld * t.element_size(), n, cols, ld, t.scalar_type()};
}
DType dtype_of(at::ScalarType t) { return t == at::kFloat ? DType::F32 : DType::BF16; }

// out (+)= scale * A B (+ bias per column), the sums in a fixed order.  With
// `before`, a bf16 out = the fp32 sum of that and the product, rounded once.
void product(const Operand& A, const Operand& B, const Out& out, const float* scale, bool accumulate,
             const at::TensorOptions& f32, const float* bias = nullptr, const Out* before = nullptr) {
  GemmArgs a;
  a.A = A.p;
  a.B = B.p;
  a.C = out.p;
  a.M = A.rows;
  a.K = A.cols;
  a.N = B.cols;
  a.sam = A.rs;
  a.sak = A.cs;
  a.sbk = B.rs;
  a.sbn = B.cs;
  a.ldc = out.ld;
  a.beta = accumulate ? 1.f : 0.f;
  a.bias = bias;
  a.bias_dtype = (int)DType::F32;
  a.ordered = true;
  a.parts = A.pitch > 0;
  a.pitch_a = A.pitch;
  a.pitch_b = B.pitch;
  const DType odt = dtype_of(out.type);
  if (before != nullptr) {
    a.residual = before->p;
    a.ldr = before->ld;
    a.residual_f32 = true;
  }
  if (a.parts && a.K > GEMM_PARTS_K) {  // pieces of K, each added to those before
    const int64_t piece = round_up(ceil_div(a.K, ceil_div(a.K, GEMM_PARTS_K)), 64);
    for (int64_t k = 0; k < A.cols; k += piece) {
      Operand x = A, w = B;
      x.p += 2 * k * A.cs;
      w.p += 2 * k * B.rs;
      x.cols = w.rows = std::min(piece, A.cols - k);
      x.done = w.done = k;
      product(x, w, out, scale, accumulate || k > 0, f32, k == 0 ? bias : nullptr);
    }
    return;
  }
  a.k_done = A.done;
  if (A.type == at::kBFloat16 && gemm_tc_supported(a)) {
    a.alpha_ptr = scale;
    const int64_t n = gemm_tc_workspace_floats(a, 0, odt);
    const at::Tensor ws = n > 0 ? at::empty({n}, f32) : at::Tensor();
    gemm_tc(odt, a, stream(), device_error_word(), 0, n > 0 ? ws.data_ptr<float>() : nullptr, n);
    return;
  }
  TORCH_INTERNAL_ASSERT(scale == nullptr && !a.parts && before == nullptr);
  if (A.type == at::kFloat && out.type == at::kFloat) {
    const float *pa = reinterpret_cast<const float*>(A.p), *pb = reinterpret_cast<const float*>(B.p);
    float* po = reinterpret_cast<float*>(out.p);
    if (A.rows <= FEW_ROWS && A.cols <= FEW_ROWS_K && A.cs == 1 && (B.cs == 1 || B.rs == 1) && !accumulate) {
      const bool turned = B.cs != 1;
      const int64_t n = few_rows_scratch_floats(A.rows, A.cols, B.cols, turned);
      const at::Tensor ws = n > 0 ? at::empty({n}, f32) : at::Tensor();
      few_rows_product(pa, A.rs, pb, turned ? B.cs : B.rs, turned, bias, po, out.ld, A.rows, A.cols, B.cols,
                       n > 0 ? ws.data_ptr<float>() : nullptr, stream());
      return;
    }
    if (A.cols <= FEW_ROWS && A.rs == 1 && B.cs == 1 && bias == nullptr) {
      few_rows_outer(pa, A.cs, pb, B.rs, po, out.ld, A.cols, A.rows, B.cols, accumulate, stream());
      return;
    }
  }
  for (int64_t r = 0; r < A.rows; r += GRID_ROWS) {  // more rows than a launch has blocks for
    a.M = std::min<int64_t>(GRID_ROWS, A.rows - r);
    a.A = A.p + r * A.rs * (int64_t)c10::elementSize(A.type);
    a.C = out.p + r * out.ld * (int64_t)c10::elementSize(out.type);
    const int64_t n = gemm_simt_workspace_floats(a);
    const at::Tensor ws = n > 0 ? at::empty({n}, f32) : at::Tensor();
    gemm_simt(dtype_of(A.type), odt, a, stream(), n > 0 ? ws.data_ptr<float>() : nullptr, n);
  }
}

// dst (+)= scale * A B.  On the tensor cores output rows that are no whole
// 16-byte steps go through a padded copy: the products store whole boxes.
// `room`: B's memory is this function's own and may be read up to its row pitch.
void product_into(const Operand& A, const Operand& B, const Out& dst, const float* scale, bool accumulate, bool room,
                  const at::TensorOptions& f32) {
  const int64_t step = 16 / (int64_t)c10::elementSize(dst.type);
  if (A.type == at::kFloat || (dst.ld % step == 0 && reinterpret_cast<uintptr_t>(dst.p) % 16 == 0)) {
    product(A, B, dst, scale, accumulate, f32);
    return;
  }
  const int64_t ld = round_up(dst.cols, step);
  const at::Tensor c = at::empty({dst.rows, ld}, f32.dtype(dst.type));
  // where B's rows have room for the padding, its columns too: whole steps all the way
  Operand b = B;
  if (room && B.cs == 1 && (B.pitch > 0 ? B.pitch : B.rs) >= ld) b.cols = ld;
  product(A, b, rows_out(c, 0, dst.rows, b.cols, ld), scale, false, f32);
  copy_matrix(dtype_of(dst.type), dtype_of(dst.type), c.data_ptr(), ld, 1, dst.p, dst.ld, dst.rows, dst.cols, dst.cols,
              accumulate, stream());
}

}  // namespace

// Rows of one block: `room` elements of [rows, classes] (rows of whole lines
// of 64), at least 2048 (every block reads and writes the fp32 sums of dW once:
// 8 bytes per element of W for 6 flops per row and element, 14% of the products'
// time at 2048) and at most GRID_ROWS, in equal blocks of whole tiles.
int64_t linear_ce_block_rows(int64_t rows, int64_t classes, int64_t room) {
  const int64_t most = std::min(GRID_ROWS, std::max<int64_t>(2048, room / round_up(classes, 64)));
  return std::min(rows, round_up(ceil_div(rows, ceil_div(rows, most)), 256));
}

LinearCeResult linear_ce_op(const at::Tensor& x, const at::Tensor& w, const at::Tensor& target,
                            c10::optional<at::Tensor> bias, int64_t ignore_index, bool mean, bool want_grad,
                            c10::optional<at::Tensor> grad_scale, c10::optional<at::Tensor> dw_out, bool dw_accumulate,
                            c10::optional<at::Tensor> db_out, bool db_accumulate, c10::optional<at::Tensor> correct,
                            c10::optional<at::Tensor> counted, c10::optional<at::Tensor> loss_sum) {
  check_cuda(x, "hidden");
  const at::Device dev = x.device();
  const auto dt = x.scalar_type();
  TORCH_CHECK(dt == at::kFloat || dt == at::kBFloat16, "dlvk.linear_ce: hidden is fp32 or bf16, got ", dt);
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && w.size(0) == x.size(1), "dlvk.linear_ce: hidden ", x.sizes(),
              " needs a weight [", x.dim() == 2 ? x.size(1) : -1, ", classes], got ", w.sizes());
  TORCH_CHECK(w.scalar_type() == dt && w.device() == dev, "dlvk.linear_ce: hidden is ", dt, " on ", dev,
              ", the weight ", w.scalar_type(), " on ", w.device());
  const int64_t N = x.size(0), E = x.size(1), V = w.size(1);
  TORCH_CHECK(E >= 1 && V >= 1, "dlvk.linear_ce: an empty weight ", w.sizes());
  TORCH_CHECK(N < (1LL << 31) - 256 && V < (1LL << 30) && E < (1LL << 31) - 64, "dlvk.linear_ce: sizes above 2^30");
  TORCH_CHECK((target.scalar_type() == at::kInt || target.scalar_type() == at::kLong) && target.device() == dev &&
                  target.dim() == 1 && target.size(0) == N,
              "dlvk.linear_ce: target must be int32 or int64 [", N, "] on ", dev, ", got ", target.scalar_type(), " ",
              target.sizes(), " on ", target.device());
  auto scalar = [&](const c10::optional<at::Tensor>& t, at::ScalarType st, const char* name) {
    TORCH_CHECK(!t.has_value() || (t->scalar_type() == st && t->numel() == 1 && t->device() == dev), "dlvk.linear_ce: ",
                name, " must be one ", st, " on ", dev);
  };
  scalar(grad_scale, at::kFloat, "grad_scale");
  scalar(correct, at::kLong, "correct");
  scalar(counted, at::kLong, "counted");
  scalar(loss_sum, at::kFloat, "loss_sum");
  if (bias.has_value())
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == V && bias->device() == dev &&
                    (bias->scalar_type() == at::kFloat || bias->scalar_type() == at::kBFloat16),
                "dlvk.linear_ce: bias must be fp32 or bf16 [", V, "] on ", dev);
  if (dw_out.has_value())
    TORCH_CHECK(dw_out->sizes() == w.sizes() && dw_out->device() == dev && (dw_out->stride(1) == 1 || V == 1 ||
                dw_out->stride(0) == 1 || E == 1) &&
                    (dw_out->scalar_type() == at::kFloat || (dw_out->scalar_type() == dt && !dw_accumulate)),
                "dlvk.linear_ce: the weight gradient must be fp32 (or, overwritten, of the weight's type) ", w.sizes(),
                " with one unit stride on ", dev);
  if (dw_out.has_value()) {
    const int64_t se = dw_out->stride(0), sv = dw_out->stride(1);
    TORCH_CHECK((V == 1 || sv >= 1) && (E == 1 || se >= 1) && (V == 1 || E == 1 || sv + se > (sv == 1 ? V : E)),
                "dlvk.linear_ce: the weight gradient repeats its elements, strides ", dw_out->strides());
  }
  // blocks of rows write the gradients before the next ones read the operands
  const auto apart = [&](const c10::optional<at::Tensor>& t) {
    if (!t.has_value()) return;
    at::assert_no_overlap(*t, w);
    at::assert_no_overlap(*t, x);
    at::assert_no_overlap(*t, target);
    if (bias.has_value()) at::assert_no_overlap(*t, *bias);
  };
  apart(dw_out);
  apart(db_out);
  if (dw_out.has_value() && db_out.has_value()) at::assert_no_overlap(*dw_out, *db_out);
  if (db_out.has_value())
    TORCH_CHECK(bias.has_value() && db_out->scalar_type() == at::kFloat && db_out->is_contiguous() &&
                    db_out->numel() == V && db_out->device() == dev,
                "dlvk.linear_ce: the bias gradient must be contiguous fp32 [", V, "] on ", dev);
  c10::cuda::CUDAGuard g(dev);
  const PdlScope pdl;  // each launch starts up while the one before it ends
  at::AutoDispatchBelowADInplaceOrView below;  // no autograd bookkeeping for what follows
  const auto f32 = x.options().dtype(at::kFloat);
  const bool bf = dt == at::kBFloat16;

  LinearCeResult out;
  out.loss = at::empty({}, f32);
  out.rows = at::empty({N}, f32);
  if (want_grad) {
    out.dx = at::empty({N, E}, x.options());
    if (dw_out.has_value()) out.dw = *dw_out;
    else out.dw = (w.stride(1) == 1 || w.stride(0) != 1) ? at::empty({E, V}, w.options())
                                                         : at::empty({V, E}, w.options()).t();
    if (bias.has_value()) out.dbias = db_out.has_value() ? *db_out : at::empty({V}, f32);
  }
  if (N == 0) {
    out.loss.zero_();
    if (want_grad && !dw_accumulate) out.dw.zero_();
    if (want_grad && bias.has_value() && !db_accumulate) out.dbias.zero_();
    return out;
  }

  const at::Tensor tc = target.contiguous();
  at::Tensor bc = bias.has_value() ? bias->to(at::kFloat).contiguous() : at::Tensor();
  if (bc.defined() && !bf && V % 4 != 0) {  // room for whole 16-byte steps
    const at::Tensor padded = at::empty({round_up(V, 4)}, f32);
    copy_matrix(DType::F32, DType::F32, bc.data_ptr(), V, 1, padded.data_ptr(), padded.size(0), 1, V, padded.size(0),
                false, stream());
    bc = padded;
  }
  const float* biasp = bc.defined() ? bc.data_ptr<float>() : nullptr;
  const CeRows all{N, V, ignore_index, tc.data_ptr(), tc.scalar_type() == at::kLong};
  at::Tensor xq, wq;
  bool w_k;  // classes are rows: W^T is what memory holds
  CeProjection c;
  // fp32 operands of some size run as six products of bf16 parts; few rows read
  // the weight as it is, and a small or narrow product, which would be mostly
  // padding, stays on the SIMT kernel
  const bool parts = !bf && fp32_gemm_mode() != 0 && N > FEW_ROWS && E >= 16 && V >= 64 &&
                     (double)N * E * V >= 4194304.0;
  if (parts) {
    const at::Tensor xs = x.stride(1) == 1 ? x : x.contiguous();
    const at::Tensor wr = (w.stride(0) == 1 || w.stride(1) == 1) ? w : w.contiguous();
    w_k = wr.stride(1) != 1;
    const at::Tensor wm = w_k ? wr.t() : wr;  // rows of unit stride
    const auto b16 = x.options().dtype(at::kBFloat16);
    const int64_t ep = round_up(E, 64), wp = round_up(wm.size(1), 64);
    xq = at::empty({N, 3 * ep}, b16);
    wq = at::empty({w_k ? round_up(V, 4) : E, 3 * wp}, b16);
    // rows that do not count are zeros, whatever they hold (see x_clean below)
    split_parts(xs.data_ptr<float>(), xs.stride(0), N, E, reinterpret_cast<__nv_bfloat16*>(xq.data_ptr()), ep, &all,
                stream());
    split_parts(wm.data_ptr<float>(), wm.stride(0), wm.size(0), wm.size(1),
                reinterpret_cast<__nv_bfloat16*>(wq.data_ptr()), wp, nullptr, stream());
    c.parts = true;
    c.pitch_x = ep;
    c.pitch_w = wp;
    c.ldx = 3 * ep;
    c.ldw = 3 * wp;
  } else {
    wq = (w.stride(0) == 1 || w.stride(1) == 1) ? w : w.contiguous();
    xq = x.stride(1) == 1 ? x : x.contiguous();  // the products read x by rows
    if (bf) {
      wq = rows_of_16(wq);
      xq = rows_of_16(xq);
      if (xq.stride(1) != 1) xq = rows_of_16(xq.contiguous());
    }
    w_k = wq.stride(1) != 1;
    c.ldx = xq.stride(0);
    c.ldw = w_k ? wq.stride(1) : wq.stride(0);
  }
  Operand wo = operand(wq);  // [E, V]
  if (parts) {
    wo = parts_operand(wq, 0, w_k ? V : E, w_k ? E : V);
    if (w_k) wo = wo.t();
  }
  c.x = reinterpret_cast<const __nv_bfloat16*>(xq.data_ptr());
  c.w = reinterpret_cast<const __nv_bfloat16*>(wq.data_ptr());
  c.rows = N;
  c.width = E;
  c.classes = V;
  c.w_k = w_k;
  c.bias = biasp;
  c.labels64 = all.labels64;
  c.ignore = ignore_index;
  // Where the logits are: in the accumulators (bf16, and the loss alone of
  // fp32 parts), else a block of them in memory as fp32.
  const bool tc_ok = (bf || parts) && E >= 16 && ce_tc_supported(c);
  // (fp32: while one accumulator may hold the whole width, which the epilogue
  // that reduces the logits does not split)
  const bool fused = tc_ok && (bf || (!want_grad && E <= GEMM_PARTS_ACC));
  const bool keep = fused && want_grad && !bias.has_value();  // exponentials kept, not made again

  // Room for 256 MB of a block's exponentials (2 bytes), or logits that become
  // gradients (4), of which linear_ce_block_rows() takes at least 2048 rows: with
  // V words max(256 MB, 2048 V times that).  fp32 gradients in parts are 6 bytes
  // a logit beside it, x and W in parts 6 bytes an element, and the split sums of
  // a product up to 32 of its outputs.  The loss alone keeps the statistics, 8
  // bytes for 128 logits, on the tensor cores.
  const int64_t rows = linear_ce_block_rows(N, V, !fused ? (64LL << 20) : want_grad ? (128LL << 20) : (1LL << 30));
  const int64_t blocks = ceil_div(N, rows);
  const auto stat_cols_of = [&](int64_t n) { return fused ? ce_tc_stat_cols(n, V, parts) : ce_memory_stat_cols(n, V); };
  // a last, smaller block may be cut into more statistics for each of fewer rows
  int64_t stat_room = rows * stat_cols_of(rows);
  if (N % rows != 0) stat_room = std::max<int64_t>(stat_room, N % rows * stat_cols_of(N % rows));
  const int groups = (int)ceil_div(N, 32), lab_size = c.labels64 ? 8 : 4;
  // scratch: 8-byte items first (sums, statistics, norms), then floats, then the counter
  const at::Tensor ws = at::empty({6LL * groups + 2 * stat_room + 3 * rows + 2}, f32);
  double* partial = reinterpret_cast<double*>(ws.data_ptr<float>());
  float2* stats = reinterpret_cast<float2*>(ws.data_ptr<float>() + 6LL * groups);
  float2* norm = stats + stat_room;
  float* zlabel = reinterpret_cast<float*>(norm + rows);
  float* gscale = zlabel + rows;
  unsigned* done = reinterpret_cast<unsigned*>(gscale + 1);
  const float* gsp = grad_scale.has_value() ? grad_scale->data_ptr<float>() : nullptr;
  c.stats = stats;
  c.zlabel = zlabel;
  c.norm = norm;
  c.gscale = gscale;

  // rows of whole 128-byte lines: a box of the tiles' stores is one line a row
  const int64_t ldv = round_up(V, 64), vp = ldv;
  const int64_t ldx = round_up(E, 16 / x.element_size());
  at::Tensor z, dl, xc, part, dw32;
  if (!fused) z = at::empty({rows, ldv}, f32);
  bool dw_k = false;
  if (want_grad) {
    dl = parts ? at::empty({rows, 3 * vp}, xq.options()) : bf ? at::empty({rows, ldv}, x.options()) : z;
    // dW = x^T dz reads x once more, with zeros in the rows that do not count:
    // their dz is 0, but 0 times an infinity or NaN left there would not be.
    if (!parts) xc = at::empty({rows, ldx}, x.options());
    dw_k = out.dw.stride(1) != 1 && V > 1;  // the gradient's rows are classes too
    // sums over several blocks are fp32 until the last
    if (blocks > 1 && out.dw.scalar_type() != at::kFloat)
      dw32 = dw_k ? at::empty({V, round_up(E, 4)}, f32).narrow(1, 0, E).t()
                  : at::empty({E, round_up(V, 4)}, f32).narrow(1, 0, V);
    if (out.dbias.defined()) part = at::empty({fused ? ceil_div(rows, 32) * V : ldv}, f32);
  }
  const auto dw_rows = [&](const at::Tensor& t) {  // [E, V], or of classes by width (dw_k)
    return Out{static_cast<char*>(t.data_ptr()), dw_k ? V : E, dw_k ? E : V, dw_k ? t.stride(1) : t.stride(0),
               t.scalar_type()};
  };
  Out dw{}, dw_last{};
  if (want_grad) dw = dw_last = dw_rows(dw32.defined() ? dw32 : out.dw);
  // the last of several blocks adds to the others' sums and rounds, where its output has whole 16-byte rows
  bool round_last = false;
  if (dw32.defined()) {
    const Out o = dw_rows(out.dw);
    round_last = fused && o.ld % 8 == 0 && reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && dw.cols >= 16;
    if (round_last) dw_last = o;
  }
  if (blocks > 1) ce_count(all, mean, gsp, gscale, done, stream());

  for (int64_t k = 0; k < blocks; ++k) {
    const int64_t r0 = k * rows, n = std::min(rows, N - r0);
    CeRows r = all;
    r.rows = n;
    r.labels = static_cast<const char*>(tc.data_ptr()) + r0 * lab_size;
    Operand xo = parts ? parts_operand(xq, r0, n, E) : rows_operand(xq, r0, n, E, xq.stride(0));
    c.rows = n;
    c.x = reinterpret_cast<const __nv_bfloat16*>(xo.p);
    c.labels = r.labels;
    c.done = blocks == 1 ? done : nullptr;
    if (keep) {
      ce_exp_tc(c, dl.data_ptr(), ldv, stream(), device_error_word());
    } else if (fused) {
      ce_stats_tc(c, stream(), device_error_word());
    } else {
      // parts: columns up to whole 16-byte steps, which wq and the bias have room for
      Operand wl = wo;
      if (parts) wl.cols = round_up(V, 4);
      product(xo, wl, rows_out(z, 0, n, wl.cols, ldv), nullptr, false, f32, biasp);
      ce_memory_stats(r, z.data_ptr<float>(), ldv, stats, zlabel, c.done, stream());
    }
    CeFinish f{};
    f.stats = stats;
    f.stat_cols = stat_cols_of(n);
    f.zlabel = zlabel;
    f.rows_loss = out.rows.data_ptr<float>() + r0;
    f.norm = norm;
    f.mean = mean;
    f.set_gscale = blocks == 1;
    f.grad_scale = gsp;
    f.loss = out.loss.data_ptr<float>();
    f.gscale = gscale;
    f.loss_sum = loss_sum.has_value() ? loss_sum->data_ptr<float>() : nullptr;
    f.counted = counted.has_value() ? reinterpret_cast<unsigned long long*>(counted->data_ptr<int64_t>()) : nullptr;
    f.correct = correct.has_value() ? reinterpret_cast<unsigned long long*>(correct->data_ptr<int64_t>()) : nullptr;
    f.partial = partial;
    f.done = done;
    f.first_group = (int)(r0 / 32);  // blocks are whole tiles, the last apart
    f.total_groups = groups;
    if (xc.defined()) {
      f.x = xo.p;
      f.ldx = xo.rs;
      f.width = E;
      f.x_clean = xc.data_ptr();
      f.ldc = ldx;
      xo = rows_operand(xc, 0, n, E, ldx);
    }
    const bool join = keep && ce_rescale_joins(n, V, f.stat_cols);
    if (!join) ce_finish(r, f, to_dtype(x), stream());
    if (!want_grad) continue;

    const Operand d = parts ? parts_operand(dl, 0, n, V) : rows_operand(dl, 0, n, V, ldv);
    const float* scale = gscale;  // dz holds softmax - onehot, the products its factor
    if (keep) {
      ce_rescale(r, f, ce_tc_stat_width(n, V), join, dl.data_ptr(), ldv, stream());
    } else if (fused) {
      ce_grad_tc(c, reinterpret_cast<__nv_bfloat16*>(dl.data_ptr()), ldv,
                 part.defined() ? part.data_ptr<float>() : nullptr, stream(), device_error_word());
      if (part.defined())
        colsum_partials(part.data_ptr<float>(), ceil_div(n, 32), V, 1.f, out.dbias.data_ptr<float>(),
                        db_accumulate || k > 0, stream());
    } else {
      ce_memory_grad(r, z.data_ptr<float>(), ldv, norm, gscale,
                     dl.is_same(z) ? nullptr : reinterpret_cast<__nv_bfloat16*>(dl.data_ptr()), parts ? vp : 0,
                     !parts || part.defined(), stream());
      if (!parts) scale = nullptr;  // these carry it
      if (part.defined()) {  // the padding's columns are summed too and left out of the copy
        const int64_t ns = colsum_scratch_floats(n, ldv);
        const at::Tensor scr = ns > 0 ? at::empty({ns}, f32) : at::Tensor();
        colsum(DType::F32, DType::F32, z.data_ptr(), n, ldv, 1.f, part.data_ptr<float>(), false,
               ns > 0 ? scr.data_ptr<float>() : nullptr, stream());
        copy_matrix(DType::F32, DType::F32, part.data_ptr(), 0, 1, out.dbias.data_ptr<float>(), V, 1, V, V,
                    db_accumulate || k > 0, stream());
      }
    }
    product_into(d, wo.t(), rows_out(out.dx, r0, n, E, E), scale, false, !wq.is_same(w), f32);
    const Operand left = dw_k ? d.t() : xo.t(), right = dw_k ? xo : d;
    if (round_last && k == blocks - 1) product(left, right, dw_last, scale, false, f32, nullptr, &dw);
    else product_into(left, right, dw, scale, dw32.defined() ? k > 0 : (dw_accumulate || k > 0), true, f32);
  }
  if (dw32.defined() && !round_last) {
    const at::Tensor src = dw_k ? dw32.t() : dw32, dst = dw_k ? out.dw.t() : out.dw;
    copy_matrix(to_dtype(dst), DType::F32, src.data_ptr(), src.stride(0), 1, dst.data_ptr(), dst.stride(0),
                dst.size(0), dst.size(1), dst.size(1), false, stream());
  }
  return out;
}

}  // namespace aten
}  // namespace dlvk
