// ATen-level softmax cross entropy of a vocabulary projection: loss and
// gradients from x [rows, width] and W [width, classes] without an array of
// logits (gemm_tc.cu EPI 3 / 4, vocab_loss.cu).
#include <ATen/ATen.h>
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

// An operand of the products: an fp32 one with its two TF32 parts where the
// products run on the tensor cores (three of them: 3xTF32), made once.
struct Operand {
  at::Tensor v, hi, lo;
  Operand t() const { return hi.defined() ? Operand{v.t(), hi.t(), lo.t()} : Operand{v.t(), {}, {}}; }
  Operand columns(int64_t at, int64_t n) const {
    return hi.defined() ? Operand{v.narrow(1, at, n), hi.narrow(1, at, n), lo.narrow(1, at, n)}
                        : Operand{v.narrow(1, at, n), {}, {}};
  }
};

// `t` (one unit stride, rows of whole 16-byte steps) and its parts.
Operand split(const at::Tensor& t) {
  const bool turn = t.stride(1) != 1;
  at::Tensor v = turn ? t.t() : t;
  const int64_t rows = v.size(0), cols = v.size(1), ld = round_up(cols, 4);
  if (v.stride(0) != ld) {  // gaps between the rows: the parts are made of a dense copy
    const at::Tensor c = at::empty({rows, ld}, t.options());
    copy_matrix(DType::F32, DType::F32, v.data_ptr(), v.stride(0), 1, c.data_ptr(), ld, rows, cols, ld, false, stream());
    v = c.narrow(1, 0, cols);
  }
  // the last row's padding may lie past the end of t's memory: split up to its last element
  const int64_t n = (rows - 1) * ld + cols;
  const at::Tensor hi = at::empty({rows, ld}, t.options()), lo = at::empty({rows, ld}, t.options());
  tf32_split(v.data_ptr<float>(), hi.data_ptr<float>(), lo.data_ptr<float>(), n, stream());
  const Operand o{t, hi.narrow(1, 0, cols), lo.narrow(1, 0, cols)};
  return turn ? Operand{t, o.hi.t(), o.lo.t()} : o;
}

constexpr double kTf32Macs = 67108864.0;  // as gemm_op: smaller products stay on the SIMT kernel

// out (+)= A B (+ bias per column), sums in a fixed order.
void product(const Operand& A, const Operand& B, const at::Tensor& out, bool accumulate,
             const c10::optional<at::Tensor>& bias = c10::nullopt) {
  const double macs = (double)out.size(0) * out.size(1) * A.v.size(1);
  if (A.hi.defined() && B.hi.defined() && macs >= kTf32Macs) {
    GemmArgs ll = fill_args(A.lo, B.hi, out), lh = fill_args(A.hi, B.lo, out), hh = fill_args(A.hi, B.hi, out);
    if (gemm_tf32_tc_supported(ll) && gemm_tf32_tc_supported(lh) && gemm_tf32_tc_supported(hh)) {
      if (bias.has_value()) hh.bias = bias->data_ptr();
      int pass = 0;
      for (GemmArgs* a : {&ll, &lh, &hh}) {  // the small terms first
        a->ordered = true;
        a->beta = (pass++ > 0 || accumulate) ? 1.f : 0.f;
        const int64_t n = gemm_tc_workspace_floats(*a, 0, DType::F32, true);
        const at::Tensor ws = n > 0 ? at::empty({n}, out.options()) : at::Tensor();
        gemm_tf32_tc(DType::F32, *a, stream(), device_error_word(), 0, n > 0 ? ws.data_ptr<float>() : nullptr, n);
      }
      return;
    }
  }
  const bool simt = A.v.scalar_type() == at::kFloat && fp32_gemm_mode() != 1;
  gemm_op(A.v, B.v, bias, ACT_NONE, 1.0, accumulate ? 1.0 : 0.0, out, c10::nullopt, simt ? 2 : 0, 0, c10::nullopt,
          c10::nullopt, c10::nullopt, 1.0, false, c10::nullopt, c10::nullopt, true);
}

// dst (+)= A B.  Output rows that are no whole 16-byte steps go through a
// padded copy: the products store whole boxes.
void product_into(const Operand& A, const Operand& B, const at::Tensor& dst, bool accumulate) {
  const int64_t n = dst.size(1), step = 16 / dst.element_size();
  if (dst.stride(0) % step == 0 && reinterpret_cast<uintptr_t>(dst.data_ptr()) % 16 == 0) {
    product(A, B, dst, accumulate);
    return;
  }
  const at::Tensor c = at::empty({dst.size(0), round_up(n, step)}, dst.options());
  product(A, B, c.narrow(1, 0, n), false);
  copy_matrix(to_dtype(dst), to_dtype(c), c.data_ptr(), c.size(1), 1, dst.data_ptr(), dst.stride(0), dst.size(0), n, n,
              accumulate, stream());
}

// Classes of one piece of the gradient: `room` elements of [rows, piece], at
// least 4096, in equal pieces of whole tiles.  A larger piece costs memory, a
// smaller one another pass over the fp32 sums of dx.
int64_t piece_of(int64_t rows, int64_t classes, int64_t room) {
  const int64_t most = std::max<int64_t>(4096, room / std::max<int64_t>(rows, 1));
  return std::min(round_up(ceil_div(classes, ceil_div(classes, most)), 256), round_up(classes, 256));
}

}  // namespace

LinearCeResult linear_ce_op(const at::Tensor& x, const at::Tensor& w, const at::Tensor& target,
                            c10::optional<at::Tensor> bias, int64_t ignore_index, bool mean, bool want_grad,
                            c10::optional<at::Tensor> grad_scale, c10::optional<at::Tensor> dw_out, bool dw_accumulate,
                            c10::optional<at::Tensor> db_out, bool db_accumulate, c10::optional<at::Tensor> correct) {
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
  if (db_out.has_value())
    TORCH_CHECK(bias.has_value() && db_out->scalar_type() == at::kFloat && db_out->is_contiguous() &&
                    db_out->numel() == V && db_out->device() == dev,
                "dlvk.linear_ce: the bias gradient must be contiguous fp32 [", V, "] on ", dev);
  c10::cuda::CUDAGuard g(dev);
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
  const at::Tensor bc = bias.has_value() ? bias->to(at::kFloat).contiguous() : at::Tensor();
  at::Tensor xq = rows_of_16(x);
  if (xq.stride(1) != 1) xq = rows_of_16(x.contiguous());  // the products read x by rows
  at::Tensor wq = rows_of_16((w.stride(0) == 1 || w.stride(1) == 1) ? w : w.contiguous());
  const bool w_k = wq.stride(1) != 1;  // classes are rows: W^T is what memory holds

  CeProjection c;
  if (bf) {
    c.x = reinterpret_cast<const __nv_bfloat16*>(xq.data_ptr());
    c.w = reinterpret_cast<const __nv_bfloat16*>(wq.data_ptr());
  }
  c.rows = N;
  c.width = E;
  c.classes = V;
  c.ldx = xq.stride(0);
  c.ldw = w_k ? wq.stride(1) : wq.stride(0);
  c.w_k = w_k;
  c.bias = bc.defined() ? bc.data_ptr<float>() : nullptr;
  c.labels = tc.data_ptr();
  c.labels64 = tc.scalar_type() == at::kLong;
  c.ignore = ignore_index;
  CeRows r{N, V, ignore_index, c.labels, c.labels64};
  const bool tensor = bf && ce_tc_supported(c);  // else the logits of one piece at a time in memory

  const int64_t piece = piece_of(N, V, tensor ? (128 << 20) : (64 << 20));
  const int64_t pieces = ceil_div(V, piece);
  const int stat_cols = tensor ? ce_tc_stat_cols(N, V) : (int)pieces;
  const int64_t blocks = ceil_div(N, 32);
  // scratch: 8-byte items first (sums, statistics), then floats, then the counter
  const at::Tensor ws = at::empty({6 * blocks + 2 * N * stat_cols + 3 * N + 2}, f32);
  double* partial = reinterpret_cast<double*>(ws.data_ptr<float>());
  float2* stats = reinterpret_cast<float2*>(ws.data_ptr<float>() + 6 * blocks);
  float2* norm = stats + N * stat_cols;
  float* zlabel = reinterpret_cast<float*>(norm + N);
  float* gscale = zlabel + N;
  unsigned* done = reinterpret_cast<unsigned*>(gscale + 1);
  c.stats = stats;
  c.zlabel = zlabel;
  c.norm = norm;
  c.gscale = gscale;
  c.done = done;

  const bool parts = !bf && fp32_gemm_mode() == 3 && (double)N * E * V >= kTf32Macs;
  const Operand xo = parts ? split(xq) : Operand{xq, {}, {}}, wo = parts ? split(wq) : Operand{wq, {}, {}};
  at::Tensor z;  // fp32 logits of a piece, where they do go through memory
  auto logits = [&](int64_t col0, int64_t n) {
    const at::Tensor zn = z.narrow(1, 0, n);
    product(xo, wo.columns(col0, n), zn, false,
            bc.defined() ? c10::optional<at::Tensor>(bc.narrow(0, col0, n)) : c10::nullopt);
  };
  if (tensor) {
    ce_stats_tc(c, stream(), device_error_word());
  } else {
    z = at::empty({N, piece}, f32);
    for (int64_t k = 0; k < pieces; ++k) {
      const int64_t col0 = k * piece, n = std::min(piece, V - col0);
      logits(col0, n);
      ce_piece_stats(r, z.data_ptr<float>(), piece, col0, n, stats + k * N, zlabel, done, stream());
    }
  }
  // dW = x^T dz reads x once more, with zeros in the rows that do not count:
  // their dz is 0, but 0 times an infinity or NaN left there would not be.
  at::Tensor xc;
  if (want_grad) {
    const int64_t ld = round_up(E, 16 / x.element_size());
    xc = at::empty({N, ld}, x.options()).narrow(1, 0, E);
  }
  ce_finish(r, stats, stat_cols, zlabel, out.rows.data_ptr<float>(), norm, mean,
            grad_scale.has_value() ? grad_scale->data_ptr<float>() : nullptr, out.loss.data_ptr<float>(), gscale,
            correct.has_value() ? reinterpret_cast<unsigned long long*>(correct->data_ptr<int64_t>()) : nullptr, partial,
            done, to_dtype(x), xq.data_ptr(), xq.stride(0), E, xc.defined() ? xc.data_ptr() : nullptr,
            xc.defined() ? xc.stride(0) : 0, stream());
  if (!want_grad) return out;

  const Operand xco = parts ? split(xc) : Operand{xc, {}, {}};
  const bool dw_k = out.dw.stride(1) != 1 && V > 1;  // the gradient's rows are classes too
  at::Tensor dl = bf ? at::empty({N, piece}, x.options()) : z;
  at::Tensor sum;  // dx of several pieces, fp32
  if (pieces > 1) sum = at::empty({N, E}, f32);
  at::Tensor part;
  if (out.dbias.defined()) part = at::empty({tensor ? blocks * piece : piece}, f32);
  for (int64_t k = 0; k < pieces; ++k) {
    const int64_t col0 = k * piece, n = std::min(piece, V - col0);
    if (tensor) {
      ce_grad_tc(c, (int)col0, (int)n, reinterpret_cast<__nv_bfloat16*>(dl.data_ptr()), piece,
                 part.defined() ? part.data_ptr<float>() : nullptr, stream(), device_error_word());
      if (part.defined())
        colsum_partials(part.data_ptr<float>(), blocks, n, 1.f, out.dbias.data_ptr<float>() + col0, db_accumulate,
                        stream());
    } else {
      if (pieces > 1) logits(col0, n);
      ce_piece_grad(r, z.data_ptr<float>(), piece, col0, n, norm, gscale,
                    bf ? reinterpret_cast<__nv_bfloat16*>(dl.data_ptr()) : nullptr, stream());
      if (part.defined()) {  // the columns past n are left over from nothing: only n of the sums are kept
        const int64_t ns = colsum_scratch_floats(N, piece);
        const at::Tensor scr = ns > 0 ? at::empty({ns}, f32) : at::Tensor();
        colsum(DType::F32, DType::F32, z.data_ptr(), N, piece, 1.f, part.data_ptr<float>(), false,
               ns > 0 ? scr.data_ptr<float>() : nullptr, stream());
        copy_matrix(DType::F32, DType::F32, part.data_ptr(), 0, 1, out.dbias.data_ptr<float>() + col0, n, 1, n, n,
                    db_accumulate, stream());
      }
    }
    const Operand d = parts ? split(dl.narrow(1, 0, n)) : Operand{dl.narrow(1, 0, n), {}, {}};
    const Operand wp = wo.columns(col0, n);
    if (pieces == 1) product_into(d, wp.t(), out.dx, false);
    else product_into(d, wp.t(), sum, k > 0);
    const at::Tensor dwp = out.dw.narrow(1, col0, n);
    if (dw_k) product_into(d.t(), xco, dwp.t(), dw_accumulate);
    else product_into(xco.t(), d, dwp, dw_accumulate);
  }
  if (pieces > 1) unary(DType::F32, to_dtype(x), sum.data_ptr(), out.dx.data_ptr(), N * E, UN_COPY, 0.f, 0.f, stream());
  return out;
}

}  // namespace aten
}  // namespace dlvk
