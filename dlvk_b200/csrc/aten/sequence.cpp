// ATen-level wrappers of the operators over sequences with a state (short
// causal convolution, selective state space scan) and of the choice of the next
// word (declared in dlvk/aten_ops.h).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "dlvk/aten_ops.h"
#include "dlvk/kernels.h"
#include "dlvk/overlap.h"

namespace dlvk {
namespace aten {
namespace {

using OptTensor = c10::optional<at::Tensor>;

// What the tensors of one call have in common.  `one`: a token of each sequence,
// whose tensors have no dimension of tokens.
struct Call {
  const char* what;
  at::Device device;
  at::ScalarType type;
  int64_t B, T, D;
  bool one = false;
};

Call call_of(const at::Tensor& x, const char* what, const char* name, bool one) {
  TORCH_CHECK(x.is_cuda(), "dlvk.", what, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(x.dim() == (one ? 2 : 3), "dlvk.", what, ": ", name, one ? " is [sequences, channels], got " :
              " is [sequences, tokens, channels], got ", x.sizes());
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, "dlvk.", what, ": ", name,
              " is fp32 or bf16, got ", x.scalar_type());
  const int64_t D = x.size(one ? 1 : 2);
  TORCH_CHECK(D < (1LL << 31) - 4096, "dlvk.", what, ": ", D, " channels");
  return {what, x.device(), x.scalar_type(), x.size(0), one ? 1 : x.size(1), D, one};
}

// Sizes [B, T, rest...], without T for one token.
using Sizes = c10::SmallVector<int64_t, 4>;
Sizes sizes_of(const Call& c, std::initializer_list<int64_t> rest) {
  Sizes s{c.B};
  if (!c.one) s.push_back(c.T);
  s.append(rest.begin(), rest.end());
  return s;
}

void check(const Call& c, const at::Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef sizes) {
  TORCH_CHECK(t.device() == c.device, "dlvk.", c.what, ": ", name, " is on ", t.device(), ", the call on ", c.device);
  TORCH_CHECK(t.scalar_type() == type, "dlvk.", c.what, ": ", name, " is ", t.scalar_type(), ", expected ", type);
  TORCH_CHECK(t.layout() == at::kStrided, "dlvk.", c.what, ": ", name, " is not strided");
  TORCH_CHECK(t.sizes() == sizes, "dlvk.", c.what, ": ", name, " is ", t.sizes(), ", expected ", sizes);
}

// Whether what follows the tokens (channels, or groups of states) is one run.
bool runs(const Call& c, const at::Tensor& t) {
  const int64_t d = t.dim(), groups = c.one ? 1 : 2;
  return t.numel() == 0 || ((t.size(d - 1) <= 1 || t.stride(d - 1) == 1) &&
                            (d <= groups + 1 || t.size(groups) <= 1 || t.stride(groups) == t.size(groups + 1)));
}
SeqRef ref(const Call& c, const at::Tensor& t) { return {t.data_ptr(), t.stride(0), c.one ? 0 : t.stride(1)}; }

// A tensor that is read; a copy where its rows are no runs.  `keep` holds it.
SeqRef read(const Call& c, const at::Tensor& t, const char* name, std::initializer_list<int64_t> rest, at::Tensor& keep) {
  check(c, t, name, c.type, sizes_of(c, rest));
  keep = runs(c, t) ? t : t.contiguous();
  return ref(c, keep);
}

const float* read_param(const Call& c, const OptTensor& t, const char* name, at::IntArrayRef sizes, at::Tensor& keep) {
  if (!t.has_value()) return nullptr;
  check(c, *t, name, at::kFloat, sizes);
  keep = t->contiguous();
  return keep.data_ptr<float>();
}

const int32_t* read_lengths(const Call& c, const OptTensor& t, at::Tensor& keep) {
  if (!t.has_value()) return nullptr;
  check(c, *t, "lengths", at::kInt, {c.B});
  keep = t->contiguous();
  return keep.data_ptr<int32_t>();
}

// A tensor that is written: given by the caller, or a new one.
at::Tensor written(const Call& c, const OptTensor& out, const char* name, at::ScalarType type, at::IntArrayRef sizes) {
  if (!out.has_value()) return at::empty(sizes, at::TensorOptions().dtype(type).device(c.device));
  check(c, *out, name, type, sizes);
  TORCH_CHECK(!may_repeat(*out), "dlvk.", c.what, ": ", name, " repeats its elements (an expanded tensor)");
  return *out;
}
SeqRef written_rows(const Call& c, const at::Tensor& t, const char* name) {
  TORCH_CHECK(runs(c, t), "dlvk.", c.what, ": ", name, " needs a contiguous last dimension");
  return ref(c, t);
}
// The convolution's state [B, taps - 1, D], whatever the call's tensors have.
SeqRef conv_state(const Call& c, const at::Tensor& t, int64_t taps, const char* name, bool write, at::Tensor& keep) {
  check(c, t, name, c.type, {c.B, taps - 1, c.D});
  const bool rows = t.numel() == 0 || c.D <= 1 || t.stride(2) == 1;
  TORCH_CHECK(rows || !write, "dlvk.", c.what, ": ", name, " needs a contiguous last dimension");
  TORCH_CHECK(!write || !may_repeat(t), "dlvk.", c.what, ": ", name, " repeats its elements (an expanded tensor)");
  keep = rows ? t : t.contiguous();
  return {keep.data_ptr(), keep.stride(0), keep.stride(1)};
}
float* written_param(const Call& c, const OptTensor& t, const char* name, at::IntArrayRef sizes) {
  if (!t.has_value()) return nullptr;
  check(c, *t, name, at::kFloat, sizes);
  TORCH_CHECK(t->is_contiguous(), "dlvk.", c.what, ": ", name, " must be contiguous");
  return t->data_ptr<float>();
}
bool share(const at::Tensor& a, const at::Tensor& b) {
  return a.defined() && b.defined() && a.numel() > 0 && b.numel() > 0 && share_bytes(extent_of(a, 0), extent_of(b, 0));
}
// What is written lies apart from the other outputs and from what is read.
void apart(const Call& c, const std::vector<at::Tensor>& out, const std::vector<at::Tensor>& in) {
  for (size_t i = 0; i < out.size(); ++i) {
    for (size_t j = 0; j < i; ++j)
      TORCH_CHECK(!share(out[i], out[j]), "dlvk.", c.what, ": two outputs share memory");
    for (const at::Tensor& t : in)
      TORCH_CHECK(!share(out[i], t), "dlvk.", c.what, ": an output shares memory with an operand");
  }
}
// A state moves on in place, or into memory apart from it.
void in_place_or_apart(const Call& c, const at::Tensor& out, const at::Tensor& state) {
  const bool same = state.defined() && out.data_ptr() == state.data_ptr() && out.strides() == state.strides();
  TORCH_CHECK(same || !share(out, state), "dlvk.", c.what, ": out_state lies partly on state");
}

struct Conv {
  Call call;
  ShortConv a;
  at::Tensor x, weight, bias, state, lengths;
};
Conv conv_of(const char* what, const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
             const OptTensor& state, const OptTensor& lengths, bool silu, bool one = false) {
  Conv v{call_of(x, what, "x", one), {}, {}, {}, {}, {}, {}};
  const Call& c = v.call;
  TORCH_CHECK(weight.dim() == 2 && weight.size(1) >= 2 && weight.size(1) <= 4, "dlvk.", what,
              ": weight is [channels, 2 to 4 taps], got ", weight.sizes());
  const int64_t taps = weight.size(1);
  v.a.dt = to_dtype(x);
  v.a.B = c.B;
  v.a.T = c.T;
  v.a.D = (int)c.D;
  v.a.taps = (int)taps;
  v.a.silu = silu;
  v.a.x = read(c, x, "x", {c.D}, v.x);
  v.a.weight = read_param(c, weight, "weight", {c.D, taps}, v.weight);
  v.a.bias = read_param(c, bias, "bias", {c.D}, v.bias);
  if (state.has_value()) v.a.state = conv_state(c, *state, taps, "state", false, v.state);
  v.a.lengths = read_lengths(c, lengths, v.lengths);
  return v;
}

struct Scan {
  Call call;
  StateScan a;
  at::Tensor u, dt, b, c, z, a_log, skip, dt_bias, state, lengths;
  Sizes bc;  // sizes of b and c as given
  std::vector<at::Tensor> inputs() const { return {u, dt, b, c, z, a_log, skip, dt_bias, lengths}; }
};
Scan scan_of(const char* what, const at::Tensor& u, const at::Tensor& dt, const at::Tensor& a_log, const at::Tensor& b,
             const at::Tensor& c, const OptTensor& skip, const OptTensor& z, const OptTensor& dt_bias,
             const OptTensor& state, const OptTensor& lengths, bool one = false) {
  Scan v{call_of(u, what, "u", one)};
  const Call& k = v.call;
  TORCH_CHECK(a_log.dim() == 2 && a_log.size(1) >= 1 && a_log.size(1) <= STATE_SCAN_STATES, "dlvk.", what,
              ": a_log is [channels, 1 to ", STATE_SCAN_STATES, " states], got ", a_log.sizes());
  const int64_t N = a_log.size(1), flat = one ? 2 : 3;  // dimensions of b without groups
  TORCH_CHECK(b.dim() == flat || b.dim() == flat + 1, "dlvk.", what, ": b is [sequences, ", one ? "" : "tokens, ",
              "states] or the same with groups before the states, got ", b.sizes());
  const bool grouped = b.dim() > flat;
  const int64_t G = grouped ? b.size(flat - 1) : 1;
  TORCH_CHECK(G >= 1 && k.D % G == 0, "dlvk.", what, ": ", k.D, " channels in ", G, " groups");
  v.a.type = to_dtype(u);
  v.a.B = k.B;
  v.a.T = k.T;
  v.a.D = (int)k.D;
  v.a.N = (int)N;
  v.a.G = (int)G;
  v.a.u = read(k, u, "u", {k.D}, v.u);
  v.a.dt = read(k, dt, "dt", {k.D}, v.dt);
  if (grouped) {
    v.bc = sizes_of(k, {G, N});
    v.a.b = read(k, b, "b", {G, N}, v.b);
    v.a.c = read(k, c, "c", {G, N}, v.c);
  } else {
    v.bc = sizes_of(k, {N});
    v.a.b = read(k, b, "b", {N}, v.b);
    v.a.c = read(k, c, "c", {N}, v.c);
  }
  if (z.has_value()) v.a.z = read(k, *z, "z", {k.D}, v.z);
  v.a.a_log = read_param(k, a_log, "a_log", {k.D, N}, v.a_log);
  v.a.skip = read_param(k, skip, "skip", {k.D}, v.skip);
  v.a.dt_bias = read_param(k, dt_bias, "dt_bias", {k.D}, v.dt_bias);
  v.a.state = read_param(k, state, "state", {k.B, k.D, N}, v.state);
  v.a.lengths = read_lengths(k, lengths, v.lengths);
  return v;
}

}  // namespace

std::vector<OptTensor> short_conv_fwd_op(const at::Tensor& x, const at::Tensor& weight, OptTensor bias, OptTensor state,
                                         OptTensor lengths, bool silu, bool want_state, OptTensor out_state) {
  Conv v = conv_of("short_conv_fwd", x, weight, bias, state, lengths, silu);
  const Call& c = v.call;
  c10::cuda::CUDAGuard g(c.device);
  at::AutoDispatchBelowADInplaceOrView below;
  at::Tensor y = at::empty({c.B, c.T, c.D}, x.options()), last;
  SeqRef to;
  if (want_state || out_state.has_value()) {
    at::Tensor keep;
    last = out_state.has_value() ? *out_state : at::empty({c.B, v.a.taps - 1, c.D}, x.options());
    to = conv_state(c, last, v.a.taps, "out_state", true, keep);
    apart(c, {last}, {v.x, v.weight, v.bias, v.lengths});
    in_place_or_apart(c, last, v.state);
  }
  short_conv_fwd(v.a, {y.data_ptr(), y.stride(0), y.stride(1)}, to, stream());
  return {y, last.defined() ? OptTensor(last) : c10::nullopt};
}

at::Tensor short_conv_step_op(const at::Tensor& x, const at::Tensor& weight, OptTensor bias, const at::Tensor& state,
                              bool silu, OptTensor out_state) {
  Conv v = conv_of("short_conv_step", x, weight, bias, state, c10::nullopt, silu, true);
  const Call& c = v.call;
  c10::cuda::CUDAGuard g(c.device);
  at::AutoDispatchBelowADInplaceOrView below;
  at::Tensor y = at::empty({c.B, c.D}, x.options()), keep;
  const at::Tensor& last = out_state.has_value() ? *out_state : state;
  const SeqRef to = conv_state(c, last, v.a.taps, "out_state", true, keep);
  apart(c, {last}, {v.x, v.weight, v.bias});
  if (out_state.has_value()) in_place_or_apart(c, last, v.state);
  short_conv_fwd(v.a, ref(c, y), to, stream());
  return y;
}

std::vector<OptTensor> short_conv_bwd_op(const at::Tensor& x, const at::Tensor& weight, OptTensor bias,
                                         const at::Tensor& dy, OptTensor state, OptTensor lengths, bool silu,
                                         OptTensor dx, OptTensor dweight, OptTensor dbias, bool accumulate) {
  Conv v = conv_of("short_conv_bwd", x, weight, bias, state, lengths, silu);
  const Call& c = v.call;
  TORCH_CHECK(!accumulate || (dweight.has_value() && (dbias.has_value() || !bias.has_value())),
              "dlvk.short_conv_bwd: accumulate needs dweight (and dbias where there is a bias)");
  TORCH_CHECK(bias.has_value() || !dbias.has_value(), "dlvk.short_conv_bwd: dbias without a bias");
  c10::cuda::CUDAGuard g(c.device);
  at::AutoDispatchBelowADInplaceOrView below;
  at::Tensor dyk;
  const SeqRef go = read(c, dy, "dy", {c.D}, dyk);
  at::Tensor gx = written(c, dx, "dx", c.type, {c.B, c.T, c.D});
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(c.device);
  if (!dweight.has_value()) dweight = at::empty({c.D, v.a.taps}, f32);
  if (bias.has_value() && !dbias.has_value()) dbias = at::empty({c.D}, f32);
  float* gw = written_param(c, dweight, "dweight", {c.D, v.a.taps});
  float* gb = written_param(c, dbias, "dbias", {c.D});
  apart(c, {gx, *dweight, dbias.value_or(at::Tensor())}, {v.x, v.weight, v.bias, v.state, v.lengths, dyk});
  at::Tensor part = at::empty({std::max<int64_t>(1, short_conv_part_floats(v.a))}, f32);
  short_conv_bwd(v.a, go, written_rows(c, gx, "dx"), gw, gb, accumulate, part.data_ptr<float>(), stream());
  return {gx, dweight, dbias};
}

std::vector<OptTensor> state_scan_fwd_op(const at::Tensor& u, const at::Tensor& dt, const at::Tensor& a_log,
                                         const at::Tensor& b, const at::Tensor& c, OptTensor skip, OptTensor z,
                                         OptTensor dt_bias, OptTensor state, OptTensor lengths, bool want_state,
                                         bool save, OptTensor out_state) {
  Scan v = scan_of("state_scan_fwd", u, dt, a_log, b, c, skip, z, dt_bias, state, lengths);
  const Call& k = v.call;
  c10::cuda::CUDAGuard g(k.device);
  at::AutoDispatchBelowADInplaceOrView below;
  at::Tensor y = at::empty({k.B, k.T, k.D}, u.options()), last, saved, scratch;
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(k.device);
  if (want_state || out_state.has_value()) {
    last = written(k, out_state, "out_state", at::kFloat, {k.B, k.D, v.a.N});
    TORCH_CHECK(last.is_contiguous(), "dlvk.state_scan_fwd: out_state must be contiguous");
    apart(k, {last}, v.inputs());
    in_place_or_apart(k, last, v.state);
  }
  if (save) saved = at::empty({k.B, (k.T + STATE_SCAN_SPAN - 1) / STATE_SCAN_SPAN, k.D, v.a.N}, f32);
  const int64_t floats = state_scan_fwd_scratch_floats(v.a);
  if (floats > 0) scratch = at::empty({floats}, f32);
  state_scan_fwd(v.a, {y.data_ptr(), y.stride(0), y.stride(1)}, last.defined() ? last.data_ptr<float>() : nullptr,
                 save ? saved.data_ptr<float>() : nullptr, floats > 0 ? scratch.data_ptr<float>() : nullptr, stream());
  return {y, last.defined() ? OptTensor(last) : c10::nullopt, save ? OptTensor(saved) : c10::nullopt};
}

at::Tensor state_scan_step_op(const at::Tensor& u, const at::Tensor& dt, const at::Tensor& a_log, const at::Tensor& b,
                              const at::Tensor& c, const at::Tensor& state, OptTensor skip, OptTensor z,
                              OptTensor dt_bias, OptTensor out_state) {
  Scan v = scan_of("state_scan_step", u, dt, a_log, b, c, skip, z, dt_bias, state, c10::nullopt, true);
  const Call& k = v.call;
  c10::cuda::CUDAGuard g(k.device);
  at::AutoDispatchBelowADInplaceOrView below;
  const at::Tensor& last = out_state.has_value() ? *out_state : state;
  check(k, last, "out_state", at::kFloat, {k.B, k.D, v.a.N});
  TORCH_CHECK(last.is_contiguous(), "dlvk.state_scan_step: ", out_state.has_value() ? "out_state" : "state",
              " must be contiguous");
  for (const at::Tensor& t : {v.u, v.dt, v.b, v.c, v.z, v.a_log, v.skip, v.dt_bias})
    TORCH_CHECK(!share(last, t), "dlvk.state_scan_step: the state shares memory with an operand");
  if (out_state.has_value()) in_place_or_apart(k, last, v.state);
  at::Tensor y = at::empty({k.B, k.D}, u.options());
  state_scan_fwd(v.a, ref(k, y), last.data_ptr<float>(), nullptr, nullptr, stream());
  return y;
}

std::vector<OptTensor> state_scan_bwd_op(const at::Tensor& u, const at::Tensor& dt, const at::Tensor& a_log,
                                         const at::Tensor& b, const at::Tensor& c, OptTensor skip, OptTensor z,
                                         OptTensor dt_bias, const at::Tensor& dy, const at::Tensor& saved,
                                         OptTensor lengths, OptTensor du, OptTensor ddt, OptTensor db, OptTensor dc,
                                         OptTensor dz, OptTensor da_log, OptTensor dskip, OptTensor ddt_bias,
                                         bool accumulate) {
  Scan v = scan_of("state_scan_bwd", u, dt, a_log, b, c, skip, z, dt_bias, c10::nullopt, lengths);
  const Call& k = v.call;
  TORCH_CHECK(!accumulate || (da_log.has_value() && (dskip.has_value() || !skip.has_value()) &&
                              (ddt_bias.has_value() || !dt_bias.has_value())),
              "dlvk.state_scan_bwd: accumulate needs the parameters' gradients");
  TORCH_CHECK((z.has_value() || !dz.has_value()) && (skip.has_value() || !dskip.has_value()) &&
                  (dt_bias.has_value() || !ddt_bias.has_value()),
              "dlvk.state_scan_bwd: a gradient of an operand that is not there");
  check(k, saved, "saved", at::kFloat, {k.B, (k.T + STATE_SCAN_SPAN - 1) / STATE_SCAN_SPAN, k.D, v.a.N});
  TORCH_CHECK(saved.is_contiguous(), "dlvk.state_scan_bwd: saved must be contiguous");
  c10::cuda::CUDAGuard g(k.device);
  at::AutoDispatchBelowADInplaceOrView below;
  at::Tensor dyk;
  const SeqRef go = read(k, dy, "dy", {k.D}, dyk);
  const std::vector<int64_t> rows{k.B, k.T, k.D};
  at::Tensor gu = written(k, du, "du", k.type, rows), gdt = written(k, ddt, "ddt", k.type, rows);
  at::Tensor gb = written(k, db, "db", k.type, v.bc), gc = written(k, dc, "dc", k.type, v.bc), gz;
  if (z.has_value()) gz = written(k, dz, "dz", k.type, rows);
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(k.device);
  if (!da_log.has_value()) da_log = at::empty({k.D, v.a.N}, f32);
  if (skip.has_value() && !dskip.has_value()) dskip = at::empty({k.D}, f32);
  if (dt_bias.has_value() && !ddt_bias.has_value()) ddt_bias = at::empty({k.D}, f32);
  StateScanGrads r;
  r.du = written_rows(k, gu, "du");
  r.ddt = written_rows(k, gdt, "ddt");
  r.db = written_rows(k, gb, "db");
  r.dc = written_rows(k, gc, "dc");
  if (gz.defined()) r.dz = written_rows(k, gz, "dz");
  r.da_log = written_param(k, da_log, "da_log", {k.D, v.a.N});
  r.dskip = written_param(k, dskip, "dskip", {k.D});
  r.ddt_bias = written_param(k, ddt_bias, "ddt_bias", {k.D});
  r.accumulate = accumulate;
  std::vector<at::Tensor> in = v.inputs();
  in.push_back(dyk);
  in.push_back(saved);
  apart(k, {gu, gdt, gb, gc, gz, *da_log, dskip.value_or(at::Tensor()), ddt_bias.value_or(at::Tensor())}, in);
  at::Tensor scratch = at::empty({std::max<int64_t>(1, state_scan_bwd_scratch_floats(v.a))}, f32);
  state_scan_bwd(v.a, saved.data_ptr<float>(), go, r, scratch.data_ptr<float>(), stream());
  return {gu, gdt, da_log, gb, gc, dskip, gz.defined() ? OptTensor(gz) : c10::nullopt, ddt_bias};
}

at::Tensor sample_tokens_op(const at::Tensor& logits, const at::Tensor& uniform, double temperature, int64_t top_k,
                            double top_p, double min_p, OptTensor temperatures, OptTensor top_ks, OptTensor top_ps,
                            OptTensor min_ps) {
  TORCH_CHECK(logits.is_cuda(), "dlvk.sample_tokens: logits must be a CUDA tensor");
  TORCH_CHECK(logits.dim() == 2, "dlvk.sample_tokens: logits are [rows, words], got ", logits.sizes());
  TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16,
              "dlvk.sample_tokens: logits are fp32 or bf16, got ", logits.scalar_type());
  const int64_t rows = logits.size(0), words = logits.size(1);
  TORCH_CHECK(words >= 1 && words <= SAMPLING_WORDS, "dlvk.sample_tokens: 1 to ", SAMPLING_WORDS, " words, got ", words);
  const Call c{"sample_tokens", logits.device(), logits.scalar_type(), rows, words, 0};
  c10::cuda::CUDAGuard g(c.device);
  at::AutoDispatchBelowADInplaceOrView below;
  at::Tensor keep[6];
  Sampling a;
  check(c, logits, "logits", c.type, {rows, words});
  keep[0] = words == 1 || logits.stride(1) == 1 ? logits : logits.contiguous();
  a.dt = to_dtype(logits);
  a.logits = keep[0].data_ptr();
  a.ld = keep[0].stride(0);
  a.rows = rows;
  a.words = words;
  a.uniform = read_param(c, uniform, "uniform", {rows}, keep[1]);
  a.temperature = {read_param(c, temperatures, "temperature", {rows}, keep[2]), temperature};
  a.top_p = {read_param(c, top_ps, "top_p", {rows}, keep[3]), top_p};
  a.min_p = {read_param(c, min_ps, "min_p", {rows}, keep[4]), min_p};
  a.top_k.one = top_k;
  if (top_ks.has_value()) {
    check(c, *top_ks, "top_k", at::kInt, {rows});
    keep[5] = top_ks->contiguous();
    a.top_k.rows = keep[5].data_ptr<int32_t>();
  }
  at::Tensor tokens = at::empty({rows}, logits.options().dtype(at::kInt));
  sample_tokens(a, tokens.data_ptr<int32_t>(), stream());
  return tokens;
}

}  // namespace aten
}  // namespace dlvk
