// Torch binding of the 8-bit kernels: buffers, launches and backward passes without Python between them.
//
// A training step of one 8-bit linear layer is seven launches and about sixteen buffers; driven from Python it costs
// several times what the kernels take on a short batch (measured on 1021 x 1000 x 2056: 350 us of host time against
// 40 us of kernels).  The functions here allocate with torch's allocator on every call and keep nothing between calls.
// The kernel library is loaded by Python, which hands its entry points over in init(): the binding links against torch
// only.
#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <atomic>
#include <cmath>
#include <optional>

#include "scaled_abi.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

struct Api {
  decltype(&jb_scaled_gemm) gemm = nullptr;
  decltype(&jb_quantize) quantize = nullptr;
  decltype(&jb_column_sum) column_sum = nullptr;
  decltype(&jb_rms_max_cols) rms_max_cols = nullptr;
  decltype(&jb_rms_norm_fwd) rms_fwd = nullptr;
  decltype(&jb_rms_bwd_parts) rms_bwd_parts = nullptr;
  decltype(&jb_rms_norm_bwd) rms_bwd = nullptr;
} api;

std::atomic<long long> launches{0};

constexpr auto CODES = at::kFloat8_e4m3fn;
constexpr auto SCALES = at::kFloat8_e8m0fnu;

int type_of(at::ScalarType t) {
  if (t == at::kFloat) return 0;
  if (t == at::kBFloat16) return 1;
  TORCH_CHECK_TYPE(t == at::kHalf, "the 8-bit kernels take fp32, bf16 and fp16, got ", t);
  return 2;
}
at::ScalarType scalar_of(int64_t type) { return type == 0 ? at::kFloat : type == 1 ? at::kBFloat16 : at::kHalf; }

void done(int rc, const char* what, int n = 1) {
  TORCH_CHECK(rc == 0, "jigsaw_b200 kernel launcher ", what, " failed with code ", rc);
  launches.fetch_add(n, std::memory_order_relaxed);
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType t, const Tensor& like) {
  return at::detail::empty_cuda(sizes, t, like.device(), std::nullopt);
}
void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int sm_count(const Tensor& t) { return at::cuda::getDeviceProperties(t.device().index())->multiProcessorCount; }
int checked(int64_t n) {
  TORCH_CHECK_VALUE(n <= 0x7fffff00LL, "an axis of ", n, " elements is longer than the kernels address");
  return static_cast<int>(n);
}
int64_t pitch_of(int64_t n) { return (n + 15) / 16 * 16; }

std::array<Tensor, 64> status_words;                 // per device, set by Python when it first meets one
void set_status(int64_t device, const Tensor& word) { status_words.at(device) = word; }
const Tensor& status_of(const Tensor& t) {
  const Tensor& w = status_words.at(t.device().index());
  TORCH_CHECK(w.defined(), "no status word for device ", t.device().index());
  return w;
}

// A tensor as rows of its last axis, `ld` elements apart; copied only if its strides do not allow that.
struct Rows {
  Tensor t;
  int64_t rows, cols, ld;
};
Rows rows_of(const Tensor& x) {
  const int64_t c = x.size(-1), r = x.numel() / c;
  if (x.is_contiguous()) return {x, r, c, c};
  if (x.dim() == 2 && (x.stride(1) == 1 || c == 1) && x.stride(0) >= 0) return {x, r, c, x.stride(0)};
  return {x.contiguous(), r, c, c};
}

// Codes [rows, pitch] and scales of a quantised matrix.
struct Codes {
  Tensor codes, scales;
  int64_t rows = 0, cols = 0, scale_row = 0, scale_k = 0;
  bool square = false;
  bool turned = false;       // `scales` are those of the transpose

  JbScaledOperand operand() const {
    return {codes.data_ptr(), codes.size(1), scales.data_ptr(), scale_row, scale_k, static_cast<int>(rows), square ? 1 : 0};
  }
  // The public forms: [rows, cols] and [scale rows, blocks].
  Tensor code_view() const { return codes.size(1) == cols ? codes : codes.narrow(1, 0, cols); }
  Tensor scale_view() const {
    const int64_t blocks = ((turned ? rows : cols) + 127) / 128;
    const Tensor s = scales.size(1) == blocks ? scales : scales.narrow(1, 0, blocks);
    return turned ? s.t() : s;
  }
};
// The scales of a row start on a whole word: the product reads those of four blocks at once.
int64_t words_of(int64_t blocks) { return (blocks + 3) / 4 * 4; }
Codes new_codes(int64_t rows, int64_t cols, const Tensor& like) {
  Codes q;
  q.rows = rows;
  q.cols = cols;
  q.codes = empty({rows, pitch_of(cols)}, CODES, like);
  return q;
}
void new_row_scales(Codes& q) {
  q.scales = empty({q.rows, words_of((q.cols + 127) / 128)}, SCALES, q.codes);
  q.scale_row = q.scales.size(1);
  q.scale_k = 1;
}

struct Quantized {
  std::optional<Codes> rows, cols;
  Tensor sums;
};

// Codes of x (of x * rstd * gain) along its rows and / or of its transpose along the columns, read once; `sum_type` >= 0
// asks for the column sums.
Quantized quantize(const Tensor& input, bool square, bool want_rows, bool want_cols, const Tensor& rstd, const Tensor& gain,
                   int sum_type) {
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows x = rows_of(input);
  const int64_t rb = (x.rows + 127) / 128, cb = (x.cols + 127) / 128;
  JbQuant q{};
  q.x = x.t.const_data_ptr();
  q.ldx = x.ld;
  q.rows = checked(x.rows);
  q.cols = checked(x.cols);
  q.type = type_of(x.t.scalar_type());
  q.square = square;
  Quantized out;
  Tensor shared;
  if (square) {
    shared = empty({rb, words_of(cb)}, SCALES, x.t);
    q.scales = shared.data_ptr();
    q.scale_row = shared.size(1);
    q.scale_k = 1;
  }
  if (want_rows) {
    Codes c = new_codes(x.rows, x.cols, x.t);
    q.codes = c.codes.data_ptr();
    q.pitch = c.codes.size(1);
    if (square) {
      c.scales = shared;
      c.scale_row = shared.size(1);
      c.scale_k = 1;
      c.square = true;
    } else {
      new_row_scales(c);
      q.scales = c.scales.data_ptr();
      q.scale_row = c.scale_row;
      q.scale_k = c.scale_k;
    }
    out.rows = std::move(c);
  }
  if (want_cols) {
    Codes c = new_codes(x.cols, x.rows, x.t);
    q.codes_t = c.codes.data_ptr();
    q.pitch_t = c.codes.size(1);
    if (square) {
      c.scales = shared;
      c.scale_row = 1;
      c.scale_k = shared.size(1);
      c.square = c.turned = true;
    } else {
      new_row_scales(c);
      q.scales_t = c.scales.data_ptr();
      q.scale_t_row = c.scale_row;
      q.scale_t_k = c.scale_k;
    }
    out.cols = std::move(c);
  }
  Tensor gain_c;
  if (rstd.defined()) {
    q.rstd = rstd.const_data_ptr();
    if (gain.defined()) {
      gain_c = gain.contiguous();
      q.gain = gain_c.const_data_ptr();
      q.gain_type = type_of(gain_c.scalar_type());
    }
  }
  Tensor part;
  if (sum_type >= 0) {
    part = empty({rb, x.cols}, at::kFloat, x.t);
    q.colsum = part.data_ptr();
  }
  done(api.quantize(&q, sm_count(x.t), stream_of(x.t)), "quantize");
  if (sum_type >= 0) {
    out.sums = empty({x.cols}, scalar_of(sum_type), x.t);
    done(api.column_sum(part.const_data_ptr<float>(), checked(rb), q.cols, out.sums.data_ptr(), sum_type, stream_of(x.t)), "column_sum");
  }
  return out;
}

// a [M, K] b [N, K]^T + bias, as a tensor of the given sizes (M N elements).
Tensor product(const JbScaledOperand& a, const JbScaledOperand& b, int64_t K, const Tensor& bias, int out_type,
               at::IntArrayRef sizes, const Tensor& like) {
  Tensor out = empty(sizes, scalar_of(out_type), like);
  Tensor bias_c;
  if (bias.defined()) bias_c = bias.contiguous();
  done(api.gemm(&a, &b, K, out.data_ptr(), b.rows, out_type, bias.defined() ? bias_c.const_data_ptr() : nullptr,
                bias.defined() ? type_of(bias_c.scalar_type()) : 0, sm_count(like), status_of(like).data_ptr<int>(), stream_of(like)),
       "scaled_gemm");
  return out;
}

struct Normed {
  Tensor y, sum, rstd;
  std::optional<Codes> codes;
};

Normed rms_forward(const Tensor& input, const Tensor& gain, double eps, const Tensor& residual, int y_type, bool want_codes,
                   bool want_rstd) {
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows x = rows_of(input);
  JbRms q{};
  q.x = x.t.const_data_ptr();
  q.ldx = x.ld;
  q.rows = checked(x.rows);
  q.cols = checked(x.cols);
  q.type = type_of(x.t.scalar_type());
  q.eps = static_cast<float>(eps);
  Tensor gain_c;
  if (gain.defined()) {
    gain_c = gain.contiguous();
    q.gain = gain_c.const_data_ptr();
    q.gain_type = type_of(gain_c.scalar_type());
  }
  Normed out;
  Rows r;
  if (residual.defined()) {
    r = rows_of(residual);
    q.residual = r.t.const_data_ptr();
    q.ldr = r.ld;
    out.sum = empty(input.sizes(), x.t.scalar_type(), x.t);
    q.sum = out.sum.data_ptr();
  }
  if (want_rstd) {
    out.rstd = empty({x.rows}, at::kFloat, x.t);
    q.rstd = out.rstd.data_ptr();
  }
  if (y_type >= 0) {
    out.y = empty(input.sizes(), scalar_of(y_type), x.t);
    q.y = out.y.data_ptr();
    q.y_type = y_type;
  }
  if (want_codes) {
    Codes c = new_codes(x.rows, x.cols, x.t);
    new_row_scales(c);
    q.codes = c.codes.data_ptr();
    q.pitch = c.codes.size(1);
    q.scales = c.scales.data_ptr();
    q.scale_row = c.scale_row;
    q.scale_k = c.scale_k;
    out.codes = std::move(c);
  }
  done(api.rms_fwd(&q, sm_count(x.t), stream_of(x.t)), "rms_norm_fwd");
  return out;
}

// Gradients of the normalised sum t and of the gain; g has the type of t or fp32.
std::pair<Tensor, Tensor> rms_backward(const Tensor& sum, const Tensor& gain, const Tensor& rstd, const Tensor& grad,
                                       const Tensor& grad_sum, bool want_gain) {
  const c10::cuda::CUDAGuard guard(sum.device());
  const Rows t = rows_of(sum);
  Tensor g = grad, gs = grad_sum, gain_c;
  if (g.scalar_type() != sum.scalar_type() && g.scalar_type() != at::kFloat) g = g.to(at::kFloat);
  g = g.contiguous();
  JbRmsBwd q{};
  q.t = t.t.const_data_ptr();
  q.ldt = t.ld;
  q.rows = checked(t.rows);
  q.cols = checked(t.cols);
  q.type = type_of(t.t.scalar_type());
  q.g = g.const_data_ptr();
  q.g_f32 = g.scalar_type() == at::kFloat;
  if (gs.defined()) {
    gs = gs.to(sum.scalar_type()).contiguous();
    q.gsum = gs.const_data_ptr();
  }
  q.rstd = rstd.const_data_ptr();
  if (gain.defined()) {
    gain_c = gain.contiguous();
    q.gain = gain_c.const_data_ptr();
    q.gain_type = type_of(gain_c.scalar_type());
  }
  Tensor dx = empty(sum.sizes(), sum.scalar_type(), sum), dgain, part;
  q.dx = dx.data_ptr();
  const int sm = sm_count(sum);
  if (want_gain) {
    part = empty({api.rms_bwd_parts(&q, sm), t.cols}, at::kFloat, sum);
    q.part = part.data_ptr();
  }
  done(api.rms_bwd(&q, sm, status_of(sum).data_ptr<int>(), stream_of(sum)), "rms_norm_bwd");
  if (want_gain) {
    dgain = empty({t.cols}, gain.scalar_type(), sum);
    done(api.column_sum(part.const_data_ptr<float>(), checked(part.size(0)), q.cols, dgain.data_ptr(), q.gain_type, stream_of(sum)),
         "column_sum");
  }
  return {dx, dgain};
}

// ------------------------------------------------------------------------------------------------ autograd
using Optional = std::optional<Tensor>;
Tensor opt(const Optional& t) { return t.has_value() ? *t : Tensor(); }

// The backward passes are kernels without a derivative of their own: with create_graph=True the gradients carry a node
// that raises when it is differentiated.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list real;
  for (auto& g : grads)
    if (g.defined()) real.push_back(g.detach().requires_grad_(true));
  if (real.empty()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that is differentiable once (8-bit path)", static_cast<int64_t>(real.size()));
  variable_list marked = (*error)(std::move(real));
  size_t k = 0;
  for (auto& g : grads)
    if (g.defined()) g = marked[k++];
  return grads;
}

// Its memory does not hold its values as they are, or it has none: wrapped by a transform or a subclass, lazily negated, zeros.
bool wrapped(const Tensor& t) {
  const c10::DispatchKeySet k = t.unsafeGetTensorImpl()->key_set();
  return k.has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Python,
                                        c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor}));
}

// A gradient in memory that holds its values: autograd hands over lazily negated tensors too (the imaginary part of a
// conjugate), whose memory has the other sign, and zeros without memory.
// Tensors that a transform or a subclass wraps have none at all and are refused.
Tensor stored(const Tensor& g) {
  if (!g.defined()) return g;
  const c10::DispatchKeySet k = g.unsafeGetTensorImpl()->key_set();
  TORCH_CHECK_NOT_IMPLEMENTED(g.layout() == at::kStrided && g.is_cuda() &&
                                  !k.has_any(c10::DispatchKeySet({c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchBatched,
                                                                  c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Python})),
                              "the 8-bit path takes output gradients that are plain strided tensors (no torch.vmap, no wrapping subclass)");
  return g._is_zerotensor() ? at::zeros(g.sizes(), g.options()) : g.resolve_neg();
}

void save_codes(variable_list& to, const std::optional<Codes>& c) {
  to.push_back(c ? c->codes : Tensor());
  to.push_back(c ? c->scales : Tensor());
}
bool float_type(const Tensor& t) {
  const at::ScalarType s = t.scalar_type();
  return s == at::kFloat || s == at::kBFloat16 || s == at::kHalf;
}
// What the forward pass saved, as it comes back: saved-tensor hooks may hand over another tensor in its place, at other
// strides (then it is copied), or one that the kernels must not be given.
Tensor restored(const Tensor& t, at::ScalarType type, at::IntArrayRef sizes, const Tensor& g) {
  TORCH_CHECK(t.defined() && t.device() == g.device() && t.layout() == at::kStrided && !wrapped(t) && t.scalar_type() == type && t.sizes() == sizes,
              "a tensor that the 8-bit path saved for its backward pass came back from a saved-tensor hook as another one (device, type or shape)");
  return t.contiguous();
}
// The same for a tensor that the kernels take at any strides and in any of their types.
const Tensor& restored(const Tensor& t, int64_t rows, int64_t cols, const Tensor& g) {
  TORCH_CHECK(t.defined() && t.device() == g.device() && t.layout() == at::kStrided && !wrapped(t) && float_type(t) && t.dim() >= 1 &&
                  t.size(-1) == cols && t.numel() == rows * cols,
              "a tensor that the 8-bit path saved for its backward pass came back from a saved-tensor hook as another one (device, type or shape)");
  return t;
}
// The transposed weight, or the activations in blocks along the tokens, as saved by the forward pass.
Codes saved_codes(const Tensor& codes, const Tensor& scales, int64_t rows, int64_t cols, bool square, const Tensor& g) {
  const int64_t rb = (rows + 127) / 128, cb = (cols + 127) / 128;
  Codes c;
  c.codes = restored(codes, CODES, {rows, pitch_of(cols)}, g);
  // of a square the scales are those of the matrix that was not turned
  c.scales = square ? restored(scales, SCALES, {cb, words_of(rb)}, g) : restored(scales, SCALES, {rows, words_of(cb)}, g);
  c.rows = rows;
  c.cols = cols;
  c.square = c.turned = square;
  c.scale_row = square ? 1 : c.scales.size(1);
  c.scale_k = square ? c.scales.size(1) : 1;
  return c;
}
std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = n;
  return s;
}

struct LinearGrads {
  Tensor dx, dw, db;
};
// The two gradient products of a layer whose transposed weight and column-quantised input are given (absent: not wanted).
LinearGrads linear_backward(const Tensor& g, const std::optional<Codes>& w_t, const std::optional<Codes>& x_t, int dx_type,
                            at::IntArrayRef dx_sizes, int dw_type, int bias_type) {
  LinearGrads out;
  const Quantized q = quantize(g, false, w_t.has_value(), x_t.has_value(), Tensor(), Tensor(), bias_type);
  const int64_t N = g.size(-1), M = g.numel() / N;
  if (w_t) out.dx = product(q.rows->operand(), w_t->operand(), N, Tensor(), dx_type, dx_sizes, g);
  if (x_t) out.dw = product(q.cols->operand(), x_t->operand(), M, Tensor(), dw_type, {N, x_t->rows}, g);
  out.db = q.sums;
  return out;
}
Tensor bias_sum(const Tensor& g, int type) {
  return at::sum(g.reshape({-1, g.size(-1)}), {0}, false, at::kFloat).to(scalar_of(type));
}

// y = q(x) q(w)^T + b; dx = q(g) q(w); dw = q(g^T) q(x^T)^T with blocks along the tokens.  x and w are read once and
// written in the layouts that all three products want.
struct ScaledLinear : public Function<ScaledLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Optional& bias, int64_t out_type, bool need_x,
                        bool need_w) {
    const Tensor b = opt(bias);
    const c10::cuda::CUDAGuard guard(x.device());
    const Quantized qx = quantize(x, false, true, need_w, Tensor(), Tensor(), -1);
    const Quantized qw = quantize(w, true, true, need_x, Tensor(), Tensor(), -1);
    variable_list save;
    save_codes(save, qx.cols);
    save_codes(save, qw.cols);
    ctx->save_for_backward(save);
    ctx->saved_data["x"] = x.sizes().vec();
    ctx->saved_data["n"] = w.size(0);
    ctx->saved_data["types"] = std::vector<int64_t>{type_of(x.scalar_type()), type_of(w.scalar_type()),
                                                    b.defined() ? type_of(b.scalar_type()) : -1};
    ctx->set_materialize_grads(false);
    return product(qx.rows->operand(), qw.rows->operand(), x.size(-1), b, static_cast<int>(out_type), with_last(x, w.size(0)), x);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    const Tensor g = stored(grads[0]);
    if (!g.defined()) return out;
    const c10::cuda::CUDAGuard guard(g.device());
    const variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> xs = ctx->saved_data["x"].toIntVector(), types = ctx->saved_data["types"].toIntVector();
    const int64_t N = ctx->saved_data["n"].toInt(), K = xs.back();
    int64_t M = 1;
    for (size_t i = 0; i + 1 < xs.size(); ++i) M *= xs[i];
    std::optional<Codes> x_t, w_t;
    if (s[0].defined() && ctx->needs_input_grad(1)) x_t = saved_codes(s[0], s[1], K, M, false, g);
    if (s[2].defined() && ctx->needs_input_grad(0)) w_t = saved_codes(s[2], s[3], K, N, true, g);
    const int bias_type = types[2] >= 0 && ctx->needs_input_grad(2) ? static_cast<int>(types[2]) : -1;
    if (x_t || w_t) {
      LinearGrads l = linear_backward(g, w_t, x_t, static_cast<int>(types[0]), xs, static_cast<int>(types[1]), bias_type);
      out[0] = l.dx;
      out[1] = l.dw;
      out[2] = l.db;
    } else if (bias_type >= 0) {
      out[2] = bias_sum(g, bias_type);
    }
    return once(std::move(out));
  }
};

// y = t r gain, t = x + residual; outputs (y, t), or y alone.
struct RmsNorm : public Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Optional& gain_in, const Optional& residual_in, double eps,
                               int64_t y_type, bool need) {
    const Tensor gain = opt(gain_in), residual = opt(residual_in);
    Normed n = rms_forward(x, gain, eps, residual, static_cast<int>(y_type), false, need);
    ctx->set_materialize_grads(false);
    if (need) ctx->save_for_backward({residual.defined() ? n.sum : x, gain, n.rstd});
    ctx->saved_data["residual"] = residual.defined();
    return residual.defined() ? variable_list{n.y, n.sum} : variable_list{n.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    const variable_list s = ctx->get_saved_variables();
    const bool residual = ctx->saved_data["residual"].toBool();
    const Tensor g = stored(grads[0]), gsum = residual ? stored(grads[1]) : Tensor();
    const bool want_gain = s[1].defined() && ctx->needs_input_grad(1);
    if (g.defined()) {
      const int64_t cols = g.size(-1), rows = g.numel() / cols;
      if (s[1].defined()) restored(s[1], 1, cols, g);
      std::tie(out[0], out[1]) = rms_backward(restored(s[0], rows, cols, g), s[1], restored(s[2], at::kFloat, {rows}, g), g, gsum, want_gain);
    } else {                                   // only the sum was used
      if (gsum.defined()) out[0] = gsum.to(s[0].scalar_type());
      if (want_gain) out[1] = at::zeros_like(s[1]);
    }
    if (residual) out[2] = out[0];
    return once(std::move(out));
  }
};

// The norm's output exists as codes only; the backward pass normalises the stored sum again, straight into the column
// blocks of the weight gradient, and keeps the gradient of the normalised rows in fp32 between product and norm.
struct RmsNormLinear : public Function<RmsNormLinear> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Optional& gain_in, const Tensor& w, const Optional& bias,
                               const Optional& residual_in, double eps, int64_t out_type, bool need_h, bool need_w) {
    const Tensor gain = opt(gain_in), b = opt(bias), residual = opt(residual_in);
    const c10::cuda::CUDAGuard guard(x.device());
    Normed n = rms_forward(x, gain, eps, residual, -1, true, need_h || need_w);
    const Quantized qw = quantize(w, true, true, need_h, Tensor(), Tensor(), -1);
    ctx->set_materialize_grads(false);
    variable_list save;
    if (need_h || need_w) {
      save = {residual.defined() ? n.sum : x, gain, n.rstd};
      save_codes(save, qw.cols);
    }
    ctx->save_for_backward(save);
    ctx->saved_data["flags"] = std::vector<int64_t>{need_h, need_w, residual.defined(), w.size(0), type_of(w.scalar_type()),
                                                    b.defined() ? type_of(b.scalar_type()) : -1, gain.defined(), x.size(-1)};
    Tensor y = product(n.codes->operand(), qw.rows->operand(), x.size(-1), b, static_cast<int>(out_type), with_last(x, w.size(0)), x);
    return residual.defined() ? variable_list{y, n.sum} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    const std::vector<int64_t> f = ctx->saved_data["flags"].toIntVector();
    const bool need_h = f[0], need_w = f[1], residual = f[2];
    const int64_t N = f[3];
    const Tensor g = stored(grads[0]), gsum = residual ? stored(grads[1]) : Tensor();
    // edges count the tensors that were given: x, [gain], w, [bias], [residual]
    const size_t w_edge = f[6] ? 2 : 1, residual_edge = w_edge + (f[5] >= 0 ? 2 : 1);
    const int bias_type = f[5] >= 0 && ctx->needs_input_grad(w_edge + 1) ? static_cast<int>(f[5]) : -1;
    const variable_list s = ctx->get_saved_variables();
    if (!need_h && !need_w) {
      if (g.defined() && bias_type >= 0) out[3] = bias_sum(g, bias_type);
      return once(std::move(out));
    }
    const Tensor &t = s[0], &gain = s[1];
    const int64_t K = f[7];
    const bool want_gain = gain.defined() && ctx->needs_input_grad(1);
    const bool want_h = need_h && (want_gain || ctx->needs_input_grad(0) || (residual && ctx->needs_input_grad(residual_edge)));
    Tensor dh, rstd;
    if (g.defined()) {
      const c10::cuda::CUDAGuard guard(g.device());
      const int64_t M = g.numel() / N;
      restored(t, M, K, g);
      if (gain.defined()) restored(gain, 1, K, g);
      rstd = restored(s[2], at::kFloat, {M}, g);
      std::optional<Codes> w_t, h_t;
      if (want_h) w_t = saved_codes(s[3], s[4], K, N, true, g);
      if (need_w && ctx->needs_input_grad(w_edge)) h_t = quantize(t, false, false, true, rstd, gain, -1).cols;
      if (w_t || h_t) {
        LinearGrads l = linear_backward(g, w_t, h_t, 0, t.sizes(), static_cast<int>(f[4]), bias_type);
        dh = l.dx;
        out[2] = l.dw;
        out[3] = l.db;
      } else if (bias_type >= 0) {
        out[3] = bias_sum(g, bias_type);
      }
    }
    if (dh.defined()) {
      std::tie(out[0], out[1]) = rms_backward(t, gain, rstd, dh, gsum, want_gain);
    } else {
      if (gsum.defined()) out[0] = gsum.to(t.scalar_type());
      if (want_gain) out[1] = at::zeros_like(gain);
    }
    if (residual) out[4] = out[0];
    return once(std::move(out));
  }
};

// ------------------------------------------------------------------------------------------------ Python
// Every entry point answers None to a call that is not an ordinary one for the kernels: other types, devices or shapes that
// do not fit, empty tensors, tensors wrapped by a transform or whose memory does not hold their values as they are.  The
// caller then takes its general path, which raises the error or computes the call in torch operations.
py::object give(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

bool ordinary(const Tensor& t, const Tensor& like) {
  return t.layout() == at::kStrided && t.device() == like.device() && t.is_cuda() && !wrapped(t) && t.numel() > 0;
}
bool vector_of(const Optional& t, int64_t n, const Tensor& like) {
  return !t.has_value() || (float_type(*t) && ordinary(*t, like) && t->dim() == 1 && t->size(0) == n);
}
bool matrix_codes(const Tensor& codes, const Tensor& scales, bool square, const Tensor& like) {
  if (codes.scalar_type() != CODES || scales.scalar_type() != SCALES || !ordinary(codes, like) || !ordinary(scales, like)) return false;
  const int64_t nb = (codes.size(-1) + 127) / 128;
  if (square) return codes.dim() == 2 && scales.dim() == 2 && scales.size(0) == (codes.size(0) + 127) / 128 && scales.size(1) == nb;
  return codes.dim() >= 1 && scales.dim() == codes.dim() && scales.size(-1) == nb && scales.numel() / nb == codes.numel() / codes.size(-1);
}
bool norm_args(const Tensor& x, const Optional& gain, const Optional& residual, double eps) {
  if (!float_type(x) || x.dim() < 1 || !ordinary(x, x) || x.size(-1) > api.rms_max_cols() || !(eps >= 0.0) || std::isinf(eps)) return false;
  if (!vector_of(gain, x.size(-1), x)) return false;
  return !residual.has_value() || (residual->scalar_type() == x.scalar_type() && ordinary(*residual, x) && residual->sizes() == x.sizes());
}
bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const Optional& t) { return t.has_value() && t->requires_grad(); }
// A derivative is asked for, by reverse or by forward mode.
bool traced(const Tensor& t) { return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined(); }
bool traced(const Optional& t) { return t.has_value() && traced(*t); }

// Type of a layer's output: that of autocast where it is on.
int autocast_type(const Tensor& x) {
  if (!at::autocast::is_autocast_enabled(at::kCUDA)) return type_of(x.scalar_type());
  const at::ScalarType t = at::autocast::get_autocast_dtype(at::kCUDA);
  return t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : type_of(x.scalar_type());
}

py::object py_quantize(const Tensor& x, bool square, bool rows, bool cols, const Optional& rstd, const Optional& gain, int sum_type) {
  if (!float_type(x) || x.dim() < 1 || !ordinary(x, x) || (square && x.dim() != 2) || (cols && x.dim() != 2)) return py::none();
  if (rstd.has_value() && (x.dim() != 2 || rstd->scalar_type() != at::kFloat || !rstd->is_contiguous() || !vector_of(rstd, x.size(0), x))) return py::none();
  if (!vector_of(gain, x.size(-1), x)) return py::none();
  const Quantized q = quantize(x, square, rows, cols, opt(rstd), opt(gain), sum_type);
  return py::make_tuple(q.rows ? give(q.rows->code_view()) : py::none(), q.rows ? give(q.rows->scale_view()) : py::none(),
                        q.cols ? give(q.cols->code_view()) : py::none(), q.cols ? give(q.cols->scale_view()) : py::none(),
                        give(q.sums));
}

py::object py_quantize_any(const Tensor& x, bool square) {
  if (!float_type(x) || x.dim() < 1 || !ordinary(x, x) || (square && x.dim() != 2)) return py::none();
  const Quantized q = quantize(x, square, true, false, Tensor(), Tensor(), -1);
  Tensor codes = q.rows->code_view(), scales = q.rows->scale_view();
  if (x.dim() != 2) {              // splitting the rows of a strided matrix is a view
    codes = codes.view(x.sizes());
    scales = scales.view(with_last(x, scales.size(1)));
  }
  return py::make_tuple(give(codes), give(scales));
}

// A public operand: codes that TMA cannot address (rows not on 16-byte boundaries, or not contiguous) are copied once.
Codes operand_of(const Tensor& codes, const Tensor& scales, bool square) {
  Codes c;
  c.rows = codes.numel() / codes.size(-1);
  c.cols = codes.size(-1);
  checked(c.rows);
  Tensor m = codes;
  if (m.dim() != 2) m = m.reshape({c.rows, c.cols});
  const int64_t pitch = c.rows > 1 ? m.stride(0) : pitch_of(c.cols);
  if ((m.stride(1) != 1 && c.cols > 1) || pitch % 16 || pitch < c.cols || reinterpret_cast<uintptr_t>(m.const_data_ptr()) % 16) {
    c.codes = empty({c.rows, pitch_of(c.cols)}, CODES, m);
    c.codes.narrow(1, 0, c.cols).view(at::kByte).copy_(m.view(at::kByte));
  } else {
    // rows `pitch` bytes apart, as JbScaledOperand wants them; the view is never read through torch
    c.codes = m;
  }
  c.scales = scales.dim() == 2 ? scales : scales.reshape({c.rows, scales.size(-1)});
  c.scale_row = c.scales.stride(0);
  c.scale_k = c.scales.stride(1);
  c.square = square;
  return c;
}
JbScaledOperand describe(const Codes& c) {
  JbScaledOperand o = c.operand();
  o.pitch = c.rows > 1 ? c.codes.stride(0) : pitch_of(c.cols);
  return o;
}

py::object py_scaled_matmul(const Tensor& a_codes, const Tensor& a_scales, bool a_square, const Tensor& b_codes, const Tensor& b_scales,
                            bool b_square, const Optional& bias, int out_type) {
  if (!matrix_codes(a_codes, a_scales, a_square, a_codes) || !matrix_codes(b_codes, b_scales, b_square, a_codes) || b_codes.dim() != 2 ||
      a_codes.size(-1) != b_codes.size(1) || !vector_of(bias, b_codes.size(0), a_codes))
    return py::none();
  const c10::cuda::CUDAGuard guard(a_codes.device());
  const Codes a = operand_of(a_codes, a_scales, a_square), b = operand_of(b_codes, b_scales, b_square);
  return give(product(describe(a), describe(b), a.cols, opt(bias), out_type, with_last(a_codes, b.rows), a_codes));
}

py::object py_rms_quantize(const Tensor& x, const Optional& gain, double eps, const Optional& residual, bool want_rstd) {
  if (!norm_args(x, gain, residual, eps)) return py::none();
  const Normed n = rms_forward(x, opt(gain), eps, opt(residual), -1, true, want_rstd);
  Tensor codes = n.codes->code_view(), scales = n.codes->scale_view();
  if (x.dim() != 2) {
    codes = codes.view(x.sizes());
    scales = scales.view(with_last(x, scales.size(1)));
  }
  return py::make_tuple(give(codes), give(scales), give(n.sum), give(n.rstd));
}

// Inference forms with a prepared weight: quantisation (with or without the norm) and product, two launches.
py::object py_linear_prepared(const Tensor& x, const Tensor& w_codes, const Tensor& w_scales, bool w_square, const Optional& bias) {
  if (!float_type(x) || x.dim() < 1 || !ordinary(x, x) || !matrix_codes(w_codes, w_scales, w_square, x) || w_codes.dim() != 2 ||
      w_codes.size(1) != x.size(-1) || !vector_of(bias, w_codes.size(0), x) || traced(x) || traced(bias))
    return py::none();
  const c10::cuda::CUDAGuard guard(x.device());
  const Quantized q = quantize(x, false, true, false, Tensor(), Tensor(), -1);
  const Codes w = operand_of(w_codes, w_scales, w_square);
  return give(product(q.rows->operand(), describe(w), w.cols, opt(bias), autocast_type(x), with_last(x, w.rows), x));
}
py::object py_norm_linear_prepared(const Tensor& x, const Optional& gain, double eps, const Optional& residual, const Tensor& w_codes,
                                   const Tensor& w_scales, bool w_square, const Optional& bias) {
  if (!norm_args(x, gain, residual, eps) || !matrix_codes(w_codes, w_scales, w_square, x) || w_codes.dim() != 2 ||
      w_codes.size(1) != x.size(-1) || !vector_of(bias, w_codes.size(0), x) ||
      traced(x) || traced(gain) || traced(residual) || traced(bias))
    return py::none();
  const c10::cuda::CUDAGuard guard(x.device());
  const Normed n = rms_forward(x, opt(gain), eps, opt(residual), -1, true, false);
  const Codes w = operand_of(w_codes, w_scales, w_square);
  return py::make_tuple(give(product(n.codes->operand(), describe(w), w.cols, opt(bias), autocast_type(x), with_last(x, w.rows), x)),
                        give(n.sum));
}

bool weight_args(const Tensor& x, const Tensor& w, const Optional& b) {
  return float_type(w) && ordinary(w, x) && w.dim() == 2 && w.size(1) == x.size(-1) && vector_of(b, w.size(0), x);
}
py::object py_scaled_linear(const Tensor& x, const Tensor& w, const Optional& b) {
  if (!float_type(x) || x.dim() < 1 || !ordinary(x, x) || !weight_args(x, w, b)) return py::none();
  const bool grad = at::GradMode::is_enabled();
  return give(ScaledLinear::apply(x, w, b, static_cast<int64_t>(autocast_type(x)), grad && wants(x), grad && wants(w)));
}
py::tuple pair_of(const variable_list& v) { return py::make_tuple(give(v[0]), v.size() > 1 ? give(v[1]) : py::none()); }
py::object py_rms_norm(const Tensor& x, const Optional& gain, const Optional& residual, double eps) {
  if (!norm_args(x, gain, residual, eps)) return py::none();
  const bool need = at::GradMode::is_enabled() && (wants(x) || wants(gain) || wants(residual));
  const int64_t y_type = at::autocast::is_autocast_enabled(at::kCUDA) ? 0 : type_of(x.scalar_type());
  return pair_of(RmsNorm::apply(x, gain, residual, eps, y_type, need));
}
py::object py_rms_norm_linear(const Tensor& x, const Optional& gain, const Tensor& w, const Optional& b, const Optional& residual,
                              double eps) {
  if (!norm_args(x, gain, residual, eps) || !weight_args(x, w, b)) return py::none();
  const bool grad = at::GradMode::is_enabled();
  return pair_of(RmsNormLinear::apply(x, gain, w, b, residual, eps, static_cast<int64_t>(autocast_type(x)),
                                      grad && (wants(x) || wants(gain) || wants(residual)), grad && wants(w)));
}

void init(const py::dict& entry) {
  auto take = [&](auto& slot, const char* name) {
    slot = reinterpret_cast<std::decay_t<decltype(slot)>>(entry[name].cast<uintptr_t>());
  };
  take(api.gemm, "jb_scaled_gemm");
  take(api.quantize, "jb_quantize");
  take(api.column_sum, "jb_column_sum");
  take(api.rms_max_cols, "jb_rms_max_cols");
  take(api.rms_fwd, "jb_rms_norm_fwd");
  take(api.rms_bwd_parts, "jb_rms_bwd_parts");
  take(api.rms_bwd, "jb_rms_norm_bwd");
}

}  // namespace

PYBIND11_MODULE(_jb_torch, m) {
  m.def("init", &init);
  m.def("set_status", &set_status);
  m.def("quantize_any", &py_quantize_any);
  m.def("launches", [] { return launches.load(std::memory_order_relaxed); });
  m.def("quantize", &py_quantize);
  m.def("scaled_matmul", &py_scaled_matmul);
  m.def("rms_quantize", &py_rms_quantize);
  m.def("linear_prepared", &py_linear_prepared);
  m.def("norm_linear_prepared", &py_norm_linear_prepared);
  m.def("scaled_linear", &py_scaled_linear);
  m.def("rms_norm", &py_rms_norm);
  m.def("rms_norm_linear", &py_rms_norm_linear);
}
