// Python bindings of the preference-tuning kernels declared in tuning_api.h.  Outputs and workspaces are allocated here, for the call
// alone: two calls on two streams, or two captured graphs, share nothing.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "ops_api.h"
#include "tuning_api.h"

const unsigned long long* nmtg_seed_word(int device);       // bindings.cpp

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
void ck(const char* err) {
  if (err) throw std::runtime_error(std::string("nmtgminor_b200 kernel launch failed: ") + err);
}
int dtype_code(const Tensor& t, const char* name) {
  if (t.scalar_type() == at::kFloat) return 0;
  if (t.scalar_type() == at::kBFloat16) return 1;
  if (t.scalar_type() == at::kHalf) return 2;
  TORCH_CHECK(false, name, " must be float32, bfloat16 or float16");
  return -1;
}
uintptr_t address(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }
void need(const Tensor& t, const Tensor& like, at::ScalarType ty, int64_t n, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.is_contiguous() && t.scalar_type() == ty && t.numel() == n, name,
              ": wrong device, layout, dtype or size");
}
const float* opt_f32(const OptTensor& t, const Tensor& like, int64_t n, const char* name) {
  if (!t.has_value()) return nullptr;
  need(*t, like, at::kFloat, n, name);
  return t->data_ptr<float>();
}

// logits [rows, vocab] with adjacent elements in rows that do not overlap, labels [rows]
NmtgRows rows_of(const Tensor& logits, const Tensor& labels, int64_t pad, double temperature) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(1) >= 1 && (logits.stride(1) == 1 || logits.size(1) == 1 || logits.numel() == 0),
              "logits must be rows of adjacent elements on a GPU");
  TORCH_CHECK(logits.size(0) <= 1 || logits.stride(0) >= logits.size(1), "the rows of the logits overlap");
  TORCH_CHECK(logits.size(0) < (1 << 30) && logits.size(1) < (1LL << 31) - 64, "logits: too many rows or words");
  need(labels, logits, at::kLong, logits.size(0), "labels");
  TORCH_CHECK(temperature > 0.0 && std::isfinite(1.0 / temperature), "temperature must be positive");
  NmtgRows r = {};
  r.logits = logits.data_ptr();
  r.labels = labels.data_ptr<int64_t>();
  r.rows = static_cast<int>(logits.size(0));
  r.vocab = static_cast<int>(logits.size(1));
  r.dtype = dtype_code(logits, "logits");
  r.ld = logits.size(0) > 1 ? logits.stride(0) : logits.size(1);
  r.inv_temperature = static_cast<float>(1.0 / temperature);
  r.pad = pad;
  r.grad_scale = 1.f;
  TORCH_CHECK(address(logits) % logits.element_size() == 0, "logits: misaligned elements");
  return r;
}

// a gradient laid out as the logits are: the same row stride, the same address modulo 16 bytes
Tensor grad_like(const Tensor& logits, const NmtgRows& r) {
  const int64_t before = static_cast<int64_t>(address(logits) % 16) / logits.element_size();
  const int64_t n = r.rows > 0 ? (r.rows - 1) * r.ld + r.vocab : 0;
  return at::empty({before + n}, logits.options().requires_grad(false)).as_strided({r.rows, r.vocab}, {r.ld, 1}, before);
}

Tensor workspace(const Tensor& logits, NmtgRows& r, int pairs) {
  Tensor t = at::empty({nmtg_rows_workspace(r.rows, r.vocab, r.dtype, pairs)}, logits.options().dtype(at::kByte).requires_grad(false));
  r.workspace = t.data_ptr();
  return t;
}

// -> log-probabilities, and where `keep_stat` what their gradient needs
std::tuple<Tensor, OptTensor> row_scores(const Tensor& logits, const Tensor& labels, int64_t pad, double temperature, bool keep_stat) {
  NmtgRows r = rows_of(logits, labels, pad, temperature);
  c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  Tensor lp = at::empty({r.rows}, f32);
  OptTensor stat;
  if (keep_stat) {
    stat = at::empty({r.rows, 2}, f32);
    r.stat = reinterpret_cast<float2*>(stat->data_ptr<float>());
  }
  r.logprobs = lp.data_ptr<float>();
  const Tensor work = workspace(logits, r, 0);
  ck(nmtg_row_scores(&r, cur_stream()));
  return {lp, stat};
}

Tensor row_scores_grad(const Tensor& logits, const Tensor& labels, const Tensor& stat, const Tensor& weight, int64_t pad, double temperature) {
  NmtgRows r = rows_of(logits, labels, pad, temperature);
  c10::cuda::CUDAGuard guard(logits.device());
  need(stat, logits, at::kFloat, 2 * static_cast<int64_t>(r.rows), "stat");
  need(weight, logits, at::kFloat, r.rows, "weight");
  Tensor grad = grad_like(logits, r);
  r.grad = grad.data_ptr();
  r.stat = reinterpret_cast<float2*>(stat.data_ptr<float>());
  const Tensor work = workspace(logits, r, 0);
  ck(nmtg_row_scores_grad(&r, weight.data_ptr<float>(), cur_stream()));
  return grad;
}

// grad: 0 none, 1 a new tensor, 2 over the logits
Tensor grad_of(const Tensor& logits, NmtgRows& r, int64_t grad, const OptTensor& scale_at, double scale) {
  r.grad_scale = static_cast<float>(scale);
  r.grad_scale_at = opt_f32(scale_at, logits, 1, "grad_scale");
  Tensor g;
  if (grad == 0) return g;
  g = grad == 2 ? logits.detach() : grad_like(logits, r);
  r.grad = g.data_ptr();
  return g;
}

// What a gradient that is made in the backward pass takes from the forward pass beside the logits
struct Later { Tensor stat, coef, work; };

// -> loss, words clipped, KL, log-probabilities, gradient (or nothing)
std::tuple<Tensor, Tensor, Tensor, Tensor, OptTensor> policy_loss(const Tensor& logits, const Tensor& labels, const Tensor& old_logprobs,
                                                                  const Tensor& advantages, const OptTensor& ref_logprobs, double clip_low,
                                                                  double clip_high, double kl_coef, int64_t pad, double temperature,
                                                                  int64_t grad, const OptTensor& scale_at, double scale, Later* later) {
  NmtgRows r = rows_of(logits, labels, pad, temperature);
  c10::cuda::CUDAGuard guard(logits.device());
  NmtgPolicy p = {};
  need(old_logprobs, logits, at::kFloat, r.rows, "old_logprobs");
  need(advantages, logits, at::kFloat, r.rows, "advantages");
  p.old_logprobs = old_logprobs.data_ptr<float>();
  p.advantages = advantages.data_ptr<float>();
  p.ref_logprobs = opt_f32(ref_logprobs, logits, r.rows, "ref_logprobs");
  p.clip_low = static_cast<float>(1.0 - clip_low);
  p.clip_high = static_cast<float>(1.0 + clip_high);
  p.kl_coef = static_cast<float>(kl_coef);
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  Tensor lp = at::empty({r.rows}, f32), loss = at::empty({1}, f32), kl = at::empty({1}, f32), clipped = at::empty({1}, f32);
  const Tensor work = workspace(logits, r, 0);
  Tensor g = grad_of(logits, r, grad, scale_at, scale);
  r.logprobs = lp.data_ptr<float>();
  p.loss = loss.data_ptr<float>();
  p.kl = kl.data_ptr<float>();
  p.clipped = clipped.data_ptr<float>();
  if (later) {
    later->stat = at::empty({r.rows, 2}, f32);
    later->coef = at::empty({r.rows}, f32);
    r.stat = reinterpret_cast<float2*>(later->stat.data_ptr<float>());
    p.coef = later->coef.data_ptr<float>();
  }
  ck(nmtg_policy_loss(&r, &p, cur_stream()));
  return {loss, clipped, kl, lp, g.defined() ? OptTensor(g) : OptTensor()};
}

// -> loss, pairs ranked as preferred, sequences' log-probabilities, gradient (or nothing)
std::tuple<Tensor, Tensor, Tensor, OptTensor> preference_loss(const Tensor& logits, const Tensor& labels, const Tensor& cu, const OptTensor& ref,
                                                              int64_t kind, double beta, double smoothing, double margin, double nll_weight,
                                                              bool average, int64_t pad, double temperature, int64_t grad,
                                                              const OptTensor& scale_at, double scale, Later* later) {
  NmtgRows r = rows_of(logits, labels, pad, temperature);
  c10::cuda::CUDAGuard guard(logits.device());
  TORCH_CHECK(cu.numel() % 2 == 1 && cu.numel() < (1 << 28), "cu must hold 2 * pairs + 1 offsets");
  need(cu, logits, at::kInt, cu.numel(), "cu");
  NmtgPairs p = {};
  p.pairs = static_cast<int>(cu.numel() / 2);
  p.cu = cu.data_ptr<int>();
  p.ref = opt_f32(ref, logits, 2 * static_cast<int64_t>(p.pairs), "ref_logprobs");
  p.kind = static_cast<int>(kind);
  p.average = average;
  p.beta = static_cast<float>(beta);
  p.smoothing = static_cast<float>(smoothing);
  p.margin = static_cast<float>(margin);
  p.nll_weight = static_cast<float>(nll_weight);
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  Tensor seq = at::empty({2 * static_cast<int64_t>(p.pairs)}, f32), loss = at::empty({1}, f32), ranked = at::empty({1}, f32);
  const Tensor work = workspace(logits, r, p.pairs);
  Tensor g = grad_of(logits, r, grad, scale_at, scale);
  p.seq_logprobs = seq.data_ptr<float>();
  p.loss = loss.data_ptr<float>();
  p.ranked = ranked.data_ptr<float>();
  if (later) later->work = work;
  ck(nmtg_preference_loss(&r, &p, cur_stream()));
  return {loss, ranked, seq, g.defined() ? OptTensor(g) : OptTensor()};
}

// grad [rows, vocab] of one of the losses times the one element of `factor`
void scale_rows(Tensor& grad, const Tensor& factor) {
  TORCH_CHECK(grad.is_cuda() && grad.dim() == 2 && (grad.stride(1) == 1 || grad.size(1) == 1), "grad must be rows of adjacent elements on a GPU");
  need(factor, grad, at::kFloat, 1, "factor");
  c10::cuda::CUDAGuard guard(grad.device());
  NmtgRows r = {};
  r.grad = grad.data_ptr();
  r.rows = static_cast<int>(grad.size(0));
  r.vocab = static_cast<int>(grad.size(1));
  r.dtype = dtype_code(grad, "grad");
  r.ld = grad.size(0) > 1 ? grad.stride(0) : grad.size(1);
  ck(nmtg_scale_rows(&r, factor.data_ptr<float>(), cur_stream()));
}

// ---- embedding -----------------------------------------------------------------------------------------------------------
void need_dense(const Tensor& t, const Tensor& like, int64_t rows, int64_t width, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.is_contiguous() && t.dim() == 2 && t.size(0) == rows && t.size(1) == width,
              name, ": wrong device, layout or size");
}

Tensor embed_rows(const Tensor& tokens, const Tensor& table, double scale) {
  TORCH_CHECK(table.is_cuda() && table.dim() == 2 && table.is_contiguous(), "table must be a dense matrix on a GPU");
  need(tokens, table, at::kLong, tokens.numel(), "tokens");
  TORCH_CHECK(tokens.numel() < (1 << 30) && table.size(0) < (1LL << 31) && table.size(1) < (1 << 30), "embedding: too large");
  c10::cuda::CUDAGuard guard(table.device());
  Tensor out = at::empty({tokens.numel(), table.size(1)}, table.options().requires_grad(false));
  ck(nmtg_embed_rows(tokens.data_ptr<int64_t>(), table.data_ptr(), out.data_ptr(), static_cast<int>(tokens.numel()),
                     static_cast<int>(table.size(0)), static_cast<int>(table.size(1)), dtype_code(table, "table"), static_cast<float>(scale),
                     cur_stream()));
  return out;
}

// dropout(table[tokens] * scale + pos_table[positions]) of bf16 tables whose width is a multiple of 16
Tensor embed_flat(const Tensor& tokens, const OptTensor& positions, const Tensor& table, const OptTensor& pos_table, double scale, double p,
                  int64_t seed, int64_t stream_id) {
  if (!pos_table.has_value() && p == 0.0) return embed_rows(tokens, table, scale);
  TORCH_CHECK(table.is_cuda() && table.dim() == 2 && table.is_contiguous() && table.scalar_type() == at::kBFloat16, "table must be a dense bf16 matrix on a GPU");
  const int64_t rows = tokens.numel(), width = table.size(1);
  need(tokens, table, at::kLong, rows, "tokens");
  if (positions.has_value()) need(*positions, table, at::kLong, rows, "positions");
  if (pos_table.has_value()) {
    need(*pos_table, table, at::kBFloat16, pos_table->numel(), "pos_table");
    TORCH_CHECK(pos_table->dim() == 2 && pos_table->size(1) == width && pos_table->size(0) >= 1, "pos_table: wrong size");
  }
  TORCH_CHECK(rows < (1 << 30) && table.size(0) >= 1 && table.size(0) < (1LL << 31) && width < (1 << 30), "embedding: too large");
  c10::cuda::CUDAGuard guard(table.device());
  Tensor out = at::empty({rows, width}, table.options().requires_grad(false));
  if (rows > 0)
    ck(nmtg_embed_fwd(tokens.data_ptr<int64_t>(), positions.has_value() ? positions->data_ptr<int64_t>() : nullptr, table.data_ptr(),
                      pos_table.has_value() ? pos_table->data_ptr() : nullptr, out.data_ptr(), static_cast<int>(rows), static_cast<int>(width),
                      static_cast<int>(table.size(0)), pos_table.has_value() ? static_cast<int>(pos_table->size(0)) : 1, static_cast<float>(scale),
                      static_cast<float>(p), static_cast<unsigned long long>(seed), static_cast<unsigned long long>(stream_id),
                      nmtg_seed_word(table.get_device()), cur_stream()));
  return out;
}

// Into `grad` (fp32 [keys, width], added to), or a new [keys, width] matrix of dy's type
Tensor embed_grad(const Tensor& tokens, const OptTensor& positions, const Tensor& dy, const OptTensor& grad, int64_t vocab, int64_t keys,
                  double scale, double p, int64_t seed, int64_t stream_id, int64_t pad) {
  TORCH_CHECK(dy.is_cuda() && dy.dim() == 2, "dy must be a matrix on a GPU");
  const int64_t rows = tokens.numel(), width = dy.size(1);
  need(tokens, dy, at::kLong, rows, "tokens");
  need_dense(dy, dy, rows, width, "dy");
  if (positions.has_value()) need(*positions, dy, at::kLong, rows, "positions");
  TORCH_CHECK(rows < (1 << 30) && vocab >= 0 && vocab < (1LL << 31) && keys >= 0 && keys < (1 << 30) && width < (1 << 30), "embedding: too large");
  TORCH_CHECK(p >= 0.0 && p < 1.0, "embedding: dropout must be in [0, 1)");
  c10::cuda::CUDAGuard guard(dy.device());
  NmtgEmbedGrad e = {};
  Tensor out;
  if (grad.has_value()) {
    out = *grad;
    need_dense(out, dy, keys, width, "grad");
    TORCH_CHECK(out.scalar_type() == at::kFloat, "grad must be float32");
  } else {
    out = at::empty({keys, width}, dy.options().requires_grad(false));
  }
  e.tokens = tokens.data_ptr<int64_t>();
  e.positions = positions.has_value() ? positions->data_ptr<int64_t>() : nullptr;
  e.dy = dy.data_ptr();
  e.grad = out.data_ptr();
  e.rows = static_cast<int>(rows);
  e.vocab = static_cast<int>(vocab);
  e.keys = static_cast<int>(keys);
  e.width = static_cast<int>(width);
  e.dtype = dtype_code(dy, "dy");
  e.accumulate = grad.has_value();
  e.pad = pad;
  e.scale = static_cast<float>(scale);
  e.p = static_cast<float>(p);
  e.seed = static_cast<unsigned long long>(seed);
  e.stream_id = static_cast<unsigned long long>(stream_id);
  e.seed_dev = nmtg_seed_word(dy.get_device());
  Tensor work = at::empty({nmtg_embed_grad_workspace(e.rows, e.keys, e.width)}, dy.options().dtype(at::kByte).requires_grad(false));
  e.workspace = work.data_ptr();
  e.stream = cur_stream();
  ck(nmtg_embed_grad(&e));
  return out;
}

// ---- activations kept in 8 bits ------------------------------------------------------------------------------------------
NmtgKept kept_of(const Tensor& like, int64_t rows, int64_t width, int64_t act, double p, int64_t seed, int64_t stream_id) {
  TORCH_CHECK(p >= 0.0 && p < 1.0, "kept: dropout must be in [0, 1)");
  NmtgKept k = {};
  k.rows = rows;
  k.width = k.ld_in = width;
  k.act = static_cast<int>(act);
  k.p = static_cast<float>(p);
  k.seed = static_cast<unsigned long long>(seed);
  k.stream_id = static_cast<unsigned long long>(stream_id);
  k.seed_dev = nmtg_seed_word(like.get_device());
  k.stream = cur_stream();
  return k;
}
void codes_of(NmtgKept& k, const Tensor& codes, const Tensor& scales) {
  const int64_t blocks = (k.width + 31) / 32;
  TORCH_CHECK(codes.is_cuda() && codes.is_contiguous() && codes.scalar_type() == at::kByte && codes.numel() == k.rows * blocks * 32 &&
              address(codes) % 8 == 0, "codes: wrong device, layout, dtype or size");
  need(scales, codes, at::kByte, k.rows * blocks, "scales");
  k.codes = codes.data_ptr<uint8_t>();
  k.scales = scales.data_ptr<uint8_t>();
}
void matrix(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (t.numel() == 0 || ((t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) == 1 || t.stride(0) >= t.size(1)))), name,
              " must be rows of adjacent elements on a GPU");
}
std::tuple<Tensor, Tensor> new_codes(const Tensor& x) {
  const int64_t blocks = (x.size(1) + 31) / 32;
  const auto o = x.options().dtype(at::kByte).requires_grad(false);
  return {at::empty({x.size(0), blocks * 32}, o), at::empty({x.size(0), blocks}, o)};
}

// x [rows, width] -> codes [rows, 32 * blocks], scales [rows, blocks]
std::tuple<Tensor, Tensor> kept_quantise(const Tensor& x) {
  matrix(x, "x");
  c10::cuda::CUDAGuard guard(x.device());
  NmtgKept k = kept_of(x, x.size(0), x.size(1), 0, 0.0, 0, 0);
  auto [codes, scales] = new_codes(x);
  codes_of(k, codes, scales);
  k.in = x.data_ptr();
  k.ld_in = x.size(0) > 1 ? x.stride(0) : x.size(1);
  k.dtype = dtype_code(x, "x");
  ck(nmtg_kept_quantise(&k));
  return {codes, scales};
}

// -> x' (where `plain`), dropout(act(x')) (where act is not negative)
std::tuple<OptTensor, OptTensor> kept_restore(const Tensor& codes, const Tensor& scales, int64_t width, at::ScalarType dtype, bool plain, int64_t act,
                                              double p, int64_t seed, int64_t stream_id) {
  TORCH_CHECK(codes.is_cuda() && codes.dim() == 2, "codes must be a matrix on a GPU");
  c10::cuda::CUDAGuard guard(codes.device());
  NmtgKept k = kept_of(codes, codes.size(0), width, act < 0 ? 0 : act, act < 0 ? 0.0 : p, seed, stream_id);
  codes_of(k, codes, scales);
  const auto o = codes.options().dtype(dtype);
  OptTensor x, h;
  if (plain) { x = at::empty({k.rows, width}, o); k.out = x->data_ptr(); k.dtype = dtype_code(*x, "x"); }
  if (act >= 0) { h = at::empty({k.rows, width}, o); k.out2 = h->data_ptr(); k.dtype = dtype_code(*h, "h"); }
  if (plain || act >= 0) ck(nmtg_kept_restore(&k));
  return {x, h};
}

// -> dropout(act(z)), codes and scales where `keep`
std::tuple<Tensor, OptTensor, OptTensor> kept_forward(const Tensor& z, int64_t act, bool keep, double p, int64_t seed, int64_t stream_id) {
  matrix(z, "z");
  c10::cuda::CUDAGuard guard(z.device());
  NmtgKept k = kept_of(z, z.size(0), z.size(1), act, p, seed, stream_id);
  Tensor y = at::empty({z.size(0), z.size(1)}, z.options().requires_grad(false));
  OptTensor codes, scales;
  if (keep) {
    auto [c, s] = new_codes(z);
    codes_of(k, c, s);
    codes = c;
    scales = s;
  }
  k.in = z.data_ptr();
  k.ld_in = z.size(0) > 1 ? z.stride(0) : z.size(1);
  k.out = y.data_ptr();
  k.dtype = dtype_code(z, "z");
  ck(nmtg_kept_forward(&k));
  return {y, codes, scales};
}

Tensor kept_backward(const Tensor& dy, const Tensor& codes, const Tensor& scales, int64_t act, double p, int64_t seed, int64_t stream_id) {
  matrix(dy, "dy");
  TORCH_CHECK(codes.device() == dy.device(), "codes and dy are on different devices");
  c10::cuda::CUDAGuard guard(dy.device());
  NmtgKept k = kept_of(dy, dy.size(0), dy.size(1), act, p, seed, stream_id);
  codes_of(k, codes, scales);
  Tensor dz = at::empty({dy.size(0), dy.size(1)}, dy.options().requires_grad(false));
  k.in = dy.data_ptr();
  k.ld_in = dy.size(0) > 1 ? dy.stride(0) : dy.size(1);
  k.out = dz.data_ptr();
  k.dtype = dtype_code(dy, "dy");
  ck(nmtg_kept_backward(&k));
  return dz;
}

// ---- autograd nodes ------------------------------------------------------------------------------------------------------
// In C++, because a node in Python costs about as much as the kernels of a small call (forward and backward pass of an empty one 57 us).
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

Tensor plain_rows(const Tensor& t) {
  const bool rows = t.dim() != 2 || (t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) >= t.size(1)));
  return rows ? t : t.contiguous();
}

// The kernels' gradients are not differentiable again: create_graph would leave their part out without a word
void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": no second derivative (create_graph)");
}

struct ScoresNode : Function<ScoresNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, int64_t pad, double temperature) {
    auto [lp, stat] = row_scores(logits, labels, pad, temperature, true);
    ctx->save_for_backward({logits, labels, *stat});
    ctx->saved_data["pad"] = pad;
    ctx->saved_data["temperature"] = temperature;
    return lp;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("token_logprobs");
    const auto saved = ctx->get_saved_variables();
    const Tensor weight = g[0].to(at::kFloat).contiguous();
    return {row_scores_grad(saved[0], saved[1], saved[2], weight, ctx->saved_data["pad"].toInt(), ctx->saved_data["temperature"].toDouble()),
            Tensor(), Tensor(), Tensor()};
  }
};

// The two losses: the gradient is made with the loss and belongs to the first backward pass.  Not that of fp16 logits whose upstream factor is still to
// come: rounded to fp16 without it, entries below 2^-25 would be 0 (a tenth of a vocabulary of 51865 words), whatever the loss is scaled by.  It
// is made in the backward pass, with the factor, from the rows' sums and coefficients: the second of the paired loss's two passes as before, and one
// more pass of the policy loss.  bf16 has the range of 32 bits: its entries are rounded once more by a factor that is no power of two.
bool made_later(const Tensor& logits, bool prescaled) { return !prescaled && logits.scalar_type() == at::kHalf; }

variable_list loss_backward(AutogradContext* ctx, const variable_list& g, size_t inputs) {
  once("preference or policy loss");
  variable_list out(inputs);
  if (!g[0].defined()) return out;
  TORCH_CHECK(!ctx->saved_data["spent"].toBool(), "a second backward pass through a preference or policy loss: its gradient went to the first one");
  if (!ctx->saved_data["later"].toBool()) {
    Tensor grad = ctx->get_saved_variables()[0].detach();
    if (!ctx->saved_data["prescaled"].toBool()) scale_rows(grad, g[0].to(at::kFloat).contiguous());
    out[0] = grad;
  } else {
    const auto saved = ctx->get_saved_variables();                // logits, labels, and statistics and coefficients or the workspace
    const Tensor logits = saved[0].detach(), factor = g[0].to(at::kFloat).contiguous();
    NmtgRows r = rows_of(logits, saved[1], ctx->saved_data["pad"].toInt(), ctx->saved_data["temperature"].toDouble());
    c10::cuda::CUDAGuard guard(logits.device());
    const bool inplace = ctx->saved_data["inplace"].toBool();
    out[0] = grad_of(logits, r, inplace ? 2 : 1, factor, 1.0);
    if (saved.size() == 4) {
      r.stat = reinterpret_cast<float2*>(saved[2].data_ptr<float>());
      const Tensor work = workspace(logits, r, 0);
      ck(nmtg_row_scores_grad(&r, saved[3].data_ptr<float>(), cur_stream()));
    } else {
      r.workspace = saved[2].data_ptr();
      ck(nmtg_preference_grad(&r, static_cast<int>(ctx->saved_data["pairs"].toInt()), cur_stream()));
    }
    if (inplace) logits.unsafeGetTensorImpl()->bump_version();
  }
  ctx->saved_data["spent"] = true;
  return out;
}
void loss_forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, const OptTensor& grad, const Later& later, int64_t pairs, int64_t pad,
                  double temperature, bool inplace, bool prescaled, const variable_list& plain) {
  ctx->saved_data["spent"] = false;
  ctx->saved_data["later"] = !grad.has_value();
  if (grad.has_value()) {
    ctx->saved_data["prescaled"] = prescaled;
    if (inplace) logits.unsafeGetTensorImpl()->bump_version();    // what another node has saved of the logits is gone
    ctx->save_for_backward({*grad});                              // as the logits' version is now: a change behind the call is refused
  } else {
    if (later.work.defined()) ctx->save_for_backward({logits, labels, later.work});
    else ctx->save_for_backward({logits, labels, later.stat, later.coef});
    ctx->saved_data["pairs"] = pairs;
    ctx->saved_data["pad"] = pad;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["inplace"] = inplace;
  }
  ctx->mark_non_differentiable(plain);
  ctx->set_materialize_grads(false);
}

struct PolicyNode : Function<PolicyNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, const Tensor& old_logprobs, const Tensor& advantages,
                               const OptTensor& ref, double clip_low, double clip_high, double kl_coef, int64_t pad, double temperature, bool inplace,
                               const OptTensor& scale_at, double scale, bool prescaled) {
    Later later;
    const bool wait = made_later(logits, prescaled);
    auto [loss, clipped, kl, lp, grad] = policy_loss(logits, labels, old_logprobs, advantages, ref, clip_low, clip_high, kl_coef, pad, temperature,
                                                     wait ? 0 : inplace ? 2 : 1, scale_at, scale, wait ? &later : nullptr);
    loss_forward(ctx, logits, labels, grad, later, 0, pad, temperature, inplace, prescaled, {clipped, kl, lp});
    return {loss, clipped, kl, lp};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) { return loss_backward(ctx, g, 14); }
};

struct PreferenceNode : Function<PreferenceNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, const Tensor& cu, const OptTensor& ref, int64_t kind,
                               double beta, double smoothing, double margin, double nll_weight, bool average, int64_t pad, double temperature,
                               bool inplace, const OptTensor& scale_at, double scale, bool prescaled) {
    Later later;
    const bool wait = made_later(logits, prescaled);
    auto [loss, ranked, seq, grad] = preference_loss(logits, labels, cu, ref, kind, beta, smoothing, margin, nll_weight, average, pad, temperature,
                                                     wait ? 0 : inplace ? 2 : 1, scale_at, scale, wait ? &later : nullptr);
    loss_forward(ctx, logits, labels, grad, later, cu.numel() / 2, pad, temperature, inplace, prescaled, {ranked, seq});
    return {loss, ranked, seq};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) { return loss_backward(ctx, g, 16); }
};

struct EmbedNode : Function<EmbedNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& tokens, double scale, int64_t pad) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = pad;
    ctx->saved_data["words"] = table.size(0);
    return embed_rows(tokens, table, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("embedding with a sorted gradient");
    const auto saved = ctx->get_saved_variables();
    const int64_t words = ctx->saved_data["words"].toInt();
    return {embed_grad(saved[0], OptTensor(), g[0].contiguous(), OptTensor(), words, words, ctx->saved_data["scale"].toDouble(), 0.0, 0, 0,
                       ctx->saved_data["pad"].toInt()),
            Tensor(), Tensor(), Tensor()};
  }
};

// A table of the flat store: gradients are added to the store's buffers.  `anchor` is an empty tensor with a gradient that makes autograd record the node:
// one of the call's own, since a leaf that an eager graph holds, too, could not be passed in a backward pass that is being captured.
struct FlatEmbedNode : Function<FlatEmbedNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& /*anchor*/, const Tensor& tokens, const OptTensor& positions, const Tensor& table,
                        const OptTensor& pos_table, const OptTensor& gtable, const OptTensor& gpos, double scale, double p, int64_t seed,
                        int64_t stream_id, int64_t pad) {
    ctx->save_for_backward({tokens, positions.has_value() ? *positions : Tensor()});      // the buffers are added to, and so not among them
    ctx->saved_data["gtable"] = gtable;
    ctx->saved_data["gpos"] = gpos;
    ctx->saved_data["words"] = table.size(0);
    ctx->saved_data["numbers"] = std::vector<double>{scale, p};
    ctx->saved_data["ids"] = std::vector<int64_t>{seed, stream_id, pad};
    ctx->set_materialize_grads(false);
    return embed_flat(tokens, positions, table, pos_table, scale, p, seed, stream_id);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(12);
    if (!g[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor dy = g[0].contiguous(), tokens = saved[0];
    const OptTensor positions = saved[1].defined() ? OptTensor(saved[1]) : OptTensor();
    const int64_t words = ctx->saved_data["words"].toInt();
    const auto numbers = ctx->saved_data["numbers"].toDoubleVector();
    const auto ids = ctx->saved_data["ids"].toIntVector();
    const auto optional = [&](const char* name) { const c10::IValue& v = ctx->saved_data[name]; return v.isNone() ? OptTensor() : OptTensor(v.toTensor()); };
    const OptTensor gtable = optional("gtable"), gpos = optional("gpos");
    if (gtable.has_value()) embed_grad(tokens, OptTensor(), dy, gtable, words, words, numbers[0], numbers[1], ids[0], ids[1], ids[2]);
    if (gpos.has_value())
      embed_grad(tokens, positions.has_value() ? positions : OptTensor(at::zeros_like(tokens)), dy, gpos, words, gpos->size(0), 1.0, numbers[1], ids[0],
                 ids[1], ids[2]);
    return out;
  }
};

struct ActivationNode : Function<ActivationNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, int64_t act, double p, int64_t seed, int64_t stream_id) {
    auto [y, codes, scales] = kept_forward(z, act, true, p, seed, stream_id);
    ctx->save_for_backward({*codes, *scales});
    ctx->saved_data["act"] = act;
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["stream"] = stream_id;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("activation kept in 8 bits");
    const auto saved = ctx->get_saved_variables();
    return {kept_backward(plain_rows(g[0]), saved[0], saved[1], ctx->saved_data["act"].toInt(), ctx->saved_data["p"].toDouble(),
                          ctx->saved_data["seed"].toInt(), ctx->saved_data["stream"].toInt()),
            Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

}  // namespace

void bind_tuning_ops(pybind11::module& m) {
  m.def("row_scores", &row_scores);
  m.def("row_scores_grad", &row_scores_grad);
  m.def("policy_loss", [](const Tensor& logits, const Tensor& labels, const Tensor& old_logprobs, const Tensor& advantages, const OptTensor& ref,
                          double clip_low, double clip_high, double kl_coef, int64_t pad, double temperature, int64_t grad, const OptTensor& scale_at,
                          double scale) {
    return policy_loss(logits, labels, old_logprobs, advantages, ref, clip_low, clip_high, kl_coef, pad, temperature, grad, scale_at, scale, nullptr);
  });
  m.def("preference_loss", [](const Tensor& logits, const Tensor& labels, const Tensor& cu, const OptTensor& ref, int64_t kind, double beta,
                              double smoothing, double margin, double nll_weight, bool average, int64_t pad, double temperature, int64_t grad,
                              const OptTensor& scale_at, double scale) {
    return preference_loss(logits, labels, cu, ref, kind, beta, smoothing, margin, nll_weight, average, pad, temperature, grad, scale_at, scale, nullptr);
  });
  m.def("scale_rows", &scale_rows);
  m.def("row_scores_node", [](const Tensor& logits, const Tensor& labels, int64_t pad, double temperature) {
    return ScoresNode::apply(logits, labels, pad, temperature);
  });
  m.def("policy_loss_node", [](const Tensor& logits, const Tensor& labels, const Tensor& old_logprobs, const Tensor& advantages, const OptTensor& ref,
                               double clip_low, double clip_high, double kl_coef, int64_t pad, double temperature, bool inplace,
                               const OptTensor& scale_at, double scale, bool prescaled) {
    auto o = PolicyNode::apply(logits, labels, old_logprobs, advantages, ref, clip_low, clip_high, kl_coef, pad, temperature, inplace, scale_at, scale,
                               prescaled);
    return std::make_tuple(o[0], o[1], o[2], o[3]);
  });
  m.def("preference_loss_node", [](const Tensor& logits, const Tensor& labels, const Tensor& cu, const OptTensor& ref, int64_t kind, double beta,
                                   double smoothing, double margin, double nll_weight, bool average, int64_t pad, double temperature, bool inplace,
                                   const OptTensor& scale_at, double scale, bool prescaled) {
    auto o = PreferenceNode::apply(logits, labels, cu, ref, kind, beta, smoothing, margin, nll_weight, average, pad, temperature, inplace, scale_at,
                                   scale, prescaled);
    return std::make_tuple(o[0], o[1], o[2]);
  });
  m.def("embed_rows_node", [](const Tensor& table, const Tensor& tokens, double scale, int64_t pad) {
    return EmbedNode::apply(table, tokens, scale, pad);
  });
  m.def("embed_flat_node", [](const Tensor& tokens, const OptTensor& positions, const Tensor& table, const OptTensor& pos_table,
                              const OptTensor& gtable, const OptTensor& gpos, double scale, double p, int64_t seed, int64_t stream_id, int64_t pad) {
    const Tensor anchor = at::empty({0}, table.options().dtype(at::kFloat)).requires_grad_(true);
    return FlatEmbedNode::apply(anchor, tokens, positions, table, pos_table, gtable, gpos, scale, p, seed, stream_id, pad);
  });
  m.def("activation_node", [](const Tensor& z, int64_t act, double p, int64_t seed, int64_t stream_id) {
    return ActivationNode::apply(z, act, p, seed, stream_id);
  });
  m.def("embed_rows", &embed_rows);
  m.def("embed_grad", &embed_grad);
  m.def("kept_quantise", &kept_quantise);
  m.def("kept_restore", [](const Tensor& codes, const Tensor& scales, int64_t width, pybind11::object dtype, bool plain, int64_t act, double p,
                           int64_t seed, int64_t stream_id) {
    return kept_restore(codes, scales, width, torch::python::detail::py_object_to_dtype(dtype), plain, act, p, seed, stream_id);
  });
  m.def("kept_forward", &kept_forward);
  m.def("kept_backward", &kept_backward);
}
