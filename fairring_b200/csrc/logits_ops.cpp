#include "logits_ops.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <cmath>
#include <limits>
#include <optional>
#include <tuple>

#include "kernels/local_kernels.h"

namespace fairring {
namespace {
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int multiprocessors() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

void checkLogits(const at::Tensor& logits) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() >= 1, "logits must be a CUDA tensor of at least one dimension");
  TORCH_CHECK_VALUE(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16 ||
                        logits.scalar_type() == at::kHalf,
                    "logits must be fp32, bf16 or fp16");
  TORCH_CHECK_VALUE(logits.size(-1) > 0 && logits.size(-1) <= kMostVocab, "logits must have from 1 to ", kMostVocab,
                    " columns, not ", logits.size(-1));
  TORCH_CHECK_VALUE(logits.numel() / logits.size(-1) <= INT32_MAX, "too many rows");
}

void checkTemperature(double t) {
  TORCH_CHECK_VALUE(t >= 1e-30 && t <= 1e30, "temperature must be positive and finite, from 1e-30 to 1e30, not ", t);
}

// Logits whose rows the kernels can walk, and how: the leading dimensions as two levels of strides, the last
// dimension without gaps and, where a gradient is laid out alike, no row over another.  Others are copied.
struct Rows {
  at::Tensor t;
  LogitRows x;
};

std::optional<LogitRows> walk(const at::Tensor& t) {
  const int64_t vocab = t.size(-1);
  if (vocab > 1 && t.stride(-1) != 1) return std::nullopt;
  // Levels from the inside out; a level that continues the one inside it is part of it.
  int64_t count[2] = {1, 1}, stride[2] = {vocab, 0};
  int levels = 0;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    const int64_t n = t.size(d), s = t.stride(d);
    if (n == 1) continue;
    if (levels > 0 && s == count[levels - 1] * stride[levels - 1]) {
      count[levels - 1] *= n;
    } else if (levels < 2) {
      count[levels] = n;
      stride[levels++] = s;
    } else {
      return std::nullopt;
    }
  }
  // No row over another, whichever level is the outer one in memory.
  const int near = count[1] > 1 && stride[1] < stride[0] ? 1 : 0, far = 1 - near;
  if (count[near] > 1 && stride[near] < vocab) return std::nullopt;
  if (count[far] > 1 && stride[far] < (count[near] - 1) * stride[near] + vocab) return std::nullopt;
  LogitRows x;
  x.rows = count[0] * count[1];
  x.inner = count[0];
  x.outer_stride = stride[1];
  x.row_stride = stride[0];
  x.vocab = (int)vocab;
  x.type = t.scalar_type() == at::kFloat      ? LogitType::kFloat
           : t.scalar_type() == at::kBFloat16 ? LogitType::kBFloat16
                                              : LogitType::kHalf;
  return x;
}

Rows rowsOf(const at::Tensor& logits) {
  if (const auto x = walk(logits)) return {logits, *x};
  const at::Tensor t = logits.clone(at::MemoryFormat::Contiguous);
  return {t, *walk(t)};
}

// Where the logits' gradient goes: laid out as they are, so that a vector of the one is a vector of the other,
// unless they lie in a much larger tensor; those are copied first.
at::Tensor gradientFor(Rows& rows) {
  const auto extent = [](const LogitRows& x) {
    return (x.rows / x.inner - 1) * x.outer_stride + (x.inner - 1) * x.row_stride + x.vocab;
  };
  if (rows.x.rows > 0 && extent(rows.x) > rows.t.numel() + rows.t.numel() / 2) {
    rows.t = rows.t.clone(at::MemoryFormat::Contiguous);
    rows.x = *walk(rows.t);
  }
  if (rows.x.rows == 0) return at::empty(rows.t.sizes(), rows.t.options());
  const int64_t phase =
      (int64_t)(reinterpret_cast<uintptr_t>(rows.t.data_ptr()) % 16 / (uintptr_t)rows.t.element_size());
  const at::Tensor memory = at::empty({extent(rows.x) + phase}, rows.t.options());
  if (phase == 0 && rows.t.is_contiguous()) return memory.view(rows.t.sizes());
  return memory.as_strided(rows.t.sizes(), rows.t.strides(), phase);
}

// One value per row as a kernel reads it: fp32, and the distance between two rows' values, 0 for one value for all.
std::tuple<at::Tensor, int64_t> perRow(const at::Tensor& g) {
  at::Tensor t = g.scalar_type() == at::kFloat ? g : g.to(at::kFloat);
  bool same = true;
  for (int64_t d = 0; d < t.dim(); ++d) same = same && (t.size(d) == 1 || t.stride(d) == 0);
  if (same) return std::make_tuple(t, 0);
  return std::make_tuple(t.contiguous(), 1);
}

// Saved-tensor hooks may have brought it back in another layout.
at::Tensor dense(const at::Tensor& saved) { return saved.defined() ? saved.contiguous() : saved; }

// int64, contiguous, from integers of that shape on the logits' device.
at::Tensor checkTokens(const at::Tensor& tokens, const at::Tensor& logits, at::IntArrayRef sizes, const char* name) {
  TORCH_CHECK_VALUE(at::isIntegralType(tokens.scalar_type(), false), name, " must be integers, not ", tokens.scalar_type());
  TORCH_CHECK_VALUE(tokens.sizes() == sizes && tokens.device() == logits.device(), name, " must be ", sizes, " on ",
                    logits.device(), ", not ", tokens.sizes(), " on ", tokens.device());
  return tokens.to(at::kLong).contiguous();
}

// ---- log probabilities -----------------------------------------------------------
struct TokenLogProbs {
  at::Tensor log_probs, entropy, top_log_probs, top_tokens, stats;
};

TokenLogProbs tokenLogProbsForward(const Rows& rows, const std::optional<at::Tensor>& tokens, double temperature,
                                   bool entropy, int64_t top_k, bool keep) {
  const at::IntArrayRef lead = rows.t.sizes().slice(0, rows.t.dim() - 1);
  const auto fopt = rows.t.options().dtype(at::kFloat);
  std::vector<int64_t> wide(lead.begin(), lead.end());
  wide.push_back(top_k);
  TokenLogProbs out;
  if (tokens.has_value()) out.log_probs = at::empty(lead, fopt);
  if (entropy) out.entropy = at::empty(lead, fopt);
  if (top_k > 0) {
    out.top_log_probs = at::empty(wide, fopt);
    out.top_tokens = at::empty(wide, fopt.dtype(at::kLong));
  }
  if (keep) out.stats = at::empty({rows.x.rows, 2}, fopt);
  TokenLogProbsArgs a = {};
  a.tokens = tokens.has_value() ? tokens->data_ptr<int64_t>() : nullptr;
  a.temperature = temperature;
  a.log_probs = tokens.has_value() ? out.log_probs.data_ptr<float>() : nullptr;
  a.entropy = entropy ? out.entropy.data_ptr<float>() : nullptr;
  a.stats = keep ? out.stats.data_ptr<float>() : nullptr;
  a.k = (int)top_k;
  a.top_log_probs = top_k > 0 ? out.top_log_probs.data_ptr<float>() : nullptr;
  a.top_tokens = top_k > 0 ? out.top_tokens.data_ptr<int64_t>() : nullptr;
  const cudaError_t e =
      launchTokenLogProbs(rows.t.data_ptr(), rows.x, a, multiprocessors(), c10::cuda::getCurrentCUDAStream());
  TORCH_CHECK(e == cudaSuccess, "token_log_probs launch failed: ", cudaGetErrorString(e));
  return out;
}

// The gradient of the logits from torch's ops, where its own graph is wanted.
at::Tensor tokenLogProbsBackwardGraph(const at::Tensor& logits, const at::Tensor& tokens, double temperature,
                                      const at::Tensor& g_log_probs, const at::Tensor& g_entropy) {
  at::Tensor counts, known, wide = logits.to(at::kFloat);
  if (tokens.defined()) {  // a row that does not count is not looked at, be it NaN
    counts = tokens.ge(0).unsqueeze(-1);
    known = counts.logical_and(tokens.lt(logits.size(-1)).unsqueeze(-1));
    wide = wide.masked_fill(counts.logical_not(), 0.0);
  }
  const at::Tensor logp = at::log_softmax(wide / temperature, -1), p = logp.exp();
  at::Tensor grad = at::zeros_like(p);
  if (g_log_probs.defined()) {
    const at::Tensor at = tokens.unsqueeze(-1).where(known, at::zeros_like(tokens).unsqueeze(-1));
    const at::Tensor g = g_log_probs.unsqueeze(-1);
    grad = (at::zeros_like(p).scatter_(-1, at, 1.0) - p) * g;
  }
  if (g_entropy.defined()) {
    const at::Tensor finite = logp.masked_fill(p.eq(0), 0.0);
    const at::Tensor h = -(p * finite).sum(-1, true);
    grad = grad - p * (finite + h) * g_entropy.unsqueeze(-1);
  }
  if (counts.defined()) {
    grad = grad.masked_fill(known.logical_not(), std::numeric_limits<double>::quiet_NaN());
    grad = at::where(counts, grad, at::zeros_like(grad));
  }
  return (grad / temperature).to(logits.scalar_type());
}

struct TokenLogProbsNode : torch::autograd::Function<TokenLogProbsNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const std::optional<at::Tensor>& tokens,
                               double temperature, bool entropy, int64_t top_k) {
    const Rows rows = rowsOf(logits);
    const TokenLogProbs out = tokenLogProbsForward(rows, tokens, temperature, entropy, top_k, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, tokens.value_or(at::Tensor()), out.stats, out.entropy});
    ctx->saved_data["temperature"] = temperature;
    variable_list result, values;
    if (out.log_probs.defined()) result.push_back(out.log_probs);
    if (entropy) result.push_back(out.entropy);
    if (top_k > 0) {
      values = {out.top_log_probs, out.top_tokens};
      ctx->mark_non_differentiable(values);
      result.insert(result.end(), values.begin(), values.end());
    }
    return result;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], tokens = dense(saved[1]), stats = dense(saved[2]), entropy = dense(saved[3]);
    const double temperature = ctx->saved_data["temperature"].toDouble();
    at::Tensor g, h;
    size_t i = 0;
    if (tokens.defined()) g = grads[i++];
    if (entropy.defined()) h = grads[i++];
    const at::Tensor none;
    if (!g.defined() && !h.defined()) return {none, none, none, none, none};
    if (at::GradMode::is_enabled())
      return {tokenLogProbsBackwardGraph(logits, tokens, temperature, g, h), none, none, none, none};
    c10::cuda::CUDAGuard guard(logits.device());
    Rows rows = rowsOf(logits);
    const at::Tensor grad = gradientFor(rows);
    TokenLogProbsGrads a = {};
    at::Tensor g_rows, h_rows;
    if (g.defined()) std::tie(g_rows, a.g_stride) = perRow(g);
    if (h.defined()) std::tie(h_rows, a.h_stride) = perRow(h);
    a.tokens = tokens.defined() ? tokens.data_ptr<int64_t>() : nullptr;
    a.temperature = temperature;
    a.stats = stats.data_ptr<float>();
    a.entropy = entropy.defined() ? entropy.data_ptr<float>() : nullptr;
    a.g_log_probs = g.defined() ? g_rows.data_ptr<float>() : nullptr;
    a.g_entropy = h.defined() ? h_rows.data_ptr<float>() : nullptr;
    const cudaError_t e = launchTokenLogProbsBackward(rows.t.data_ptr(), rows.x, grad.data_ptr(), a,
                                                      c10::cuda::getCurrentCUDAStream());
    TORCH_CHECK(e == cudaSuccess, "token_log_probs backward launch failed: ", cudaGetErrorString(e));
    return {grad, none, none, none, none};
  }
};

// (log probabilities, entropy, top log probabilities, top tokens), None for what was not asked.
std::tuple<std::optional<at::Tensor>, std::optional<at::Tensor>, std::optional<at::Tensor>, std::optional<at::Tensor>>
tokenLogProbs(const at::Tensor& logits, std::optional<at::Tensor> tokens, double temperature, bool entropy,
              int64_t top_k) {
  checkLogits(logits);
  checkTemperature(temperature);
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= kMostTopTokens && top_k <= logits.size(-1),
                    "top_k must be from 0 to the vocabulary, ", logits.size(-1), ", and here to ", kMostTopTokens, ", not ", top_k);
  TORCH_CHECK_VALUE(tokens.has_value() || entropy || top_k > 0, "nothing is asked for: give tokens, entropy=True or top_k");
  c10::cuda::CUDAGuard guard(logits.device());
  if (tokens.has_value()) tokens = checkTokens(*tokens, logits, logits.sizes().slice(0, logits.dim() - 1), "tokens");
  std::tuple<std::optional<at::Tensor>, std::optional<at::Tensor>, std::optional<at::Tensor>, std::optional<at::Tensor>> out;
  if (at::GradMode::is_enabled() && logits.requires_grad() && (tokens.has_value() || entropy)) {
    const variable_list got = TokenLogProbsNode::apply(logits, tokens, temperature, entropy, top_k);
    size_t i = 0;
    if (tokens.has_value()) std::get<0>(out) = got[i++];
    if (entropy) std::get<1>(out) = got[i++];
    if (top_k > 0) {
      std::get<2>(out) = got[i++];
      std::get<3>(out) = got[i++];
    }
  } else {
    const TokenLogProbs got = tokenLogProbsForward(rowsOf(logits.detach()), tokens, temperature, entropy, top_k, false);
    if (tokens.has_value()) std::get<0>(out) = got.log_probs;
    if (entropy) std::get<1>(out) = got.entropy;
    if (top_k > 0) {
      std::get<2>(out) = got.top_log_probs;
      std::get<3>(out) = got.top_tokens;
    }
  }
  return out;
}

// ---- distillation ----------------------------------------------------------------
// `kept`: of every row 4 floats and, for the backward, its tokens' pairs; the number of rows that count, for the mean.
struct Distillation {
  at::Tensor loss, kept;
};
struct Kept {
  float* count;
  float* stats;
  void* pairs;
  Kept(const at::Tensor& kept, int64_t rows)
      : count(kept.data_ptr<float>()), stats(count + 4), pairs(stats + 4 * rows) {}  // 16-byte steps
};

Distillation distillationForward(const Rows& rows, const at::Tensor& tokens, const at::Tensor& log_probs,
                                 double temperature, bool rest, bool mean, bool keep) {
  const auto fopt = rows.t.options().dtype(at::kFloat);
  const auto stream = c10::cuda::getCurrentCUDAStream();
  const int64_t n = rows.x.rows, k = tokens.size(-1);
  Distillation out;
  out.kept = at::empty({4 + 4 * n + (keep ? 2 * k * n : 0) + (mean ? n : 0)}, fopt);
  const Kept kept(out.kept, n);
  out.loss = mean ? at::empty({}, fopt) : at::empty(rows.t.sizes().slice(0, rows.t.dim() - 1), fopt);
  float* losses = mean ? kept.stats + 4 * n + (keep ? 2 * k * n : 0) : out.loss.data_ptr<float>();
  DistillationArgs a;
  a.tokens = tokens.data_ptr<int64_t>();
  a.log_probs = log_probs.data_ptr<float>();
  a.k = (int)k;
  a.temperature = temperature;
  a.rest = rest;
  cudaError_t e = launchDistillation(rows.t.data_ptr(), rows.x, a, losses, kept.stats, keep ? kept.pairs : nullptr,
                                     multiprocessors(), stream);
  TORCH_CHECK(e == cudaSuccess, "distillation launch failed: ", cudaGetErrorString(e));
  if (mean) {
    e = launchDistillationMean(losses, kept.stats, n, out.loss.data_ptr<float>(), kept.count, stream);
    TORCH_CHECK(e == cudaSuccess, "distillation mean launch failed: ", cudaGetErrorString(e));
  }
  return out;
}

// The gradient of the logits from torch's ops, where its own graph is wanted.
at::Tensor distillationBackwardGraph(const at::Tensor& logits, const at::Tensor& tokens, const at::Tensor& log_probs,
                                     double temperature, bool rest, bool mean, const at::Tensor& g, const at::Tensor& kept) {
  const at::Tensor there = tokens.ge(0), bad = tokens.ge(logits.size(-1)).any(-1, true);
  const at::Tensor known = there.logical_and(tokens.lt(logits.size(-1)));
  const double low = -std::numeric_limits<double>::infinity();
  const at::Tensor at = tokens.where(known, at::zeros_like(tokens));
  const at::Tensor counts = (rest ? there : there.logical_and(log_probs.eq(low).logical_not())).any(-1, true);
  const at::Tensor z = logits.to(at::kFloat).masked_fill(counts.logical_not(), 0.0) / temperature;
  at::Tensor grad = at::softmax(z, -1), q;
  if (rest) {
    q = at::where(known, log_probs.exp(), at::zeros_like(log_probs));
    const at::Tensor mass = q.to(at::kDouble).sum(-1, true), some = 1 - mass;
    const at::Tensor left = at::where(some.ge(kLeastRest), some, at::zeros_like(some));
    const at::Tensor listed = at::zeros_like(z).scatter_add_(-1, at, known.to(z.scalar_type())).gt(0);
    const at::Tensor gone = listed.logical_or(z.eq(low)).all(-1, true);  // no other token has any probability
    const at::Tensor share =
        at::softmax(z.masked_fill(listed.logical_and(gone.logical_not()), low), -1).masked_fill(listed.logical_or(gone), 0.0);
    grad = grad * (mass + left).to(at::kFloat) - at::where(left.gt(0), share * left.to(at::kFloat), at::zeros_like(share));
  } else {
    // A row without any mass does not count; its softmax is NaN, which a factor of zero would hand on.
    const at::Tensor none = known.logical_not().logical_or(counts.logical_not());
    q = at::softmax((log_probs / temperature).masked_fill(known.logical_not(), low), -1).masked_fill(none, 0.0);
  }
  grad = grad.scatter_add(-1, at, -q);
  grad = grad.masked_fill(bad, std::numeric_limits<double>::quiet_NaN());
  const at::Tensor up = mean ? g.to(at::kFloat) / kept.select(0, 0) : g.to(at::kFloat).unsqueeze(-1);
  grad = at::where(counts, grad * (up / temperature), at::zeros_like(grad));
  return grad.to(logits.scalar_type());
}

struct DistillationNode : torch::autograd::Function<DistillationNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& tokens,
                            const at::Tensor& log_probs, double temperature, bool rest, bool mean) {
    const Distillation out = distillationForward(rowsOf(logits), tokens, log_probs, temperature, rest, mean, true);
    ctx->save_for_backward({logits, tokens, log_probs, out.kept});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["rest"] = rest;
    ctx->saved_data["mean"] = mean;
    return out.loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], memory = dense(saved[3]), none;
    const double temperature = ctx->saved_data["temperature"].toDouble();
    const bool mean = ctx->saved_data["mean"].toBool();
    if (at::GradMode::is_enabled())
      return {distillationBackwardGraph(logits, saved[1], saved[2], temperature, ctx->saved_data["rest"].toBool(), mean, grads[0],
                                        memory),
              none, none, none, none, none};
    c10::cuda::CUDAGuard guard(logits.device());
    Rows rows = rowsOf(logits);
    const at::Tensor grad = gradientFor(rows);
    const auto [g, stride] = perRow(grads[0]);
    const Kept kept(memory, rows.x.rows);
    const cudaError_t e = launchDistillationBackward(rows.t.data_ptr(), rows.x, grad.data_ptr(), kept.stats, kept.pairs,
                                                     (int)saved[1].size(-1), temperature, g.data_ptr<float>(), stride,
                                                     mean ? kept.count : nullptr, c10::cuda::getCurrentCUDAStream());
    TORCH_CHECK(e == cudaSuccess, "distillation backward launch failed: ", cudaGetErrorString(e));
    return {grad, none, none, none, none, none};
  }
};

// The divergence of every row, or with `mean` its mean over the rows that count.
at::Tensor distillation(const at::Tensor& logits, at::Tensor tokens, at::Tensor log_probs, double temperature, bool rest,
                        bool mean) {
  checkLogits(logits);
  checkTemperature(temperature);
  const int64_t k = tokens.dim() > 0 ? tokens.size(-1) : 0;
  TORCH_CHECK_VALUE(k >= 1 && k <= kMostTeacherTokens, "a row has from 1 to ", kMostTeacherTokens, " teacher tokens");
  TORCH_CHECK_VALUE(!rest || logits.size(-1) <= kMostRestVocab, "with the rest the vocabulary is at most ", kMostRestVocab);
  std::vector<int64_t> sizes(logits.sizes().begin(), logits.sizes().end());
  sizes.back() = k;
  c10::cuda::CUDAGuard guard(logits.device());
  tokens = checkTokens(tokens, logits, sizes, "teacher_tokens");
  TORCH_CHECK_VALUE(at::isFloatingType(log_probs.scalar_type()) && log_probs.sizes() == tokens.sizes() &&
                        log_probs.device() == logits.device(),
                    "teacher_log_probs must be floating-point ", tokens.sizes(), " on ", logits.device(), ", not ",
                    log_probs.scalar_type(), " ", log_probs.sizes(), " on ", log_probs.device());
  TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && log_probs.requires_grad()), "teacher_log_probs are constants: detach them");
  log_probs = (log_probs.requires_grad() ? log_probs.detach() : log_probs).to(at::kFloat).contiguous();
  if (at::GradMode::is_enabled() && logits.requires_grad())
    return DistillationNode::apply(logits, tokens, log_probs, temperature, rest, mean);
  return distillationForward(rowsOf(logits.detach()), tokens, log_probs, temperature, rest, mean, false).loss;
}

}  // namespace

void bindLogitsOps(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("token_log_probs", &tokenLogProbs, py::arg("logits"), py::arg("tokens"), py::arg("temperature"),
        py::arg("entropy"), py::arg("top_k"));
  m.def("distillation", &distillation, py::arg("logits"), py::arg("tokens"), py::arg("log_probs"), py::arg("temperature"),
        py::arg("rest"), py::arg("mean"));
  m.attr("MOST_VOCAB") = kMostVocab;
  m.attr("MOST_TOP_TOKENS") = kMostTopTokens;
  m.attr("MOST_TEACHER_TOKENS") = kMostTeacherTokens;
  m.attr("MOST_REST_VOCAB") = kMostRestVocab;
  m.attr("LEAST_REST") = kLeastRest;
}

}  // namespace fairring
