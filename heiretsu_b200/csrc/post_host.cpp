// Torch-facing entry points of the post-training losses (post_loss.cu): argument checks, stream
// selection, then the raw launchers. Refused calls raise before anything is launched. Numbers go into
// the messages as strings: an extension whose linker brought its own static libstdc++ faults when it streams them.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <string>

#include "host_utils.h"
#include "ops.h"
#include "post_args.h"

namespace hb {

long logit_row_limit(int type);
long policy_scratch_doubles();
long preference_scratch_doubles(int P, int T);
void token_logprobs_launch(const LogitRows& a, cudaStream_t s);
void policy_loss_launch(const LogitRows& a, const PolicyTerms& p, double* scratch, float* loss, float* stats,
                        cudaStream_t s);
void preference_loss_launch(const float* logp, const float* ref, const int64_t* targets, int64_t ignore_index, int P,
                            int T, double beta, double smoothing, float* loss, float* rewards, float* dlogp,
                            double* scratch, cudaStream_t s);

namespace {

constexpr int64_t kIntMax = std::numeric_limits<int>::max();

bool given(const c10::optional<at::Tensor>& t) { return t && t->defined(); }

int logit_type(const at::Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return kLogitBf16;
    case at::kHalf: return kLogitF16;
    case at::kFloat: return kLogitF32;
    default: TORCH_CHECK(false, op, ": logits must be bf16, fp16 or fp32");
  }
}

// A contiguous tensor of one type with exactly n elements on the logits' device.
void check_vec(const at::Tensor& t, at::ScalarType dt, int64_t n, const at::Device& dev, const char* op,
               const char* name) {
  TORCH_CHECK(t.device() == dev, op, ": ", name, " must be on ", dev.str());
  TORCH_CHECK(t.scalar_type() == dt, op, ": ", name, " has the wrong dtype");
  TORCH_CHECK(t.is_contiguous(), op, ": ", name, " must be contiguous");
  TORCH_CHECK(t.numel() == n, op, ": ", name, " must hold ", std::to_string(n), " elements, got ",
              std::to_string(t.numel()));
}

// First byte and one past the last byte that a 2-D row-strided tensor reaches.
std::pair<uintptr_t, uintptr_t> extent(const at::Tensor& t) {
  const auto p = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.numel() == 0) return {p, p};
  return {p, p + ((t.size(0) - 1) * t.stride(0) + t.size(1)) * t.element_size()};
}

LogitRows logit_rows(const at::Tensor& logits, int64_t V, const at::Tensor& targets, int64_t ignore_index,
                     const at::Tensor& logp, const c10::optional<at::Tensor>& lse,
                     const c10::optional<at::Tensor>& grad, const char* op) {
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1), op,
              ": logits must be 2-D with contiguous rows");
  LogitRows a{};
  a.type = logit_type(logits, op);
  const int64_t M = logits.size(0);
  TORCH_CHECK(V >= 1 && V <= logits.size(1), op, ": V must be in [1, row width]");
  TORCH_CHECK(M <= kIntMax / 2, op, ": too many rows");
  const int64_t widest = logit_row_limit(a.type);  // what the shared memory of one cluster holds
  TORCH_CHECK(V <= widest, op, ": V must be at most ", std::to_string(widest), " for this dtype");
  TORCH_CHECK(logits.stride(0) >= 0, op, ": logits need a row stride that is not negative");
  const at::Device dev = logits.device();
  check_vec(targets, at::kLong, M, dev, op, "targets");
  check_vec(logp, at::kFloat, M, dev, op, "logp");
  a.x = logits.data_ptr();
  a.ld = logits.stride(0);
  a.M = static_cast<int>(M);
  a.V = static_cast<int>(V);
  a.targets = targets.data_ptr<int64_t>();
  a.ignore_index = ignore_index;
  a.logp = logp.data_ptr<float>();
  if (given(lse)) {
    check_vec(*lse, at::kFloat, M, dev, op, "lse");
    a.lse = lse->data_ptr<float>();
  }
  if (given(grad)) {
    const at::Tensor& g = *grad;
    TORCH_CHECK(g.device() == dev && g.scalar_type() == logits.scalar_type() && g.dim() == 2 && g.size(0) == M &&
                    (g.size(1) <= 1 || g.stride(1) == 1),
                op, ": grad must be a matrix with contiguous rows like logits, of its dtype, rows and device");
    TORCH_CHECK(g.size(1) >= V && g.size(1) <= widest, op, ": grad must be at least V wide and at most ",
                std::to_string(widest));
    TORCH_CHECK(M <= 1 || g.stride(0) >= g.size(1), op, ": grad rows must not overlap");
    const bool same = g.data_ptr() == logits.data_ptr() && (M <= 1 || g.stride(0) == logits.stride(0));
    const auto x = extent(logits), y = extent(g);
    TORCH_CHECK(same || x.second <= y.first || y.second <= x.first, op,
                ": grad must be the logits themselves or not overlap them");
    a.grad = g.data_ptr();
    a.gld = g.stride(0);
    a.W = static_cast<int>(g.size(1));
  } else {
    a.W = static_cast<int>(std::max(V, std::min(widest, logits.size(1))));  // rows are dealt out as with a gradient
  }
  a.status = device_status_ptr(logits.get_device());
  return a;
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> token_logprobs(const at::Tensor& logits, int64_t V, const at::Tensor& targets,
                                                  int64_t ignore_index, const c10::optional<at::Tensor>& grad) {
  const char* op = "token_logprobs";
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, op, ": logits must be a CUDA matrix");
  c10::cuda::CUDAGuard g(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor logp = at::empty({logits.size(0)}, f32), lse = at::empty({logits.size(0)}, f32);
  const LogitRows a = logit_rows(logits, V, targets, ignore_index, logp, lse, grad, op);
  token_logprobs_launch(a, at::cuda::getCurrentCUDAStream());
  return {logp, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> policy_loss(
    const at::Tensor& logits, int64_t V, const at::Tensor& targets, const at::Tensor& old_logp,
    const at::Tensor& advantages, const c10::optional<at::Tensor>& ref_logp, const c10::optional<at::Tensor>& weights,
    double clip_low, double clip_high, double kl_coef, const c10::optional<at::Tensor>& grad_scale,
    int64_t ignore_index, const c10::optional<at::Tensor>& grad_out) {
  const char* op = "policy_loss";
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, op, ": logits must be a CUDA matrix");
  c10::cuda::CUDAGuard g(logits.device());
  const at::Device dev = logits.device();
  const int64_t M = logits.size(0);
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor logp = at::empty({M}, f32), loss = at::empty({}, f32), stats = at::empty({2}, f32);
  at::Tensor grad = given(grad_out) ? *grad_out : at::empty_like(logits);
  const LogitRows a = logit_rows(logits, V, targets, ignore_index, logp, c10::nullopt, grad, op);
  PolicyTerms p{};
  check_vec(old_logp, at::kFloat, M, dev, op, "old_logp");
  const int64_t n_adv = advantages.numel();
  TORCH_CHECK(M == 0 || (n_adv >= 1 && M % n_adv == 0), op,
              ": advantages must hold one value per row or per equal run of rows");
  check_vec(advantages, at::kFloat, n_adv, dev, op, "advantages");
  TORCH_CHECK(clip_low >= 0 && clip_low <= 1 && clip_high >= 0 && std::isfinite(clip_high), op,
              ": clip_low must be in [0, 1] and clip_high finite and not negative");
  TORCH_CHECK(std::isfinite(kl_coef), op, ": kl_coef must be finite");
  p.old_logp = old_logp.data_ptr<float>();
  p.adv = advantages.data_ptr<float>();
  p.adv_rows = M == 0 ? 1 : static_cast<int>(M / n_adv);
  if (given(ref_logp)) {
    check_vec(*ref_logp, at::kFloat, M, dev, op, "ref_logp");
    p.ref_logp = ref_logp->data_ptr<float>();
  }
  if (given(weights)) {
    check_vec(*weights, at::kFloat, M, dev, op, "weights");
    p.weights = weights->data_ptr<float>();
  }
  if (given(grad_scale)) {
    check_vec(*grad_scale, at::kFloat, 1, dev, op, "grad_scale");
    p.grad_scale = grad_scale->data_ptr<float>();
  }
  p.clip_lo = static_cast<float>(1.0 - clip_low);
  p.clip_hi = static_cast<float>(1.0 + clip_high);
  p.kl_coef = static_cast<float>(kl_coef);
  at::Tensor scratch = at::empty({policy_scratch_doubles()}, logits.options().dtype(at::kDouble));
  policy_loss_launch(a, p, scratch.data_ptr<double>(), loss.data_ptr<float>(), stats.data_ptr<float>(),
                     at::cuda::getCurrentCUDAStream());
  return {loss, stats, logp, grad};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> preference_loss(const at::Tensor& logp, const at::Tensor& targets,
                                                               const c10::optional<at::Tensor>& ref_logp, double beta,
                                                               double label_smoothing, int64_t ignore_index) {
  const char* op = "preference_loss";
  TORCH_CHECK(logp.is_cuda(), op, ": logp must be a CUDA tensor");
  TORCH_CHECK(logp.dim() == 2 && logp.size(0) % 2 == 0, op,
              ": logp must be [2 * pairs, T], the chosen sequences before the rejected ones");
  const int64_t n = logp.numel(), P = logp.size(0) / 2, T = logp.size(1);
  TORCH_CHECK(P <= kIntMax / 2 && T <= kIntMax / 2, op, ": too many pairs or tokens");
  TORCH_CHECK(std::isfinite(beta), op, ": beta must be finite");
  TORCH_CHECK(label_smoothing >= 0 && label_smoothing <= 1, op, ": label_smoothing must be in [0, 1]");
  c10::cuda::CUDAGuard g(logp.device());
  const at::Device dev = logp.device();
  check_vec(logp, at::kFloat, n, dev, op, "logp");
  check_vec(targets, at::kLong, n, dev, op, "targets");
  if (given(ref_logp)) check_vec(*ref_logp, at::kFloat, n, dev, op, "ref_logp");
  const auto f32 = logp.options();
  at::Tensor loss = at::empty({}, f32), rewards = at::empty({2, P}, f32), dlogp = at::empty(logp.sizes(), f32);
  const long doubles = preference_scratch_doubles(static_cast<int>(P), static_cast<int>(T));
  at::Tensor scratch;
  if (doubles > 0) scratch = at::empty({doubles}, f32.dtype(at::kDouble));
  preference_loss_launch(logp.data_ptr<float>(), given(ref_logp) ? ref_logp->data_ptr<float>() : nullptr,
                         targets.data_ptr<int64_t>(), ignore_index, static_cast<int>(P), static_cast<int>(T), beta,
                         label_smoothing, loss.data_ptr<float>(), rewards.data_ptr<float>(), dlogp.data_ptr<float>(),
                         doubles > 0 ? scratch.data_ptr<double>() : nullptr, at::cuda::getCurrentCUDAStream());
  return {loss, rewards, dlogp};
}

}  // namespace hb
