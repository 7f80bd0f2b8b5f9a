// Post-training losses: target log-probabilities of vocabulary logits, the clipped policy loss with a
// KL term, and the paired log-ratio (preference) loss, each with its gradient.
//
// For a row x of V logits with target t:
//   lse  = log sum_j exp(x_j),  logp = x_t - lse,  d logp / d x_j = [j == t] - exp(x_j - lse)
// Policy loss of a token, with d = logp - old, r = e^d, advantage A, u = ref - logp:
//   l = -min(r A, clip(r) A) + kl (e^u - u - 1)
//   dl / dlogp = (r A <= clip(r) A ? -r A : 0) + kl (1 - e^u)
// Rows whose target is `ignore_index` are not read: their log-probability is 0 and their gradient row zero.
// A target outside [0, V) gives NaN and the bad-argument status, as in the cross-entropy kernels.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "host_utils.h"
#include "post_args.h"

namespace hb {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

template <int TYPE>
__device__ __forceinline__ float load1(const void* base, long i) {
  if constexpr (TYPE == kLogitF32) return static_cast<const float*>(base)[i];
  else return to_f32<TYPE == kLogitF16>(static_cast<const uint16_t*>(base)[i]);
}
template <int TYPE>
__device__ __forceinline__ void store1(void* base, long i, float v) {
  if constexpr (TYPE == kLogitF32) static_cast<float*>(base)[i] = v;
  else static_cast<uint16_t*>(base)[i] = from_f32<TYPE == kLogitF16>(v);
}

// (max, sum of exp(x - max)) pairs; an empty pair is (-inf, 0).
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
  const float nm = fmaxf(m, m2);
  // s == 0 keeps an empty side out (its max is -inf, and exp(-inf - -inf) would be NaN)
  const float a = s == 0.f ? 0.f : s * __expf(m - nm);
  const float b = s2 == 0.f ? 0.f : s2 * __expf(m2 - nm);
  m = nm;
  s = a + b;
}

// What one row adds to the loss and its statistics, and the factor of its gradient.
struct RowTerm {
  float coef, loss, kl, clipped;
};
__device__ __forceinline__ RowTerm policy_term(const PolicyTerms& p, int row, float logp, float w) {
  RowTerm t{0.f, 0.f, 0.f, 0.f};
  const float a = p.adv[row / p.adv_rows];
  const float r = expf(logp - p.old_logp[row]);
  const float c = fminf(fmaxf(r, p.clip_lo), p.clip_hi);
  // written so that a NaN ratio is not clipped and reaches the loss and the gradient
  const bool clipped = c * a < r * a;
  t.loss = clipped ? -c * a : -r * a;
  t.coef = clipped ? 0.f : -r * a;
  t.clipped = clipped ? w : 0.f;
  if (p.ref_logp) {
    const float u = p.ref_logp[row] - logp;
    const float e = expm1f(u);
    t.kl = e - u;
    t.loss = fmaf(p.kl_coef, t.kl, t.loss);
    t.coef = fmaf(-p.kl_coef, e, t.coef);
  }
  t.loss *= w;
  t.kl *= w;
  t.coef *= w;
  return t;
}

enum Mode : int { kLogp = 0, kUnit = 1, kPolicy = 2 };

// One CTA per row; two passes over it.
template <int TYPE, int MODE>
__global__ void __launch_bounds__(kThreads) logit_rows_kernel(LogitRows a, PolicyTerms p, const double* __restrict__ head,
                                                              double* __restrict__ part) {
  __shared__ float sm[kWarps], ss[kWarps];
  const int row = blockIdx.x;
  const int64_t t = a.targets[row];
  const bool counted = t != a.ignore_index;
  const bool bad = counted && (t < 0 || t >= a.V);
  if (bad && threadIdx.x == 0) record_error(a.status, kBadArg, 410);
  const long base = (long)row * a.ld;
  float m = -INFINITY, s = 0.f, xt = 0.f;
  if (counted) {
    if (!bad) xt = load1<TYPE>(a.x, base + t);
    for (int j = threadIdx.x; j < a.V; j += kThreads) {
      const float v = load1<TYPE>(a.x, base + j);
      merge(m, s, v, v == -INFINITY ? 0.f : 1.f);
      if (isnan(v)) s = v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    if ((threadIdx.x & 31) == 0) {
      sm[threadIdx.x >> 5] = m;
      ss[threadIdx.x >> 5] = s;
    }
    __syncthreads();  // also: every thread has read the row (and its target) before any of it is overwritten
    m = sm[0];
    s = ss[0];
    for (int w = 1; w < kWarps; ++w) merge(m, s, sm[w], ss[w]);
  }
  const float lse = counted ? m + logf(s) : 0.f;
  const float logp = bad ? NAN : (counted ? (xt - m) - logf(s) : 0.f);
  if (threadIdx.x == 0) {
    a.logp[row] = logp;
    if (a.lse) a.lse[row] = lse;
  }
  if constexpr (MODE == kLogp) return;
  float coef = counted ? 1.f : 0.f;
  if constexpr (MODE == kPolicy) {
    RowTerm r{0.f, 0.f, 0.f, 0.f};
    if (counted) r = policy_term(p, row, logp, p.weights ? p.weights[row] : (float)head[0]);
    if (threadIdx.x == 0) {
      part[3L * row] = r.loss;
      part[3L * row + 1] = r.kl;
      part[3L * row + 2] = r.clipped;
    }
    coef = r.coef * (p.grad_scale ? *p.grad_scale : 1.f);
  }
  if (bad) coef = NAN;
  const long gbase = (long)row * a.gld;
  for (int j = threadIdx.x; j < a.W; j += kThreads) {
    float g = 0.f;
    if (counted && j < a.V) {
      const float pj = __expf(load1<TYPE>(a.x, base + j) - lse);
      g = coef * ((j == t ? 1.f : 0.f) - pj);
    }
    store1<TYPE>(a.grad, gbase + j, g);
  }
}

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) v += sh[w];
  __syncthreads();
  return v;
}

__global__ void __launch_bounds__(1024) count_rows_kernel(const int64_t* __restrict__ targets, int M,
                                                          int64_t ignore_index, double* __restrict__ head) {
  __shared__ double sh[32];
  int n = 0;
  for (int i = threadIdx.x; i < M; i += 1024) n += targets[i] != ignore_index;
  const double c = block_sum((double)n, sh);
  if (threadIdx.x == 0) head[0] = 1.0 / fmax(c, 1.0);
}

// loss and statistics: the rows' terms added in a fixed order, in 64 bits.
__global__ void __launch_bounds__(1024) policy_sum_kernel(const double* __restrict__ part, int n,
                                                          float* __restrict__ loss, float* __restrict__ stats) {
  __shared__ double sh[32];
  double s[3] = {0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < n; i += 1024)
    for (int k = 0; k < 3; ++k) s[k] += part[3L * i + k];
  for (int k = 0; k < 3; ++k) s[k] = block_sum(s[k], sh);
  if (threadIdx.x == 0) {
    loss[0] = (float)s[0];
    stats[0] = (float)s[1];
    stats[1] = (float)s[2];
  }
}

// log(1 + e^t) without overflow.
__device__ __forceinline__ double softplus(double t) { return fmax(t, 0.0) + log1p(exp(-fabs(t))); }

// One CTA per pair: sums both sequences, then writes both gradient rows.
__global__ void __launch_bounds__(256) preference_kernel(const float* __restrict__ logp, const float* __restrict__ ref,
                                                         const int64_t* __restrict__ targets, int64_t ignore_index,
                                                         int P, int T, double beta, double smoothing,
                                                         float* __restrict__ rewards, float* __restrict__ dlogp,
                                                         double* __restrict__ part) {
  __shared__ double sh[32];
  const int i = blockIdx.x;
  double sum[2];
  for (int h = 0; h < 2; ++h) {
    const long base = (long)(i + h * P) * T;
    double v = 0.0;
    for (int j = threadIdx.x; j < T; j += blockDim.x)
      if (targets[base + j] != ignore_index) v += (double)logp[base + j] - (ref ? (double)ref[base + j] : 0.0);
    sum[h] = beta * block_sum(v, sh);
  }
  const double z = sum[0] - sum[1];
  const double c = beta / P * (smoothing / (1.0 + exp(-z)) - (1.0 - smoothing) / (1.0 + exp(z)));
  if (threadIdx.x == 0) {
    rewards[i] = (float)sum[0];
    rewards[P + i] = (float)sum[1];
    part[i] = (1.0 - smoothing) * softplus(-z) + smoothing * softplus(z);
  }
  for (int h = 0; h < 2; ++h) {
    const long base = (long)(i + h * P) * T;
    const float g = (float)(h ? -c : c);
    for (int j = threadIdx.x; j < T; j += blockDim.x) dlogp[base + j] = targets[base + j] != ignore_index ? g : 0.f;
  }
}

__global__ void __launch_bounds__(256) preference_sum_kernel(const double* __restrict__ part, int P,
                                                             float* __restrict__ loss) {
  __shared__ double sh[32];
  double v = 0.0;
  for (int i = threadIdx.x; i < P; i += 256) v += part[i];
  v = block_sum(v, sh);
  if (threadIdx.x == 0) loss[0] = P > 0 ? (float)(v / P) : 0.f;
}

template <int MODE>
void launch_rows(const LogitRows& a, const PolicyTerms& p, const double* head, double* part, cudaStream_t s) {
  if (a.M == 0) return;
  auto* k = a.type == kLogitF32   ? logit_rows_kernel<kLogitF32, MODE>
            : a.type == kLogitF16 ? logit_rows_kernel<kLogitF16, MODE>
                                  : logit_rows_kernel<kLogitBf16, MODE>;
  k<<<a.M, kThreads, 0, s>>>(a, p, head, part);
  HB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace

long policy_scratch_doubles(int M) { return 1 + 3L * M; }
long preference_scratch_doubles(int P) { return P; }

void token_logprobs_launch(const LogitRows& a, cudaStream_t s) {
  const PolicyTerms none{};
  if (a.grad) launch_rows<kUnit>(a, none, nullptr, nullptr, s);
  else launch_rows<kLogp>(a, none, nullptr, nullptr, s);
}

void policy_loss_launch(const LogitRows& a, const PolicyTerms& p, double* scratch, float* loss, float* stats,
                        cudaStream_t s) {
  if (!p.weights) {
    count_rows_kernel<<<1, 1024, 0, s>>>(a.targets, a.M, a.ignore_index, scratch);
    HB_CUDA_CHECK(cudaGetLastError());
  }
  launch_rows<kPolicy>(a, p, scratch, scratch + 1, s);
  policy_sum_kernel<<<1, 1024, 0, s>>>(scratch + 1, a.M, loss, stats);
  HB_CUDA_CHECK(cudaGetLastError());
}

void preference_loss_launch(const float* logp, const float* ref, const int64_t* targets, int64_t ignore_index, int P,
                            int T, double beta, double smoothing, float* loss, float* rewards, float* dlogp,
                            double* scratch, cudaStream_t s) {
  if (P > 0) {
    preference_kernel<<<P, 256, 0, s>>>(logp, ref, targets, ignore_index, P, T, beta, smoothing, rewards, dlogp,
                                        scratch);
    HB_CUDA_CHECK(cudaGetLastError());
  }
  preference_sum_kernel<<<1, 256, 0, s>>>(scratch, P, loss);
  HB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace hb
