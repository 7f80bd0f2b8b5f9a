// A token per row of logits from a given uniform number.
//
// With top = max x and temperature T > 0 a token weighs w_i = e^((x_i - top) / T). In the order by logit, descending, equal
// ones by index, the tokens kept are: the first top_k; of these the shortest start whose weight reaches top_p of
// theirs (token i is kept if what precedes it weighs less); of these the ones with w_i >= min_p. The first always is.
// All three cut the same order, so what is kept is every logit above a threshold and the first `ties` equal to it. The
// token drawn is the first kept one, by index, at which the running weight exceeds u times the kept weight.
//
// Weights are whole numbers of 2^-44, rounded once from a 64-bit exponential: sums have no order, the same token comes
// out whatever the launch, and equal logits weigh exactly the same. A sum over the 2^19 columns allowed stays below 2^63.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "decode_args.h"
#include "host_utils.h"

namespace hb {

namespace {

using u64 = unsigned long long;
constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr double kOne = 17592186044416.0;  // 2^44

// Unsigned whole numbers in the order of the logits (-0 counts as 0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (static_cast<int>(b) < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key ^ (static_cast<int>(key) < 0 ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ u64 weight(float x, float top, double inv_t) {
  if (x == top) return static_cast<u64>(kOne);
  if (x == -INFINITY) return 0;
  return __double2ull_rn(exp((static_cast<double>(x) - top) * inv_t) * kOne);
}

template <int TYPE>
__device__ __forceinline__ float logit(const SampleArgs& a, int row, int i) {
  const long at = row * a.ld + i;
  if constexpr (TYPE == 2) return static_cast<const float*>(a.x)[at];
  else return to_f32<TYPE == 1>(static_cast<const uint16_t*>(a.x)[at]);
}

__device__ __forceinline__ u64 block_sum(u64 v, u64* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// What the threads before this one hold.
__device__ __forceinline__ u64 block_before(u64 v, u64* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += x;
  }
  __syncthreads();
  if (lane == 31) buf[warp] = run;
  __syncthreads();
  u64 before = run - v;
  for (int w = 0; w < warp; ++w) before += buf[w];
  return before;
}

// One CTA per row; a thread takes consecutive columns.
template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
  __shared__ u64 buf[kWarps];
  __shared__ uint32_t s_max;
  __shared__ int s_bad, s_pick;
  const int row = blockIdx.x, tid = threadIdx.x;
  const int each = (a.V + kThreads - 1) / kThreads, c0 = min(tid * each, a.V), c1 = min(c0 + each, a.V);
  const double T = a.temperature ? a.temperature[row] : a.temperature0;
  const double top_p = a.top_p ? a.top_p[row] : a.top_p0, min_p = a.min_p ? a.min_p[row] : a.min_p0;
  const int64_t top_k = a.top_k ? a.top_k[row] : a.top_k0;
  const double u = a.u[row];

  if (tid == 0) s_max = 0, s_bad = T != T || top_p != top_p || min_p != min_p || u != u, s_pick = a.V;
  __syncthreads();
  uint32_t mx = 0;
  bool bad = false;
  for (int i = c0; i < c1; ++i) {
    const float x = logit<TYPE>(a, row, i);
    bad |= !(x < INFINITY);
    mx = max(mx, key_of(x));
  }
  atomicMax(&s_max, mx);
  if (bad) s_bad = 1;
  __syncthreads();
  const uint32_t kmax = s_max;
  const float top = logit_of(kmax);
  if (s_bad || top == -INFINITY) {  // NaN or +inf among the logits, nothing but -inf, a setting that is no number
    if (tid == 0) a.tokens[row] = -1;
    return;
  }
  if (T <= 0 || min_p > 1 || top_p <= 0) {  // the first token of the order
    for (int i = c0; i < c1; ++i)
      if (key_of(logit<TYPE>(a, row, i)) == kmax) {
        atomicMin(&s_pick, i);
        break;
      }
    __syncthreads();
    if (tid == 0) a.tokens[row] = s_pick;
    return;
  }
  const double inv_t = 1.0 / T;
  const auto mass = [&](uint32_t from) {  // weight of the keys >= from
    u64 m = 0;
    for (int i = c0; i < c1; ++i) {
      const float x = logit<TYPE>(a, row, i);
      if (key_of(x) >= from) m += weight(x, top, inv_t);
    }
    return block_sum(m, buf);
  };
  const auto count = [&](uint32_t from) {
    u64 n = 0;
    for (int i = c0; i < c1; ++i) n += key_of(logit<TYPE>(a, row, i)) >= from;
    return block_sum(n, buf);
  };
  uint32_t t = 0;       // kept: keys above t, and the first `ties` equal to it
  u64 ties = ~0ull;
  if (top_k > 0 && top_k < a.V) {
    for (int bit = 31; bit >= 0; --bit)
      if (count(t | (1u << bit)) >= static_cast<u64>(top_k)) t |= 1u << bit;
    ties = top_k - (t == ~0u ? 0 : count(t + 1));
  }
  if (top_p < 1) {
    const u64 above = mass(t + 1);
    const u64 total = t == 0 ? above : above + ties * weight(logit_of(t), top, inv_t);
    const u64 need = max(__double2ull_ru(top_p * static_cast<double>(total)), 1ull);
    uint32_t t2 = t;
    if (above >= need) {
      t2 = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = t2 | (1u << bit);
        if (c <= t || mass(c) >= need) t2 = c;
      }
    }
    const u64 w = weight(logit_of(t2), top, inv_t);
    if (w > 0) {
      const u64 n = (need - min(mass(t2 + 1), need) + w - 1) / w;
      ties = t2 == t ? min(ties, n) : n;
    }
    t = t2;
  }
  if (min_p > 0) {
    const float from = T == INFINITY ? -INFINITY : __double2float_ru(static_cast<double>(top) + T * log(min_p));
    const uint32_t k = key_of(from);
    if (k > t) t = k, ties = ~0ull;
  }
  u64 equal = 0;
  for (int i = c0; i < c1; ++i) equal += key_of(logit<TYPE>(a, row, i)) == t;
  const u64 tie0 = block_before(equal, buf);
  const auto kept = [&](uint32_t k, u64& tie) { return k > t || (k == t && tie++ < ties); };
  u64 mine = 0, tie = tie0;
  for (int i = c0; i < c1; ++i) {
    const float x = logit<TYPE>(a, row, i);
    if (kept(key_of(x), tie)) mine += weight(x, top, inv_t);
  }
  const u64 total = block_sum(mine, buf);
  u64 run = block_before(mine, buf);
  const u64 target = min(static_cast<u64>(max(u, 0.0) * static_cast<double>(total)), total - 1);
  if (run <= target && target < run + mine) {
    tie = tie0;
    for (int i = c0; i < c1; ++i) {
      const float x = logit<TYPE>(a, row, i);
      if (kept(key_of(x), tie)) run += weight(x, top, inv_t);
      if (run > target) {
        a.tokens[row] = i;
        break;
      }
    }
  }
}

}  // namespace

void sample_tokens_launch(const SampleArgs& a, cudaStream_t s) {
  if (a.rows == 0) return;
  if (a.type == 0) sample_kernel<0><<<a.rows, kThreads, 0, s>>>(a);
  else if (a.type == 1) sample_kernel<1><<<a.rows, kThreads, 0, s>>>(a);
  else sample_kernel<2><<<a.rows, kThreads, 0, s>>>(a);
  HB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace hb
