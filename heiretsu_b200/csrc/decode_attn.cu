// Attention of one new token per sequence over a paged key/value cache:
//   s_j = scale q.k_j,  j < length;  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m);  lse = m + log sum_j e^(s_j - m)
// A sequence of length 0 gives 0 and -inf. A length outside [0, width * page size] or a page outside the cache gives NaN in
// the sequence's rows, and the bad-argument status.
#include "act8.cuh"
#include "common.cuh"
#include "decode_args.h"
#include "host_utils.h"

namespace hb {

namespace {

constexpr int kWarps = 8;
constexpr int kSite = 430;  // status site
constexpr float kLog2e = 1.4426950408889634f;

// One CTA per sequence and query head; warp w takes the tokens w, w + 8, ..., a lane every 32nd channel.
template <bool F16>
__global__ void __launch_bounds__(kWarps * 32) decode_attn_kernel(const DecodeArgs a) {
  __shared__ float sm_m[kWarps], sm_l[kWarps], sm_o[kWarps][128];
  const int b = blockIdx.x / a.heads_q, hq = blockIdx.x - b * a.heads_q;
  const KvPool& p = a.pool;
  const int h = hq / (a.heads_q / p.heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = a.lengths[b];
  bool bad = len < 0 || len > static_cast<long>(a.width) * p.size;
  float q[4] = {}, o[4] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < p.dim)
      q[i] = to_f32<F16>(static_cast<const uint16_t*>(a.q)[b * a.qt + hq * a.qh + lane + 32 * i]);
  for (int j = warp; !bad && j < len; j += kWarps) {
    const int pg = a.table[b * a.tt + j / p.size], at = j % p.size;
    if (pg < 0 || pg >= p.pages) {
      bad = true;
      break;
    }
    const long ki = pg * p.kp + h * p.kh + at * p.ks, vi = pg * p.vp + h * p.vh + at * p.vs;
    float ksc = 1.f, vsc = 1.f;
    if (p.type == kKvCodes) {
      ksc = act8_scale(p.ke[pg * p.kep + h * p.keh + at]);
      vsc = act8_scale(p.ve[pg * p.vep + h * p.veh + at]);
    }
    float s = 0.f, v[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      if (d >= p.dim) continue;
      float k;
      if (p.type == kKvCodes) {
        k = static_cast<const int8_t*>(p.k)[ki + d];
        v[i] = static_cast<const int8_t*>(p.v)[vi + d] * vsc;
      } else {
        k = to_f32<F16>(static_cast<const uint16_t*>(p.k)[ki + d]);
        v[i] = to_f32<F16>(static_cast<const uint16_t*>(p.v)[vi + d]);
      }
      s = fmaf(q[i], k, s);
    }
    s = warp_sum(s) * ksc * a.scale;
    const float top = fmaxf(m, s), ref = top == -INFINITY ? 0.f : top;
    const float w = exp2f((s - ref) * kLog2e), c = exp2f((m - ref) * kLog2e);
    l = l * c + w;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * c + w * v[i];
    m = top;
  }
  if (lane == 0) sm_m[warp] = bad ? __uint_as_float(0x7FC00000u) : m, sm_l[warp] = l;
#pragma unroll
  for (int i = 0; i < 4; ++i) sm_o[warp][lane + 32 * i] = o[i];
  if (bad && lane == 0) record_error(a.status, kBadArg, kSite);
  __syncthreads();
  float top = -INFINITY, sum = 0.f, acc = 0.f;
  bool nan = false;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w]), nan |= sm_m[w] != sm_m[w];
  const float ref = nan ? __uint_as_float(0x7FC00000u) : top == -INFINITY ? 0.f : top;
  const int d = threadIdx.x;
  for (int w = 0; w < kWarps; ++w) {
    const float c = exp2f((sm_m[w] - ref) * kLog2e);
    sum += sm_l[w] * c;
    if (d < p.dim) acc += sm_o[w][d] * c;
  }
  const long row = static_cast<long>(b) * a.heads_q + hq;
  if (d < p.dim)
    static_cast<uint16_t*>(a.out)[row * p.dim + d] = from_f32<F16>(len == 0 ? 0.f : acc / sum);
  if (d == 0) a.lse[row] = len == 0 ? -INFINITY : ref + logf(sum);
}

}  // namespace

void decode_attention_launch(const DecodeArgs& a, cudaStream_t s) {
  if (a.seqs == 0) return;
  const unsigned grid = static_cast<unsigned>(a.seqs) * a.heads_q;
  if (a.f16) decode_attn_kernel<true><<<grid, kWarps * 32, 0, s>>>(a);
  else decode_attn_kernel<false><<<grid, kWarps * 32, 0, s>>>(a);
  HB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace hb
