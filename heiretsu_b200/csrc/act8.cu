// Activations kept in 8 bits between forward and backward (format: act8.cuh), and the LayerNorm that keeps
// its normalised input that way.
//
//   pack         x -> codes, exponent bytes
//   unpack       codes, bytes -> x in fp32, bf16 or fp16 (values beyond the type's range become its largest)
//   unpack_gelu  the same, and GELU (tanh form) of the restored value: the MLP's pre-activation is kept once
//                and both operands of its backward come from it
//   LayerNorm    forward: y = xh w + b with xh = (x - mean) rstd, keeping codes(xh) and rstd; backward from those:
//                gw = dy w, dx = rstd (gw - mean(gw) - xh mean(gw xh)), dgamma += sum dy xh, dbeta += sum dy, and
//                y again, which the weight gradient of the layer behind the norm reads
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "act8.cuh"
#include "common.cuh"
#include "host_utils.h"

namespace hb {

// Element types of an activation.
enum ActType : int { kActBf16 = 0, kActF16 = 1, kActF32 = 2 };

namespace {

template <int TYPE>
__device__ __forceinline__ float act_load(const void* p, long i) {
  if constexpr (TYPE == kActF32) return static_cast<const float*>(p)[i];
  else return to_f32<TYPE == kActF16>(static_cast<const uint16_t*>(p)[i]);
}
template <int TYPE>
__device__ __forceinline__ float act_clamp(float v) {
  // a code rounded up can stand for 2^128 (or, in 16 bits, for more than the type holds): keep it finite.
  constexpr float kMax = TYPE == kActF16 ? 65504.f : TYPE == kActBf16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
  return isnan(v) ? v : fminf(fmaxf(v, -kMax), kMax);
}
template <int TYPE>
__device__ __forceinline__ void act_store(void* p, long i, float v) {
  if constexpr (TYPE == kActF32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = from_f32<TYPE == kActF16>(v);
}

// x / (1 + e^(-2u)), u = sqrt(2/pi) (x + 0.044715 x^3): GELU's tanh form through 1 + tanh(u) = 2 / (1 + e^(-2u)).
__device__ __forceinline__ float gelu_full(float x) {
  const float u = 0.7978845608028654f * fmaf(0.044715f * x, x * x, x);
  return x / (1.f + __expf(-2.f * u));
}

// One warp per block of 128 columns.
template <int TYPE>
__global__ void __launch_bounds__(256) act8_pack_kernel(const void* __restrict__ x, long ld, int8_t* __restrict__ q,
                                                        uint8_t* __restrict__ e, long M, int N, int nb) {
  const long blk = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (blk >= M * nb) return;
  const long row = blk / nb;
  const int c0 = (int)(blk % nb) * kAct8Block + (threadIdx.x & 31);
  float v[4];
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = c0 + 32 * k < N ? act_load<TYPE>(x, row * ld + c0 + 32 * k) : 0.f;
    top = max(top, __float_as_uint(v[k]) & 0x7FFFFFFFu);
  }
  const uint32_t byte = act8_byte(__reduce_max_sync(0xffffffffu, top));
  const float inv = act8_inv_scale(byte);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (c0 + 32 * k < N) q[row * N + c0 + 32 * k] = static_cast<int8_t>(byte == kAct8Nan ? 0u : act8_code(v[k], inv));
  if ((threadIdx.x & 31) == 0) e[blk] = static_cast<uint8_t>(byte);
}

template <int TYPE, bool GELU>
__global__ void __launch_bounds__(256) act8_unpack_kernel(const int8_t* __restrict__ q, const uint8_t* __restrict__ e,
                                                          void* __restrict__ x, void* __restrict__ h, long M, int N,
                                                          int nb) {
  const long n = M * N;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long row = i / N;
    const float v = act_clamp<TYPE>(act8_value((uint8_t)q[i], act8_scale(e[row * nb + (i - row * N) / kAct8Block])));
    act_store<TYPE>(x, i, v);
    if constexpr (GELU) act_store<TYPE>(h, i, gelu_full(v));
  }
}

// One warp per row, two passes over it.
template <bool F16>
__global__ void __launch_bounds__(256) ln_fwd_act8_kernel(const float* __restrict__ x, const float* __restrict__ w,
                                                          const float* __restrict__ b, uint16_t* __restrict__ y,
                                                          int8_t* __restrict__ q, uint8_t* __restrict__ e,
                                                          float* __restrict__ rstd_out, int M, int H, int nb, float eps) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= M) return;
  const float* xr = x + (long)row * H;
  float s = 0.f;
  for (int j = lane; j < H; j += 32) s += xr[j];
  const float mu = warp_sum(s) / H;
  float ss = 0.f;
  for (int j = lane; j < H; j += 32) ss = fmaf(xr[j] - mu, xr[j] - mu, ss);
  const float rstd = rsqrtf(warp_sum(ss) / H + eps);
  for (int k = 0; k < nb; ++k) {
    float v[4];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = k * kAct8Block + 32 * i + lane;
      v[i] = j < H ? (xr[j] - mu) * rstd : 0.f;
      top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    }
    const uint32_t byte = act8_byte(__reduce_max_sync(0xffffffffu, top));
    const float inv = act8_inv_scale(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = k * kAct8Block + 32 * i + lane;
      if (j < H) {
        q[(long)row * H + j] = static_cast<int8_t>(byte == kAct8Nan ? 0u : act8_code(v[i], inv));
        y[(long)row * H + j] = from_f32<F16>(fmaf(v[i], w[j], b[j]));
      }
    }
    if (lane == 0) e[(long)row * nb + k] = static_cast<uint8_t>(byte);
  }
  if (lane == 0) rstd_out[row] = rstd;
}

// One warp per row; the per-column sums are a second kernel, one partial row ([2, H]: dgamma, dbeta) per CTA.
template <bool F16>
__global__ void __launch_bounds__(256) ln_bwd_act8_kernel(const float* __restrict__ dy, const int8_t* __restrict__ q,
                                                          const uint8_t* __restrict__ e, const float* __restrict__ rstd,
                                                          const float* __restrict__ w, const float* __restrict__ b,
                                                          const float* dres_in, float* dres,
                                                          uint16_t* __restrict__ dres16, uint16_t* __restrict__ y,
                                                          int M, int H, int nb) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= M) return;
  const long base = (long)row * H;
  float s1 = 0.f, s2 = 0.f;
  for (int j = lane; j < H; j += 32) {
    const float xh = act8_value((uint8_t)q[base + j], act8_scale(e[(long)row * nb + j / kAct8Block]));
    const float g = dy[base + j] * w[j];
    s1 += g;
    s2 = fmaf(g, xh, s2);
  }
  const float m1 = warp_sum(s1) / H, m2 = warp_sum(s2) / H, rs = rstd[row];
  for (int j = lane; j < H; j += 32) {
    const float xh = act8_value((uint8_t)q[base + j], act8_scale(e[(long)row * nb + j / kAct8Block]));
    const float o = fmaf(rs, dy[base + j] * w[j] - m1 - xh * m2, dres_in[base + j]);
    dres[base + j] = o;
    dres16[base + j] = from_f32<F16>(o);
    y[base + j] = from_f32<F16>(fmaf(xh, w[j], b[j]));
  }
}

__global__ void __launch_bounds__(256) ln_cols_act8_kernel(const float* __restrict__ dy, const int8_t* __restrict__ q,
                                                           const uint8_t* __restrict__ e, float* __restrict__ part, int M,
                                                           int H, int nb) {
  for (int j = threadIdx.x; j < H; j += 256) {
    float g = 0.f, s = 0.f;
    for (int r = blockIdx.x; r < M; r += gridDim.x) {
      const float d = dy[(long)r * H + j];
      g = fmaf(d, act8_value((uint8_t)q[(long)r * H + j], act8_scale(e[(long)r * nb + j / kAct8Block])), g);
      s += d;
    }
    part[(long)blockIdx.x * 2 * H + j] = g;
    part[(long)blockIdx.x * 2 * H + H + j] = s;
  }
}

}  // namespace

// Adds the partial rows of a LayerNorm backward to dgamma and dbeta in a fixed order (norm.cu).
void ln_reduce_partials_launch(const float* part, int rows, int H, float* dgamma, float* dbeta, cudaStream_t s);

static int blocks_of(long N) { return (int)((N + kAct8Block - 1) / kAct8Block); }

void act8_pack_launch(const void* x, long ld, int type, int8_t* q, uint8_t* e, long M, int N, cudaStream_t s) {
  if (M == 0 || N == 0) return;
  const int nb = blocks_of(N);
  const long ctas = (M * nb + 7) / 8;
  if (ctas > 0x7FFFFFFFL) throw std::runtime_error("act8_pack: too many rows");
  auto* k = type == kActF32 ? act8_pack_kernel<kActF32> : type == kActF16 ? act8_pack_kernel<kActF16> : act8_pack_kernel<kActBf16>;
  k<<<(unsigned)ctas, 256, 0, s>>>(x, ld, q, e, M, N, nb);
  HB_CUDA_CHECK(cudaGetLastError());
}

void act8_unpack_launch(const int8_t* q, const uint8_t* e, int type, void* x, void* h, long M, int N, cudaStream_t s) {
  if (M == 0 || N == 0) return;
  const int nb = blocks_of(N);
  const int ctas = (int)std::min<long>((M * N + 255) / 256, 8L * num_sms(current_device()));
#define HB_UNPACK(T) (h ? act8_unpack_kernel<T, true> : act8_unpack_kernel<T, false>)
  auto* k = type == kActF32 ? HB_UNPACK(kActF32) : type == kActF16 ? HB_UNPACK(kActF16) : HB_UNPACK(kActBf16);
#undef HB_UNPACK
  k<<<ctas, 256, 0, s>>>(q, e, x, h, M, N, nb);
  HB_CUDA_CHECK(cudaGetLastError());
}

void ln_fwd_act8_launch(const float* x, const float* w, const float* b, void* y, int8_t* q, uint8_t* e, float* rstd,
                        int M, int H, float eps, bool f16, cudaStream_t s) {
  if (M == 0) return;
  (f16 ? ln_fwd_act8_kernel<true> : ln_fwd_act8_kernel<false>)<<<(M + 7) / 8, 256, 0, s>>>(
      x, w, b, static_cast<uint16_t*>(y), q, e, rstd, M, H, blocks_of(H), eps);
  HB_CUDA_CHECK(cudaGetLastError());
}

int ln_bwd_act8_ctas(int M, int device) {
  const int full = 2 * num_sms(device), need = (M + 7) / 8;
  return need < 1 ? 1 : need < full ? need : full;
}

void ln_bwd_act8_launch(const float* dy, const int8_t* q, const uint8_t* e, const float* rstd, const float* w,
                        const float* b, const float* dres_in, float* dres, void* dres16, void* y, float* part, int ctas,
                        float* dgamma, float* dbeta, int M, int H, bool f16, cudaStream_t s) {
  if (M == 0) return;
  (f16 ? ln_bwd_act8_kernel<true> : ln_bwd_act8_kernel<false>)<<<(M + 7) / 8, 256, 0, s>>>(
      dy, q, e, rstd, w, b, dres_in, dres, static_cast<uint16_t*>(dres16), static_cast<uint16_t*>(y), M, H, blocks_of(H));
  HB_CUDA_CHECK(cudaGetLastError());
  ln_cols_act8_kernel<<<ctas, 256, 0, s>>>(dy, q, e, part, M, H, blocks_of(H));
  HB_CUDA_CHECK(cudaGetLastError());
  ln_reduce_partials_launch(part, ctas, H, dgamma, dbeta, s);
}

}  // namespace hb
