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

#include <algorithm>
#include <atomic>

#include "act8.cuh"
#include "common.cuh"
#include "host_utils.h"

namespace hb {

// Element types of an activation.
enum ActType : int { kActBf16 = 0, kActF16 = 1, kActF32 = 2 };

namespace {

// Four consecutive elements: one lane's share of a block of 128 columns.
template <int TYPE>
__device__ __forceinline__ void load4(const void* p, long i, float (&v)[4]) {
  if constexpr (TYPE == kActF32) {
    const float4 r = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w;
  } else {
    const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    v[0] = lo16<TYPE == kActF16>(r.x), v[1] = hi16<TYPE == kActF16>(r.x);
    v[2] = lo16<TYPE == kActF16>(r.y), v[3] = hi16<TYPE == kActF16>(r.y);
  }
}
template <int TYPE>
__device__ __forceinline__ float load1(const void* p, long i) {
  if constexpr (TYPE == kActF32) return static_cast<const float*>(p)[i];
  else return to_f32<TYPE == kActF16>(static_cast<const uint16_t*>(p)[i]);
}
template <int TYPE>
__device__ __forceinline__ void store4(void* p, long i, const float (&v)[4]) {
  if constexpr (TYPE == kActF32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
        make_uint2(pack16<TYPE == kActF16>(v[0], v[1]), pack16<TYPE == kActF16>(v[2], v[3]));
  }
}
template <int TYPE>
__device__ __forceinline__ void store1(void* p, long i, float v) {
  if constexpr (TYPE == kActF32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = from_f32<TYPE == kActF16>(v);
}

// A code rounded up can stand for 2^128 or, in fp16, for more than 65504: such values become the largest finite one.
// Only blocks whose exponent byte is at least kClampByte hold any; NaN stays.
template <int TYPE>
struct Range {
  static constexpr float kMax =
      TYPE == kActF16 ? 65504.f : TYPE == kActBf16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
  static constexpr uint32_t kClampByte = TYPE == kActF16 ? 127 + 9 : 127 + 121;  // 127 * 2^8 < 65504, 127 * 2^120 < 2^127
};
template <int TYPE>
__device__ __forceinline__ void decode4(uint32_t codes, uint32_t byte, float (&v)[4]) {
  act8_values(codes, act8_scale(byte), v);
  if (byte >= Range<TYPE>::kClampByte && byte != kAct8Nan) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fminf(fmaxf(v[i], -Range<TYPE>::kMax), Range<TYPE>::kMax);
  }
}

// x / (1 + e^(-2u)), u = sqrt(2/pi) (x + 0.044715 x^3): GELU's tanh form through 1 + tanh(u) = 2 / (1 + e^(-2u)), with
// one exponential and one reciprocal (both within 2 units in the last place), not the epilogues' tanh
// approximation: the kernel is bound by memory, and h is the operand of a weight gradient.
__device__ __forceinline__ float gelu_full(float x) {
  const float k0 = -2.f * 0.7978845608028654f * 1.4426950408889634f;  // -2 sqrt(2/pi) log2 e
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * fmaf(k0 * 0.044715f, x * x, k0)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return x * r;
}

constexpr int kPackBlocks = 4;  // consecutive blocks of one warp: their loads are in flight together

// One warp per kPackBlocks blocks; a lane holds 4 consecutive columns of a block (VEC: N and the row stride are
// multiples of 4 and every row starts on a boundary of 4 elements), else columns lane + 32 k. Bound by memory: one
// load and one store of each value.
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(256) act8_pack_kernel(const void* __restrict__ x, long ld, uint8_t* __restrict__ q,
                                                        uint8_t* __restrict__ e, uint32_t blocks, int N, uint32_t nb) {
  const int lane = threadIdx.x & 31;
  const uint32_t b0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kPackBlocks;
  if (b0 >= blocks) return;
  long row[kPackBlocks];
  int col[kPackBlocks];
  float v[kPackBlocks][4];
  uint32_t r0 = b0 / nb, k0 = b0 - r0 * nb;
#pragma unroll
  for (int u = 0; u < kPackBlocks; ++u) {
    row[u] = r0;
    col[u] = b0 + u < blocks ? static_cast<int>(k0) * kAct8Block + (VEC ? 4 * lane : lane) : N;
    if (++k0 == nb) k0 = 0, ++r0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[u][i] = 0.f;
    if constexpr (VEC) {
      if (col[u] < N) load4<TYPE>(x, row[u] * ld + col[u], v[u]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col[u] + 32 * i < N) v[u][i] = load1<TYPE>(x, row[u] * ld + col[u] + 32 * i);
    }
  }
  uint32_t mine = 0;  // lane u keeps the byte of block u
#pragma unroll
  for (int u = 0; u < kPackBlocks; ++u) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(v[u][i]) & 0x7FFFFFFFu);
    const uint32_t byte = act8_byte(__reduce_max_sync(0xffffffffu, top));
    if (lane == u) mine = byte;
    const uint32_t codes = act8_codes(v[u], byte);
    if constexpr (VEC) {
      if (col[u] < N) *reinterpret_cast<uint32_t*>(q + row[u] * N + col[u]) = codes;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col[u] + 32 * i < N) q[row[u] * N + col[u] + 32 * i] = static_cast<uint8_t>(codes >> (8 * i));
    }
  }
  if (lane < kPackBlocks && b0 + lane < blocks) e[b0 + lane] = static_cast<uint8_t>(mine);
}

template <int TYPE, bool GELU, bool VEC>
__global__ void __launch_bounds__(256) act8_unpack_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e,
                                                          void* __restrict__ x, void* __restrict__ h, uint32_t blocks,
                                                          int N, uint32_t nb) {
  const int lane = threadIdx.x & 31;
  const uint32_t b0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kPackBlocks;
  if (b0 >= blocks) return;
  long at[kPackBlocks];
  int col[kPackBlocks];
  uint32_t codes[kPackBlocks], byte[kPackBlocks];
  uint32_t r0 = b0 / nb, k0 = b0 - r0 * nb;
#pragma unroll
  for (int u = 0; u < kPackBlocks; ++u) {
    col[u] = b0 + u < blocks ? static_cast<int>(k0) * kAct8Block + (VEC ? 4 * lane : lane) : N;
    at[u] = static_cast<long>(r0) * N + col[u];
    if (++k0 == nb) k0 = 0, ++r0;
    byte[u] = b0 + u < blocks ? e[b0 + u] : 0;
    codes[u] = 0;
    if constexpr (VEC) {
      if (col[u] < N) codes[u] = *reinterpret_cast<const uint32_t*>(q + at[u]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col[u] + 32 * i < N) codes[u] |= static_cast<uint32_t>(q[at[u] + 32 * i]) << (8 * i);
    }
  }
#pragma unroll
  for (int u = 0; u < kPackBlocks; ++u) {
    float v[4], g[4];
    decode4<TYPE>(codes[u], byte[u], v);
    if constexpr (GELU) {
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = gelu_full(v[i]);
    }
    if constexpr (VEC) {
      if (col[u] < N) {
        store4<TYPE>(x, at[u], v);
        if constexpr (GELU) store4<TYPE>(h, at[u], g);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (col[u] + 32 * i < N) {
          store1<TYPE>(x, at[u] + 32 * i, v[i]);
          if constexpr (GELU) store1<TYPE>(h, at[u] + 32 * i, g[i]);
        }
      }
    }
  }
}

// LayerNorm forward: one warp per row, the row in registers (V4 float4 a lane; float4 i of the 32 lanes is block i),
// statistics in two passes over the registers. One read of x, one write of y and of the codes.
template <int V4, bool F16>
__global__ void __launch_bounds__(256) ln_fwd_act8_kernel(const float* __restrict__ x, const float* __restrict__ w,
                                                          const float* __restrict__ b, uint16_t* __restrict__ y,
                                                          uint8_t* __restrict__ q, uint8_t* __restrict__ e,
                                                          float* __restrict__ rstd_out, int M, int H, int nb,
                                                          float eps) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= M) return;
  const long base = static_cast<long>(row) * H;
  float v[V4][4];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < V4; ++i) {
    const int j = kAct8Block * i + 4 * lane;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[i][k] = 0.f;
    if (j < H) load4<kActF32>(x, base + j, v[i]);
    s += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
  }
  const float mu = warp_sum(s) / H;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < V4; ++i) {
    const bool in = kAct8Block * i + 4 * lane < H;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[i][k] = in ? v[i][k] - mu : 0.f;
      ss = fmaf(v[i][k], v[i][k], ss);
    }
  }
  const float rstd = rsqrtf(warp_sum(ss) / H + eps);
  uint32_t mine = 0;  // lane i keeps the byte of block i
#pragma unroll
  for (int i = 0; i < V4; ++i) {
    const int j = kAct8Block * i + 4 * lane;
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[i][k] *= rstd;
      top = max(top, __float_as_uint(v[i][k]) & 0x7FFFFFFFu);
    }
    const uint32_t byte = act8_byte(__reduce_max_sync(0xffffffffu, top));
    if (lane == i) mine = byte;
    if (j < H) {
      *reinterpret_cast<uint32_t*>(q + base + j) = act8_codes(v[i], byte);
      float ww[4], bb[4], o[4];
      load4<kActF32>(w, j, ww);
      load4<kActF32>(b, j, bb);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = fmaf(v[i][k], ww[k], bb[k]);
      store4<F16 ? kActF16 : kActBf16>(y, base + j, o);
    }
  }
  if (lane < nb) e[static_cast<long>(row) * nb + lane] = static_cast<uint8_t>(mine);
  if (lane == 0) rstd_out[row] = rstd;
}

// LayerNorm backward: warps stride over rows; a lane keeps the row's codes (4 to a register, decoded twice: that is
// cheaper than four registers each) and dy, and its columns' dgamma / dbeta sums. All loads of a row are issued
// before its arithmetic, the incoming residual gradient before the first store (dres may be dres_in). Each CTA adds
// its warps' sums in a fixed order and leaves one partial row.
constexpr int kLnWarps = 8;
constexpr int ln_ctas_per_sm(int v4) { return v4 <= 4 ? 2 : 1; }  // 17 V4 registers and about 20 more a thread

template <int V4, bool F16>
__global__ void __launch_bounds__(256, ln_ctas_per_sm(V4))
    ln_bwd_act8_kernel(const float* __restrict__ dy, const uint8_t* __restrict__ q, const uint8_t* __restrict__ e,
                       const float* __restrict__ rstd, const float* __restrict__ w, const float* __restrict__ b,
                       const float* dres_in, float* dres, uint16_t* __restrict__ dres16, uint16_t* __restrict__ y,
                       float* __restrict__ part, int M, int H, int nb) {
  constexpr int kOut = F16 ? kActF16 : kActBf16;
  extern __shared__ float sums[];  // [kLnWarps][2][H]
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float ga[V4][4], ba[V4][4];
#pragma unroll
  for (int i = 0; i < V4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) ga[i][k] = ba[i][k] = 0.f;
#pragma unroll 1
  for (int r = blockIdx.x * kLnWarps + warp; r < M; r += gridDim.x * kLnWarps) {
    const long base = static_cast<long>(r) * H;
    uint32_t codes[V4];
    float d[V4][4];
#pragma unroll
    for (int i = 0; i < V4; ++i) {
      const int j = kAct8Block * i + 4 * lane;
      codes[i] = j < H ? *reinterpret_cast<const uint32_t*>(q + base + j) : 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) d[i][k] = 0.f;
      if (j < H) load4<kActF32>(dy, base + j, d[i]);
    }
    const uint32_t bytes = lane < nb ? e[static_cast<long>(r) * nb + lane] : 0u;
    const float rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < V4; ++i) {
      const int j = kAct8Block * i + 4 * lane;
      const float scale = act8_scale(__shfl_sync(0xffffffffu, bytes, i));
      if (j < H) {
        float xh[4], ww[4], bb[4], o[4];
        act8_values(codes[i], scale, xh);
        load4<kActF32>(w, j, ww);
        load4<kActF32>(b, j, bb);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          ga[i][k] = fmaf(d[i][k], xh[k], ga[i][k]);
          ba[i][k] += d[i][k];
          o[k] = fmaf(xh[k], ww[k], bb[k]);
          d[i][k] *= ww[k];
          s1 += d[i][k];
          s2 = fmaf(d[i][k], xh[k], s2);
        }
        store4<kOut>(y, base + j, o);
      }
    }
    const float m1 = warp_sum(s1) / H, m2 = warp_sum(s2) / H;
    float in[V4][4];
#pragma unroll
    for (int i = 0; i < V4; ++i) {
      const int j = kAct8Block * i + 4 * lane;
      if (j < H) load4<kActF32>(dres_in, base + j, in[i]);
    }
#pragma unroll
    for (int i = 0; i < V4; ++i) {
      const int j = kAct8Block * i + 4 * lane;
      const float scale = act8_scale(__shfl_sync(0xffffffffu, bytes, i));
      if (j < H) {
        float xh[4], o[4];
        act8_values(codes[i], scale, xh);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(rs, d[i][k] - m1 - xh[k] * m2, in[i][k]);
        store4<kActF32>(dres, base + j, o);
        store4<kOut>(dres16, base + j, o);
      }
    }
  }
  float* to = sums + static_cast<long>(warp) * 2 * H;
#pragma unroll
  for (int i = 0; i < V4; ++i) {
    const int j = kAct8Block * i + 4 * lane;
    if (j < H) {
      store4<kActF32>(to, j, ga[i]);
      store4<kActF32>(to, H + j, ba[i]);
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * H; c += 256) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kLnWarps; ++k) v += sums[static_cast<long>(k) * 2 * H + c];
    part[static_cast<long>(blockIdx.x) * 2 * H + c] = v;
  }
}

// dgamma / dbeta += the column sums of the CTAs' partial rows: 32 columns x 32 row slices a block, fixed order. Launched
// beside the backward kernel (programmatic dependent launch).
__global__ void __launch_bounds__(1024) ln_sum_act8_kernel(const float* __restrict__ part, int rows, int H,
                                                           float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < 2 * H) {
#pragma unroll 5
    for (int r = slice; r < rows; r += 32) v += __ldcg(part + static_cast<long>(r) * 2 * H + c);
  }
  red[slice][lane] = v;
  __syncthreads();
  if (slice == 0 && c < 2 * H) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += red[k][lane];
    if (c < H) dgamma[c] += s;
    else dbeta[c - H] += s;
  }
}

int blocks_of(long N) { return static_cast<int>((N + kAct8Block - 1) / kAct8Block); }
bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// CTAs of a pack or unpack launch over `blocks` blocks.
unsigned pack_ctas(long blocks) { return static_cast<unsigned>((blocks + 8 * kPackBlocks - 1) / (8 * kPackBlocks)); }

// Row widths in float4 a lane that kernels are built for.
#define HB_ACT8_WIDTHS(V4, ...)                                  \
  switch (V4) {                                                  \
    case 1: { constexpr int kV = 1; __VA_ARGS__; } break;        \
    case 2: { constexpr int kV = 2; __VA_ARGS__; } break;        \
    case 4: { constexpr int kV = 4; __VA_ARGS__; } break;        \
    case 6: { constexpr int kV = 6; __VA_ARGS__; } break;        \
    case 8: { constexpr int kV = 8; __VA_ARGS__; } break;        \
    case 10: { constexpr int kV = 10; __VA_ARGS__; } break;      \
    case 12: { constexpr int kV = 12; __VA_ARGS__; } break;      \
    default: { constexpr int kV = 16; __VA_ARGS__; } break;      \
  }
int width_v4(int H) {
  const int v = blocks_of(H);
  for (int a : {1, 2, 4, 6, 8, 10, 12})
    if (a >= v) return a;
  return 16;
}

}  // namespace

void act8_pack_launch(const void* x, long ld, int type, int8_t* q, uint8_t* e, long M, int N, cudaStream_t s) {
  if (M == 0 || N == 0) return;
  const int nb = blocks_of(N), bytes = type == kActF32 ? 4 : 2;
  const long blocks = M * nb;
  const bool vec = N % 4 == 0 && (M == 1 || ld % 4 == 0) && aligned(x, 4 * bytes) && aligned(q, 4);
#define HB_PACK(T) (vec ? act8_pack_kernel<T, true> : act8_pack_kernel<T, false>)
  auto* k = type == kActF32 ? HB_PACK(kActF32) : type == kActF16 ? HB_PACK(kActF16) : HB_PACK(kActBf16);
#undef HB_PACK
  k<<<pack_ctas(blocks), 256, 0, s>>>(x, ld, reinterpret_cast<uint8_t*>(q), e, static_cast<uint32_t>(blocks), N, nb);
  HB_CUDA_CHECK(cudaGetLastError());
}

void act8_unpack_launch(const int8_t* q, const uint8_t* e, int type, void* x, void* h, long M, int N, cudaStream_t s) {
  if (M == 0 || N == 0) return;
  const int nb = blocks_of(N), bytes = type == kActF32 ? 4 : 2;
  const long blocks = M * nb;
  const bool vec = N % 4 == 0 && aligned(q, 4) && aligned(x, 4 * bytes) && (!h || aligned(h, 4 * bytes));
#define HB_UNPACK(T)                                                                      \
  (h ? (vec ? act8_unpack_kernel<T, true, true> : act8_unpack_kernel<T, true, false>)     \
     : (vec ? act8_unpack_kernel<T, false, true> : act8_unpack_kernel<T, false, false>))
  auto* k = type == kActF32 ? HB_UNPACK(kActF32) : type == kActF16 ? HB_UNPACK(kActF16) : HB_UNPACK(kActBf16);
#undef HB_UNPACK
  k<<<pack_ctas(blocks), 256, 0, s>>>(reinterpret_cast<const uint8_t*>(q), e, x, h, static_cast<uint32_t>(blocks), N, nb);
  HB_CUDA_CHECK(cudaGetLastError());
}

void ln_fwd_act8_launch(const float* x, const float* w, const float* b, void* y, int8_t* q, uint8_t* e, float* rstd,
                        int M, int H, float eps, bool f16, cudaStream_t s) {
  if (M == 0) return;
  HB_ACT8_WIDTHS(width_v4(H),
                 (f16 ? ln_fwd_act8_kernel<kV, true> : ln_fwd_act8_kernel<kV, false>)<<<(M + 7) / 8, 256, 0, s>>>(
                     x, w, b, static_cast<uint16_t*>(y), reinterpret_cast<uint8_t*>(q), e, rstd, M, H, blocks_of(H), eps));
  HB_CUDA_CHECK(cudaGetLastError());
}

int ln_bwd_act8_ctas(int M, int H, int device) {
  const int full = ln_ctas_per_sm(width_v4(H)) * num_sms(device), need = (M + kLnWarps - 1) / kLnWarps;
  return std::max(1, std::min(need, full));
}

void ln_bwd_act8_launch(const float* dy, const int8_t* q, const uint8_t* e, const float* rstd, const float* w,
                        const float* b, const float* dres_in, float* dres, void* dres16, void* y, float* part, int ctas,
                        float* dgamma, float* dbeta, int M, int H, bool f16, cudaStream_t s) {
  if (M == 0) return;
  const size_t smem = static_cast<size_t>(kLnWarps) * 2 * H * sizeof(float);  // 128 KB at most
  HB_ACT8_WIDTHS(width_v4(H), {
    auto* k = f16 ? ln_bwd_act8_kernel<kV, true> : ln_bwd_act8_kernel<kV, false>;
    if (smem > 48 * 1024) {
      static std::atomic<uint64_t> ready[2];  // devices whose shared-memory limit is raised
      const uint64_t bit = uint64_t{1} << current_device();
      if (!(ready[f16].load(std::memory_order_relaxed) & bit)) {
        HB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kV * kLnWarps * 1024));
        ready[f16].fetch_or(bit, std::memory_order_relaxed);
      }
    }
    k<<<ctas, 256, smem, s>>>(dy, reinterpret_cast<const uint8_t*>(q), e, rstd, w, b, dres_in, dres,
                              static_cast<uint16_t*>(dres16), static_cast<uint16_t*>(y), part, M, H, blocks_of(H));
  });
  HB_CUDA_CHECK(cudaGetLastError());
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((2 * H + 31) / 32);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  HB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, ln_sum_act8_kernel, static_cast<const float*>(part), ctas, H, dgamma, dbeta));
}

}  // namespace hb
