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
// 16 bytes of an activation.
template <int TYPE, int E>
__device__ __forceinline__ void store_share(void* p, long i, const float (&v)[E]) {
  if constexpr (TYPE == kActF32) {
    store4<TYPE>(p, i, v);
  } else {
    constexpr bool F16 = TYPE == kActF16;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(pack16<F16>(v[0], v[1]), pack16<F16>(v[2], v[3]), pack16<F16>(v[4], v[5]), pack16<F16>(v[6], v[7]));
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
  // 127 * 2^8 < 65504, 127 * 2^120 < 2^127
  static constexpr uint32_t kClampByte = TYPE == kActF16 ? 127 + 9 : 127 + 121;
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

// One lane's share of a step of pack or unpack: 16 bytes of the activation, so 4 (fp32) or 8 consecutive columns, and
// a warp covers 1 or 2 blocks of 128 columns a step.
template <int TYPE>
struct Share {
  static constexpr int kElems = TYPE == kActF32 ? 4 : 8;
  static constexpr int kLanes = kAct8Block / kElems;  // lanes of a block
  static constexpr int kBlocks = 32 / kLanes;         // blocks of a step
};
template <int STEP>
__device__ __forceinline__ void next_block(uint32_t& row, uint32_t& k, uint32_t nb) {
  k += STEP;
#pragma unroll
  for (int i = 0; i < STEP; ++i)
    if (k >= nb) k -= nb, ++row;
}
// The bits of |x| in fp32 from those in its type.
template <int TYPE>
__device__ __forceinline__ uint32_t bits32(uint32_t b) {
  if constexpr (TYPE == kActF32) return b;
  else return __float_as_uint(to_f32<TYPE == kActF16>(static_cast<uint16_t>(b)));
}
constexpr int kPackSteps = 4;  // steps of one warp: their loads are in flight together

// Each warp takes kPackSteps * kBlocks consecutive blocks. VEC: N and the row stride are multiples of the share and
// rows start on 16-byte boundaries; else the lane's columns are kLanes apart and move one by one. Bound by memory:
// each value is loaded and stored once (8192 x 5120 bf16: pack 126 MB in 25 us, unpack with GELU 210 MB in 35 us, 6.0
// TB/s; 2 or 8 steps a warp, or a resident grid that loops, measured the same or slower).
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(256) act8_pack_kernel(const void* __restrict__ x, long ld, uint8_t* __restrict__ q,
                                                        uint8_t* __restrict__ e, uint32_t blocks, int N, uint32_t nb) {
  using S = Share<TYPE>;
  constexpr int E = S::kElems;
  const int lane = threadIdx.x & 31, part = lane / S::kLanes, sub = lane % S::kLanes;
  const uint32_t first = (blockIdx.x * 8 + (threadIdx.x >> 5)) * (kPackSteps * S::kBlocks);
  uint32_t r = (first + part) / nb, k = first + part - r * nb;  // row, and block of the row
  long row[kPackSteps];
  int col[kPackSteps];  // first column of the lane's share; N: none
  float v[kPackSteps][E];
#pragma unroll
  for (int u = 0; u < kPackSteps; ++u) {
    row[u] = r;
    col[u] = first + part + u * S::kBlocks < blocks ? static_cast<int>(k) * kAct8Block + (VEC ? E * sub : sub) : N;
    next_block<S::kBlocks>(r, k, nb);
#pragma unroll
    for (int i = 0; i < E; ++i) v[u][i] = 0.f;
    if constexpr (VEC) {
      if (col[u] < N) {
#pragma unroll
        for (int i = 0; i < E; i += 4)
          load4<TYPE>(x, row[u] * ld + col[u] + i, *reinterpret_cast<float(*)[4]>(&v[u][i]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (col[u] + S::kLanes * i < N) v[u][i] = load1<TYPE>(x, row[u] * ld + col[u] + S::kLanes * i);
    }
  }
  uint32_t mine = 0;  // lane i keeps the byte of block i
#pragma unroll
  for (int u = 0; u < kPackSteps; ++u) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) top = max(top, __float_as_uint(v[u][i]) & 0x7FFFFFFFu);
    if constexpr (S::kBlocks == 1) {
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == u) mine = top;
    } else {
      const uint32_t t0 = __reduce_max_sync(0xffffffffu, part == 0 ? top : 0u);
      const uint32_t t1 = __reduce_max_sync(0xffffffffu, part == 1 ? top : 0u);
      top = part == 0 ? t0 : t1;
      if (lane / 2 == u) mine = lane & 1 ? t1 : t0;
    }
    const uint32_t byte = act8_byte(top);
    uint32_t codes[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) codes[i] = act8_codes(*reinterpret_cast<float(*)[4]>(&v[u][4 * i]), byte);
    uint8_t* to = q + row[u] * N + col[u];
    if constexpr (VEC) {
      if (col[u] < N) {
        if constexpr (E == 8) *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
        else *reinterpret_cast<uint32_t*>(to) = codes[0];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (col[u] + S::kLanes * i < N) to[S::kLanes * i] = static_cast<uint8_t>(codes[i / 4] >> (8 * (i & 3)));
    }
  }
  if (lane < kPackSteps * S::kBlocks && first + lane < blocks) e[first + lane] = static_cast<uint8_t>(act8_byte(mine));
}

// Flat pack: rows that follow one another without a gap and hold whole blocks are one long row. Without the row and
// column of every step, and with the maximum of 16-bit types taken on their bits, two at a time (|x| orders like its
// bits), the warps' instructions no longer hold up the memory: 8192 x 5120 bf16 in 21.8 us, 5.8 TB/s (25.0 as above),
// fp32 in 31.7 (35.4); 8192 x 1280 bf16, in L2, 5.7 (7.1). The same for unpack gains nothing from DRAM (21.1, 35.0).
template <int TYPE>
__global__ void __launch_bounds__(256) act8_pack_flat_kernel(const uint4* __restrict__ x, uint8_t* __restrict__ q,
                                                             uint8_t* __restrict__ e, uint32_t blocks) {
  using S = Share<TYPE>;
  constexpr int E = S::kElems;
  const int lane = threadIdx.x & 31, part = lane / S::kLanes;
  const uint32_t first = (blockIdx.x * 8 + (threadIdx.x >> 5)) * (kPackSteps * S::kBlocks);
  const long base = static_cast<long>(first) * S::kLanes + lane;
  uint4 raw[kPackSteps];
#pragma unroll
  for (int u = 0; u < kPackSteps; ++u) {
    raw[u] = make_uint4(0u, 0u, 0u, 0u);
    if (first + part + u * S::kBlocks < blocks) raw[u] = x[base + 32 * u];
  }
  uint32_t mine = 0;  // lane i keeps the byte of block i
#pragma unroll
  for (int u = 0; u < kPackSteps; ++u) {
    uint32_t top;
    float v[E];
    if constexpr (TYPE == kActF32) {
      v[0] = __uint_as_float(raw[u].x), v[1] = __uint_as_float(raw[u].y);
      v[2] = __uint_as_float(raw[u].z), v[3] = __uint_as_float(raw[u].w);
      top = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    } else {
      constexpr bool F16 = TYPE == kActF16;
      const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t = __vmaxu2(t, w[i] & 0x7FFF7FFFu);
        v[2 * i] = lo16<F16>(w[i]), v[2 * i + 1] = hi16<F16>(w[i]);
      }
      top = max(t & 0xFFFFu, t >> 16);
    }
    if constexpr (S::kBlocks == 1) {
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == u) mine = top;
    } else {
      const uint32_t t0 = __reduce_max_sync(0xffffffffu, part == 0 ? top : 0u);
      const uint32_t t1 = __reduce_max_sync(0xffffffffu, part == 1 ? top : 0u);
      top = part == 0 ? t0 : t1;
      if (lane / 2 == u) mine = lane & 1 ? t1 : t0;
    }
    const uint32_t byte = act8_byte(bits32<TYPE>(top));
    uint32_t codes[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) codes[i] = act8_codes(*reinterpret_cast<float(*)[4]>(&v[4 * i]), byte);
    if (first + part + u * S::kBlocks < blocks) {
      if constexpr (E == 8) reinterpret_cast<uint2*>(q)[base + 32 * u] = make_uint2(codes[0], codes[1]);
      else reinterpret_cast<uint32_t*>(q)[base + 32 * u] = codes[0];
    }
  }
  if (lane < kPackSteps * S::kBlocks && first + lane < blocks)
    e[first + lane] = static_cast<uint8_t>(act8_byte(bits32<TYPE>(mine)));
}

template <int TYPE, bool GELU, bool VEC>
__global__ void __launch_bounds__(256) act8_unpack_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e,
                                                          void* __restrict__ x, void* __restrict__ h, uint32_t blocks,
                                                          int N, uint32_t nb) {
  using S = Share<TYPE>;
  constexpr int E = S::kElems;
  const int lane = threadIdx.x & 31, part = lane / S::kLanes, sub = lane % S::kLanes;
  const uint32_t first = (blockIdx.x * 8 + (threadIdx.x >> 5)) * (kPackSteps * S::kBlocks) + part;
  uint32_t r = first / nb, k = first - r * nb;
  long at[kPackSteps];
  int col[kPackSteps];
  uint32_t codes[kPackSteps][E / 4], byte[kPackSteps];
#pragma unroll
  for (int u = 0; u < kPackSteps; ++u) {
    const uint32_t blk = first + u * S::kBlocks;
    col[u] = blk < blocks ? static_cast<int>(k) * kAct8Block + (VEC ? E * sub : sub) : N;
    at[u] = static_cast<long>(r) * N + col[u];
    byte[u] = blk < blocks ? e[blk] : 0;
    next_block<S::kBlocks>(r, k, nb);
#pragma unroll
    for (int i = 0; i < E / 4; ++i) codes[u][i] = 0;
    if constexpr (VEC) {
      if (col[u] < N) {
        if constexpr (E == 8) {
          const uint2 c = *reinterpret_cast<const uint2*>(q + at[u]);
          codes[u][0] = c.x, codes[u][1] = c.y;
        } else {
          codes[u][0] = *reinterpret_cast<const uint32_t*>(q + at[u]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (col[u] + S::kLanes * i < N)
          codes[u][i / 4] |= static_cast<uint32_t>(q[at[u] + S::kLanes * i]) << (8 * (i & 3));
    }
  }
#pragma unroll
  for (int u = 0; u < kPackSteps; ++u) {
    float v[E], g[E];
#pragma unroll
    for (int i = 0; i < E; i += 4) decode4<TYPE>(codes[u][i / 4], byte[u], *reinterpret_cast<float(*)[4]>(&v[i]));
    if constexpr (GELU) {
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = gelu_full(v[i]);
    }
    if constexpr (VEC) {
      if (col[u] < N) {
        store_share<TYPE>(x, at[u], v);
        if constexpr (GELU) store_share<TYPE>(h, at[u], g);
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (col[u] + S::kLanes * i < N) {
          store1<TYPE>(x, at[u] + S::kLanes * i, v[i]);
          if constexpr (GELU) store1<TYPE>(h, at[u] + S::kLanes * i, g[i]);
        }
      }
    }
  }
}

// LayerNorm forward: one warp per row, the row in registers (V4 float4 a lane; float4 i of the 32 lanes is block i),
// statistics in two passes over the registers, in the order of ln_fwd_kernel (norm.cu): y has the same bits, so keeping
// activations in 8 bits leaves the forward pass as it is. One read of x, one write of y and of the codes: 8192 x 1280,
// 73 MB in 17.6 us of a graph of such calls (the 16-bit LayerNorm, 63 MB: 11.2).
// xh in 32 bits is off by up to 3 units in its last place, 4e-5 of a step, and by the rounding of the row's mean (5e-6 of
// a standard deviation, 2e-4 of a step, where the mean is 100 of them). So where it lies closer to the middle between
// two codes than 2^-14 and the mean's rounding (one value in 8000 of centred rows), the four codes are taken again from
// x, with a mean and rstd to about 1e-8: 0.1 to 0.2 codes of a million then differ from those of xh in 64 bits, without
// it 1.5 (and 3 us less), and without the mean's part of it 46 at a mean of 100 standard deviations (0.4 us less: a
// register spills; the mean and rstd kept in fewer registers take 18.2 us, their conversions move in front of the rows).
// The second look kept for the end of the row takes 3 us more (the row read again) or 19 (held in registers, which spill).
constexpr float kNearTie = 0.5f - 0x1p-14f;
__device__ __forceinline__ uint32_t ln_act8_tie(const float* __restrict__ x, double mean, double scaled) {
  float v[4];
  load4<kActF32>(x, 0, v);
  uint32_t codes = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const double t = fmin(fmax((v[k] - mean) * scaled, -127.0), 127.0);
    codes |= (static_cast<uint32_t>(__double2int_rn(t)) & 0xFFu) << (8 * k);
  }
  return codes;
}
// CTAs an SM that the registers are held to (64 a thread and 4 CTAs at 1280 columns; 80 and 3 took 20.7 us).
constexpr int ln_fwd_ctas(int v4) { return v4 <= 2 ? 8 : v4 <= 4 ? 6 : v4 <= 6 ? 5 : v4 <= 10 ? 4 : v4 <= 12 ? 3 : 2; }
template <int V4, bool F16>
__global__ void __launch_bounds__(256, ln_fwd_ctas(V4))
    ln_fwd_act8_kernel(const float* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                       uint16_t* __restrict__ y, uint8_t* __restrict__ q, uint8_t* __restrict__ e,
                       float* __restrict__ rstd_out, int M, int H, int nb, float eps) {
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
    s += v[i][0] + v[i][1] + v[i][2] + v[i][3];
  }
  const float mu = warp_sum(s) / H;
  float ss = 0.f, rest = 0.f;
  double wide = 0.0;
#pragma unroll
  for (int i = 0; i < V4; ++i) {
    if (kAct8Block * i + 4 * lane < H) {
      const float a = v[i][0] - mu, c = v[i][1] - mu, d = v[i][2] - mu, f = v[i][3] - mu;
      const float sq = a * a + c * c + d * d + f * f;
      ss += sq;
      wide += sq;
      rest += (a + c) + (d + f);
    }
  }
  const float rstd = rsqrtf(warp_sum(ss) / H + eps);
  // for the ties: what the sum of x - mu leaves of the mean, and rstd by a Newton step on the squares' 64-bit sum
  const double part = 1.0 / H, off = warp_sum(rest) * part, mean = mu + off;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wide += __shfl_xor_sync(0xffffffffu, wide, o);
  const double r = rstd, rstd_wide = r * (1.5 - 0.5 * (wide * part - off * off + eps) * r * r);
  const float lean = fabsf(static_cast<float>(off)) * rstd;  // what the mean's rounding moves every xh by
  uint32_t mine = 0;  // lane i keeps the byte of block i
#pragma unroll
  for (int i = 0; i < V4; ++i) {
    const int j = kAct8Block * i + 4 * lane;
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[i][k] = j < H ? (v[i][k] - mu) * rstd : 0.f;
      top = max(top, __float_as_uint(v[i][k]) & 0x7FFFFFFFu);
    }
    const uint32_t byte = act8_byte(__reduce_max_sync(0xffffffffu, top));
    if (lane == i) mine = byte;
    if (j < H) {
      uint32_t codes = act8_codes(v[i], byte);
      if (byte != kAct8Nan && fmaf(lean, act8_inv_scale(byte), act8_off_code(v[i], byte)) > kNearTie)
        codes = ln_act8_tie(x + base + j, mean, rstd_wide * act8_inv_scale(byte));
      *reinterpret_cast<uint32_t*>(q + base + j) = codes;
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

// LayerNorm backward: groups of WPR warps stride over rows, each warp with V4 of the row's blocks of 128 columns (at
// most 6, so that 16 warps fit an SM's registers; they join their two sums through shared memory, one barrier of the
// group a row). Every lane copies its own columns of a row (dy, codes, the incoming residual
// gradient) into shared memory of its own with asynchronous copies, the next row's dy and codes as soon as this row's
// are in registers and its residual gradient once this row's is used, so copies are in flight all the time and need
// no barrier (with plain loads the few warps that the registers allow waited for memory: 40 us at 8192 x 1280). The
// column sums of dgamma and dbeta stay in registers; codes are decoded twice, which is cheaper than four registers
// each. 8192 x 1280: 178 MB in 31 us, 5.7 TB/s; 8192 x 2048 in 47 us, 6.1 TB/s (one warp a row and 8 warps an SM: 36 and
// 60 us). Each CTA adds its groups' sums in a fixed order and leaves one partial row. dres may be dres_in: a row's
// residual gradient is read before its outputs are stored, by the same lane.
constexpr int kLnWarps = 8;
constexpr int kLnCtasPerSm = 2;
constexpr int ln_slot_bytes(int v4) { return v4 * 32 * 36; }      // of one warp: 16 + 16 + 4 bytes a lane and block

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits for all but the newest group.
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
__device__ __forceinline__ void read16(uint32_t from, float (&v)[4]) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
               : "r"(from)
               : "memory");
}
__device__ __forceinline__ uint32_t read4(uint32_t from) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
  return v;
}

template <int V4, int WPR, bool F16>
__global__ void __launch_bounds__(256, kLnCtasPerSm)
    ln_bwd_act8_kernel(const float* __restrict__ dy, const uint8_t* __restrict__ q, const uint8_t* __restrict__ e,
                       const float* __restrict__ rstd, const float* __restrict__ w, const float* __restrict__ b,
                       const float* dres_in, float* dres, uint16_t* __restrict__ dres16, uint16_t* __restrict__ y,
                       float* __restrict__ part, int M, int H, int nb) {
  constexpr int kOut = F16 ? kActF16 : kActBf16;
  constexpr int kGroups = kLnWarps / WPR;
  extern __shared__ __align__(16) float sums[];  // the warps' slots; after the rows, [kGroups][2][H]
  __shared__ float joint[2][kLnWarps][2];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = warp / WPR;
  const int blk0 = warp % WPR * V4;                // this warp's first block
  const int col0 = kAct8Block * blk0 + 4 * lane;  // this lane's first column
  // this lane's slots of block i: dy, residual gradient, codes
  const uint32_t slot = smem_u32(sums) + warp * ln_slot_bytes(V4) + lane * 16;
  const uint32_t slot_in = slot + V4 * 512, slot_q = slot + V4 * 1024 - lane * 12;
  const int stride = gridDim.x * kGroups;
  const auto copy_dy = [&](int r) {
    const long base = static_cast<long>(r) * H + col0;
#pragma unroll
    for (int i = 0; i < V4; ++i) {
      if (kAct8Block * i + col0 < H) {
        copy16(slot + 512 * i, dy + base + kAct8Block * i);
        copy4(slot_q + 128 * i, q + base + kAct8Block * i);
      }
    }
  };
  const auto copy_in = [&](int r) {
    const long base = static_cast<long>(r) * H + col0;
#pragma unroll
    for (int i = 0; i < V4; ++i)
      if (kAct8Block * i + col0 < H) copy16(slot_in + 512 * i, dres_in + base + kAct8Block * i);
  };
  float ga[V4][4], ba[V4][4];
#pragma unroll
  for (int i = 0; i < V4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) ga[i][k] = ba[i][k] = 0.f;
  int r = blockIdx.x * kGroups + group, parity = 0;
  uint32_t bytes = 0;
  float rs = 0.f;
  if (r < M) {
    copy_dy(r);
    copies_commit();
    copy_in(r);
    copies_commit();
    bytes = lane < nb ? e[static_cast<long>(r) * nb + lane] : 0u;
    rs = rstd[r];
  }
#pragma unroll 1
  for (; r < M; r += stride) {
    const long base = static_cast<long>(r) * H;
    const int next = r + stride;
    uint32_t codes[V4];
    float d[V4][4];
    copies_wait();  // dy and codes; the residual gradient may be on its way
#pragma unroll
    for (int i = 0; i < V4; ++i) {
      codes[i] = 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) d[i][k] = 0.f;
      if (kAct8Block * i + col0 < H) {
        read16(slot + 512 * i, d[i]);
        codes[i] = read4(slot_q + 128 * i);
      }
    }
    uint32_t next_bytes = 0;
    float next_rs = 0.f;
    if (next < M) {
      copy_dy(next);
      next_bytes = lane < nb ? e[static_cast<long>(next) * nb + lane] : 0u;
      next_rs = rstd[next];
    }
    copies_commit();
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < V4; ++i) {
      const int j = kAct8Block * i + col0;
      const float scale = act8_scale(__shfl_sync(0xffffffffu, bytes, blk0 + i));
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
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if constexpr (WPR > 1) {
      if (lane == 0) {
        joint[parity][warp][0] = s1;
        joint[parity][warp][1] = s2;
      }
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(32 * WPR) : "memory");
      s1 = s2 = 0.f;
#pragma unroll
      for (int k = 0; k < WPR; ++k) {
        s1 += joint[parity][group * WPR + k][0];
        s2 += joint[parity][group * WPR + k][1];
      }
      parity ^= 1;  // the next row writes the other half: no second barrier
    }
    const float m1 = s1 / H, m2 = s2 / H;
    copies_wait();  // the residual gradient; the next row's dy may be on its way
#pragma unroll
    for (int i = 0; i < V4; ++i) {
      const int j = kAct8Block * i + col0;
      const float scale = act8_scale(__shfl_sync(0xffffffffu, bytes, blk0 + i));
      if (j < H) {
        float xh[4], in[4], o[4];
        act8_values(codes[i], scale, xh);
        read16(slot_in + 512 * i, in);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(rs, d[i][k] - m1 - xh[k] * m2, in[k]);
        store4<kActF32>(dres, base + j, o);
        store4<kOut>(dres16, base + j, o);
      }
    }
    if (next < M) copy_in(next);
    copies_commit();
    bytes = next_bytes;
    rs = next_rs;
  }
  __syncthreads();  // the slots become the sums
  float* to = sums + static_cast<long>(group) * 2 * H;
#pragma unroll
  for (int i = 0; i < V4; ++i) {
    const int j = kAct8Block * i + col0;
    if (j < H) {
      store4<kActF32>(to, j, ga[i]);
      store4<kActF32>(to, H + j, ba[i]);
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * H; c += 256) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) v += sums[static_cast<long>(k) * 2 * H + c];
    part[static_cast<long>(blockIdx.x) * 2 * H + c] = v;
  }
}

// dgamma / dbeta += the column sums of the CTAs' partial rows: 32 columns x 32 row slices a block, fixed order, in 64
// bits (some 300 rows in 32 bits double the sums' error: 1.3e-5 root mean square for 6.2e-6, 8192 x 1280 normal values;
// the time is the same). Launched beside the backward kernel (programmatic dependent launch).
__global__ void __launch_bounds__(1024) ln_sum_act8_kernel(const float* __restrict__ part, int rows, int H,
                                                           float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ double red[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  double v = 0.0;
  if (c < 2 * H) {
#pragma unroll 5
    for (int r = slice; r < rows; r += 32) v += __ldcg(part + static_cast<long>(r) * 2 * H + c);
  }
  red[slice][lane] = v;
  __syncthreads();
  if (slice == 0 && c < 2 * H) {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += red[k][lane];
    float* to = c < H ? dgamma + c : dbeta + c - H;
    *to = static_cast<float>(*to + s);
  }
}

int blocks_of(long N) { return static_cast<int>((N + kAct8Block - 1) / kAct8Block); }
bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// CTAs of a pack or unpack launch over `blocks` blocks.
unsigned pack_ctas(long blocks, int type) {
  const long per_cta = 8L * kPackSteps * (type == kActF32 ? 1 : 2);
  return static_cast<unsigned>((blocks + per_cta - 1) / per_cta);
}

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
  const int nb = blocks_of(N), share = type == kActF32 ? 4 : 8;
  const long blocks = M * nb;
  const bool vec = N % share == 0 && (M == 1 || ld % share == 0) && aligned(x, 16) && aligned(q, share);
  if (vec && (M == 1 || ld == N) && N % kAct8Block == 0) {
    auto* k = type == kActF32   ? act8_pack_flat_kernel<kActF32>
              : type == kActF16 ? act8_pack_flat_kernel<kActF16>
                                : act8_pack_flat_kernel<kActBf16>;
    k<<<pack_ctas(blocks, type), 256, 0, s>>>(static_cast<const uint4*>(x), reinterpret_cast<uint8_t*>(q), e,
                                              static_cast<uint32_t>(blocks));
    HB_CUDA_CHECK(cudaGetLastError());
    return;
  }
#define HB_PACK(T) (vec ? act8_pack_kernel<T, true> : act8_pack_kernel<T, false>)
  auto* k = type == kActF32 ? HB_PACK(kActF32) : type == kActF16 ? HB_PACK(kActF16) : HB_PACK(kActBf16);
#undef HB_PACK
  k<<<pack_ctas(blocks, type), 256, 0, s>>>(x, ld, reinterpret_cast<uint8_t*>(q), e, static_cast<uint32_t>(blocks), N,
                                            nb);
  HB_CUDA_CHECK(cudaGetLastError());
}

void act8_unpack_launch(const int8_t* q, const uint8_t* e, int type, void* x, void* h, long M, int N, cudaStream_t s) {
  if (M == 0 || N == 0) return;
  const int nb = blocks_of(N), share = type == kActF32 ? 4 : 8;
  const long blocks = M * nb;
  const bool vec = N % share == 0 && aligned(q, share) && aligned(x, 16) && (!h || aligned(h, 16));
#define HB_UNPACK(T)                                                                      \
  (h ? (vec ? act8_unpack_kernel<T, true, true> : act8_unpack_kernel<T, true, false>)     \
     : (vec ? act8_unpack_kernel<T, false, true> : act8_unpack_kernel<T, false, false>))
  auto* k = type == kActF32 ? HB_UNPACK(kActF32) : type == kActF16 ? HB_UNPACK(kActF16) : HB_UNPACK(kActBf16);
#undef HB_UNPACK
  k<<<pack_ctas(blocks, type), 256, 0, s>>>(reinterpret_cast<const uint8_t*>(q), e, x, h,
                                            static_cast<uint32_t>(blocks), N, nb);
  HB_CUDA_CHECK(cudaGetLastError());
}

void ln_fwd_act8_launch(const float* x, const float* w, const float* b, void* y, int8_t* q, uint8_t* e, float* rstd,
                        int M, int H, float eps, bool f16, cudaStream_t s) {
  if (M == 0) return;
  HB_ACT8_WIDTHS(width_v4(H),
                 (f16 ? ln_fwd_act8_kernel<kV, true> : ln_fwd_act8_kernel<kV, false>)<<<(M + 7) / 8, 256, 0, s>>>(
                     x, w, b, static_cast<uint16_t*>(y), reinterpret_cast<uint8_t*>(q), e, rstd, M, H, blocks_of(H),
                     eps));
  HB_CUDA_CHECK(cudaGetLastError());
}

// Warps that share a row of the backward, and the blocks each of them takes: at most 6.
static int ln_bwd_warps(int H) { return width_v4(H) <= 6 ? 1 : width_v4(H) <= 12 ? 2 : 4; }

int ln_bwd_act8_ctas(int M, int H, int device) {
  const int groups = kLnWarps / ln_bwd_warps(H);
  return std::max(1, std::min((M + groups - 1) / groups, kLnCtasPerSm * num_sms(device)));
}

void ln_bwd_act8_launch(const float* dy, const int8_t* q, const uint8_t* e, const float* rstd, const float* w,
                        const float* b, const float* dres_in, float* dres, void* dres16, void* y, float* part, int ctas,
                        float* dgamma, float* dbeta, int M, int H, bool f16, cudaStream_t s) {
  if (M == 0) return;
  HB_ACT8_WIDTHS(width_v4(H), {
    constexpr int kWpr = kV <= 6 ? 1 : kV <= 12 ? 2 : 4;
    constexpr int kSmem = kLnWarps * ln_slot_bytes(kV / kWpr);  // the sums, 8 / kWpr * 2 H floats, need less
    static_assert(kLnWarps / kWpr * 2 * kV * kAct8Block * 4 <= kSmem, "the sums take the place of the slots");
    auto* k = f16 ? ln_bwd_act8_kernel<kV / kWpr, kWpr, true> : ln_bwd_act8_kernel<kV / kWpr, kWpr, false>;
    if (kSmem > 48 * 1024) {
      static std::atomic<uint64_t> ready[2];  // devices whose shared-memory limit is raised
      const uint64_t bit = uint64_t{1} << current_device();
      if (!(ready[f16].load(std::memory_order_relaxed) & bit)) {
        HB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        ready[f16].fetch_or(bit, std::memory_order_relaxed);
      }
    }
    k<<<ctas, 256, kSmem, s>>>(dy, reinterpret_cast<const uint8_t*>(q), e, rstd, w, b, dres_in, dres,
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
