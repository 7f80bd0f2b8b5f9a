// A paged key/value cache: K and V of new tokens into their slots, in 16 bits or quantised to 8 as they are
// written (the format of act8.cuh with a block per head of a token), and back.
#include "act8.cuh"
#include "common.cuh"
#include "decode_args.h"
#include "host_utils.h"

namespace hb {

namespace {

constexpr int kThreads = 256;
constexpr int kSiteWrite = 420, kSiteRead = 421;  // status sites

// Eight consecutive 16-bit elements.
__device__ __forceinline__ uint4 load8(const void* p, long i, bool vec) {
  const uint16_t* s = static_cast<const uint16_t*>(p) + i;
  if (vec) return *reinterpret_cast<const uint4*>(s);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = s[2 * j] | (static_cast<uint32_t>(s[2 * j + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Codes of eight elements whose head is held by LANES neighbouring lanes; `byte`: the head's exponent byte.
template <int LANES>
__device__ __forceinline__ uint2 quantise8(const uint4& r, bool f16, uint32_t& byte) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  float x[8];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = f16 ? lo16<true>(w[j]) : lo16<false>(w[j]);
    x[2 * j + 1] = f16 ? hi16<true>(w[j]) : hi16<false>(w[j]);
    top = max(top, max(__float_as_uint(x[2 * j]) & 0x7FFFFFFFu, __float_as_uint(x[2 * j + 1]) & 0x7FFFFFFFu));
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  byte = act8_byte(top);
  const float a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
  return make_uint2(act8_codes(a, byte), act8_codes(b, byte));
}

// LANES = dim / 8 neighbouring threads take one head of one token, K and V.
template <int LANES, bool CODES>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvTokens t, const KvPool p, int* status) {
  const long id = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
  const int row = static_cast<int>(min(id / LANES, static_cast<long>(t.n) * p.heads - 1));
  const int part = threadIdx.x % LANES, token = row / p.heads, head = row - token * p.heads;
  const int64_t slot = t.slots[token];
  const bool in = slot >= 0 && slot < static_cast<int64_t>(p.pages) * p.size;
  const bool live = in && id / LANES == row;  // threads behind the last row only take part in the exchange of lanes
  if (slot >= 0 && !in && part == 0 && head == 0) record_error(status, kBadArg, kSiteWrite);
  const uint4 k = load8(t.k, token * t.kt + head * t.kh + part * 8, t.vec);
  const uint4 v = load8(t.v, token * t.vt + head * t.vh + part * 8, t.vec);
  const long page = in ? slot / p.size : 0, at = in ? slot - page * p.size : 0;
  const long ki = page * p.kp + head * p.kh + at * p.ks + part * 8, vi = page * p.vp + head * p.vh + at * p.vs + part * 8;
  if constexpr (CODES) {
    uint32_t kb, vb;
    const uint2 kc = quantise8<LANES>(k, t.f16, kb), vc = quantise8<LANES>(v, t.f16, vb);
    if (live) {
      *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.k) + ki) = kc;
      *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.v) + vi) = vc;
      if (part == 0) {
        p.ke[page * p.kep + head * p.keh + at] = static_cast<uint8_t>(kb);
        p.ve[page * p.vep + head * p.veh + at] = static_cast<uint8_t>(vb);
      }
    }
  } else if (live) {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.k) + ki) = k;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.v) + vi) = v;
  }
}

// Types of the values read back.
enum OutType : int { kOutBf16 = 0, kOutF16 = 1, kOutF32 = 2 };

// The largest finite value of each: a code rounded up can stand for more than the type holds.
template <int OUT>
__device__ __forceinline__ float largest() {
  return OUT == kOutF16 ? 65504.f : OUT == kOutBf16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
}
template <int OUT>
__device__ __forceinline__ void store8(void* p, long i, const float (&v)[8]) {
  if constexpr (OUT == kOutF32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    constexpr bool F16 = OUT == kOutF16;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(pack16<F16>(v[0], v[1]), pack16<F16>(v[2], v[3]), pack16<F16>(v[4], v[5]), pack16<F16>(v[6], v[7]));
  }
}
template <int OUT>
__device__ __forceinline__ void decode8(const uint2& codes, uint32_t byte, float (&v)[8]) {
  float a[4], b[4];
  act8_values(codes.x, act8_scale(byte), a);
  act8_values(codes.y, act8_scale(byte), b);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  if (byte != kAct8Nan) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fminf(fmaxf(v[j], -largest<OUT>()), largest<OUT>());
  }
}

// OUT: type of the codes' values; a 16-bit cache is copied. Tokens without a slot read as zeros, those whose slot is
// outside the cache as NaN.
template <int LANES, bool CODES, int OUT>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const int64_t* __restrict__ slots, const KvPool p, void* k,
                                                           void* v, int n, int* status) {
  const long id = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
  if (id / LANES >= static_cast<long>(n) * p.heads) return;
  const int row = static_cast<int>(id / LANES);
  const int part = threadIdx.x % LANES, token = row / p.heads, head = row - token * p.heads;
  const int64_t slot = slots[token];
  const bool in = slot >= 0 && slot < static_cast<int64_t>(p.pages) * p.size;
  if (slot >= 0 && !in && part == 0 && head == 0) record_error(status, kBadArg, kSiteRead);
  const long page = in ? slot / p.size : 0, at = in ? slot - page * p.size : 0, o = id * 8;
  const long ki = page * p.kp + head * p.kh + at * p.ks + part * 8, vi = page * p.vp + head * p.vh + at * p.vs + part * 8;
  if (!in) {
    const float x = slot < 0 ? 0.f : __uint_as_float(0x7FC00000u);
    const float none[8] = {x, x, x, x, x, x, x, x};
    store8<OUT>(k, o, none);
    store8<OUT>(v, o, none);
  } else if constexpr (CODES) {
    const uint2 kc = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p.k) + ki);
    const uint2 vc = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p.v) + vi);
    const uint32_t kb = p.ke[page * p.kep + head * p.keh + at], vb = p.ve[page * p.vep + head * p.veh + at];
    float x[8];
    decode8<OUT>(kc, kb, x);
    store8<OUT>(k, o, x);
    decode8<OUT>(vc, vb, x);
    store8<OUT>(v, o, x);
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.k) + ki);
    const uint4 b = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.v) + vi);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(k) + o) = a;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(v) + o) = b;
  }
}

unsigned blocks_for(long threads) { return static_cast<unsigned>((threads + kThreads - 1) / kThreads); }

template <int LANES>
void write_dim(const KvTokens& t, const KvPool& p, int* status, cudaStream_t s) {
  const unsigned grid = blocks_for(static_cast<long>(t.n) * p.heads * LANES);
  if (p.type == kKvCodes) kv_write_kernel<LANES, true><<<grid, kThreads, 0, s>>>(t, p, status);
  else kv_write_kernel<LANES, false><<<grid, kThreads, 0, s>>>(t, p, status);
}
template <int LANES>
void read_dim(const int64_t* slots, const KvPool& p, void* k, void* v, int n, int out, int* status, cudaStream_t s) {
  const unsigned grid = blocks_for(static_cast<long>(n) * p.heads * LANES);
  const auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, s>>>(slots, p, k, v, n, status); };
  if (p.type == kKvBf16) go(kv_read_kernel<LANES, false, kOutBf16>);
  else if (p.type == kKvF16) go(kv_read_kernel<LANES, false, kOutF16>);
  else if (out == kOutBf16) go(kv_read_kernel<LANES, true, kOutBf16>);
  else if (out == kOutF16) go(kv_read_kernel<LANES, true, kOutF16>);
  else go(kv_read_kernel<LANES, true, kOutF32>);
}

}  // namespace

void kv_write_launch(const KvTokens& t, const KvPool& p, int* status, cudaStream_t s) {
  if (t.n == 0) return;
  switch (p.dim) {
    case 16: write_dim<2>(t, p, status, s); break;
    case 32: write_dim<4>(t, p, status, s); break;
    case 64: write_dim<8>(t, p, status, s); break;
    default: write_dim<16>(t, p, status, s); break;
  }
  HB_CUDA_CHECK(cudaGetLastError());
}

void kv_read_launch(const int64_t* slots, const KvPool& p, void* k, void* v, int n, int out, int* status,
                    cudaStream_t s) {
  if (n == 0) return;
  switch (p.dim) {
    case 16: read_dim<2>(slots, p, k, v, n, out, status, s); break;
    case 32: read_dim<4>(slots, p, k, v, n, out, status, s); break;
    case 64: read_dim<8>(slots, p, k, v, n, out, status, s); break;
    default: read_dim<16>(slots, p, k, v, n, out, status, s); break;
  }
  HB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace hb
