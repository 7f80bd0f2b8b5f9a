// A paged key/value cache: K and V of new tokens into their slots, in 16 bits or quantised to 8 as they are
// written (the format of act8.cuh with a block per head of a token), and back:
//   byte = e + 127, e >= -126 the least with max |x| <= 127 * 2^e over a head of a token;  code = rint(x / 2^e);  x' = code * 2^e
// Bound by memory (one pass, 16 bytes a load), and for a step's few tokens by the launch. B200, write and read together:
// 8192 tokens of 20 heads of 64 into 8 bits and back 27.0 us (126 MB, 4.7 TB/s), 4099 of 12 heads in 16 bits 9.5 us,
// 16 tokens into 8 bits 4.2 us.
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
template <int LANES, bool F16>
__device__ __forceinline__ uint2 quantise8(const uint4& r, uint32_t& byte) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  uint32_t top = 0;  // of the magnitudes' bits, two 16-bit numbers at a time
#pragma unroll
  for (int j = 0; j < 4; ++j) top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
  byte = act8_byte(__float_as_uint(to_f32<F16>(static_cast<uint16_t>(max(top & 0xFFFFu, top >> 16)))));
  const float a[4] = {lo16<F16>(w[0]), hi16<F16>(w[0]), lo16<F16>(w[1]), hi16<F16>(w[1])};
  const float b[4] = {lo16<F16>(w[2]), hi16<F16>(w[2]), lo16<F16>(w[3]), hi16<F16>(w[3])};
  return make_uint2(act8_codes(a, byte), act8_codes(b, byte));
}

// x / d and what remains, from 2^32 / d rounded down (at most 2^32 - 1): x times that, over 2^32, is less than 1 below x / d, so
// the quotient is right or one too small. Shorter than a division (8192 tokens 28.4 -> 26.2 us).
__device__ __forceinline__ uint32_t divide(uint32_t x, uint32_t d, uint32_t per, uint32_t& left) {
  uint32_t q = __umulhi(x, per);
  left = x - q * d;
  if (left >= d) ++q, left -= d;
  return q;
}

// Where a token's slot is.
struct Place {
  bool in;
  uint32_t page, at;
  __device__ __forceinline__ Place(int64_t slot, const KvPool& p) {
    in = slot >= 0 && slot < static_cast<int64_t>(p.pages) * p.size;
    page = at = 0;
    if (in && slot <= 0xFFFFFFFFll) page = divide(static_cast<uint32_t>(slot), p.size, p.per_slot, at);
    else if (in) page = static_cast<uint32_t>(slot / p.size), at = static_cast<uint32_t>(slot % p.size);
  }
};
// Strides are below 2^32 elements: one instruction a product.
__device__ __forceinline__ long times(uint32_t a, long stride) {
  return static_cast<long>(static_cast<uint64_t>(a) * static_cast<uint32_t>(stride));
}

// LANES = dim / 8 neighbouring threads take a head of a token: the largest magnitude takes a few exchanges between lanes. (Four
// tokens to a thread, whose loads are in flight together, gained 1.5% at best and lost 36% at 2048 tokens of 12 heads of 64.)
struct Share {
  int part, head, token;
  template <int LANES>
  __device__ __forceinline__ static Share of(const KvPool& p) {
    const uint32_t row = (blockIdx.x * kThreads + threadIdx.x) / LANES;
    Share s;
    s.part = threadIdx.x % LANES;
    uint32_t head;
    s.token = divide(row, p.heads, p.per_head, head);
    s.head = head;
    return s;
  }
};

template <int LANES, bool CODES, bool F16>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvTokens t, const KvPool p, int* status) {
  const Share me = Share::of<LANES>(p);
  const int token = min(me.token, t.n - 1);  // threads without a token only take part in the exchange of lanes
  const int64_t slot = t.slots[token];
  const uint4 k = load8(t.k, times(token, t.kt) + times(me.head, t.kh) + me.part * 8, t.vec);
  const uint4 v = load8(t.v, times(token, t.vt) + times(me.head, t.vh) + me.part * 8, t.vec);
  const Place s(slot, p);
  if (slot >= 0 && !s.in && me.part == 0 && me.head == 0) record_error(status, kBadArg, kSiteWrite);
  const bool store = s.in && me.token < t.n;
  const long ki = times(s.page, p.kp) + times(me.head, p.kh) + times(s.at, p.ks) + me.part * 8;
  const long vi = times(s.page, p.vp) + times(me.head, p.vh) + times(s.at, p.vs) + me.part * 8;
  if constexpr (CODES) {
    uint32_t kb, vb;
    const uint2 kc = quantise8<LANES, F16>(k, kb), vc = quantise8<LANES, F16>(v, vb);
    if (store) {
      *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.k) + ki) = kc;
      *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.v) + vi) = vc;
      if (me.part == 0) {
        p.ke[times(s.page, p.kep) + times(me.head, p.keh) + s.at] = static_cast<uint8_t>(kb);
        p.ve[times(s.page, p.vep) + times(me.head, p.veh) + s.at] = static_cast<uint8_t>(vb);
      }
    }
  } else if (store) {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.k) + ki) = k;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.v) + vi) = v;
  }
}

// Types of the values read back.
enum OutType : int { kOutBf16 = 0, kOutF16 = 1, kOutF32 = 2 };

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
// A code rounded up can stand for more than the type holds, in blocks whose byte is large: it becomes the largest finite value.
template <int OUT>
__device__ __forceinline__ void decode8(const uint2& codes, uint32_t byte, float (&v)[8]) {
  constexpr float kMost = OUT == kOutF16 ? 65504.f : OUT == kOutBf16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
  constexpr uint32_t kLarge = OUT == kOutF16 ? 127 + 9 : 127 + 121;  // 127 * 2^8 < 65504, 127 * 2^120 < 2^127
  float a[4], b[4];
  act8_values(codes.x, act8_scale(byte), a);
  act8_values(codes.y, act8_scale(byte), b);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  if (byte >= kLarge && byte != kAct8Nan) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fminf(fmaxf(v[j], -kMost), kMost);
  }
}

// OUT: type of the codes' values; a 16-bit cache is copied. Tokens without a slot read as zeros, those whose slot is
// outside the cache as NaN.
template <int LANES, bool CODES, int OUT>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const int64_t* __restrict__ slots, const KvPool p, void* k,
                                                           void* v, int n, int* status) {
  const Share me = Share::of<LANES>(p);
  if (me.token >= n) return;
  const int64_t slot = slots[me.token];
  const Place s(slot, p);
  if (slot >= 0 && !s.in && me.part == 0 && me.head == 0) record_error(status, kBadArg, kSiteRead);
  const long o = (static_cast<long>(me.token) * p.heads + me.head) * (LANES * 8) + me.part * 8;
  if (!s.in) {
    const float x = slot < 0 ? 0.f : __uint_as_float(0x7FC00000u);
    const float none[8] = {x, x, x, x, x, x, x, x};
    store8<OUT>(k, o, none);
    store8<OUT>(v, o, none);
    return;
  }
  const long ki = times(s.page, p.kp) + times(me.head, p.kh) + times(s.at, p.ks) + me.part * 8;
  const long vi = times(s.page, p.vp) + times(me.head, p.vh) + times(s.at, p.vs) + me.part * 8;
  if constexpr (CODES) {
    const uint2 kc = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p.k) + ki);
    const uint2 vc = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p.v) + vi);
    const uint32_t kb = p.ke[times(s.page, p.kep) + times(me.head, p.keh) + s.at];
    const uint32_t vb = p.ve[times(s.page, p.vep) + times(me.head, p.veh) + s.at];
    float x[8];
    decode8<OUT>(kc, kb, x);
    store8<OUT>(k, o, x);
    decode8<OUT>(vc, vb, x);
    store8<OUT>(v, o, x);
  } else {
    const uint4 kr = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.k) + ki);
    const uint4 vr = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.v) + vi);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(k) + o) = kr;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(v) + o) = vr;
  }
}

unsigned blocks_for(int n, int heads, int lanes) {
  return static_cast<unsigned>((static_cast<long>(n) * heads * lanes + kThreads - 1) / kThreads);
}

template <int LANES>
void write_dim(const KvTokens& t, const KvPool& p, int* status, cudaStream_t s) {
  const auto go = [&](auto kernel) { kernel<<<blocks_for(t.n, p.heads, LANES), kThreads, 0, s>>>(t, p, status); };
  if (p.type != kKvCodes) go(kv_write_kernel<LANES, false, false>);
  else if (t.f16) go(kv_write_kernel<LANES, true, true>);
  else go(kv_write_kernel<LANES, true, false>);
}
template <int LANES>
void read_dim(const int64_t* slots, const KvPool& p, void* k, void* v, int n, int out, int* status, cudaStream_t s) {
  const auto go = [&](auto kernel) {
    kernel<<<blocks_for(n, p.heads, LANES), kThreads, 0, s>>>(slots, p, k, v, n, status);
  };
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
