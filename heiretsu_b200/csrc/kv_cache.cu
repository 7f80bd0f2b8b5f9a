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

// Where a token's slot is. (A division in 64 bits costs five times one in 32.)
struct Place {
  bool in;
  uint32_t page, at;
  __device__ __forceinline__ Place(int64_t slot, const KvPool& p) {
    in = slot >= 0 && slot < static_cast<int64_t>(p.pages) * p.size;
    const uint32_t size = p.size;
    page = !in ? 0 : slot <= 0xFFFFFFFFll ? static_cast<uint32_t>(slot) / size : static_cast<uint32_t>(slot / p.size);
    at = in ? static_cast<uint32_t>(slot - static_cast<int64_t>(page) * p.size) : 0;
  }
};
// Strides are below 2^32 elements: one instruction a product.
__device__ __forceinline__ long times(uint32_t a, long stride) {
  return static_cast<long>(static_cast<uint64_t>(a) * static_cast<uint32_t>(stride));
}

// LANES = dim / 8 neighbouring threads take a head of ROWS tokens, `step` tokens apart: head and place in the head are worked
// out once, and the loads of all are in flight together.
struct Share {
  int part, head, token;
  template <int LANES>
  __device__ __forceinline__ static Share of(int heads) {
    const uint32_t row = (blockIdx.x * kThreads + threadIdx.x) / LANES;
    Share s;
    s.part = threadIdx.x % LANES;
    s.token = row / static_cast<uint32_t>(heads);
    s.head = row - s.token * heads;
    return s;
  }
};

template <int LANES, bool CODES, bool F16, int ROWS>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvTokens t, const KvPool p, const int step, int* status) {
  const Share me = Share::of<LANES>(p.heads);
  uint4 k[ROWS], v[ROWS];
  int64_t slot[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int token = min(me.token + u * step, t.n - 1);  // threads without a token only take part in the exchange of lanes
    slot[u] = t.slots[token];
    k[u] = load8(t.k, times(token, t.kt) + times(me.head, t.kh) + me.part * 8, t.vec);
    v[u] = load8(t.v, times(token, t.vt) + times(me.head, t.vh) + me.part * 8, t.vec);
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const Place s(slot[u], p);
    if (slot[u] >= 0 && !s.in && me.part == 0 && me.head == 0) record_error(status, kBadArg, kSiteWrite);
    const bool store = s.in && me.token < step && me.token + u * step < t.n;
    const long ki = times(s.page, p.kp) + times(me.head, p.kh) + times(s.at, p.ks) + me.part * 8;
    const long vi = times(s.page, p.vp) + times(me.head, p.vh) + times(s.at, p.vs) + me.part * 8;
    if constexpr (CODES) {
      uint32_t kb, vb;
      const uint2 kc = quantise8<LANES, F16>(k[u], kb), vc = quantise8<LANES, F16>(v[u], vb);
      if (store) {
        *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.k) + ki) = kc;
        *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.v) + vi) = vc;
        if (me.part == 0) {
          p.ke[times(s.page, p.kep) + times(me.head, p.keh) + s.at] = static_cast<uint8_t>(kb);
          p.ve[times(s.page, p.vep) + times(me.head, p.veh) + s.at] = static_cast<uint8_t>(vb);
        }
      }
    } else if (store) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.k) + ki) = k[u];
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.v) + vi) = v[u];
    }
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
template <int LANES, bool CODES, int OUT, int ROWS>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const int64_t* __restrict__ slots, const KvPool p, void* k,
                                                           void* v, int n, const int step, int* status) {
  const Share me = Share::of<LANES>(p.heads);
  if (me.token >= step) return;
  uint4 kr[ROWS], vr[ROWS];
  uint32_t kb[ROWS], vb[ROWS];
  int64_t slot[ROWS];
  bool in[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) slot[u] = me.token + u * step < n ? slots[me.token + u * step] : -1;
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const Place s(slot[u], p);
    in[u] = s.in;
    if (slot[u] >= 0 && !s.in && me.part == 0 && me.head == 0) record_error(status, kBadArg, kSiteRead);
    if (!s.in) continue;
    const long ki = times(s.page, p.kp) + times(me.head, p.kh) + times(s.at, p.ks) + me.part * 8;
    const long vi = times(s.page, p.vp) + times(me.head, p.vh) + times(s.at, p.vs) + me.part * 8;
    if constexpr (CODES) {
      const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p.k) + ki);
      const uint2 b = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p.v) + vi);
      kr[u] = make_uint4(a.x, a.y, 0, 0), vr[u] = make_uint4(b.x, b.y, 0, 0);
      kb[u] = p.ke[times(s.page, p.kep) + times(me.head, p.keh) + s.at];
      vb[u] = p.ve[times(s.page, p.vep) + times(me.head, p.veh) + s.at];
    } else {
      kr[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.k) + ki);
      vr[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.v) + vi);
    }
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int token = me.token + u * step;
    if (token >= n) break;
    const long o = (static_cast<long>(token) * p.heads + me.head) * (LANES * 8) + me.part * 8;
    if (!in[u]) {
      const float x = slot[u] < 0 ? 0.f : __uint_as_float(0x7FC00000u);
      const float none[8] = {x, x, x, x, x, x, x, x};
      store8<OUT>(k, o, none);
      store8<OUT>(v, o, none);
    } else if constexpr (CODES) {
      float x[8];
      decode8<OUT>(make_uint2(kr[u].x, kr[u].y), kb[u], x);
      store8<OUT>(k, o, x);
      decode8<OUT>(make_uint2(vr[u].x, vr[u].y), vb[u], x);
      store8<OUT>(v, o, x);
    } else {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(k) + o) = kr[u];
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(v) + o) = vr[u];
    }
  }
}

// Tokens a thread takes: several where that still leaves every SM with 4 full sets of threads.
constexpr int kMany = 4;
bool many(int n, int heads, int lanes) {
  return static_cast<long>(n) * heads * lanes >= 4l * 2048 * num_sms(current_device());
}
unsigned blocks_for(int step, int heads, int lanes) {
  return static_cast<unsigned>((static_cast<long>(step) * heads * lanes + kThreads - 1) / kThreads);
}

template <int LANES, int ROWS>
void write_rows(const KvTokens& t, const KvPool& p, int* status, cudaStream_t s) {
  const int step = (t.n + ROWS - 1) / ROWS;
  const auto go = [&](auto kernel) { kernel<<<blocks_for(step, p.heads, LANES), kThreads, 0, s>>>(t, p, step, status); };
  if (p.type != kKvCodes) go(kv_write_kernel<LANES, false, false, ROWS>);
  else if (t.f16) go(kv_write_kernel<LANES, true, true, ROWS>);
  else go(kv_write_kernel<LANES, true, false, ROWS>);
}
template <int LANES>
void write_dim(const KvTokens& t, const KvPool& p, int* status, cudaStream_t s) {
  if (many(t.n, p.heads, LANES)) write_rows<LANES, kMany>(t, p, status, s);
  else write_rows<LANES, 1>(t, p, status, s);
}
template <int LANES, int ROWS>
void read_rows(const int64_t* slots, const KvPool& p, void* k, void* v, int n, int out, int* status, cudaStream_t s) {
  const int step = (n + ROWS - 1) / ROWS;
  const auto go = [&](auto kernel) {
    kernel<<<blocks_for(step, p.heads, LANES), kThreads, 0, s>>>(slots, p, k, v, n, step, status);
  };
  if (p.type == kKvBf16) go(kv_read_kernel<LANES, false, kOutBf16, ROWS>);
  else if (p.type == kKvF16) go(kv_read_kernel<LANES, false, kOutF16, ROWS>);
  else if (out == kOutBf16) go(kv_read_kernel<LANES, true, kOutBf16, ROWS>);
  else if (out == kOutF16) go(kv_read_kernel<LANES, true, kOutF16, ROWS>);
  else go(kv_read_kernel<LANES, true, kOutF32, ROWS>);
}
template <int LANES>
void read_dim(const int64_t* slots, const KvPool& p, void* k, void* v, int n, int out, int* status, cudaStream_t s) {
  if (many(n, p.heads, LANES)) read_rows<LANES, kMany>(slots, p, k, v, n, out, status, s);
  else read_rows<LANES, 1>(slots, p, k, v, n, out, status, s);
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
