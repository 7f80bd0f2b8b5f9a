// A token per row of logits from a given uniform number.
//
// With top = max x and temperature T > 0 a token weighs w_i = e^((x_i - top) / T). In the order by logit, descending, equal
// ones by index, the tokens kept are: the first top_k; of these the shortest start whose weight reaches top_p of
// theirs (token i is kept if what precedes it weighs less); of these the ones with w_i >= min_p. The first always is.
// All three cut the same order, so what is kept is every logit above a threshold and the first `ties` equal to it. The
// token drawn is the first kept one, by index, at which the running weight exceeds u times the kept weight.
//
// Weights are whole numbers of 2^-44, rounded once from a 64-bit exponential: sums have no order, the same token comes
// out whatever the launch, and equal logits weigh exactly the same. A sum over the 2^19 columns allowed stays below 2^64.
// 32-bit exponentials would not do: the chance that a number falls on another token is twice the error of the running
// weights times the number of tokens in play, about 5% a row for 10,000 tokens at 2^-18.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "decode_args.h"
#include "host_utils.h"

namespace hb {

namespace {

using u64 = unsigned long long;
constexpr uint32_t kFull = 0xffffffffu;
constexpr int kEach = 4;   // candidates a thread holds
constexpr int kBins = 256; // of the histogram of weights, 8 to a factor of 2
constexpr int kTable = 32; // of 2^(j / 32)
constexpr float kFaint = -46.f;  // 2^kFaint is no more than half of 2^-44, with room for the rounding of the exponent

// Element types as the host numbers them; keys are unsigned numbers in the order of the logits (-0 counts as 0).
template <int TYPE>
struct Type {
  static constexpr bool kWide = TYPE == 2;
  static constexpr int kElems = kWide ? 4 : 8, kBytes = kWide ? 4 : 2;  // of a 16-byte piece, of an element
  static constexpr int kBits = kWide ? 32 : 16;                         // of a key
  static __device__ __forceinline__ uint32_t key(uint32_t b) {
    if constexpr (kWide) {
      if (b == 0x80000000u) b = 0;
      return b ^ (static_cast<int>(b) < 0 ? 0xFFFFFFFFu : 0x80000000u);
    } else {
      if (b == 0x8000u) b = 0;
      return b ^ (b & 0x8000u ? 0xFFFFu : 0x8000u);
    }
  }
  static __device__ __forceinline__ float value(uint32_t b) {
    if constexpr (kWide) return __uint_as_float(b);
    else return to_f32<TYPE == 1>(static_cast<uint16_t>(b));
  }
  static __device__ __forceinline__ float logit(uint32_t key) {
    if constexpr (kWide) return value(key ^ (static_cast<int>(key) < 0 ? 0x80000000u : 0xFFFFFFFFu));
    else return value(key ^ (key & 0x8000u ? 0x8000u : 0xFFFFu));
  }
  // the least key of a logit >= x, x finite or -inf
  static __device__ __forceinline__ uint32_t key_from(float x) {
    if constexpr (kWide) {
      return key(__float_as_uint(x));
    } else {
      const uint16_t b = TYPE == 1 ? __half_as_ushort(__float2half_ru(x)) : __bfloat16_as_ushort(__float2bfloat16_ru(x));
      return key(b);
    }
  }
  static __device__ __forceinline__ uint32_t bits(const uint4& r, int e) {  // element e, known when compiled
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    if constexpr (kWide) return w[e];
    else return e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu;
  }
};

// The weight of a logit in units of 2^-44. 2^(d log2 e / T), d = x - top, is 2^n 2^(j / 32) 2^r with |r| <= 1 / 64; the last
// factor is e^(r ln 2) by its series to degree 5, whose remainder is below (ln 2 / 64)^6 / 720 < 3e-15.
struct Weigher {
  double top, by;    // by: log2 e / T
  float top32, by32;
  const double* table;  // 2^(44 + j / 32)
  __device__ __forceinline__ float exponent(float x) const { return (x - top32) * by32; }  // about; monotone
  __device__ __forceinline__ u64 operator()(float x) const {
    if (x == top32) return 1ull << 44;
    if (!(exponent(x) > kFaint)) return 0;
    const double t = (static_cast<double>(x) - top) * by, shift = 211106232532992.0;  // 1.5 * 2^47
    const double s = t + shift, r = t - (s - shift);
    const int k = __double2loint(s);
    double p = fma(r, 1.3333558146428443e-3, 9.6181291076284772e-3);  // (ln 2)^5/5!, (ln 2)^4/4!
    p = fma(r, p, 5.5504108664821580e-2);                             // (ln 2)^3/3!
    p = fma(r, p, 2.4022650695910071e-1);                             // (ln 2)^2/2!
    p = fma(r, p, 6.9314718055994531e-1);                             // ln 2
    p = fma(r, p, 1.0);
    p *= table[k & (kTable - 1)];
    p = __hiloint2double(__double2hiint(p) + (k >> 5 << 20), __double2loint(p));
    return __double_as_longlong(p + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;  // 2^52: the fraction is the number
  }
};

template <int WARPS>
struct Block {
  u64 buf[WARPS];
  __device__ __forceinline__ u64 sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = buf[threadIdx.x % WARPS];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
  }
};

// A row as a block sees it: pieces of 16 bytes from the 16-byte boundary at or before its start, `off` elements of the first
// lying before the row. Warp w has the pieces [w per, (w + 1) per), 32 at a time.
template <int TYPE, int WARPS>
struct Row {
  using P = Type<TYPE>;
  static constexpr int E = P::kElems;
  const char* base;  // of the row
  uint4* copy;       // the pieces in shared memory, or null
  int V, off, pieces, per;

  __device__ __forceinline__ bool inside(int piece) const { return piece * E >= off && (piece + 1) * E <= off + V; }
  // elements outside the row read as -inf
  __device__ __forceinline__ uint4 load(int piece) const {
    if (inside(piece)) return __ldg(reinterpret_cast<const uint4*>(base + (static_cast<long>(piece) * E - off) * P::kBytes));
    constexpr uint32_t none = TYPE == 2 ? 0xFF800000u : TYPE == 1 ? 0xFC00u : 0xFF80u;
    uint32_t b[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = piece * E - off + e;
      b[e] = none;
      if (i >= 0 && i < V) {
        if constexpr (P::kWide) b[e] = reinterpret_cast<const uint32_t*>(base)[i];
        else b[e] = reinterpret_cast<const uint16_t*>(base)[i];
      }
    }
    if constexpr (P::kWide) return make_uint4(b[0], b[1], b[2], b[3]);
    else return make_uint4(b[0] | b[1] << 16, b[2] | b[3] << 16, b[4] | b[5] << 16, b[6] | b[7] << 16);
  }
  __device__ __forceinline__ uint4 again(int piece) const { return copy != nullptr ? copy[piece] : load(piece); }
  // f(bits, index) for each element of a piece that is in the row
  template <class F>
  __device__ __forceinline__ void each(const uint4& r, int piece, F f) const {
    const int i0 = piece * E - off;
    if (inside(piece)) {
#pragma unroll
      for (int e = 0; e < E; ++e) f(P::bits(r, e), i0 + e);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i0 + e >= 0 && i0 + e < V) f(P::bits(r, e), i0 + e);
    }
  }
  // f(bits, index) for each element of this thread's pieces, after the first pass
  template <class F>
  __device__ __forceinline__ void all(F f) const {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, end = min((w + 1) * per, pieces);
    for (int p = w * per + lane; p < end; p += 32) each(again(p), p, f);
  }
};

// One block per row. Passes over the row, which is kept in shared memory where it fits:
//   1. maximum; whether every logit is a number
//   2. top_k or min_p: candidates, the logits not below a bound that is sure to hold everything kept (top_k: the
//      top_k-th largest of the threads' own maxima), go to a list, and the cuts are found among them.
//      top_p alone: all weights, their sum and a histogram of them, which tells in which bins the cut lies; then the
//      sum above those bins, and the list of what is in them.
//   3. the kept weight of each warp's part of the row; the warp whose part holds u times the whole walks its part again.
// Where a list overflows, the cuts are found by halving over the whole row.
template <int TYPE, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) sample_kernel(const SampleArgs a, const bool resident) {
  constexpr int kWarps = THREADS / 32, kList = kEach * THREADS;
  using P = Type<TYPE>;
  extern __shared__ uint4 smem[];
  __shared__ Block<kWarps> block;
  __shared__ u64 warp_sums[kWarps];
  __shared__ uint32_t list[kList], hist[kBins], s_max[kWarps];
  __shared__ double table[kTable];
  __shared__ int s_bad, s_pick, s_listed, s_bins[2];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  const double T = a.temperature ? a.temperature[row] : a.temperature0;
  const double top_p = a.top_p ? a.top_p[row] : a.top_p0, min_p = a.min_p ? a.min_p[row] : a.min_p0;
  const int64_t top_k = a.top_k ? a.top_k[row] : a.top_k0;
  const double u = a.u[row];
  Row<TYPE, kWarps> x;
  x.base = static_cast<const char*>(a.x) + row * a.ld * P::kBytes;
  x.copy = resident ? smem : nullptr;
  x.V = a.V;
  x.off = static_cast<int>(reinterpret_cast<uintptr_t>(x.base) & 15) / P::kBytes;
  x.pieces = (x.off + a.V + x.E - 1) / x.E;
  x.per = ((x.pieces + kWarps - 1) / kWarps + 31) / 32 * 32;
  if (x.per * (kWarps - 1) >= x.pieces) x.per = (x.pieces + kWarps - 1) / kWarps;

  if (tid == 0) s_bad = T != T || top_p != top_p || min_p != min_p || u != u, s_pick = a.V, s_listed = 0;
  if (tid < kTable) table[tid] = exp2(44.0 + tid / static_cast<double>(kTable));
  for (int i = tid; i < kBins; i += THREADS) hist[i] = 0;
  uint32_t mine = 0;  // this thread's largest key
  bool bad = false;
  {
    const int end = min((warp + 1) * x.per, x.pieces);
#pragma unroll 4
    for (int p = warp * x.per + lane; p < end; p += 32) {
      const uint4 r = x.load(p);
      if (resident) smem[p] = r;
#pragma unroll
      for (int e = 0; e < x.E; ++e) {
        bad |= !(P::value(P::bits(r, e)) < INFINITY);
        mine = max(mine, P::key(P::bits(r, e)));
      }
    }
  }
  const uint32_t warp_max = __reduce_max_sync(kFull, mine);
  if (lane == 0) s_max[warp] = warp_max;
  __syncthreads();  // also: s_bad is set up
  if (bad) s_bad = 1;
  const uint32_t kmax = __reduce_max_sync(kFull, s_max[lane % kWarps]);
  __syncthreads();
  Weigher weight;
  weight.top32 = P::logit(kmax);
  if (s_bad || weight.top32 == -INFINITY) {  // NaN or +inf among the logits, nothing but -inf, a setting that is no number
    if (tid == 0) a.tokens[row] = -1;
    return;
  }
  if (T <= 0 || min_p > 1 || top_p <= 0) {  // the first token of the order
    x.all([&](uint32_t b, int i) {
      if (P::key(b) == kmax) atomicMin(&s_pick, i);
    });
    __syncthreads();
    if (tid == 0) a.tokens[row] = s_pick;
    return;
  }
  weight.top = weight.top32;
  weight.by = fmin(1.4426950408889634 / T, 1.6069380442589903e60);  // 2^200: no two logits are closer than 2^-149
  weight.by32 = static_cast<float>(fmin(weight.by, 3e38));
  weight.table = table;

  uint32_t t = 0;  // kept: keys above t, and the first `ties` equal to it
  u64 ties = ~0ull;
  const bool use_k = top_k > 0 && top_k < a.V, use_p = top_p < 1;
  uint32_t floor_key = 0;  // of min_p
  if (min_p > 0 && T < INFINITY) floor_key = P::key_from(fmaxf(__double2float_ru(weight.top + T * log(min_p)), -3.4028234663852886e38f));
  const auto need_of = [&](u64 total) { return max(__double2ull_ru(top_p * static_cast<double>(total)), 1ull); };

  // ---- candidates
  uint32_t from = 0;        // keys at or above it are listed
  bool listing = false;
  u64 above = 0, need = 0;  // top_p alone: the weight above the listed bins, and what the kept weight has to reach
  int bin0 = 0, bin1 = kBins;
  const auto bin_of = [&](float v) { return static_cast<int>(fminf(weight.exponent(v) * -8.f, static_cast<float>(kBins))); };
  if (use_k) {
    const int have = __syncthreads_count(mine != 0);
    if (top_k <= have) {
      for (int bit = P::kBits - 1; bit >= 0; --bit) {
        const uint32_t c = from | (1u << bit);
        if (__syncthreads_count(mine >= c) >= top_k) from = c;
      }
      listing = true;
    }
    if (!use_p && floor_key > from) from = floor_key, listing = true;
  } else if (use_p) {
    u64 sum = 0;
    x.all([&](uint32_t b, int) {
      const float v = P::value(b);
      const u64 w = weight(v);
      sum += w;
      const int bin = bin_of(v);
      if (bin < kBins) atomicAdd(&hist[bin], static_cast<uint32_t>(w >> (32 - (bin >> 3))));  // 11 bits or 12
    });
    need = need_of(block.sum(sum));
    if (warp == 0) {  // first bin whose end may reach `need`, first whose end does
      u64 run = 0, part[kBins / 32];
#pragma unroll
      for (int i = 0; i < kBins / 32; ++i) {
        const int bin = lane * (kBins / 32) + i;
        part[i] = static_cast<u64>(hist[bin]) << (32 - (bin >> 3));
        run += part[i];
      }
      u64 before = run;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(kFull, before, o);
        if (lane >= o) before += y;
      }
      before -= run;
      int may = kBins, does = kBins;
#pragma unroll
      for (int i = 0; i < kBins / 32; ++i) {
        before += part[i];
        const int bin = lane * (kBins / 32) + i;
        // what was cut off is less than 1 in 2^11 of a bin; 2^30: the exponent's rounding, near a bin's edge
        if (before + (before >> 10) + (1ull << 30) >= need) may = min(may, bin);
        if (before >= need) does = min(does, bin);
      }
      may = __reduce_min_sync(kFull, may), does = __reduce_min_sync(kFull, does);
      if (lane == 0) s_bins[0] = may, s_bins[1] = does;
    }
    __syncthreads();
    bin0 = s_bins[0], bin1 = s_bins[1];
    listing = true;
  } else if (floor_key > 0) {
    from = floor_key;
  }

  uint32_t key[kEach];
  int n = 0;
  if (listing) {
    const bool bins = use_p && !use_k;
    u64 sum = 0;
    x.all([&](uint32_t b, int) {
      const uint32_t k = P::key(b);
      bool take = k >= from;
      if (bins) {
        const int bin = bin_of(P::value(b));
        take = bin >= bin0 && bin <= bin1;
        if (bin < bin0) sum += weight(P::value(b));
      }
      if (take) {
        const int at = atomicAdd(&s_listed, 1);
        if (at < kList) list[at] = k;
      }
    });
    if (bins) above = block.sum(sum);
    __syncthreads();
    n = s_listed;
#pragma unroll
    for (int i = 0; i < kEach; ++i) key[i] = i * THREADS + tid < n ? list[min(i * THREADS + tid, kList - 1)] : 0;  // 0: none
  }
  const bool listed = listing && n <= kList && (!use_p || use_k || above < need);

  // ---- cuts: counts and sums over the list where there is one, else over the row
  const auto count = [&](uint32_t c) -> u64 {
    uint32_t m = 0;
    if (listed) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) m += key[i] >= c;
    } else {
      x.all([&](uint32_t b, int) { m += P::key(b) >= c; });
    }
    return block.sum(m);
  };
  u64 w[kEach];  // of the list
  const auto mass = [&](uint32_t c) -> u64 {
    u64 m = 0;
    if (listed) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) m += key[i] >= c ? w[i] : 0;
    } else {
      x.all([&](uint32_t b, int) {
        if (P::key(b) >= c) m += weight(P::value(b));
      });
    }
    return block.sum(m);
  };
  if (use_k) {
    const bool few = listed && static_cast<u64>(n) < static_cast<u64>(top_k);  // min_p leaves fewer than top_k
    if (!few) {
      for (int bit = P::kBits - 1; bit >= 0; --bit)
        if (count(t | (1u << bit)) >= static_cast<u64>(top_k)) t |= 1u << bit;
      ties = top_k - count(t + 1);
    }
  }
  if (use_p) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) w[i] = listed && key[i] != 0 ? weight(P::logit(key[i])) : 0;
    u64 over = mass(t + 1);  // of the keys above t
    if (use_k || !listed) {
      above = 0;
      const u64 total = t == 0 ? over : over + ties * weight(P::logit(t));
      need = need_of(total);
    }
    uint32_t t2 = t;
    if (above + over >= need) {
      t2 = 0;
      for (int bit = P::kBits - 1; bit >= 0; --bit) {
        const uint32_t c = t2 | (1u << bit);
        if (c <= t || above + mass(c) >= need) t2 = c;
      }
      over = mass(t2 + 1);
    }
    const u64 each = weight(P::logit(t2));
    if (each > 0 && t2 > 0) {
      const u64 m = (need - min(above + over, need) + each - 1) / each;
      ties = t2 == t ? min(ties, m) : m;
    }
    t = t2;
  }
  if (floor_key > t) t = floor_key, ties = ~0ull;

  // ---- the draw. Equal keys of the warps before this one count first
  u64 tie = 0;
  if (ties != ~0ull) {
    uint32_t m = 0;
    x.all([&](uint32_t b, int) { m += P::key(b) == t; });
    m = __reduce_add_sync(kFull, m);
    __syncthreads();
    if (lane == 0) block.buf[warp] = m;
    __syncthreads();
    for (int i = 0; i < warp; ++i) tie += block.buf[i];
  }
  const int end = min((warp + 1) * x.per, x.pieces);
  // what this thread's piece of a round holds; `seen`: equal keys before the round, which it moves behind
  const auto round = [&](const uint4& r, int piece, u64& seen, auto&& f) {
    u64 rank = seen;
    if (ties != ~0ull) {
      uint32_t m = 0;
      if (piece < end) x.each(r, piece, [&](uint32_t b, int) { m += P::key(b) == t; });
      if (__any_sync(kFull, m != 0)) {
        uint32_t run = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t y = __shfl_up_sync(kFull, run, o);
          if (lane >= o) run += y;
        }
        rank += run - m;
        seen += __shfl_sync(kFull, run, 31);
      }
    }
    if (piece < end)
      x.each(r, piece, [&](uint32_t b, int i) {
        const uint32_t k = P::key(b);
        if (k > t || (k == t && rank++ < ties)) f(P::value(b), i);
      });
  };
  u64 kept = 0, seen = tie;
  for (int p0 = warp * x.per; p0 < end; p0 += 32) {
    const int p = p0 + lane;
    round(p < end ? x.again(p) : uint4{}, p, seen, [&](float v, int) { kept += weight(v); });
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) kept += __shfl_xor_sync(kFull, kept, o);
  if (lane == 0) warp_sums[warp] = kept;
  __syncthreads();
  u64 total = 0, run = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i == warp) run = total;
    total += warp_sums[i];
  }
  const u64 target = min(static_cast<u64>(max(u, 0.0) * static_cast<double>(total)), total - 1);
  if (target < run || target >= run + kept) return;
  seen = tie;
  for (int p0 = warp * x.per; p0 < end; p0 += 32) {
    const int p = p0 + lane;
    const uint4 r = p < end ? x.again(p) : uint4{};
    u64 part = 0, old = seen;
    round(r, p, seen, [&](float v, int) { part += weight(v); });
    u64 upto = part;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(kFull, upto, o);
      if (lane >= o) upto += y;
    }
    const u64 all = __shfl_sync(kFull, upto, 31);
    if (target < run + all) {
      u64 at = run + upto - part;
      const bool here = target >= at && target < at + part;
      round(r, p, old, [&](float v, int i) {
        const u64 next = at + weight(v);
        if (here && at <= target && target < next) a.tokens[row] = i;
        at = next;
      });
      return;
    }
    run += all;
  }
}

template <int TYPE, int THREADS>
void launch(const SampleArgs& a, cudaStream_t s) {
  constexpr int kRoom = (227 * 1024 - 1024 * (1024 / THREADS)) / (1024 / THREADS) - (THREADS == 1024 ? 20 : 11) * 1024;
  const size_t bytes = (static_cast<size_t>(a.V) * Type<TYPE>::kBytes + 15 + 15) / 16 * 16 + 16;
  const bool resident = bytes <= kRoom;
  const auto kernel = sample_kernel<TYPE, THREADS>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may use that much shared memory
  const int dev = current_device();
  if (!(ready.load() >> dev & 1)) {
    HB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRoom));
    ready.fetch_or(1ull << dev);
  }
  kernel<<<a.rows, THREADS, resident ? bytes : 0, s>>>(a, resident);
  HB_CUDA_CHECK(cudaGetLastError());
}
template <int TYPE>
void launch_type(const SampleArgs& a, cudaStream_t s) {
  // More rows than SMs: two blocks of half the threads share one and overlap their passes
  if (a.rows > num_sms(current_device())) launch<TYPE, 512>(a, s);
  else launch<TYPE, 1024>(a, s);
}

}  // namespace

void sample_tokens_launch(const SampleArgs& a, cudaStream_t s) {
  if (a.rows == 0) return;
  if (a.type == 0) launch_type<0>(a, s);
  else if (a.type == 1) launch_type<1>(a, s);
  else launch_type<2>(a, s);
}

}  // namespace hb
