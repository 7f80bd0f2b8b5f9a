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
//
// The row is read once, and its passes are made in shared memory: bound by the arithmetic of the weights (10 instructions
// in 64 bits and about 20 others each) and, for few rows, by the chain of barriers. Device times on a B200, and what the
// bytes alone take: rows of 50257, 1 by top_k 15.9 us (0.02), 64 whole ones in 32 bits 17.2 us (2.0), 256 by top_p 53.7 us
// (3.9), 256 greedy 8.9 us, 256 by min_p 17.5 us; 101 of 32003 with settings of their own 30.0 us (1.0); 64 of 130000 in 32 bits,
// which shared memory does not hold, whole 37.5 us, by top_k 38 us, by top_p 79 us (5.1).
// The lists hold 2048 tokens (1024 where two rows share an SM), and a bound on the top_k-th logit comes from the threads' own
// maxima. Where that is not enough the cuts are searched for over the whole row, a pass for each bit of a key: 64 rows of 50257 by
// top_p of 0.99, whose border lies among thousands of alike tokens, 217 us (0.9: 34), by top_k 1000 54 us (800: 19.5), 256
// by top_k 500 86 us (400: 25), 64 of 1000 by top_k 200 (125 threads have a piece) 21 us (100: 15).
// Tried and slower: searches by one warp (1 row 22.5 us) or of two bits a step (17.7), tables of 256 exponentials.
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
constexpr int kEach = 2;      // candidates a thread holds
constexpr int kBins = 512;    // of the histogram of weights, 16 to a factor of 2
constexpr int kTable = 16;    // of 2^(j / 16): as many as shared memory has pairs of banks, so that no two lanes wait for each other
constexpr int kFine = 256;    // steps of a bin
constexpr float kInf = INFINITY;

// Element types as the host numbers them; keys are unsigned numbers in the order of the logits (-0 counts as 0).
template <int TYPE>
struct Type {
  static constexpr bool kWide = TYPE == 2;
  static constexpr int kElems = kWide ? 4 : 8, kBytes = kWide ? 4 : 2;  // of a 16-byte piece, of an element
  static constexpr int kBits = kWide ? 32 : 16;                         // of a key
  static constexpr uint32_t kNone = TYPE == 2 ? 0xFF800000u : TYPE == 1 ? 0xFC00u : 0xFF80u;  // -inf
  static __device__ __forceinline__ uint32_t key(float x) {
    uint32_t b;
    if constexpr (kWide) {
      b = __float_as_uint(x + 0.f);
      return b ^ (static_cast<int>(b) < 0 ? 0xFFFFFFFFu : 0x80000000u);
    } else {
      b = from_f32<TYPE == 1>(x + 0.f);
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
  // the least logit of the type that is >= x, x finite
  static __device__ __forceinline__ float round_up(float x) {
    if constexpr (kWide) return x;
    else if constexpr (TYPE == 1) return __half2float(__float2half_ru(x));
    else return __bfloat162float(__float2bfloat16_ru(x));
  }
  static __device__ __forceinline__ float at(const uint4& r, int e) {  // element e, known when compiled
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    if constexpr (kWide) return value(w[e]);
    else return e & 1 ? hi16<TYPE == 1>(w[e >> 1]) : lo16<TYPE == 1>(w[e >> 1]);
  }
  // the largest element of a piece, NaN where there is one
  static __device__ __forceinline__ float largest(const uint4& r) {
    if constexpr (kWide) {
      return max_nan(max_nan(value(r.x), value(r.y)), max_nan(value(r.z), value(r.w)));
    } else {
      const uint32_t w = max2(max2(r.x, r.y), max2(r.z, r.w));
      return max_nan(lo16<TYPE == 1>(w), hi16<TYPE == 1>(w));
    }
  }
  static __device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (TYPE == 1) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};

// 2^(44 + j / 16)
__device__ const double kPowers[kTable] = {
    17592186044416, 18371058661769.059, 19184414915921.48, 20033781527906.219,
    20920752812471.082, 21846993670708.133, 22814242715178.152, 23824315533396.16,
    24879108095803.801, 25980600314625.527, 27130859760288.855, 28332045542384.562,
    29586412362451.676, 30896314746194.609, 32264211463076.527, 33692670141584.852};

// The weight of a logit x in units of 2^-44. 2^(d log2 e / T), d = x - top, is 2^n 2^(j / 16) 2^r with |r| <= 1 / 32; the last
// factor is e^(r ln 2) by its series to degree 5, whose remainder is below (ln 2 / 32)^6 / 720 < 1.5e-13.
// x is raised to `least` first, whose weight of 2^-46 or less is rounded to 0 as that of all below it is: so n stays small,
// and -inf is like the others. That `least` is finite, and not `top`, takes
// - x and T in units of 2^56 where one of them is so large that top - 46 T ln 2 is no number of 32 bits,
// - T ln 2 of at most 2^174, which has all finite logits weigh 1 as an infinite T does, and
// - T ln 2 of at least 1 / 50 of the distance to the next number of 32 bits below top, which still weighs 0.
struct Weigher {
  double top, by;    // by: log2 e / T
  float unit, least, top32, inv32, steps;  // inv32: T ln 2; steps: of bins, to a logit
  const double* table;  // 2^(44 + j / 16), the j that k << 16 adds to its exponent field taken off
  __device__ __forceinline__ Weigher(float t, double T, const double* tab) : table(tab) {
    double inv = fmin(T * 0.69314718055994531, 2.3945242826029513e52);
    unit = t < -1e38f || t - 46 * inv < -3.4028234663852886e38 ? 1.3877787807814457e-17f : 1.f;
    top32 = t * unit, top = top32;
    const float below = nextafterf(top32, -INFINITY);
    inv = fmax(inv * unit, (top - below) * 0.02);
    by = 1 / inv;
    least = fminf(__double2float_rd(top - 46 * inv), below);
    inv32 = static_cast<float>(inv);
    steps = static_cast<float>(fmin(by * 16 * kFine, 1e38));
  }
  __device__ __forceinline__ float raised(float x) const { return fmaxf(x * unit, least); }
  __device__ __forceinline__ bool any(float largest) const { return largest * unit > least; }
  // In the histogram: 0x4B000000 + the steps below top, rounded; more where the logit is far below it.
  __device__ __forceinline__ int place(float x) const { return __float_as_int(fmaf(top32 - x * unit, steps, 8388608.f)); }
  // of a logit that has been raised
  __device__ __forceinline__ u64 raw(float x) const {
    const double d = static_cast<double>(x) - top, shift = 422212465065984.0;  // 1.5 * 2^48
    const double s = fma(d, by, shift), r = fma(d, by, shift - s);
    const int k = __double2loint(s);
    double p = fma(r, 1.3333558146428443e-3, 9.6181291076284772e-3);  // (ln 2)^5/5!, (ln 2)^4/4!
    p = fma(r, p, 5.5504108664821580e-2);                             // (ln 2)^3/3!
    p = fma(r, p, 2.4022650695910071e-1);                             // (ln 2)^2/2!
    p = fma(r, p, 6.9314718055994531e-1);                             // ln 2
    p = fma(r, p, 1.0);
    const double q = table[k & (kTable - 1)];
    const double scale = __hiloint2double(__double2hiint(q) + (k << 16), __double2loint(q));
    // 2^52 is added, whose fraction takes the number
    return static_cast<u64>(__double_as_longlong(fma(p, scale, 4503599627370496.0))) - 0x4330000000000000ull;
  }
  __device__ __forceinline__ u64 operator()(float x) const { return raw(raised(x)); }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int TYPE>
struct Row {
  using P = Type<TYPE>;
  static constexpr int E = P::kElems;
  const char* base;  // of the row
  uint4* copy;       // the pieces in shared memory, or null
  int V, off, pieces, per, first, end;  // first: this thread's first piece; end: behind its warp's last

  __device__ __forceinline__ bool inside(int piece) const { return piece * E >= off && (piece + 1) * E <= off + V; }
  __device__ __forceinline__ uint32_t bits(int i) const {  // of element i of the row
    if constexpr (P::kWide) return copy ? reinterpret_cast<const uint32_t*>(copy)[off + i] : reinterpret_cast<const uint32_t*>(base)[i];
    else return copy ? reinterpret_cast<const uint16_t*>(copy)[off + i] : reinterpret_cast<const uint16_t*>(base)[i];
  }
  // elements outside the row read as -inf
  __device__ __forceinline__ uint4 load(int piece) const {
    if (inside(piece)) return __ldg(reinterpret_cast<const uint4*>(base + (static_cast<long>(piece) * E - off) * P::kBytes));
    uint32_t b[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = piece * E - off + e;
      b[e] = P::kNone;
      if (i >= 0 && i < V) {
        if constexpr (P::kWide) b[e] = reinterpret_cast<const uint32_t*>(base)[i];
        else b[e] = reinterpret_cast<const uint16_t*>(base)[i];
      }
    }
    if constexpr (P::kWide) return make_uint4(b[0], b[1], b[2], b[3]);
    else return make_uint4(b[0] | b[1] << 16, b[2] | b[3] << 16, b[4] | b[5] << 16, b[6] | b[7] << 16);
  }
  // f(piece, its number) for this thread's pieces
  template <class F>
  __device__ __forceinline__ void pieces_of(F f) const {
    if (copy != nullptr)
      for (int p = first; p < end; p += 32) f(copy[p], p);
    else
      for (int p = first; p < end; p += 32) f(load(p), p);
  }
  // f(logit, index) for each element of a piece that is in the row and >= from
  template <class F>
  __device__ __forceinline__ void each(const uint4& r, int piece, float from, F f) const {
    if (!(P::largest(r) >= from)) return;
    const int i0 = piece * E - off;
    if (from > -kInf || inside(piece)) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (P::at(r, e) >= from) f(P::at(r, e), i0 + e);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i0 + e >= 0 && i0 + e < V) f(P::at(r, e), i0 + e);
    }
  }
  // the weight of a piece's elements, ALL or those that are not below `from` (elements outside the row weigh nothing)
  template <bool ALL = false>
  __device__ __forceinline__ u64 weigh(const uint4& r, const Weigher& weight, float from = 0) const {
    u64 sum = 0;
    if (!weight.any(P::largest(r))) return sum;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const u64 w = weight(P::at(r, e));
      if (ALL || P::at(r, e) >= from) sum += w;
    }
    return sum;
  }
};

// Sums over a block, in one barrier each: parts of 22, 22 and 20 bits that warps add up in one instruction and the
// block in shared memory (whole numbers: in any order). Each sum takes new slots, set to 0 beforehand.
constexpr int kSums = 2 * 33 + 8;  // two searches of 32 bits, and a few
struct Sums {
  uint32_t (*slots)[3];
  int used = 0;
  __device__ __forceinline__ u64 operator()(u64 v) {
    uint32_t* s = slots[used++];
    const uint32_t part[3] = {static_cast<uint32_t>(v & 0x3FFFFF), static_cast<uint32_t>(v >> 22 & 0x3FFFFF),
                              static_cast<uint32_t>(v >> 44)};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint32_t x = __reduce_add_sync(kFull, part[i]);
      if ((threadIdx.x & 31) == 0 && x != 0) atomicAdd(&s[i], x);
    }
    __syncthreads();
    return s[0] + (static_cast<u64>(s[1]) << 22) + (static_cast<u64>(s[2]) << 44);
  }
  __device__ __forceinline__ uint32_t count(uint32_t v) {
    uint32_t* s = slots[used++];
    v = __reduce_add_sync(kFull, v);
    if ((threadIdx.x & 31) == 0 && v != 0) atomicAdd(&s[0], v);
    __syncthreads();
    return s[0];
  }
};

// One block per row. Passes over the row, which is kept in shared memory where it fits:
//   1. maximum; whether every logit is a number
//   2. top_k or min_p: candidates, the logits not below a bound that is sure to hold everything kept (top_k: the
//      top_k-th largest of the threads' own maxima), go to a list, and the cuts are found among them.
//      top_p alone: all weights, their sum and a histogram of them, which tells in which bins the cut lies; then the
//      sum above those bins, and the list of what is in them.
//   3. the kept weight of each warp's part of the row; the part that holds u times the whole is looked at by all.
// Where a list overflows, the cuts are found by halving over the whole row.
template <int TYPE, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) sample_kernel(const SampleArgs a, const bool resident) {
  constexpr int kWarps = THREADS / 32, kList = kEach * THREADS;
  using P = Type<TYPE>;
  extern __shared__ uint4 smem[];
  __shared__ u64 warp_sums[kWarps];
  __shared__ __align__(16) uint2 list[kList];  // (key, index); before that the histogram, four copies of a bin side by side
  __shared__ uint32_t slots[kSums][3], warp_ties[kWarps], warp_parts[kWarps][3];
  __shared__ float warp_max[kWarps];
  __shared__ double table[kTable];
  __shared__ int s_pick, s_listed, s_bins[2];
  __shared__ uint32_t s_range[2];  // of the list's keys

  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  const double T = a.temperature ? a.temperature[row] : a.temperature0;
  const double top_p = a.top_p ? a.top_p[row] : a.top_p0, min_p = a.min_p ? a.min_p[row] : a.min_p0;
  const int64_t top_k = a.top_k ? a.top_k[row] : a.top_k0;
  const double u = a.u[row];
  Row<TYPE> x;
  x.base = static_cast<const char*>(a.x) + row * a.ld * P::kBytes;
  x.copy = resident ? smem : nullptr;
  x.V = a.V;
  x.off = static_cast<int>(reinterpret_cast<uintptr_t>(x.base) & 15) / P::kBytes;
  x.pieces = (x.off + a.V + x.E - 1) / x.E;
  x.per = (x.pieces + kWarps - 1) / kWarps;
  x.first = warp * x.per + lane;
  x.end = min((warp + 1) * x.per, x.pieces);

  if (tid == 0) s_pick = a.V, s_listed = 0, s_range[0] = ~0u, s_range[1] = 0;
  if (tid < kTable) table[tid] = __hiloint2double(__double2hiint(kPowers[tid]) - (tid << 16), __double2loint(kPowers[tid]));
  for (int i = tid; i < kSums * 3; i += THREADS) slots[i / 3][i % 3] = 0;
  float mine = -kInf;  // this thread's largest
  const auto take = [&](const uint4& r, int p) {
    if (resident) smem[p] = r;
    mine = P::max_nan(mine, P::largest(r));
  };
  if (x.inside(warp * x.per) && x.inside(x.end - 1)) {  // all of the warp's pieces: their loads are issued together
    const uint4* src = reinterpret_cast<const uint4*>(x.base - x.off * P::kBytes);
#pragma unroll 8
    for (int p = x.first; p < x.end; p += 32) take(__ldg(src + p), p);
  } else {
    for (int p = x.first; p < x.end; p += 32) take(x.load(p), p);
  }
  float top = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = P::max_nan(top, __shfl_xor_sync(kFull, top, o));
  if (lane == 0) warp_max[warp] = top;
  __syncthreads();
  top = warp_max[lane % kWarps];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = P::max_nan(top, __shfl_xor_sync(kFull, top, o));
  // NaN or +inf among the logits, nothing but -inf, a setting that is no number
  if (!(top < kInf) || top == -kInf || T != T || top_p != top_p || min_p != min_p || u != u) {
    if (tid == 0) a.tokens[row] = -1;
    return;
  }
  if (T <= 0 || min_p > 1 || top_p <= 0) {  // the first token of the order
    x.pieces_of([&](const uint4& r, int p) { x.each(r, p, top, [&](float, int i) { atomicMin(&s_pick, i); }); });
    __syncthreads();
    if (tid == 0) a.tokens[row] = s_pick;
    return;
  }
  const Weigher weight(top, T, table);
  Sums sums{slots};

  uint32_t t = 0;  // kept: keys above t, and the first `ties` equal to it
  u64 ties = ~0ull;
  const uint32_t kmax = P::key(top);
  const bool use_k = top_k > 0 && top_k < a.V, use_p = top_p < 1;
  uint32_t floor_key = 0;  // of min_p
  if (min_p > 0 && T < INFINITY)
    floor_key = min(kmax, P::key(P::round_up(fmaxf(__double2float_ru(top + T * log(min_p)), -3.4028234663852886e38f))));
  const auto need_of = [&](u64 total) { return max(__double2ull_ru(top_p * static_cast<double>(total)), 1ull); };
  // the largest key c with enough(c), which holds for `low` and not above `high`: only the bits below those they share
  const auto search = [&](uint32_t low, uint32_t high, auto&& enough) {
    if (low >= high) return low;
    const int bits = 32 - __clz(low ^ high);
    uint32_t c = bits >= 32 ? 0 : high >> bits << bits;
    for (int bit = bits - 1; bit >= 0; --bit)
      if ((c | (1u << bit)) <= low || enough(c | (1u << bit))) c |= 1u << bit;
    return c;
  };
  constexpr uint32_t kLowest = TYPE == 2 ? 0x007FFFFFu : TYPE == 1 ? 0x03FFu : 0x007Fu;  // the key of -inf

  // ---- candidates
  uint32_t from = 0;        // keys at or above it are listed
  bool listing = false;
  u64 above = 0, need = 0;  // top_p alone: the weight above the listed bins, and what the kept weight has to reach
  u64 mine_above = 0;       // this thread's part of `above`
  float listed_from = 0, listed_to = 0;  // of raised logits, those >= the first and < the second
  const bool bins = use_p && !use_k;
  if (use_k) {
    const uint32_t key = x.first < x.end ? P::key(mine) : 0;
    const uint32_t least = __reduce_min_sync(kFull, key != 0 ? key : ~0u);
    if (lane == 0) atomicMin(&s_range[0], least);
    if (top_k <= __syncthreads_count(key != 0)) {
      from = search(s_range[0], kmax, [&](uint32_t c) { return __syncthreads_count(key >= c) >= top_k; });
      listing = true;
    }
    __syncthreads();
    if (tid == 0) s_range[0] = ~0u;
    if (!use_p && floor_key > from) from = floor_key, listing = true;
  } else if (use_p) {
    // In 32 bits: which bins the cut may be in. Within a bin a weight falls from 6038 to 5783 steps of equal size, which is off
    // by no more than 1 in 2^12; the sum of 2^19 stays below 2^32. Lanes that add to one bin wait for each other: with four copies
    // of the bins few do.
    uint32_t* const hist = reinterpret_cast<uint32_t*>(list);
    static_assert(4 * kBins <= 2 * kList, "");
    for (int i = tid; i < 4 * kBins; i += THREADS) hist[i] = 0;
    __syncthreads();
    x.pieces_of([&](const uint4& r, int) {
      if (weight.place(P::largest(r)) >= 0x4B000000 + kBins * kFine) return;
#pragma unroll
      for (int e = 0; e < x.E; ++e) {
        const int at = weight.place(P::at(r, e)) - 0x4B000000;
        if (at < kBins * kFine) atomicAdd(&hist[at / kFine * 4 + (lane & 3)], 6038u - static_cast<uint32_t>(at % kFine));
      }
    });
    __syncthreads();
    if (warp == 0) {  // first bin whose end may reach top_p of the whole, first whose end is sure to
      float part[kBins / 32], run = 0.f;
#pragma unroll
      for (int i = 0; i < kBins / 32; ++i) {
        const int bin = lane * (kBins / 32) + i;
        const uint4 h = reinterpret_cast<const uint4*>(hist)[bin];
        part[i] = (h.x + h.y + h.z + h.w) * ex2(bin * -0.0625f);
        run += part[i];
      }
      float before = run;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float y = __shfl_up_sync(kFull, before, o);
        if (lane >= o) before += y;
      }
      // weights to 1 in 2^12, sums in 32 bits, and up to 2^19 logits below the bins: by 1 in 2^10
      const float all = __shfl_sync(kFull, before, 31), goal = static_cast<float>(top_p) * all;
      before -= run;
      int may = kBins, does = kBins;
#pragma unroll
      for (int i = 0; i < kBins / 32; ++i) {
        before += part[i];
        const int bin = lane * (kBins / 32) + i;
        if (before >= goal * (1.f - 1.f / 1024)) may = min(may, bin);
        if (before >= goal * (1.f + 1.f / 1024)) does = min(does, bin);
      }
      may = __reduce_min_sync(kFull, may), does = __reduce_min_sync(kFull, does);
      if (lane == 0) s_bins[0] = may, s_bins[1] = does;
    }
    __syncthreads();
    // (1 / 16 of a bin more on either side, for the roundings)
    listed_to = s_bins[0] == 0 ? kInf : __fadd_ru(weight.top32, (1.f / 256 - s_bins[0] * 0.0625f) * weight.inv32);
    listed_from = s_bins[1] >= kBins ? -kInf : __fadd_rd(weight.top32, (-1.f / 256 - (s_bins[1] + 1) * 0.0625f) * weight.inv32);
    listing = true;
  } else if (floor_key > 0) {
    from = floor_key, listing = true;
  }

  uint32_t key[kEach];
  int n = 0;
  if (listing) {
    // the elements `which` of a piece, those that are in the row
    const auto put = [&](int p, uint32_t which) {
      const int i0 = p * x.E - x.off;
      if (!x.inside(p)) {
#pragma unroll
        for (int e = 0; e < x.E; ++e)
          if (i0 + e < 0 || i0 + e >= x.V) which &= ~(1u << e);
      }
      if (which == 0) return;
      for (int at = atomicAdd(&s_listed, __popc(which)); which; which &= which - 1, ++at) {
        const int i = i0 + __ffs(which) - 1;
        if (at < kList) list[at] = make_uint2(P::key(P::value(x.bits(i))), i);
      }
    };
    if (bins) {
      u64 sum = 0;
      x.pieces_of([&](const uint4& r, int p) {
        uint32_t which = 0;
        if (weight.any(P::largest(r))) {
#pragma unroll
          for (int e = 0; e < x.E; ++e) {
            const float y = weight.raised(P::at(r, e));
            const u64 w = weight.raw(y);
            sum += w;
            if (y >= listed_to) mine_above += w;
            else if (y >= listed_from) which |= 1u << e;
          }
        } else if (weight.least >= listed_from) {
          which = (1u << x.E) - 1;
        }
        put(p, which);
      });
      need = need_of(sums(sum));
      above = sums(mine_above);
    } else {
      const float low = from == 0 ? -kInf : P::logit(from);
      x.pieces_of([&](const uint4& r, int p) {
        if (!(P::largest(r) >= low)) return;
        uint32_t which = 0;
#pragma unroll
        for (int e = 0; e < x.E; ++e)
          if (P::at(r, e) >= low) which |= 1u << e;
        put(p, which);
      });
      __syncthreads();
    }
    n = s_listed;
#pragma unroll
    for (int i = 0; i < kEach; ++i) key[i] = i * THREADS + tid < n ? list[min(i * THREADS + tid, kList - 1)].x : 0;  // 0: none
    if (bins) {
      uint32_t least = ~0u, most = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) least = min(least, key[i] != 0 ? key[i] : ~0u), most = max(most, key[i]);
      least = __reduce_min_sync(kFull, least), most = __reduce_max_sync(kFull, most);
      if (lane == 0) atomicMin(&s_range[0], least), atomicMax(&s_range[1], most);
      __syncthreads();
    }
  }
  bool listed = listing && n <= kList && (!bins || above < need);

  // ---- cuts, from count(c) and mass(c), of the keys >= c: over the list where there is one, else over the row
  u64 w[kEach] = {};  // of the list
  if (listed)
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (key[i] != 0) w[i] = weight(P::logit(key[i]));
  const auto count = [&](uint32_t c) -> uint32_t {
    uint32_t m = 0;
    if (listed) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) m += key[i] >= c;
    } else {
      const float low = P::logit(c);
      x.pieces_of([&](const uint4& r, int p) { x.each(r, p, low, [&](float, int) { ++m; }); });
    }
    return sums.count(m);
  };
  const auto mass = [&](uint32_t c) -> u64 {
    u64 m = 0;
    if (listed) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) m += key[i] >= c ? w[i] : 0;
      return sums(m);
    }
    const float low = P::logit(c);
    x.pieces_of([&](const uint4& r, int) {
      if (P::largest(r) >= low) m += x.weigh(r, weight, low);
    });
    return sums(m);
  };
  if (use_k) {
    const bool few = listed && n < top_k;  // min_p leaves fewer than top_k
    if (!few) {
      t = search(listed ? from : kLowest, kmax, [&](uint32_t c) { return count(c) >= top_k; });
      ties = top_k - (t >= kmax ? 0 : count(t + 1));
    }
  }
  if (use_p) {
    if (bins && listed && above + mass(kLowest) < need) listed = false;  // the bins did not hold the cut after all
    u64 over = t >= kmax ? 0 : mass(max(t + 1, kLowest));  // of the keys above t
    if (use_k || !listed) {
      above = 0;
      const u64 total = t == 0 ? over : over + ties * weight(P::logit(t));
      need = need_of(total);
    }
    uint32_t t2 = t;
    if (above + over >= need) {
      const bool few = bins && listed;
      t2 = search(few ? s_range[0] : max(t, kLowest), few ? s_range[1] : kmax, [&](uint32_t c) { return above + mass(c) >= need; });
      over = t2 >= kmax ? 0 : mass(t2 + 1);
    }
    const u64 each = t2 > kLowest ? weight(P::logit(t2)) : 0;
    if (each > 0) {
      const u64 m = (need - min(above + over, need) + each - 1) / each;
      ties = t2 == t ? min(ties, m) : m;
    }
    t = t2;
  }
  if (floor_key > t) t = floor_key, ties = ~0ull;

  // ---- the draw. `low`: the least logit kept; equal ones of the warps before this one count first
  const float low = t <= kLowest ? -kInf : P::logit(t);
  const bool limited = ties != ~0ull;
  u64 kept = 0;
  {
    uint32_t equal = 0;
    // Where the list holds all that is kept, or all but what has been weighed above its bins, it tells; else the row.
    if (listed && !(bins && weight.raised(low) >= listed_to)) {
      for (int i = tid; i < kWarps * 3; i += THREADS) warp_parts[i / 3][i % 3] = 0;
      if (tid < kWarps) warp_ties[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (key[i] == 0 || key[i] < t) continue;
        const int owner = (static_cast<int>(list[i * THREADS + tid].y) + x.off) / x.E / x.per;
        if (limited && key[i] == t) {
          atomicAdd(&warp_ties[owner], 1u);
        } else {  // parts of 20 bits: kList of them add up to less than 2^32
          atomicAdd(&warp_parts[owner][0], static_cast<uint32_t>(w[i] & 0xFFFFF));
          atomicAdd(&warp_parts[owner][1], static_cast<uint32_t>(w[i] >> 20 & 0xFFFFF));
          atomicAdd(&warp_parts[owner][2], static_cast<uint32_t>(w[i] >> 40));
        }
      }
      __syncthreads();
      equal = lane == 0 ? warp_ties[warp] : 0;
      kept = mine_above;
      if (lane == 0)
        kept += warp_parts[warp][0] + (static_cast<u64>(warp_parts[warp][1]) << 20) +
                (static_cast<u64>(warp_parts[warp][2]) << 40);
    } else {
      const float above_ties = !limited ? low : t >= kmax ? kInf : P::logit(t + 1);
      if (t == 0) x.pieces_of([&](const uint4& r, int) { kept += x.template weigh<true>(r, weight); });  // nothing is cut
      else x.pieces_of([&](const uint4& r, int p) {
        if (!(P::largest(r) >= low)) return;
        if (limited) x.each(r, p, low, [&](float v, int) { equal += v == low; });
        kept += x.weigh(r, weight, above_ties);
      });
    }
    if (limited) {
      equal = __reduce_add_sync(kFull, equal);
      if (lane == 0) warp_ties[warp] = equal;
      __syncthreads();
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) kept += __shfl_xor_sync(kFull, kept, o);
  }
  // of lanes: the warps' ties, weights, and both up to and with each
  const auto scan = [&](u64 v) {
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
      const u64 y = __shfl_up_sync(kFull, v, o);
      if (lane >= o) v += y;
    }
    return v;
  };
  uint32_t tie_upto = 0, tie_own = 0;
  if (limited) {
    tie_own = lane < kWarps ? warp_ties[lane] : 0;
    tie_upto = static_cast<uint32_t>(scan(tie_own));
    const uint32_t upto = __shfl_sync(kFull, tie_upto, warp), own = __shfl_sync(kFull, tie_own, warp);
    const u64 left = ties > upto - own ? ties - (upto - own) : 0;
    kept += min(left, static_cast<u64>(own)) * weight(low);
  }
  if (lane == 0) warp_sums[warp] = kept;
  __syncthreads();
  const u64 own = lane < kWarps ? warp_sums[lane] : 0, upto_all = scan(own);
  const u64 total = __shfl_sync(kFull, upto_all, kWarps - 1);
  u64 target = min(static_cast<u64>(max(u, 0.0) * static_cast<double>(total)), total - 1);
  const int owner = __ffs(__ballot_sync(kFull, lane < kWarps && target < upto_all)) - 1;
  target -= __shfl_sync(kFull, upto_all - own, owner);
  u64 tie0 = __shfl_sync(kFull, tie_upto - tie_own, owner);
  // The part of warp `owner`, kRun elements in turn to a thread: with 512 threads a part is 1 / 16 of the row, and fewer rounds
  // count (256 rows by top_p 53.5 us, with 1 element 54.7); with 1024 the first result does (1 row 15.0 us, with 4 elements 15.7).
  constexpr int kRun = THREADS == 512 ? 4 : 1;
  const int i1 = min((owner + 1) * x.per * x.E - x.off, a.V);
  __syncthreads();
  for (int i0 = max(owner * x.per * x.E - x.off, 0); i0 < i1; i0 += kRun * THREADS) {
    const int i = i0 + kRun * tid;
    u64 y[kRun];
    uint32_t equal = 0;
#pragma unroll
    for (int e = 0; e < kRun; ++e) {
      const float v = i + e < i1 ? P::value(x.bits(i + e)) : -kInf;
      y[e] = v >= low ? weight(v) : 0;
      equal |= i + e < i1 && v == low ? 1u << e : 0;
    }
    if (limited) {
      uint32_t upto = __popc(equal);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t z = __shfl_up_sync(kFull, upto, o);
        if (lane >= o) upto += z;
      }
      if (lane == 31) warp_ties[warp] = upto;
      __syncthreads();
      const uint32_t o = lane < kWarps ? warp_ties[lane] : 0, s = static_cast<uint32_t>(scan(o));
      u64 rank = tie0 + __shfl_sync(kFull, s - o, warp) + upto - __popc(equal);
      tie0 += __shfl_sync(kFull, s, kWarps - 1);
#pragma unroll
      for (int e = 0; e < kRun; ++e)
        if (equal >> e & 1 && rank++ >= ties) y[e] = 0;
    }
    u64 upto = 0;
#pragma unroll
    for (int e = 0; e < kRun; ++e) upto += y[e];
    const u64 mine_all = upto;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 z = __shfl_up_sync(kFull, upto, o);
      if (lane >= o) upto += z;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    const u64 o = lane < kWarps ? warp_sums[lane] : 0, s = scan(o), all = __shfl_sync(kFull, s, kWarps - 1);
    upto += __shfl_sync(kFull, s - o, warp);
    if (target < all) {
      u64 at = upto - mine_all;
#pragma unroll
      for (int e = 0; e < kRun; ++e) {
        if (target >= at && target < at + y[e]) a.tokens[row] = i + e;
        at += y[e];
      }
      return;
    }
    target -= all;
    __syncthreads();
  }
}

template <int TYPE, int THREADS>
void launch(const SampleArgs& a, cudaStream_t s) {
  constexpr int kRoom = (227 * 1024 - 1024 * (1024 / THREADS)) / (1024 / THREADS) - (THREADS == 1024 ? 21 : 12) * 1024;
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
  // More rows than SMs: two blocks of half the threads share one and overlap their passes (256 rows by top_p 54 us instead
  // of 68). Fewer: a row takes all threads of its SM (64 rows 17 us instead of 22, 1 row 15 instead of 17).
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
