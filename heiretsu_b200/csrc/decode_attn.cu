// Attention of one new token per sequence over a paged key/value cache:
//   s_j = scale q.k_j,  j < length;  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m);  lse = m + log sum_j e^(s_j - m)
// A sequence of length 0 gives 0 and -inf. A length outside [0, width * page size] or a page outside the cache gives NaN in
// the sequence's rows, and the bad-argument status.
#include <algorithm>
#include <atomic>

#include "act8.cuh"
#include "common.cuh"
#include "decode_args.h"
#include "host_utils.h"

namespace hb {

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kCols = 8;        // query heads of a unit: the columns of one matrix instruction
constexpr int kSite = 430;      // status site
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kFull = 0xffffffffu;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7FC00000u); }

// D += A B: A 16 x 16 (rows by lane / 4), B 16 x 8, 16-bit; D 16 x 8 in 32 bits.
template <bool F16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (F16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
// Transposes an 8 x 8 matrix of 16-bit values held two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// W words from global memory, or zeros.
template <int W>
__device__ __forceinline__ void load_words(uint32_t (&r)[W], const void* p, bool ok) {
  if constexpr (W == 4) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (ok) x = __ldg(static_cast<const uint4*>(p));
    r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
  } else if constexpr (W == 2) {
    uint2 x = make_uint2(0, 0);
    if (ok) x = __ldg(static_cast<const uint2*>(p));
    r[0] = x.x, r[1] = x.y;
  } else {
    static_assert(W == 1);
    r[0] = ok ? __ldg(static_cast<const uint32_t*>(p)) : 0u;
  }
}

// Two signed bytes (the low ones of `pair`'s halves, what lies above them is dropped) as two 16-bit floats.
// fp16: a byte with its sign flipped is code + 128; under 0x64 it reads as 1024 + 128 + code, and 1152 is taken off.
// bf16 has 7 fraction bits: under 0x43 the low 7 bits u read as 128 + u, the sign bit as 128 or 256; their difference
// is u - 128 sign.
template <bool F16>
__device__ __forceinline__ uint32_t widen_pair(uint32_t pair) {
  if constexpr (F16) {
    const uint32_t x = ((pair & 0x00FF00FFu) ^ 0x00800080u) | 0x64006400u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const uint32_t x = (pair & 0x007F007Fu) | 0x43004300u, y = (pair & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// How a warp holds a tile of 16 * KT tokens. In the matrix instructions' layout lane (g = lane / 4, t = lane % 4)
// holds, of each 16 tokens, K of the tokens g and g + 8 and V of 2t, 2t + 1, 2t + 8 and 2t + 9. Which channel an index of
// a product stands for is free as long as both operands agree, so a lane's channels are taken to be consecutive ones:
//   K: KE channels from c * 4 KE + t KE, for NKC chunks c (scores: K times q, sums over channels)
//   V: 2 VW channels from c * 16 VW + g 2 VW, for NVC chunks c (output: V^T times weights, sums over tokens)
// and tiles go from memory into registers in wide loads, with no shared memory between.
template <int D, bool CODES>
struct Shape {
  static constexpr int kBytes = CODES ? 1 : 2;
  static constexpr int KE = CODES ? (D / 4 < 16 ? D / 4 : 16) : (D / 4 < 8 ? D / 4 : 8);
  static constexpr int NKC = D / (4 * KE);
  static constexpr int KW = KE * kBytes / 4;  // words of a chunk
  static constexpr int QW = KE / 2;           // words of q of a chunk
  static constexpr int VW = CODES ? D / 16 : (D / 16 < 4 ? D / 16 : 4);
  static constexpr int NVC = D / (16 * VW);
  static constexpr int VB = 2 * VW * kBytes;  // bytes of a chunk
  static constexpr int VL = VB < 4 ? 1 : VB / 4;
  // 8 KB of K and V a tile where that is 64 registers or fewer
  static constexpr int KT = D >= 128 ? (CODES ? 2 : 1) : D == 64 ? (CODES ? 4 : 2) : 4;
  static constexpr int kTokens = 16 * KT;
};

// The share of CTA `c` of n: tiles [first(c), first(c + 1)).
__device__ __forceinline__ long first_tile(long total, int c, int n) { return total * c / n; }

constexpr int kMaxSeqs = 1024;  // of one launch: their tile counts are summed in shared memory

// Work is a list of tiles of 16 * KT tokens, ordered by sequence, then unit (a K/V head and up to 8 of its query heads),
// then token. Every CTA takes an equal run of it and every warp an equal run of the CTA's, whatever the lengths are: a
// unit may lie inside a warp's run, or be spread over warps and CTAs. A warp walks its run with a running maximum and sum
// per query head; what it has of a unit that is not wholly its own goes to shared memory, the CTA joins these, and
// what the CTA has of a unit that is not wholly its own goes to `part`, for join_kernel. Sums have a fixed order.
struct Unit {
  int b, h, chunk;  // sequence, K/V head, which 8 of its query heads
  int tiles;        // of the unit
};

template <int D>
__device__ __forceinline__ float* slot_of(float* base, int slot, int cols) {
  return base + static_cast<long>(slot) * cols * (D + 2);  // [cols] maxima, [cols] sums, [cols][D]
}

template <int D, bool F16, bool CODES>
__global__ void __launch_bounds__(kThreads, 2) decode_attn_kernel(const DecodeArgs a, const int ctas) {
  using S = Shape<D, CODES>;
  constexpr int KT = S::KT;
  constexpr bool PV16 = F16 && !CODES;  // weights times codes run in bf16: 2^e of a head's scale has any exponent
  extern __shared__ float slots[];      // two per warp
  __shared__ int prefix[kMaxSeqs + 1];  // tiles of a unit before each sequence
  __shared__ int warp_sum[kWarps];
  struct Seg {
    long unit;
    int first, last, tiles;  // tiles [first, last) of the unit's; first < 0: none
  };
  __shared__ Seg segs[2 * kWarps];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const KvPool& p = a.pool;
  const int G = a.heads_q / p.heads, chunks = (G + kCols - 1) / kCols, cols = min(G, kCols);
  const int units = p.heads * chunks;  // of a sequence
  const long longest = static_cast<long>(a.width) * p.size;

  // tiles of a unit before each sequence
  {
    int n[kMaxSeqs / kThreads], sum = 0;
#pragma unroll
    for (int i = 0; i < kMaxSeqs / kThreads; ++i) {
      const int b = tid * (kMaxSeqs / kThreads) + i;
      const int len = b < a.seqs ? a.lengths[b] : 0;
      n[i] = len > 0 && len <= longest ? (len + S::kTokens - 1) / S::kTokens : 0;
      sum += n[i];
    }
    int run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(kFull, run, o);
      if (lane >= o) run += x;
    }
    if (lane == 31) warp_sum[warp] = run;
    if (lane < 2) segs[2 * warp + lane].first = -1;
    __syncthreads();
    run -= sum;
    for (int w = 0; w < warp; ++w) run += warp_sum[w];
#pragma unroll
    for (int i = 0; i < kMaxSeqs / kThreads; ++i) {
      prefix[tid * (kMaxSeqs / kThreads) + i] = run;
      run += n[i];
    }
    if (tid == kThreads - 1) prefix[kMaxSeqs] = run;
    __syncthreads();
  }
  const long total = static_cast<long>(prefix[kMaxSeqs]) * units;
  const int busy = static_cast<int>(min(static_cast<long>(ctas), (total + kWarps - 1) / kWarps));

  // sequences without a tile: nothing cached, or a length that is none
  for (int b = blockIdx.x; b < a.seqs; b += gridDim.x) {
    if (prefix[b + 1] != prefix[b]) continue;
    const bool bad = a.lengths[b] != 0;
    if (bad && tid == 0) record_error(a.status, kBadArg, kSite);
    for (int i = tid; i < a.heads_q * D; i += kThreads)
      static_cast<uint16_t*>(a.out)[static_cast<long>(b) * a.heads_q * D + i] = from_f32<F16>(bad ? quiet_nan() : 0.f);
    for (int i = tid; i < a.heads_q; i += kThreads)
      a.lse[static_cast<long>(b) * a.heads_q + i] = bad ? quiet_nan() : -INFINITY;
  }

  const bool idle = static_cast<int>(blockIdx.x) >= busy;
  const long c0 = idle ? 0 : first_tile(total, blockIdx.x, busy), c1 = idle ? 0 : first_tile(total, blockIdx.x + 1, busy);
  const long w0 = c0 + (c1 - c0) * warp / kWarps, w1 = c0 + (c1 - c0) * (warp + 1) / kWarps;

  for (long at = w0; at < w1;) {
    // the unit that tile `at` belongs to: the last sequence whose tiles begin at or before it and that has any
    int lo = 0, hi = a.seqs;  // prefix[lo] * units <= at < prefix[hi] * units
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<long>(prefix[mid]) * units <= at) lo = mid;
      else hi = mid;
    }
    const int b = lo, tiles = prefix[lo + 1] - prefix[lo];
    const long in_seq = at - static_cast<long>(prefix[lo]) * units;
    const int u = static_cast<int>(in_seq / tiles), first = static_cast<int>(in_seq - static_cast<long>(u) * tiles);
    const int last = static_cast<int>(min(static_cast<long>(tiles), first + (w1 - at)));
    const int h = u / chunks, q0 = h * G + (u - h * chunks) * kCols, nq = min(kCols, (h + 1) * G - q0);
    const int len = a.lengths[b];

    // q of query head g of the unit, in the order of K's channels
    uint32_t q[S::NKC][S::QW];
    {
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + b * a.qt + (q0 + g) * a.qh + t * S::KE;
#pragma unroll
      for (int c = 0; c < S::NKC; ++c)
#pragma unroll
        for (int i = 0; i < S::QW; ++i) {
          const uint16_t* s = src + c * 4 * S::KE + 2 * i;
          if (g >= nq) q[c][i] = 0;
          else if (a.q_vec) q[c][i] = *reinterpret_cast<const uint32_t*>(s);
          else q[c][i] = s[0] | (static_cast<uint32_t>(s[1]) << 16);
        }
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // of columns 2t and 2t + 1, in units of log 2; l: this lane's rows
    float o[D / 16][4];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

    // Pages: lane i holds that of the 16 tokens number group0 + i.
    const int groups = (len + 15) >> 4, per_page = p.size >> 4;
    int group0 = -64, pages = 0;
    const auto page_of = [&](int group) {  // uniform over the warp
      if (group >= group0 + 32 || group < group0) {
        group0 = group;
        const int mine = group + lane;
        pages = mine < groups ? a.table[b * a.tt + mine / per_page] : 0;
        if (pages < 0 || pages >= p.pages) {
          record_error(a.status, kBadArg, kSite);
          pages = -1;
        }
      }
      return __shfl_sync(kFull, pages, group - group0);
    };

    uint32_t kr[KT][2][S::NKC][S::KW], vr[KT][4][S::NVC][S::VL];
    uint32_t ke[KT][2], ve[KT][2];  // exponent bytes of the tokens g and g + 8
    int bad = 0;                    // groups of the tile without a page
    const char* vsrc[KT];
    const auto load_k = [&](int tile) {
      bad = 0;
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const int group = tile * KT + j, tok = group * 16;
        vsrc[j] = nullptr;
        if (group < groups) {
          const int pg = page_of(group);
          const int at0 = tok % p.size;
          if (pg < 0) bad |= 1 << j;
          const char* base = static_cast<const char*>(p.k) + (pg * p.kp + h * p.kh + (at0 + g) * p.ks + t * S::KE) * S::kBytes;
          if (pg >= 0) vsrc[j] = static_cast<const char*>(p.v) + (pg * p.vp + h * p.vh + (at0 + 2 * t) * p.vs + g * 2 * S::VW) * S::kBytes;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const bool ok = pg >= 0 && tok + g + 8 * r < len;
#pragma unroll
            for (int c = 0; c < S::NKC; ++c)
              load_words<S::KW>(kr[j][r][c], base + (8 * r * p.ks + c * 4 * S::KE) * S::kBytes, ok);
            if constexpr (CODES) {
              ke[j][r] = ok ? p.ke[pg * p.kep + h * p.keh + at0 + g + 8 * r] : 0u;
              ve[j][r] = ok ? p.ve[pg * p.vep + h * p.veh + at0 + g + 8 * r] : 0u;
            }
          }
        } else {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            ke[j][r] = ve[j][r] = 0;
#pragma unroll
            for (int c = 0; c < S::NKC; ++c)
#pragma unroll
              for (int i = 0; i < S::KW; ++i) kr[j][r][c][i] = 0;
          }
        }
      }
    };
    const auto load_v = [&](int tile) {
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const int tok = (tile * KT + j) * 16 + 2 * t;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = (r & 1) + 8 * (r >> 1);
          const bool ok = vsrc[j] != nullptr && tok + row < len;
          const char* src = vsrc[j] + row * p.vs * S::kBytes;
#pragma unroll
          for (int c = 0; c < S::NVC; ++c) {
            if constexpr (S::VB >= 4) load_words<S::VL>(vr[j][r][c], src + c * 16 * S::VW * S::kBytes, ok);
            else vr[j][r][c][0] = ok ? __ldg(reinterpret_cast<const uint16_t*>(src)) : 0u;
          }
        }
      }
    };

    load_k(first);
    load_v(first);
    for (int tile = first; tile < last; ++tile) {
      // scores: rows are tokens g and g + 8, columns query heads 2t and 2t + 1
      float s[KT][4];
      const float unit = a.scale * kLog2e;
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int c = 0; c < S::NKC; ++c)
#pragma unroll
          for (int i = 0; i < S::KE / 4; ++i) {  // 16 channels
            if constexpr (CODES) {
              const uint32_t x = kr[j][0][c][i], y = kr[j][1][c][i];
              mma<F16>(s[j], widen_pair<F16>(__byte_perm(x, 0, 0x4140)), widen_pair<F16>(__byte_perm(y, 0, 0x4140)),
                       widen_pair<F16>(__byte_perm(x, 0, 0x4342)), widen_pair<F16>(__byte_perm(y, 0, 0x4342)), q[c][2 * i],
                       q[c][2 * i + 1]);
            } else {
              mma<F16>(s[j], kr[j][0][c][2 * i], kr[j][1][c][2 * i], kr[j][0][c][2 * i + 1], kr[j][1][c][2 * i + 1],
                       q[c][2 * i], q[c][2 * i + 1]);
            }
          }
        float by[2] = {unit, unit};
        if constexpr (CODES) by[0] = act8_scale(ke[j][0]) * unit, by[1] = act8_scale(ke[j][1]) * unit;
        const int tok = (tile * KT + j) * 16 + g;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[j][i] *= by[i >> 1];
          if (bad >> j & 1) s[j][i] = quiet_nan();
          if (tok + 8 * (i >> 1) >= len) s[j][i] = -INFINITY;
        }
      }
      float vs[KT][2];
#pragma unroll
      for (int j = 0; CODES && j < KT; ++j) vs[j][0] = act8_scale(ve[j][0]), vs[j][1] = act8_scale(ve[j][1]);
      if (tile + 1 < last) {  // K of the next tile is on its way during the rest of this one
        load_k(tile + 1);
      }
      // running maximum of each column
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i & 1] = fmaxf(top[i & 1], s[j][i]);
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        top[0] = fmaxf(top[0], __shfl_xor_sync(kFull, top[0], x));
        top[1] = fmaxf(top[1], __shfl_xor_sync(kFull, top[1], x));
      }
      if (__any_sync(kFull, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float f = top[x] == m[x] ? 1.f : ex2(m[x] - top[x]);
          m[x] = top[x];
          l[x] *= f;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) o[i][x] *= f, o[i][2 + x] *= f;
        }
      }
      const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        // weights, as the sum of two 16-bit numbers: what one of 8 or 11 bits leaves would show in the output
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = ex2(s[j][i] - ref[i & 1]);
          l[i & 1] += w[i];
          if constexpr (CODES) w[i] *= vs[j][i >> 1];
        }
        uint32_t hi[2], lo2[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t x = pack16<PV16>(w[2 * r], w[2 * r + 1]);
          const uint32_t y = pack16<PV16>(w[2 * r] - lo16<PV16>(x), w[2 * r + 1] - hi16<PV16>(x));
          hi[r] = transpose8(x);
          lo2[r] = transpose8(y);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int c = i / S::VW, k = i % S::VW;
          uint32_t x[4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (CODES) {
              const uint32_t e = vr[j][2 * r][c][k / 2], f = vr[j][2 * r + 1][c][k / 2];
              x[2 * r] = widen_pair<false>(__byte_perm(e, f, k & 1 ? 0x0602 : 0x0400));
              x[2 * r + 1] = widen_pair<false>(__byte_perm(e, f, k & 1 ? 0x0703 : 0x0501));
            } else {
              const uint32_t e = vr[j][2 * r][c][k], f = vr[j][2 * r + 1][c][k];
              x[2 * r] = __byte_perm(e, f, 0x5410);
              x[2 * r + 1] = __byte_perm(e, f, 0x7632);
            }
          }
          mma<PV16>(o[i], x[0], x[1], x[2], x[3], hi[0], hi[1]);
          mma<PV16>(o[i], x[0], x[1], x[2], x[3], lo2[0], lo2[1]);
        }
      }
      if (tile + 1 < last) load_v(tile + 1);
    }
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[0] += __shfl_xor_sync(kFull, l[0], x);
      l[1] += __shfl_xor_sync(kFull, l[1], x);
    }
    if (first == 0 && last == tiles) {  // the whole unit
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = 2 * t + x;
        if (col < nq) {
          const long row = static_cast<long>(b) * a.heads_q + q0 + col;
          const float inv = 1.f / l[x];
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const int d = (i / S::VW) * 16 * S::VW + g * 2 * S::VW + 2 * (i % S::VW);
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + row * D + d) =
                pack16<F16>(o[i][x] * inv, o[i][2 + x] * inv);
          }
          if (g == 0) a.lse[row] = (m[x] + log2f(l[x])) * kLn2;
        }
      }
    } else {
      const int mine = 2 * warp + (first == 0 && at != w0 ? 1 : 0);
      if (lane == 0) segs[mine] = Seg{static_cast<long>(b) * units + u, first, last, tiles};
      float* d0 = slot_of<D>(slots, mine, cols);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = 2 * t + x;
        if (col < cols) {
          if (g == 0) d0[col] = m[x], d0[cols + col] = l[x];
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const int d = (i / S::VW) * 16 * S::VW + g * 2 * S::VW + 2 * (i % S::VW);
            *reinterpret_cast<float2*>(d0 + 2 * cols + col * D + d) = make_float2(o[i][x], o[i][2 + x]);
          }
        }
      }
    }
    at += last - first;
  }
  __syncthreads();

  // Parts of units that warps share: joined in order.
  if (tid < 2 && !idle) a.record[2 * blockIdx.x + tid] = -1;
  __syncthreads();
  for (int i = 0; i < 2 * kWarps;) {
    if (segs[i].first < 0) {
      ++i;
      continue;
    }
    const long unit = segs[i].unit;
    int n = i, end = segs[i].last;  // segments [i, n) are of this unit
    while (n < 2 * kWarps && (segs[n].first < 0 || segs[n].unit == unit)) {
      if (segs[n].first >= 0) end = segs[n].last;
      ++n;
    }
    const int first = segs[i].first;
    const bool whole = first == 0 && end == segs[i].tiles;
    const int b = static_cast<int>(unit / units), u = static_cast<int>(unit - static_cast<long>(b) * units);
    const int h = u / chunks, q0 = h * G + (u - h * chunks) * kCols, nq = min(kCols, (h + 1) * G - q0);
    const int slot = 2 * blockIdx.x + (first == 0 ? 1 : 0);
    float* dst = slot_of<D>(a.part, slot, cols);
    for (int e = tid; e < nq * D; e += kThreads) {
      const int col = e / D, d = e - col * D;
      float top = -INFINITY;
      for (int k = i; k < n; ++k)
        if (segs[k].first >= 0) top = fmaxf(top, slot_of<D>(slots, k, cols)[col]);
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f, acc = 0.f;
      for (int k = i; k < n; ++k)
        if (segs[k].first >= 0) {
          const float* s = slot_of<D>(slots, k, cols);
          const float f = ex2(s[col] - ref);
          sum = fmaf(s[cols + col], f, sum);
          acc = fmaf(s[2 * cols + e], f, acc);
        }
      if (whole) {
        const long row = static_cast<long>(b) * a.heads_q + q0 + col;
        static_cast<uint16_t*>(a.out)[row * D + d] = from_f32<F16>(acc / sum);
        if (d == 0) a.lse[row] = (top + log2f(sum)) * kLn2;
      } else {
        dst[2 * cols + e] = acc;
        if (d == 0) dst[col] = top, dst[cols + col] = sum;
      }
    }
    if (!whole && tid == 0) a.record[slot] = 2 * unit + (end == segs[i].tiles ? 1 : 0);
    i = n;
  }
  if (idle && tid < 2) a.record[2 * blockIdx.x + tid] = -1;
}

// Joins the parts of the units that CTAs share. CTA (c, y): the unit that begins in CTA c of the kernel above and does not end
// there, if any; its other parts are the first ones of the CTAs behind. y: which kThreads elements of the unit.
template <int D, bool F16>
__global__ void __launch_bounds__(kThreads) join_kernel(const DecodeArgs a, const int ctas) {
  const long rec = a.record[2 * blockIdx.x + 1];
  if (rec < 0) return;
  const long unit = rec >> 1;
  const KvPool& p = a.pool;
  const int G = a.heads_q / p.heads, chunks = (G + kCols - 1) / kCols, cols = min(G, kCols), units = p.heads * chunks;
  const int b = static_cast<int>(unit / units), u = static_cast<int>(unit - static_cast<long>(b) * units);
  const int h = u / chunks, q0 = h * G + (u - h * chunks) * kCols, nq = min(kCols, (h + 1) * G - q0);
  int n = blockIdx.x + 1;  // the last CTA that has a part
  while (n + 1 < ctas && a.record[2 * n] == 2 * unit) ++n;
  const int e = blockIdx.y * kThreads + threadIdx.x;
  if (e >= nq * D) return;
  const int col = e / D, d = e - col * D;
  const float* first = slot_of<D>(a.part, 2 * blockIdx.x + 1, cols);
  float top = first[col];
  for (int k = blockIdx.x + 1; k <= n; ++k) top = fmaxf(top, slot_of<D>(a.part, 2 * k, cols)[col]);
  const float ref = top == -INFINITY ? 0.f : top;
  float f = ex2(first[col] - ref), sum = first[cols + col] * f, acc = first[2 * cols + e] * f;
#pragma unroll 4
  for (int k = blockIdx.x + 1; k <= n; ++k) {
    const float* s = slot_of<D>(a.part, 2 * k, cols);
    f = ex2(s[col] - ref);
    sum = fmaf(s[cols + col], f, sum);
    acc = fmaf(s[2 * cols + e], f, acc);
  }
  const long row = static_cast<long>(b) * a.heads_q + q0 + col;
  static_cast<uint16_t*>(a.out)[row * D + d] = from_f32<F16>(acc / sum);
  if (d == 0) a.lse[row] = (top + log2f(sum)) * kLn2;
}

template <int D, bool F16, bool CODES>
void launch(const DecodeArgs& a, int ctas, cudaStream_t s) {
  const int cols = std::min(a.heads_q / a.pool.heads, kCols);
  const size_t smem = sizeof(float) * 2 * kWarps * cols * (D + 2);
  const auto kernel = decode_attn_kernel<D, F16, CODES>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may use that much shared memory
  const int dev = current_device();
  if (!(ready.load() >> dev & 1)) {
    HB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(sizeof(float) * 2 * kWarps * kCols * (D + 2))));
    ready.fetch_or(1ull << dev);
  }
  kernel<<<ctas, kThreads, smem, s>>>(a, ctas);
  HB_CUDA_CHECK(cudaGetLastError());
  if (ctas > 1) {
    join_kernel<D, F16><<<dim3(ctas, (cols * D + kThreads - 1) / kThreads), kThreads, 0, s>>>(a, ctas);
    HB_CUDA_CHECK(cudaGetLastError());
  }
}
template <int D>
void launch_dim(const DecodeArgs& a, int ctas, cudaStream_t s) {
  if (a.pool.type == kKvCodes) a.f16 ? launch<D, true, true>(a, ctas, s) : launch<D, false, true>(a, ctas, s);
  else a.f16 ? launch<D, true, false>(a, ctas, s) : launch<D, false, false>(a, ctas, s);
}

}  // namespace

// CTAs of a launch: two on every SM, or fewer where the table cannot hold a tile for each of their warps.
int decode_attention_ctas(int seqs, int units, long longest) {
  const long tiles = static_cast<long>(seqs) * units * ((longest + 15) / 16);
  return static_cast<int>(std::max(1l, std::min(2l * num_sms(current_device()), (tiles + kWarps - 1) / kWarps)));
}
int decode_attention_seqs() { return kMaxSeqs; }

void decode_attention_launch(const DecodeArgs& a, int ctas, cudaStream_t s) {
  switch (a.pool.dim) {
    case 16: launch_dim<16>(a, ctas, s); break;
    case 32: launch_dim<32>(a, ctas, s); break;
    case 64: launch_dim<64>(a, ctas, s); break;
    default: launch_dim<128>(a, ctas, s); break;
  }
}

}  // namespace hb
