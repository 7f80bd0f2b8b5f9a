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

// W words from global memory.
template <int W>
__device__ __forceinline__ void load_words(uint32_t (&r)[W], const void* p) {
  if constexpr (W == 4) {
    const uint4 x = __ldg(static_cast<const uint4*>(p));
    r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
  } else if constexpr (W == 2) {
    const uint2 x = __ldg(static_cast<const uint2*>(p));
    r[0] = x.x, r[1] = x.y;
  } else {
    static_assert(W == 1);
    r[0] = __ldg(static_cast<const uint32_t*>(p));
  }
}

// Four signed bytes as fp16. A byte with its sign flipped is code + 128; under 0x64 it reads as 1024 + 128 + code, and 1152
// is taken off.
__device__ __forceinline__ void widen_word(uint32_t codes, uint32_t (&r)[2]) {
  codes ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = __byte_perm(codes, 0x64646464u, i ? 0x4342 : 0x4140);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    r[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
// Two signed bytes (the low ones of `pair`'s halves, whatever lies above them) as bf16, which has 7 fraction bits: under
// 0x43 the low 7 bits u read as 128 + u, the sign bit as 128 or 256, and their difference is u - 128 sign.
__device__ __forceinline__ uint32_t widen_pair(uint32_t pair) {
  const uint32_t x = (pair & 0x007F007Fu) | 0x43004300u, y = (pair & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
  return *reinterpret_cast<const uint32_t*>(&v);
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
  static constexpr int KT = D >= 128 ? 1 : D == 64 ? 2 : 4;
  static constexpr int kTokens = 16 * KT;
};

constexpr int kMaxSeqs = 1024;  // of one launch: their tile counts are summed in shared memory

// A unit: a K/V head of a sequence and up to 8 of its query heads.
struct Heads {
  int G, chunks, cols, units;  // query heads a K/V head, units a K/V head, columns in use, units of a sequence
  __device__ __forceinline__ explicit Heads(const DecodeArgs& a)
      : G(a.heads_q / a.pool.heads), chunks((G + kCols - 1) / kCols), cols(min(G, kCols)), units(a.pool.heads * chunks) {}
};
// Its query heads are q0 .. q0 + nq - 1.
struct Columns {
  int h, q0, nq;
  __device__ __forceinline__ Columns(const Heads& n, int u) : h(u / n.chunks) {
    q0 = h * n.G + (u - h * n.chunks) * kCols;
    nq = min(kCols, (h + 1) * n.G - q0);
  }
};

// Part of a unit: [cols] maxima, [cols] sums, [cols][D] weighted sums of V.
template <int D>
__device__ __forceinline__ float* part_of(float* base, int i, int cols) {
  return base + i * (cols * (D + 2));
}
// Joins element e = column * D + channel of parts: add() each, in order, twice: once for the maximum, once for the sums.
struct Join {
  float top = -INFINITY, ref = 0.f, sum = 0.f, acc = 0.f;
  __device__ __forceinline__ void look(const float* part, int col) { top = fmaxf(top, part[col]); }
  __device__ __forceinline__ void looked() { ref = top == -INFINITY ? 0.f : top; }
  __device__ __forceinline__ void add(const float* part, int cols, int col, int e) {
    const float f = ex2(part[col] - ref);
    sum = fmaf(part[cols + col], f, sum);
    acc = fmaf(part[2 * cols + e], f, acc);
  }
  template <bool F16>
  __device__ __forceinline__ void finish(const DecodeArgs& a, long row, int d, int D) const {
    static_cast<uint16_t*>(a.out)[row * D + d] = from_f32<F16>(acc / sum);
    if (d == 0) a.lse[row] = (top + log2f(sum)) * kLn2;
  }
};

// An equal share of `total` for each of n: that of number c begins here.
__device__ __forceinline__ int share(int total, int c, int n) {
  const int each = total / n, more = total - each * n;
  return c * each + min(c, more);
}

// Work is a list of tiles of 16 * KT tokens, ordered by sequence, then unit, then token. Every CTA takes an equal run of it
// and every warp an equal run of the CTA's, whatever the lengths are: a unit may lie inside a warp's run, or be
// spread over warps and CTAs. A warp walks its run with a running maximum and sum per query head; what it has of a
// unit that is not wholly its own goes to shared memory, the CTA joins these, and what the CTA has of a unit
// that is not wholly its own goes to a.part, for join_kernel. Sums have a fixed order. WHOLE: CTAs take whole
// units, and nothing is left to join.
template <int D, bool F16, bool CODES>
__global__ void __launch_bounds__(kThreads, 2) decode_attn_kernel(const DecodeArgs a, const bool whole_units) {
  using S = Shape<D, CODES>;
  constexpr int KT = S::KT;
  constexpr bool QK16 = F16 || CODES;   // codes times q run in fp16 (q scaled by a power of two): two instructions less a pair
  constexpr bool PV16 = F16 && !CODES;  // weights times codes run in bf16: 2^e of a head's scale has any exponent
  extern __shared__ float parts[];      // two per warp
  __shared__ int prefix[kMaxSeqs + 1];  // tiles of a unit before each sequence
  __shared__ int sums[kWarps];
  __shared__ int seg_unit[2 * kWarps], seg_first[2 * kWarps], seg_last[2 * kWarps], seg_tiles[2 * kWarps];

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const KvPool& p = a.pool;
  const Heads n(a);

  {  // tiles of a unit before each sequence
    const int per = (a.seqs + kThreads - 1) / kThreads, b0 = tid * per;  // at most 4
    int sum = 0;
    for (int b = b0; b < min(b0 + per, a.seqs); ++b) {
      const int len = a.lengths[b];
      prefix[b + 1] = len > 0 && len <= a.longest ? (len + S::kTokens - 1) / S::kTokens : 0;
      sum += prefix[b + 1];
    }
    int run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(kFull, run, o);
      if (lane >= o) run += x;
    }
    if (lane == 31) sums[warp] = run;
    if (lane < 2) seg_unit[2 * warp + lane] = -1;
    __syncthreads();
    run -= sum;
    for (int w = 0; w < warp; ++w) run += sums[w];
    for (int b = b0; b < min(b0 + per, a.seqs); ++b) {
      run += prefix[b + 1];
      prefix[b + 1] = run;
    }
    if (tid == 0) prefix[0] = 0;
    __syncthreads();
  }

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

  const int total = prefix[a.seqs] * n.units;
  int c0, c1, busy = gridDim.x;  // this CTA's run
  if (whole_units) {
    const auto start = [&](int c) {
      const int i = share(a.seqs * n.units, c, gridDim.x), b = i / n.units;
      return b == a.seqs ? total : prefix[b] * n.units + (i - b * n.units) * (prefix[b + 1] - prefix[b]);
    };
    c0 = start(blockIdx.x), c1 = start(blockIdx.x + 1);
  } else {
    busy = min(static_cast<int>(gridDim.x), (total + kWarps - 1) / kWarps);  // a tile for every warp at least
    const bool idle = static_cast<int>(blockIdx.x) >= busy;
    c0 = idle ? total : share(total, blockIdx.x, busy), c1 = idle ? total : share(total, blockIdx.x + 1, busy);
  }
  const int w0 = c0 + share(c1 - c0, warp, kWarps), w1 = c0 + share(c1 - c0, warp + 1, kWarps);

  for (int at = w0; at < w1;) {
    int b = 0;  // the last sequence whose tiles begin at or before `at`
    for (int hi = a.seqs; hi - b > 1;) {
      const int mid = (b + hi) >> 1;
      if (prefix[mid] * n.units <= at) b = mid;
      else hi = mid;
    }
    const int tiles = prefix[b + 1] - prefix[b], in_seq = at - prefix[b] * n.units;
    const int u = in_seq / tiles, first = in_seq - u * tiles, last = min(tiles, first + (w1 - at));
    const Columns c(n, u);
    const int len = a.lengths[b], groups = (len + 15) >> 4;  // of 16 tokens

    // Lane i knows where the group number group0 + i is: K and V in units of 16 bytes, the exponent bytes in bytes, from the
    // lane's own place in slot 0 of page 0. A page outside the cache is replaced by page 0 and noted in `lost`.
    int group0;
    uint32_t k_at, v_at, ke_at = 0, ve_at = 0, lost;
    const auto find_pages = [&](int group) {
      group0 = group;
      const int mine = min(group + lane, groups - 1);
      const int page = mine / p.groups, slot = (mine - page * p.groups) * 16;
      int id = a.table[b * a.tt + page];
      const bool bad = id < 0 || id >= p.pages;
      if (bad) id = 0;
      lost = __ballot_sync(kFull, bad);
      if (lost && lane == 0) record_error(a.status, kBadArg, kSite);
      k_at = id * p.kp16 + slot * p.ks16, v_at = id * p.vp16 + slot * p.vs16;
      if constexpr (CODES) ke_at = id * static_cast<uint32_t>(p.kep) + slot, ve_at = id * static_cast<uint32_t>(p.vep) + slot;
    };
    const char* const kb = static_cast<const char*>(p.k) + (c.h * p.kh + g * p.ks + t * S::KE) * S::kBytes;
    const char* const vb = static_cast<const char*>(p.v) + (c.h * p.vh + 2 * t * p.vs + g * 2 * S::VW) * S::kBytes;
    const uint8_t *keb = nullptr, *veb = nullptr;
    if constexpr (CODES) keb = p.ke + c.h * p.keh + g, veb = p.ve + c.h * p.veh + g;
    const long k8 = 8 * p.ks * S::kBytes, v1 = p.vs * S::kBytes;

    uint32_t kr[KT][2][S::NKC][S::KW], vr[KT][4][S::NVC][S::VL], vo[KT];
    uint32_t ke[KT][2], ve[KT][2];  // exponent bytes of the tokens g and g + 8
    // Slots behind the length are read too (they are slots of the page): K's scores and V are blanked out below.
    const auto load_k = [&](int tile) {
      if (tile * KT >= group0 + 32) find_pages(tile * KT);
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const int i = tile * KT + j - group0;
        const char* src = kb + static_cast<uint64_t>(__shfl_sync(kFull, k_at, i)) * 16;
        vo[j] = __shfl_sync(kFull, v_at, i);
#pragma unroll
        for (int x = 0; x < S::NKC; ++x) {
          load_words<S::KW>(kr[j][0][x], src + x * 4 * S::KE * S::kBytes);
          load_words<S::KW>(kr[j][1][x], src + k8 + x * 4 * S::KE * S::kBytes);
        }
        if constexpr (CODES) {
          const uint8_t* ks = keb + __shfl_sync(kFull, ke_at, i);
          const uint8_t* vs = veb + __shfl_sync(kFull, ve_at, i);
          ke[j][0] = __ldg(ks), ke[j][1] = __ldg(ks + 8);
          ve[j][0] = __ldg(vs), ve[j][1] = __ldg(vs + 8);
        }
      }
    };
    const auto load_v = [&]() {
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const char* src = vb + static_cast<uint64_t>(vo[j]) * 16;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int x = 0; x < S::NVC; ++x) {
            const char* s = src + ((r & 1) + 8 * (r >> 1)) * v1 + x * 16 * S::VW * S::kBytes;
            if constexpr (S::VB >= 4) load_words<S::VL>(vr[j][r][x], s);
            else vr[j][r][x][0] = __ldg(reinterpret_cast<const uint16_t*>(s));
          }
      }
    };
    find_pages(first * KT);
    load_k(first);
    load_v();

    // q of query head g of the unit, in the order of K's channels
    float unit = a.scale * kLog2e;
    uint32_t q[S::NKC][S::QW];
    {
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + b * a.qt + (c.q0 + g) * a.qh + t * S::KE;
#pragma unroll
      for (int x = 0; x < S::NKC; ++x)
#pragma unroll
        for (int i = 0; i < S::QW; ++i) {
          const uint16_t* s = src + x * 4 * S::KE + 2 * i;
          if (g >= c.nq) q[x][i] = 0;
          else if (a.q_vec) q[x][i] = *reinterpret_cast<const uint32_t*>(s);
          else q[x][i] = s[0] | (static_cast<uint32_t>(s[1]) << 16);
        }
    }
    float q_unit[2] = {unit, unit};  // of columns 2t and 2t + 1
    if constexpr (QK16 && !F16) {
      // bf16 q in fp16: times 2^(14 - exponent of the head's largest), so that 2^-29 of it is still exact
      uint32_t top = 0;
#pragma unroll
      for (int x = 0; x < S::NKC; ++x)
#pragma unroll
        for (int i = 0; i < S::QW; ++i) top = max(top, max(q[x][i] & 0x7FFFu, q[x][i] >> 16 & 0x7FFFu));
      top = max(top, __shfl_xor_sync(kFull, top, 1));
      top = max(top, __shfl_xor_sync(kFull, top, 2));
      const int e = min(max(static_cast<int>(top >> 7), 40), 254);  // biased; 255: infinity or NaN, which stay
      // 2^(141 - e), in two factors, which keeps q_unit out of the range below 2^-126
      const int s0 = (141 - e) / 2, s1 = 141 - e - s0;
      const float f0 = __uint_as_float((127 + s0) << 23), f1 = __uint_as_float((127 + s1) << 23);
#pragma unroll
      for (int x = 0; x < S::NKC; ++x)
#pragma unroll
        for (int i = 0; i < S::QW; ++i) q[x][i] = pack_f16(lo16<false>(q[x][i]) * f0 * f1, hi16<false>(q[x][i]) * f0 * f1);
      const float back0 = __uint_as_float((127 - s0) << 23), back1 = __uint_as_float((127 - s1) << 23);
      const float b0 = __shfl_sync(kFull, back0, 8 * t), b1 = __shfl_sync(kFull, back1, 8 * t);
      const float d0 = __shfl_sync(kFull, back0, 8 * t + 4), d1 = __shfl_sync(kFull, back1, 8 * t + 4);
      q_unit[0] = b0 * unit * b1, q_unit[1] = d0 * unit * d1;
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // of columns 2t and 2t + 1, in powers of 2; l: this lane's rows
    float o[D / 16][4];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

    for (int tile = first; tile < last; ++tile) {
      // scores: rows are tokens g and g + 8, columns query heads 2t and 2t + 1
      float s[KT][4], vs[KT][2];
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int x = 0; x < S::NKC; ++x)
#pragma unroll
          for (int i = 0; i < S::KE / 4; ++i) {  // 16 channels
            if constexpr (CODES) {
              uint32_t r0[2], r1[2];
              widen_word(kr[j][0][x][i], r0);
              widen_word(kr[j][1][x][i], r1);
              mma<true>(s[j], r0[0], r1[0], r0[1], r1[1], q[x][2 * i], q[x][2 * i + 1]);
            } else {
              mma<F16>(s[j], kr[j][0][x][2 * i], kr[j][1][x][2 * i], kr[j][0][x][2 * i + 1], kr[j][1][x][2 * i + 1],
                       q[x][2 * i], q[x][2 * i + 1]);
            }
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (CODES) s[j][i] *= act8_scale(ke[j][i >> 1]) * q_unit[i & 1];
          else s[j][i] *= unit;
        }
        if constexpr (CODES) vs[j][0] = act8_scale(ve[j][0]), vs[j][1] = act8_scale(ve[j][1]);
      }
      if (lost | (tile * KT + KT >= groups)) {  // the last tile, or pages that are none
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const int group = tile * KT + j;
          const bool none = lost >> (min(group, groups - 1) - group0) & 1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (none) s[j][i] = quiet_nan();
            if (group * 16 + g + 8 * (i >> 1) >= len) {
              s[j][i] = -INFINITY;
              if constexpr (CODES) vs[j][i >> 1] = 0.f;
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (none || group * 16 + 2 * t + (r & 1) + 8 * (r >> 1) >= len)
#pragma unroll
              for (int x = 0; x < S::NVC; ++x)
#pragma unroll
                for (int i = 0; i < S::VL; ++i) vr[j][r][x][i] = 0;
        }
      }
      if (tile + 1 < last) load_k(tile + 1);  // on its way during the rest of this tile
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
        uint32_t hi[2], rest[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t x = pack16<PV16>(w[2 * r], w[2 * r + 1]);
          rest[r] = transpose8(pack16<PV16>(w[2 * r] - lo16<PV16>(x), w[2 * r + 1] - hi16<PV16>(x)));
          hi[r] = transpose8(x);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int x = i / S::VW, k = i % S::VW;
          uint32_t v[4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (CODES) {
              const uint32_t e = vr[j][2 * r][x][k / 2], f = vr[j][2 * r + 1][x][k / 2];
              v[2 * r] = widen_pair(__byte_perm(e, f, k & 1 ? 0x0602 : 0x0400));
              v[2 * r + 1] = widen_pair(__byte_perm(e, f, k & 1 ? 0x0703 : 0x0501));
            } else {
              const uint32_t e = vr[j][2 * r][x][k], f = vr[j][2 * r + 1][x][k];
              v[2 * r] = __byte_perm(e, f, 0x5410);
              v[2 * r + 1] = __byte_perm(e, f, 0x7632);
            }
          }
          mma<PV16>(o[i], v[0], v[1], v[2], v[3], hi[0], hi[1]);
          mma<PV16>(o[i], v[0], v[1], v[2], v[3], rest[0], rest[1]);
        }
      }
      if (tile + 1 < last) load_v();
    }
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[0] += __shfl_xor_sync(kFull, l[0], x);
      l[1] += __shfl_xor_sync(kFull, l[1], x);
    }
    const auto channel = [&](int i) { return (i / S::VW) * 16 * S::VW + g * 2 * S::VW + 2 * (i % S::VW); };
    if (first == 0 && last == tiles) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = 2 * t + x;
        if (col < c.nq) {
          const long row = static_cast<long>(b) * a.heads_q + c.q0 + col;
          const float inv = 1.f / l[x];
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + row * D + channel(i)) =
                pack16<F16>(o[i][x] * inv, o[i][2 + x] * inv);
          if (g == 0) a.lse[row] = (m[x] + log2f(l[x])) * kLn2;
        }
      }
    } else {
      const int mine = 2 * warp + (at != w0 ? 1 : 0);  // a run has at most two such: where it begins, and where it ends
      if (lane == 0) seg_unit[mine] = b * n.units + u, seg_first[mine] = first, seg_last[mine] = last, seg_tiles[mine] = tiles;
      float* dst = part_of<D>(parts, mine, n.cols);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = 2 * t + x;
        if (col < n.cols) {
          if (g == 0) dst[col] = m[x], dst[n.cols + col] = l[x];
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            *reinterpret_cast<float2*>(dst + 2 * n.cols + col * D + channel(i)) = make_float2(o[i][x], o[i][2 + x]);
        }
      }
    }
    at += last - first;
  }
  if (tid < 2) a.record[2 * blockIdx.x + tid] = make_int2(-1, 0);
  __syncthreads();

  // Parts of units that warps share. Lane i looks at segment i; neighbouring ones of one unit are a set; 32 elements
  // of a set are an item, and the warps take the items in turn.
  const int unit = lane < 2 * kWarps ? seg_unit[lane] : -1;
  const uint32_t used = __ballot_sync(kFull, unit >= 0), before = used & ((1u << lane) - 1);
  const int prev = __shfl_sync(kFull, unit, before ? 31 - __clz(before) : 0);
  uint32_t starts = __ballot_sync(kFull, unit >= 0 && (before == 0 || prev != unit));
  for (int item = warp; starts; starts &= starts - 1) {
    const int i0 = __ffs(starts) - 1;
    const uint32_t rest = starts & (starts - 1);
    const uint32_t members = used & ~((1u << i0) - 1) & (rest ? (1u << (__ffs(rest) - 1)) - 1 : kFull);
    const int id = seg_unit[i0], b = id / n.units, first = seg_first[i0], end = 31 - __clz(members);
    const Columns c(n, id - b * n.units);
    const bool whole = first == 0 && seg_last[end] == seg_tiles[i0];
    const int slot = 2 * blockIdx.x + (first == 0 ? 1 : 0);
    float* dst = part_of<D>(a.part, slot, n.cols);
    const int items = c.nq * D / 32 + (c.nq * D % 32 != 0);
    for (; item < items; item += kWarps) {
      const int e = item * 32 + lane, col = e / D, d = e % D;
      if (item == 0 && lane == 0 && !whole) {
        // how many CTAs behind this one have a part of a unit that begins here
        const int left = seg_tiles[i0] - seg_last[end];
        int last_cta = blockIdx.x;
        if (left > 0) {
          const int tile = c1 + left - 1, each = total / busy, more = total - each * busy;  // who has this one
          last_cta = tile < more * (each + 1) ? tile / (each + 1) : (tile - more) / each;
        }
        a.record[slot] = make_int2(id, last_cta - blockIdx.x);
      }
      if (col >= c.nq) continue;
      Join j;
      for (uint32_t s = members; s; s &= s - 1) j.look(part_of<D>(parts, __ffs(s) - 1, n.cols), col);
      j.looked();
      for (uint32_t s = members; s; s &= s - 1) j.add(part_of<D>(parts, __ffs(s) - 1, n.cols), n.cols, col, e);
      if (whole) {
        j.finish<F16>(a, static_cast<long>(b) * a.heads_q + c.q0 + col, d, D);
      } else {
        dst[2 * n.cols + e] = j.acc;
        if (d == 0) dst[col] = j.top, dst[n.cols + col] = j.sum;
      }
    }
    item -= items;
  }
}

// Joins the parts of the units that CTAs share. CTA (c, y): the unit that begins in CTA c of the kernel above and does not end
// there, if any; its other parts are the first ones of the CTAs behind. y: which kJoin elements of the unit.
constexpr int kJoin = 128;
template <int D, bool F16>
__global__ void __launch_bounds__(kJoin) join_kernel(const DecodeArgs a) {
  const Heads n(a);
  const int e = blockIdx.y * kJoin + threadIdx.x, col = e / D, d = e % D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int2 rec = a.record[2 * blockIdx.x + 1];
  if (rec.x < 0) return;
  const int b = rec.x / n.units;
  const Columns c(n, rec.x - b * n.units);
  if (col >= c.nq) return;
  const auto part = [&](int i) { return part_of<D>(a.part, 2 * (blockIdx.x + i) + (i == 0 ? 1 : 0), n.cols); };
  Join j;
#pragma unroll 4
  for (int i = 0; i <= rec.y; ++i) j.look(part(i), col);
  j.looked();
#pragma unroll 4
  for (int i = 0; i <= rec.y; ++i) j.add(part(i), n.cols, col, e);
  j.finish<F16>(a, static_cast<long>(b) * a.heads_q + c.q0 + col, d, D);
}

template <int D, bool F16, bool CODES>
void launch(const DecodeArgs& a, int ctas, bool whole, cudaStream_t s) {
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
  kernel<<<ctas, kThreads, smem, s>>>(a, whole);
  HB_CUDA_CHECK(cudaGetLastError());
  if (whole || ctas == 1) return;
  cudaLaunchConfig_t cfg{};  // launched while the kernel above runs: it waits for its end by itself
  cfg.gridDim = dim3(ctas, (cols * D + kJoin - 1) / kJoin);
  cfg.blockDim = dim3(kJoin);
  cfg.stream = s;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = early;
  cfg.numAttrs = 1;
  HB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, join_kernel<D, F16>, a));
}
template <int D>
void launch_dim(const DecodeArgs& a, int ctas, bool whole, cudaStream_t s) {
  if (a.pool.type == kKvCodes) a.f16 ? launch<D, true, true>(a, ctas, whole, s) : launch<D, false, true>(a, ctas, whole, s);
  else a.f16 ? launch<D, true, false>(a, ctas, whole, s) : launch<D, false, false>(a, ctas, whole, s);
}

constexpr int kWholeTokens = 256;

}  // namespace

// Two CTAs on every SM, or fewer where the table cannot hold a tile for each of their warps.
DecodePlan decode_attention_plan(int seqs, int units, int longest) {
  DecodePlan d;
  const long tiles = (longest + 15) / 16, fit = (1l << 31) - 1;
  d.seqs = static_cast<int>(std::min<long>(std::min(seqs, kMaxSeqs), fit / std::max(1l, units * tiles)));
  if (d.seqs == 0) return d;
  d.whole = longest <= kWholeTokens;
  const long all = static_cast<long>(d.seqs) * units;
  d.ctas = static_cast<int>(std::max(1l, std::min(2l * num_sms(current_device()), d.whole ? all : (all * tiles + kWarps - 1) / kWarps)));
  return d;
}

void decode_attention_launch(const DecodeArgs& a, const DecodePlan& d, cudaStream_t s) {
  switch (a.pool.dim) {
    case 16: launch_dim<16>(a, d.ctas, d.whole, s); break;
    case 32: launch_dim<32>(a, d.ctas, d.whole, s); break;
    case 64: launch_dim<64>(a, d.ctas, d.whole, s); break;
    default: launch_dim<128>(a, d.ctas, d.whole, s); break;
  }
}

}  // namespace hb
