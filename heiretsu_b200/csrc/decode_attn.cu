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

// Four 8 x 8 matrices of 16-bit values from shared memory (two with X2); lane i gives the address of row i % 8 of number i / 8.
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], uint32_t at) {  // each transposed
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
// Asynchronous copies into this CTA's shared memory: a box of a 4-D tensor, and 16 bytes.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void bulk_load_16(uint32_t dst, const void* src, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], 16, [%2];" ::"r"(dst),
               "l"(src), "r"(bar)
               : "memory");
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

// A tile of 16 * KT tokens of one K/V head, as it lies in a stage of a warp's ring in shared memory: K, then V, each
// [KT groups of 16 tokens][boxes of up to 128 bytes of a token][16 tokens][box]; codes have [KT][16 exponent bytes of K, 16
// of V] besides. The copies swizzle 16-byte chunks of a box by its token, so that the 8 rows of a matrix load
// lie in different banks.
template <int D, bool CODES>
struct Shape {
  static constexpr int kRow = D * (CODES ? 1 : 2);       // bytes of a token
  static constexpr int kBox = kRow < 128 ? kRow : 128;
  static constexpr int kBoxes = kRow / kBox;
  static constexpr int kGroup = 16 * kRow;               // bytes of 16 tokens
  // 4 KB of K and V (head dim 128 in 16 bits: 8; head dim 16 in codes: 2)
  static constexpr int KT = kGroup >= 2048 ? 1 : kGroup == 1024 ? 2 : 4;
  static constexpr int kTokens = 16 * KT;
  static constexpr int kKv = KT * kGroup;                // bytes of K of a tile
  static constexpr int kStage = 2 * kKv;
  static constexpr int kExps = CODES ? KT * 32 : 0;      // exponent bytes of a tile, kept apart
  static constexpr int kCtas = kGroup >= 4096 ? 1 : 2;   // on an SM: what the shared memory holds
  static constexpr int kSteps = D / 16;                  // matrix instructions along the channels
  // byte offset of 16-byte chunk c of token r in a group
  static __device__ __forceinline__ uint32_t chunk(int r, int c) {
    constexpr int per = kBox / 16;  // chunks of a box: 8, 4, 2 or 1
    const int x = per == 8 ? r & 7 : per == 4 ? r >> 1 & 3 : per == 2 ? r >> 2 & 1 : 0;
    return (c / per) * (16 * kBox) + r * kBox + (((c % per) ^ x) << 4);
  }
};

constexpr int kMaxSeqs = 1024;  // of one launch: their tile counts are summed in shared memory
constexpr int kMaxStages = 4;

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
__global__ void __launch_bounds__(kThreads, (Shape<D, CODES>::kCtas))
    decode_attn_kernel(const DecodeArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const int stages, const bool whole_units) {
  using S = Shape<D, CODES>;
  constexpr int KT = S::KT;
  constexpr bool QK16 = F16 || CODES;   // codes times q run in fp16 (q scaled by a power of two): fewer instructions to widen
  constexpr bool PV16 = F16 && !CODES;  // weights times codes run in bf16: 2^e of a head's scale has any exponent
  extern __shared__ uint8_t smem_raw[];  // the warps' rings, exponent bytes, a part for each warp
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int prefix[kMaxSeqs + 1];  // tiles of a unit before each sequence
  __shared__ int sums[kWarps];
  __shared__ int seg_unit[2 * kWarps], seg_first[2 * kWarps], seg_last[2 * kWarps], seg_tiles[2 * kWarps];
  __shared__ uint64_t full[kWarps][kMaxStages];

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
    if (lane < stages) mbar_init(&full[warp][lane], KT);
    fence_barrier_init();
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
  // number 2 w: where the run of warp w begins; 2 w + 1: where it ends, in its ring
  const auto part = [&](int i) {
    return reinterpret_cast<float*>(smem + (i & 1 ? (i >> 1) * stages * S::kStage : kWarps * stages * (S::kStage + S::kExps) + (i >> 1) * n.cols * (D + 2) * 4));
  };
  const int w0 = c0 + share(c1 - c0, warp, kWarps), w1 = c0 + share(c1 - c0, warp + 1, kWarps);

  // The ring. The copies of a tile are issued as soon as its stage has been read, in the order of the warp's run and across
  // its units, by the lanes that know the pages: lane i knows that of group number group0 + i of the sequence.
  uint8_t* const ring = smem + warp * stages * S::kStage;
  uint8_t* const exps = smem + kWarps * stages * S::kStage + warp * stages * S::kExps;
  const uint32_t ring0 = smem_u32(ring), bar0 = smem_u32(&full[warp][0]);
  struct {
    int at, b, u, tile, tiles, groups, group0, page, slot;
  } next;  // the tile to be copied next
  next.at = w0;
  uint32_t lost_pages = 0, lost = 0;  // lanes whose page is none; of the stages' groups, KT bits each
  const auto unit_at = [&](int at, int& b, int& u, int& tile, int& tiles) {
    b = 0;  // the last sequence whose tiles begin at or before `at`
    for (int hi = a.seqs; hi - b > 1;) {
      const int mid = (b + hi) >> 1;
      if (prefix[mid] * n.units <= at) b = mid;
      else hi = mid;
    }
    tiles = prefix[b + 1] - prefix[b];
    const int in_seq = at - prefix[b] * n.units;
    u = in_seq / tiles;
    tile = in_seq - u * tiles;
  };
  const auto find_pages = [&]() {
    next.group0 = next.tile * KT;
    const int mine = min(next.group0 + lane, next.groups - 1), page = mine / p.groups;
    next.slot = (mine - page * p.groups) * 16;
    next.page = a.table[next.b * a.tt + page];
    lost_pages = __ballot_sync(kFull, next.page < 0 || next.page >= p.pages);
    if (lost_pages && lane == 0) record_error(a.status, kBadArg, kSite);
  };
  const auto copy_next = [&](int stage) {
    if (next.at >= w1) return;
    if (next.at == w0 || next.tile == next.tiles) {  // another unit
      unit_at(next.at, next.b, next.u, next.tile, next.tiles);
      next.groups = (a.lengths[next.b] + 15) >> 4;
      find_pages();
    } else if (next.tile * KT >= next.group0 + 32) {
      find_pages();
    }
    const int first = next.tile * KT - next.group0, i = lane - first;
    lost = (lost & ~(((1u << KT) - 1) << (stage * KT))) | ((lost_pages >> first & ((1u << KT) - 1)) << (stage * KT));
    if (i >= 0 && i < KT) {
      const uint32_t bar = bar0 + 8 * stage, dst = ring0 + stage * S::kStage + i * S::kGroup;
      if (next.tile * KT + i < next.groups) {
        mbar_arrive_expect_tx(&full[warp][stage], 2 * S::kGroup + (CODES ? 32 : 0));
        const int h = next.u / n.chunks;
#pragma unroll
        for (int x = 0; x < S::kBoxes; ++x) {
          tma_load_4d(dst + x * 16 * S::kBox, &k_map, bar, x * (S::kBox / (CODES ? 1 : 2)), next.slot, h, next.page);
          tma_load_4d(dst + S::kKv + x * 16 * S::kBox, &v_map, bar, x * (S::kBox / (CODES ? 1 : 2)), next.slot, h, next.page);
        }
        if constexpr (CODES) {
          const long page = next.page < 0 || next.page >= p.pages ? 0 : next.page;
          const uint32_t e = smem_u32(exps) + stage * S::kExps + i * 32;
          bulk_load_16(e, p.ke + page * p.kep + h * p.keh + next.slot, bar);
          bulk_load_16(e + 16, p.ve + page * p.vep + h * p.veh + next.slot, bar);
        }
      } else {
        mbar_arrive(&full[warp][stage]);
      }
    }
    ++next.at, ++next.tile;
  };
  for (int s = 0; s < stages; ++s) copy_next(s);

  int stage = 0;
  uint32_t parity = 0;
  bool broken = false;  // a copy that did not arrive in time
  // where this lane's rows of matrix loads are: K of the tokens and chunks, V of the same, by Shape::chunk
  const int row_k = (lane & 7) + (lane & 8), chunk_k = lane >> 4;
  const int row_v = CODES ? row_k : (lane & 7) + (lane >> 4) * 8, chunk_v = CODES ? chunk_k : lane >> 3 & 1;

  for (int at = w0; at < w1 && !broken;) {
    int b, u, first, tiles;
    unit_at(at, b, u, first, tiles);
    const int last = min(tiles, first + (w1 - at));
    const Columns c(n, u);
    const int len = a.lengths[b], groups = (len + 15) >> 4;  // of 16 tokens

    // q of query head g of the unit, in the order of K's channels: index 2t of 16 is channel 2t (codes: 4t), 2t + 8 is 2t + 8
    // (codes: 4t + 2)
    float unit = a.scale * kLog2e;
    uint32_t q[S::kSteps][2];
    {
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + b * a.qt + (c.q0 + g) * a.qh + (CODES ? 4 * t : 2 * t);
#pragma unroll
      for (int x = 0; x < S::kSteps; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint16_t* s = src + 16 * x + (CODES ? 2 : 8) * i;
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
      for (int x = 0; x < S::kSteps; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) top = max(top, max(q[x][i] & 0x7FFFu, q[x][i] >> 16 & 0x7FFFu));
      top = max(top, __shfl_xor_sync(kFull, top, 1));
      top = max(top, __shfl_xor_sync(kFull, top, 2));
      const int e = min(max(static_cast<int>(top >> 7), 40), 254);  // biased; 255: infinity or NaN, which stay
      // 2^(141 - e), in two factors, which keeps q_unit out of the range below 2^-126
      const int s0 = (141 - e) / 2, s1 = 141 - e - s0;
      const float f0 = __uint_as_float((127 + s0) << 23), f1 = __uint_as_float((127 + s1) << 23);
#pragma unroll
      for (int x = 0; x < S::kSteps; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) q[x][i] = pack_f16(lo16<false>(q[x][i]) * f0 * f1, hi16<false>(q[x][i]) * f0 * f1);
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
      const uint32_t k0 = ring0 + stage * S::kStage, v0 = k0 + S::kKv;
      if (!mbar_wait(&full[warp][stage], parity, a.status, kSite)) {
        broken = true;
        break;
      }
      // scores: rows are tokens g and g + 8, columns query heads 2t and 2t + 1
      float s[KT][4], vs[KT][2];
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
        if constexpr (CODES) {
#pragma unroll
          for (int x = 0; x < S::kSteps; x += 2) {  // a load is 2 chunks of 16 channels (head dim 16: one, twice)
            uint32_t r[4];
            load_matrices(r, k0 + j * S::kGroup + S::chunk(row_k, S::kSteps == 1 ? 0 : x + chunk_k));
            uint32_t w[4][2];
#pragma unroll
            for (int i = 0; i < 4; ++i) widen_word(r[i], w[i]);
            mma<true>(s[j], w[0][0], w[1][0], w[0][1], w[1][1], q[x][0], q[x][1]);
            if (x + 1 < S::kSteps) mma<true>(s[j], w[2][0], w[3][0], w[2][1], w[3][1], q[x + 1 < S::kSteps ? x + 1 : 0][0], q[x + 1 < S::kSteps ? x + 1 : 0][1]);
          }
        } else {
#pragma unroll
          for (int x = 0; x < S::kSteps; ++x) {
            uint32_t r[4];
            load_matrices(r, k0 + j * S::kGroup + S::chunk(row_k, 2 * x + chunk_k));
            mma<F16>(s[j], r[0], r[1], r[2], r[3], q[x][0], q[x][1]);
          }
        }
        if constexpr (CODES) {
          const uint8_t* e = exps + stage * S::kExps + j * 32 + g;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float by = act8_scale(e[8 * r]);
            vs[j][r] = act8_scale(e[16 + 8 * r]);
            s[j][2 * r] *= by * q_unit[0], s[j][2 * r + 1] *= by * q_unit[1];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j][i] *= unit;
        }
      }
      const uint32_t none = lost >> (stage * KT) & ((1u << KT) - 1);
      if (none | (tile * KT + KT >= groups)) {  // the last tile, or pages that are none
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const int token = (tile * KT + j) * 16;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (none >> j & 1) s[j][i] = quiet_nan();
            if (token + g + 8 * (i >> 1) >= len) {
              s[j][i] = -INFINITY;
              if constexpr (CODES) vs[j][i >> 1] = 0.f;
            }
          }
          if (token + (lane & 15) >= len)  // V behind the length, whatever it is, becomes 0
#pragma unroll
            for (int x = 0; x < S::kRow / 16; ++x)
              if ((x & 1) == lane >> 4 || S::kRow == 16)
                *reinterpret_cast<uint4*>(ring + stage * S::kStage + S::kKv + j * S::kGroup + (x / (S::kBox / 16)) * 16 * S::kBox +
                                          (lane & 15) * S::kBox + (x % (S::kBox / 16)) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
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
        uint32_t hi[2], rest[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t x = pack16<PV16>(w[2 * r], w[2 * r + 1]);
          rest[r] = transpose8(pack16<PV16>(w[2 * r] - lo16<PV16>(x), w[2 * r + 1] - hi16<PV16>(x)));
          hi[r] = transpose8(x);
        }
        // output: rows are channels
        if constexpr (CODES) {
#pragma unroll
          for (int i = 0; i < D / 16; i += 2) {
            uint32_t r[4];
            load_matrices_t(r, v0 + j * S::kGroup + S::chunk(row_v, S::kSteps == 1 ? 0 : i + chunk_v));
#pragma unroll
            for (int x = 0; x < 2 && i + x < D / 16; ++x) {  // a word: channels 2g and 2g + 1 of two tokens
              const uint32_t v[4] = {widen_pair(r[2 * x]), widen_pair(r[2 * x] >> 8), widen_pair(r[2 * x + 1]), widen_pair(r[2 * x + 1] >> 8)};
              mma<PV16>(o[i + x < D / 16 ? i + x : 0], v[0], v[1], v[2], v[3], hi[0], hi[1]);
              mma<PV16>(o[i + x < D / 16 ? i + x : 0], v[0], v[1], v[2], v[3], rest[0], rest[1]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t r[4];
            load_matrices_t(r, v0 + j * S::kGroup + S::chunk(row_v, 2 * i + chunk_v));
            mma<PV16>(o[i], r[0], r[1], r[2], r[3], hi[0], hi[1]);
            mma<PV16>(o[i], r[0], r[1], r[2], r[3], rest[0], rest[1]);
          }
        }
      }
      __syncwarp();  // the stage has been read
      copy_next(stage);
      if (++stage == stages) stage = 0, parity ^= 1;
    }
    if (broken) break;
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[0] += __shfl_xor_sync(kFull, l[0], x);
      l[1] += __shfl_xor_sync(kFull, l[1], x);
    }
    // channel of row g (x = 0) or g + 8 (x = 1) of output tile i
    const auto channel = [&](int i, int x) { return 16 * i + (CODES ? 2 * g + x : g + 8 * x); };
    if (first == 0 && last == tiles) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = 2 * t + x;
        if (col < c.nq) {
          const long row = static_cast<long>(b) * a.heads_q + c.q0 + col;
          const float inv = 1.f / l[x];
          uint16_t* dst = static_cast<uint16_t*>(a.out) + row * D;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            dst[channel(i, 0)] = from_f32<F16>(o[i][x] * inv);
            dst[channel(i, 1)] = from_f32<F16>(o[i][2 + x] * inv);
          }
          if (g == 0) a.lse[row] = (m[x] + log2f(l[x])) * kLn2;
        }
      }
    } else {
      // a run has at most two such: where it begins, and where it ends, when the ring is no longer used
      const int mine = 2 * warp + (at != w0 ? 1 : 0);
      if (lane == 0) seg_unit[mine] = b * n.units + u, seg_first[mine] = first, seg_last[mine] = last, seg_tiles[mine] = tiles;
      float* dst = part(mine);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = 2 * t + x;
        if (col < n.cols) {
          if (g == 0) dst[col] = m[x], dst[n.cols + col] = l[x];
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            dst[2 * n.cols + col * D + channel(i, 0)] = o[i][x];
            dst[2 * n.cols + col * D + channel(i, 1)] = o[i][2 + x];
          }
        }
      }
    }
    at += last - first;
  }
  if (broken) {  // wait (with a limit) for what is still on its way, which must not outlive the CTA
    for (int s = 0; s < stages; ++s) {
      mbar_wait(&full[warp][stage], parity, a.status, kSite);
      if (++stage == stages) stage = 0, parity ^= 1;
    }
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
      for (uint32_t s = members; s; s &= s - 1) j.look(part(__ffs(s) - 1), col);
      j.looked();
      for (uint32_t s = members; s; s &= s - 1) j.add(part(__ffs(s) - 1), n.cols, col, e);
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

// The cache as a tensor of (channel, slot, head, page), copied 16 slots at a time.
template <int D, bool CODES>
CUtensorMap cache_map(const KvPool& p, const void* base, long page, long head, long slot) {
  using S = Shape<D, CODES>;
  const uint64_t es = CODES ? 1 : 2;
  const uint64_t sizes[4] = {D, static_cast<uint64_t>(p.size), static_cast<uint64_t>(p.heads), static_cast<uint64_t>(p.pages)};
  // (the stride of a dimension of one element is whatever it was given, and of no use)
  const uint64_t strides[3] = {slot * es, p.heads > 1 ? head * es : 16, p.pages > 1 ? page * es : 16};
  const uint32_t box[4] = {S::kBox / static_cast<uint32_t>(es), 16, 1, 1};
  return make_tmap(CODES ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, sizes, strides, box,
                   S::kBox == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                   : S::kBox == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                   : S::kBox == 32 ? CU_TENSOR_MAP_SWIZZLE_32B
                                   : CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int D, bool F16, bool CODES>
void launch(const DecodeArgs& a, int ctas, bool whole, cudaStream_t s) {
  using S = Shape<D, CODES>;
  const int cols = std::min(a.heads_q / a.pool.heads, kCols), parts = kWarps * cols * (D + 2) * 4 + 1024;
  // 227 KB of an SM, less 1 KB a CTA and what the kernel declares
  constexpr int kRoom = (227 * 1024) / S::kCtas - 1024 - 5 * 1024;
  const int stages = std::min(kMaxStages, (kRoom - parts) / (kWarps * (S::kStage + S::kExps)));
  const size_t smem = static_cast<size_t>(kWarps) * stages * (S::kStage + S::kExps) + parts;
  const auto kernel = decode_attn_kernel<D, F16, CODES>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may use that much shared memory
  const int dev = current_device();
  if (!(ready.load() >> dev & 1)) {
    HB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRoom));
    ready.fetch_or(1ull << dev);
  }
  const KvPool& p = a.pool;
  CUtensorMap k_map{}, v_map{};  // a cache of no pages is not read
  if (p.pages > 0) {
    k_map = cache_map<D, CODES>(p, p.k, p.kp, p.kh, p.ks);
    v_map = cache_map<D, CODES>(p, p.v, p.vp, p.vh, p.vs);
  }
  kernel<<<ctas, kThreads, smem, s>>>(a, k_map, v_map, stages, whole);
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

// CTAs on an SM, and tokens of a tile.
struct Fit {
  int ctas, tokens;
};
template <int D>
Fit fit_dim(bool codes) {
  if (codes) return {Shape<D, true>::kCtas, Shape<D, true>::kTokens};
  return {Shape<D, false>::kCtas, Shape<D, false>::kTokens};
}

}  // namespace

// As many CTAs as the SMs hold, or fewer where the table cannot hold a tile for each of their warps.
DecodePlan decode_attention_plan(const KvPool& p, int seqs, int units, int longest) {
  const bool codes = p.type == kKvCodes;
  const Fit f = p.dim == 16 ? fit_dim<16>(codes) : p.dim == 32 ? fit_dim<32>(codes) : p.dim == 64 ? fit_dim<64>(codes) : fit_dim<128>(codes);
  DecodePlan d;
  const long tiles = (longest + f.tokens - 1) / f.tokens, most = (1l << 31) - 1;
  d.seqs = static_cast<int>(std::min<long>(std::min(seqs, kMaxSeqs), most / std::max(1l, units * tiles)));
  if (d.seqs == 0) return d;
  d.whole = longest <= kWholeTokens;
  const long all = static_cast<long>(d.seqs) * units, sms = num_sms(current_device());
  d.ctas = static_cast<int>(std::max(1l, std::min(f.ctas * sms, d.whole ? all : (all * tiles + kWarps - 1) / kWarps)));
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
