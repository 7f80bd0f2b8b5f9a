// Attention of one new token per sequence over a paged key/value cache:
//   s_j = scale q.k_j,  j < length;  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m);  lse = m + log sum_j e^(s_j - m)
// A sequence of length 0 gives 0 and -inf. A length outside [0, width * page size] or a page outside the cache gives NaN in
// the sequence's rows, and the bad-argument status.
//
// Every K and V is read once and takes part in 4 operations a query head that shares it: bound by memory. So the tiles lie where
// copies put them, and the products take the small matrix instructions (8 query heads are a column each; those of 128 rows
// would be all but empty). Device times on a B200, and what the bytes alone take at a copy's 6.5 TB/s:
//   64 sequences of up to 8192 tokens, 8 K/V heads of 128 with 4 query heads each, bf16    173 us    169
//   the same in codes                                                                      112       85
//   64 of up to 8192, 2 K/V heads of 64 with 16 query heads each (K and V read twice)       43.5     21.2
//   1 of 100003, 8 K/V heads of 128 with 4 query heads each, fp16                           71       63
//   61 of up to 1024, 12 heads of 64, bf16                                                  25.3     14.6
//   61 of up to 1024, 8 heads of 32 / 16, bf16                                              14.1 / 11.6    4.9 / 2.4
//   256 of up to 1024, 20 heads of 64, in codes                                             96.4     54
//   1 of 57, 12 heads of 64                                                                  5.9      0.03
// Long sequences are near their bytes. Short ones pay the start, the joins and the second kernel (about 3 us each); codes
// pay their widening, 5 to 7 instructions for 4 codes.
// Tried and slower, each beside the kernel of its time: tiles loaded into registers (64 x 8192 227 us instead of 191), every
// warp copying for itself (256 in codes 109 instead of 95), stages of K and of V apart (64 x 8192 184 instead of 174).
#include <algorithm>
#include <atomic>

#include "act8.cuh"
#include "common.cuh"
#include "decode_args.h"
#include "host_utils.h"

namespace hb {

namespace {

constexpr int kWarps = 8;                       // that compute
constexpr int kCols = 8;        // query heads of a unit: the columns of one matrix instruction
constexpr int kSite = 430;      // status site
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kFull = 0xffffffffu;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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
// Whether the phase with the given parity has completed.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Asynchronous copies into this CTA's shared memory: a box of a 4-D tensor, and 16 bytes.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void copy_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Four signed bytes as fp16, in pairs: bytes 0 and 1, 2 and 3. A byte with its sign flipped is code + 128; under 0x64 it reads as
// 1024 + 128 + code, and 1152 is taken off.
__device__ __forceinline__ void widen(uint32_t codes, uint32_t (&r)[2]) {
  codes ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = __byte_perm(codes, 0x64646464u, i ? 0x4342 : 0x4140);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    r[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
// Two signed bytes (the low ones of `pair`'s halves, whatever lies above them) as bf16, which has 7 fraction bits: under 0x43
// the low 7 bits u read as 128 + u, the sign bit as 128 or 256, and their difference is u - 128 sign.
__device__ __forceinline__ uint32_t widen_bf16(uint32_t pair) {
  const uint32_t x = (pair & 0x007F007Fu) | 0x43004300u, y = (pair & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
  return *reinterpret_cast<const uint32_t*>(&v);
}
// A tile of 16 * KT tokens of one K/V head, as it lies in a stage of a warp's ring in shared memory: K, then V; codes have
// 16 * KT exponent bytes of K and as many of V besides. A box is what one copy brings: rows of up to 128 bytes, whose 16-byte
// chunks are swizzled by the row, so that the 8 tokens of a matrix load lie in different banks.
template <int D, bool CODES>
struct Shape {
  static constexpr int kSize = CODES ? 1 : 2;
  static constexpr int kRow = D * kSize;                 // bytes of a token
  static constexpr int kBoxes = kRow <= 128 ? 1 : kRow / 128;  // along the channels
  static constexpr int kGroup = 16 * kRow;               // bytes of 16 tokens
  // What a warp takes at a time: 8 KB of K and V (head dim 16, and 32 in codes: 4, 16 in codes: 2). When this was chosen, 61 x up
  // to 1024 tokens of 12 heads of 64 took 26.9 us in bf16, with 4 KB 28.2 (its one stage a warp then has a second; later steps
  // brought 25.3). In codes the registers for that are there with one CTA an SM: 256 x up to 1024 tokens of 20 heads of 64
  // 96.5 us, 1 x 60000 of 2 heads 15.3; with 4 KB and two CTAs 99 and 19.1 (but 16 x up to 384 of 12 heads 9.1 instead
  // of 10.0), with 2 KB 129. Head dim 128 in codes, 64 x up to 8192 tokens of 8 heads: 115 us; 4 KB and two CTAs, which
  // have to spill, 141.
  static constexpr int KT = kGroup == 4096 ? 1 : kGroup == 2048 ? 2 : 4;
  static constexpr int kTokens = 16 * KT;
  static constexpr int kKv = KT * kGroup;                // bytes of K of a tile
  static constexpr int kStage = 2 * kKv;
  static constexpr int kExps = CODES ? 2 * kTokens : 0;
  static constexpr int kCtas = D == 128 || (CODES && D == 64) ? 1 : 2;  // on an SM: what its memory (16 bits) and registers hold
  static constexpr int kSteps = D / 16;                  // matrix instructions along the channels
  // Warps that issue copies, which a warp does one lane after the other. As many as leave the registers to the rest: 64 x up to 8192
  // tokens of 8 heads of 128 take 174.5 us (with two such warps 177.8, with one 179.6), in codes with pages of 16 tokens
  // 113 (115, 152), 256 x up to 1024 of 20 heads of 64 in codes with such pages 101 with two (114 with one).
  static constexpr int kMovers = kCtas == 1 ? 4 : 2;
  static constexpr int kThreads = 32 * (kWarps + kMovers);
};
// Where a lane's row of a matrix load is in 16 tokens, the group number j of a tile: chunk(c, j) is that of chunk c (known when
// compiled) of token r, c without its bits in `c0`. `packed`: the cache's slots follow one another, and where a token is
// shorter than 128 bytes a row of a box holds several, which the copies bring 2 to 8 times as fast; else a row is a token.
template <int ROW>
struct Place {
  uint32_t at, x, groups;
  __device__ __forceinline__ Place(int r, int c0, bool packed) : groups(0) {
    if (ROW >= 128) {
      at = r * 128, x = (r & 7) ^ c0;
    } else if (packed) {
      at = r * ROW & ~127, x = ((r * ROW & 127) >> 4) ^ (r * ROW >> 7 & 7) ^ c0;
      groups = 7;  // 16 tokens may be fewer than the 8 rows after which the swizzle repeats
    } else {
      at = r * ROW, x = (ROW == 64 ? r >> 1 & 3 : ROW == 32 ? r >> 2 & 1 : 0) ^ c0;
    }
  }
  __device__ __forceinline__ uint32_t chunk(int c, int j) const {  // 8 chunks to a box of 16 tokens
    const uint32_t y = ROW < 64 ? x ^ (j * 16 * ROW / 128 & groups) : x;
    return j * 16 * ROW + (c >> 3) * 2048 + at + ((y ^ (c & 7)) << 4);
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

// Part of a unit: [cols] maxima, [cols] sums, [cols][D] weighted sums of V; every part and row on 16-byte boundaries.
__host__ __device__ constexpr int part_head(int cols) { return (2 * cols + 3) & ~3; }
template <int D>
__device__ __forceinline__ float* part_of(float* base, int i, int cols) {
  return base + i * (part_head(cols) + cols * D);
}
// A warp joins column `col` of n parts, in order; part(i) gives the address of the i-th. Lane i works out the factor of
// part i; then each lane sums its share of the D channels, E consecutive ones.
template <int D>
struct Join {
  static constexpr int E = D >= 32 ? D / 32 : 1;  // head dim 16: half of the lanes have none
  float top = -INFINITY, sum = 0.f, acc[E] = {};
  template <class Part>
  __device__ __forceinline__ void run(int n, int cols, int col, int lane, Part part) {
    const int d = min(lane * E, D - E);
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      float m = -INFINITY, l = 0.f;
      if (i < n) m = part(i)[col], l = part(i)[cols + col];
      float t = m;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(kFull, t, o));
      t = fmaxf(t, top);
      const float ref = t == -INFINITY ? 0.f : t, f = ex2(m - ref), old = ex2(top - ref);
      l = i < n ? l * f : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(kFull, l, o);
      sum = sum * old + l;
#pragma unroll
      for (int k = 0; k < E; ++k) acc[k] *= old;
      top = t;
      const int left = min(32, n - i0);
#pragma unroll 4
      for (int k = 0; k < left; ++k) {
        const float* src = part(i0 + k) + part_head(cols) + col * D + d;
        const float by = __shfl_sync(kFull, f, k);
        if constexpr (E == 4) {
          const float4 v = *reinterpret_cast<const float4*>(src);
          acc[0] = fmaf(v.x, by, acc[0]), acc[1] = fmaf(v.y, by, acc[1]);
          acc[2] = fmaf(v.z, by, acc[2]), acc[3] = fmaf(v.w, by, acc[3]);
        } else if constexpr (E == 2) {
          const float2 v = *reinterpret_cast<const float2*>(src);
          acc[0] = fmaf(v.x, by, acc[0]), acc[1] = fmaf(v.y, by, acc[1]);
        } else {
          acc[0] = fmaf(*src, by, acc[0]);
        }
      }
    }
  }
  template <bool F16>
  __device__ __forceinline__ void finish(const DecodeArgs& a, long row, int lane) const {
    uint16_t* dst = static_cast<uint16_t*>(a.out) + row * D + lane * E;
    const float inv = rcp(sum);
    if (lane * E < D) {
      if constexpr (E == 4)
        *reinterpret_cast<uint2*>(dst) =
            make_uint2(pack16<F16>(acc[0] * inv, acc[1] * inv), pack16<F16>(acc[2] * inv, acc[3] * inv));
      else if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = pack16<F16>(acc[0] * inv, acc[1] * inv);
      else *dst = from_f32<F16>(acc[0] * inv);
    }
    if (lane == 0) a.lse[row] = (top + lg2(sum)) * kLn2;
  }
  __device__ __forceinline__ void keep(float* dst, int cols, int col, int lane) const {
    if (lane * E < D)
#pragma unroll
      for (int k = 0; k < E; ++k) dst[part_head(cols) + col * D + lane * E + k] = acc[k];
    if (lane == 0) dst[col] = top, dst[cols + col] = sum;
  }
};

// An equal share of `total` for each of n: that of number c begins here.
__device__ __forceinline__ int share(int total, int c, int n) {
  const int each = total / n, more = total - each * n;
  return c * each + min(c, more);
}

// How copies bring tiles: `packed` as in Place; `joint`: a page holds whole tiles, and one copy brings K of one.
struct Boxes {
  bool packed, joint;
};

// Work is a list of tiles of 16 * KT tokens, ordered by sequence, then unit, then token. Every CTA takes an equal run of it
// and every warp an equal run of the CTA's, whatever the lengths are: a unit may lie inside a warp's run, or be
// spread over warps and CTAs. A warp walks its run with a running maximum and sum per query head; what it has of a
// unit that is not wholly its own goes to shared memory, the CTA joins these, and what the CTA has of a unit
// that is not wholly its own goes to a.part, for join_kernel. Sums have a fixed order. Without a.record CTAs take whole
// units, and nothing is left to join.
template <int D, bool F16, bool CODES>
__global__ void __launch_bounds__((Shape<D, CODES>::kThreads), (Shape<D, CODES>::kCtas))
    decode_attn_kernel(const DecodeArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const int stages, const Boxes boxes) {
  using S = Shape<D, CODES>;
  constexpr int KT = S::KT, kThreads = S::kThreads, kEach = kWarps / S::kMovers;
  // Codes of K are widened to fp16, in fewer instructions than to bf16, and bf16 q is scaled by a power of two for it. Codes of V
  // are widened to bf16: a weight takes the scale of its head of a token with it, and these may lie further apart than fp16 goes.
  constexpr bool V16 = F16 && !CODES;
  // The scores' reference is raised only where one passes it by more than 2^kSlack: that saves the maxima across lanes of most
  // tiles (when it was brought in: 1 x 100003 73 us instead of 75, 256 x 1024 in codes 92.7 instead of 94.7, 64 x 8192
  // 180.6 instead of 181.2). fp16 weights are lifted by 2^kLift, which keeps them below 2^15 and what is 2^-31 of the largest;
  // bf16 ones are lowered to 1 at most, so that no sum of V is out of range that would not be with the largest as reference.
  constexpr float kSlack = 8.f, kLift = V16 ? 7.f : -kSlack;
  extern __shared__ uint8_t smem_raw[];  // the warps' rings, exponent bytes, a part for each warp
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int prefix[kMaxSeqs + 1], lens[kMaxSeqs];  // tiles of a unit before each sequence; their lengths
  __shared__ int sums[kWarps + S::kMovers];
  __shared__ int seg_unit[2 * kWarps], seg_first[2 * kWarps], seg_last[2 * kWarps], seg_tiles[2 * kWarps];
  __shared__ uint64_t full[kWarps][kMaxStages], empty[kWarps][kMaxStages];
  __shared__ uint32_t lost[kWarps][kMaxStages];  // groups of a stage's tile whose page is none

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x < 2) tma_prefetch_desc(threadIdx.x ? &v_map : &k_map);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const KvPool& p = a.pool;
  const Heads n(a);

  {  // tiles of a unit before each sequence
    const int per = (a.seqs + kWarps * 32 - 1) / (kWarps * 32), b0 = min(tid * per, a.seqs);  // at most 4
    int sum = 0;
    for (int b = b0; b < min(b0 + per, a.seqs); ++b) {
      const int len = a.lengths[b];
      lens[b] = len;
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
    if (tid < 2 * kWarps) seg_unit[tid] = -1;
    if (warp < kWarps && lane < stages) {
      mbar_init(&full[warp][lane], CODES ? 2 : 1);
      mbar_init(&empty[warp][lane], 1);
    }
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
    const bool bad = lens[b] != 0;
    if (bad && tid == 0) record_error(a.status, kBadArg, kSite);
    for (int i = tid; i < a.heads_q * D; i += kThreads)
      static_cast<uint16_t*>(a.out)[static_cast<long>(b) * a.heads_q * D + i] = from_f32<F16>(bad ? quiet_nan() : 0.f);
    for (int i = tid; i < a.heads_q; i += kThreads)
      a.lse[static_cast<long>(b) * a.heads_q + i] = bad ? quiet_nan() : -INFINITY;
  }

  const int total = prefix[a.seqs] * n.units;
  int c0, c1, busy = gridDim.x;  // this CTA's run
  if (a.record == nullptr) {
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
    const int w = i >> 1, behind = kWarps * stages * (S::kStage + S::kExps);  // behind the rings and exponent bytes
    return reinterpret_cast<float*>(smem + (i & 1 ? w * stages * S::kStage : behind + w * (part_head(n.cols) + n.cols * D) * 4));
  };
  // A unit on the way through a run.
  struct Walk {
    int b, u, h, chunk, tile, tiles;
  };
  const auto walk_from = [&](int at) {
    Walk w{};  // the last sequence whose tiles begin at or before `at`
    for (int hi = a.seqs; hi - w.b > 1;) {
      const int mid = (w.b + hi) >> 1;
      if (prefix[mid] * n.units <= at) w.b = mid;
      else hi = mid;
    }
    w.tiles = prefix[w.b + 1] - prefix[w.b];
    const int in_seq = at - prefix[w.b] * n.units;
    w.u = in_seq / w.tiles;
    w.tile = in_seq - w.u * w.tiles;
    w.h = w.u / n.chunks;
    w.chunk = w.u - w.h * n.chunks;
    return w;
  };
  const auto next_unit = [&](Walk& w) {
    w.tile = 0;
    ++w.u;
    if (++w.chunk == n.chunks) w.chunk = 0, ++w.h;
    if (w.u == n.units) {
      w.u = w.h = 0;
      do ++w.b;
      while (prefix[w.b + 1] == prefix[w.b]);
      w.tiles = prefix[w.b + 1] - prefix[w.b];
    }
  };

  uint8_t* const exps_at = smem + kWarps * stages * S::kStage;
  if (warp >= kWarps) {
    // Lane i of the first such warp keeps the ring of warp i filled, of the next one that of warp kEach + i: the copies of a tile
    // are issued when its stage has been read, in the order of the warp's run and across its units. The places of the next tile
    // are on their way meanwhile.
    const int run = (warp - kWarps) * kEach + min(lane, kEach - 1), w0 = c0 + share(c1 - c0, run, kWarps);
    int left = lane < kEach ? c0 + share(c1 - c0, run + 1, kWarps) - w0 : 0;
    Walk nx{};
    int len = 0, index = 0, slot = 0, page[KT];  // index, slot: of the tile's first token in the row of the table and in its page
    const auto look_ahead = [&]() {
      int i = index, s = slot;
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        page[j] = -1;
        if (nx.tile * S::kTokens + 16 * j < len) page[j] = __ldg(a.table + nx.b * a.tt + i);
        if (boxes.joint) break;
        s += 16;
        if (s == p.size) s = 0, ++i;
      }
    };
    const auto enter = [&]() {
      len = lens[nx.b];
      index = nx.tile * S::kTokens / p.size;
      slot = nx.tile * S::kTokens - index * p.size;
    };
    if (left > 0) {
      nx = walk_from(w0);
      enter();
      look_ahead();
    }
    int stage = 0;
    uint32_t parity = 1;
    uint64_t since = globaltimer_ns();
    for (uint32_t turn = 0; __any_sync(kFull, left > 0); ++turn) {
      const bool ready = left > 0 && mbar_test(&empty[run][stage], parity);
      if (ready) {
        const uint32_t dst = smem_u32(smem) + (run * stages + stage) * S::kStage, bar = smem_u32(&full[run][stage]);
        const int behind = (len + 15) / 16 - nx.tile * KT;  // groups of the sequence from here on
        uint32_t none = 0;
        int i = index, s = slot;
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const int pg = boxes.joint ? page[0] : page[j];
          const bool bad = pg < 0 || pg >= p.pages;
          if (j < behind && bad) none |= 1u << j;
        }
        if (none) record_error(a.status, kBadArg, kSite);
        lost[run][stage] = none;
        mbar_arrive_expect_tx(&full[run][stage], boxes.joint ? S::kStage : min(KT, behind) * 2 * S::kGroup);
        if (boxes.joint) {
          const int row = boxes.packed && S::kRow < 128 ? s * S::kRow / 128 : s;
#pragma unroll
          for (int x = 0; x < S::kBoxes; ++x) {
            tma_load_4d(dst + x * 2048, &k_map, bar, x * (128 / S::kSize), row, nx.h, page[0]);
            tma_load_4d(dst + S::kKv + x * 2048, &v_map, bar, x * (128 / S::kSize), row, nx.h, page[0]);
          }
        }
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          if (j >= behind) break;
          const int pg = boxes.joint ? page[0] : page[j];
          if (!boxes.joint) {
            const int row = boxes.packed && S::kRow < 128 ? s * S::kRow / 128 : s;
#pragma unroll
            for (int x = 0; x < S::kBoxes; ++x) {
              tma_load_4d(dst + j * S::kGroup + x * 2048, &k_map, bar, x * (128 / S::kSize), row, nx.h, pg);
              tma_load_4d(dst + S::kKv + j * S::kGroup + x * 2048, &v_map, bar, x * (128 / S::kSize), row, nx.h, pg);
            }
          }
          if (CODES && !(none >> j & 1)) {
            const uint32_t e = smem_u32(exps_at) + (run * stages + stage) * S::kExps + j * 16;
            copy_16(e, p.ke + pg * p.kep + nx.h * p.keh + s);
            copy_16(e + S::kTokens, p.ve + pg * p.vep + nx.h * p.veh + s);
          }
          s += 16;
          if (s == p.size) s = 0, ++i;
        }
        if constexpr (CODES) asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
        if (++stage == stages) stage = 0, parity ^= 1;
        if (--left > 0) {
          if (++nx.tile == nx.tiles) {
            next_unit(nx);
            enter();
          } else {
            index = i, slot = s;
          }
          look_ahead();
        }
      }
      if (__any_sync(kFull, ready)) {
        turn = ~0u;
      } else if (turn % 1024 == 0) {  // nothing to do: give up where that lasts
        if (turn == 0) since = globaltimer_ns();
        else if (globaltimer_ns() - since > HB_WAIT_TIMEOUT_NS) {
          record_error(a.status, kMbarTimeout, kSite);
          break;
        }
      }
    }
    __syncwarp();
  }
  const int w0 = warp < kWarps ? c0 + share(c1 - c0, warp, kWarps) : 0;
  const int w1 = warp < kWarps ? c0 + share(c1 - c0, warp + 1, kWarps) : 0;
  uint8_t* const ring = smem + warp * stages * S::kStage;
  uint8_t* const exps = exps_at + warp * stages * S::kExps;
  const uint32_t ring0 = smem_u32(ring);
  Walk w{};
  if (w0 < w1) w = walk_from(w0);
  int stage = 0;
  uint32_t parity = 0;
  bool broken = false;  // a copy that did not arrive in time
  const Place<S::kRow> k_row((lane & 7) + (lane & 8), lane >> 4, boxes.packed);
  const Place<S::kRow> v_row(CODES ? (lane & 7) + (lane & 8) : (lane & 7) + (lane >> 4) * 8,
                             CODES ? lane >> 4 : lane >> 3 & 1, boxes.packed);

  // q of query head g of a unit, in the order of K's channels: index 2t of 16 is channel 2t (codes: 4t), 2t + 8 is 2t + 8
  // (codes: 4t + 2). That of the next unit is on its way during the present one.
  uint32_t q[S::kSteps][2], q_ahead[S::kSteps][2];
  const auto load_q = [&](const Walk& f) {
    const int head = f.chunk * kCols + g;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + f.b * a.qt + (f.h * n.G + head) * a.qh + (CODES ? 4 * t : 2 * t);
#pragma unroll
    for (int x = 0; x < S::kSteps; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint16_t* s = src + 16 * x + (CODES ? 2 : 8) * i;
        q_ahead[x][i] = 0;
        if (head < n.G) {
          if (a.q_vec) q_ahead[x][i] = *reinterpret_cast<const uint32_t*>(s);
          else q_ahead[x][i] = s[0] | (static_cast<uint32_t>(s[1]) << 16);
        }
      }
  };
  if (w0 < w1) load_q(w);

  for (int at = w0; at < w1;) {
    const int first = w.tile, last = min(w.tiles, first + (w1 - at)), b = w.b, u = w.u, tiles = w.tiles;
    const int q0 = w.h * n.G + w.chunk * kCols, nq = min(kCols, n.G - w.chunk * kCols);
    const int len = lens[b];
#pragma unroll
    for (int x = 0; x < S::kSteps; ++x) q[x][0] = q_ahead[x][0], q[x][1] = q_ahead[x][1];
    if (at + last - first < w1) {
      next_unit(w);
      load_q(w);
    }
    const float unit = a.scale * kLog2e;
    float q_unit[2] = {unit, unit};  // of columns 2t and 2t + 1
    if constexpr (CODES && !F16) {
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
    float m[2] = {-INFINITY, -INFINITY};  // reference of the scores of columns 2t and 2t + 1, in powers of 2
    float l[2] = {0.f, 0.f};  // sum of the weights of this lane's rows
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
          for (int x = 0; x < S::kSteps; x += 2) {  // a load is 2 chunks of 16 channels (head dim 16: one, and what lies behind)
            uint32_t r[4], y[4][2];
            load_matrices(r, k0 + k_row.chunk(x, j));
#pragma unroll
            for (int i = 0; i < 4; ++i) widen(r[i], y[i]);
            mma<true>(s[j], y[0][0], y[1][0], y[0][1], y[1][1], q[x][0], q[x][1]);
            if constexpr (S::kSteps > 1) mma<true>(s[j], y[2][0], y[3][0], y[2][1], y[3][1], q[x + 1][0], q[x + 1][1]);
          }
          // lane i has the exponent byte of K of token i of the 16, lane 16 + i that of V; behind the length: 0
          const int i = lane & 15;
          uint32_t byte = exps[stage * S::kExps + (lane >> 4) * S::kTokens + j * 16 + i];
          if (tile * S::kTokens + j * 16 + i >= len) byte = 0;
          const float scale = act8_scale(byte);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float by = __shfl_sync(kFull, scale, g + 8 * r);
            vs[j][r] = __shfl_sync(kFull, scale, 16 + g + 8 * r);
            s[j][2 * r] *= by * q_unit[0], s[j][2 * r + 1] *= by * q_unit[1];
          }
        } else {
#pragma unroll
          for (int x = 0; x < S::kSteps; ++x) {
            uint32_t r[4];
            load_matrices(r, k0 + k_row.chunk(2 * x, j));
            mma<F16>(s[j], r[0], r[1], r[2], r[3], q[x][0], q[x][1]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j][i] *= unit;
        }
      }
      const uint32_t none = lost[warp][stage];
      if (none | (tile + 1 == tiles)) {  // pages that are none, or the sequence's last tile
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const int token = tile * S::kTokens + j * 16;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (none >> j & 1) s[j][i] = quiet_nan();
            if (token + g + 8 * (i >> 1) >= len) s[j][i] = -INFINITY;
          }
          // V behind the length, whatever it is, becomes 0 (codes are numbers whatever they are)
          const int r = lane & 15;
          if (!CODES && token + r >= len) {
            const uint32_t at0 = stage * S::kStage + S::kKv;
            const Place<S::kRow> place(r, 0, boxes.packed);
#pragma unroll
            for (int x = 0; x < S::kRow / 16; ++x)
              if (x % 2 == lane >> 4) *reinterpret_cast<uint4*>(ring + at0 + place.chunk(x, j)) = make_uint4(0, 0, 0, 0);
          }
        }
        if constexpr (!CODES) {
          fence_proxy_async_smem();  // before a copy takes the stage again
          __syncwarp();
        }
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i & 1] = fmaxf(top[i & 1], s[j][i]);
      if (__any_sync(kFull, top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          top[x] = fmaxf(top[x], m[x]);
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) top[x] = fmaxf(top[x], __shfl_xor_sync(kFull, top[x], i));
          const float f = top[x] == m[x] ? 1.f : ex2(m[x] - top[x]);
          m[x] = top[x];
          l[x] *= f;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) o[i][x] *= f, o[i][2 + x] *= f;
        }
      }
      float ref[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) ref[x] = (m[x] == -INFINITY ? 0.f : m[x]) - kLift;
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        // weights, as the sum of two 16-bit numbers: what one of 8 or 11 bits leaves would show in the output
        float wt[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          wt[i] = ex2(s[j][i] - ref[i & 1]);
          l[i & 1] += wt[i];
          if constexpr (CODES) wt[i] *= vs[j][i >> 1];
        }
        uint32_t hi[2], rest[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t x = pack16<V16>(wt[2 * r], wt[2 * r + 1]);
          rest[r] = transpose8(pack16<V16>(wt[2 * r] - lo16<V16>(x), wt[2 * r + 1] - hi16<V16>(x)));
          hi[r] = transpose8(x);
        }
        // output: rows are channels
        if constexpr (CODES) {
#pragma unroll
          for (int i = 0; i < D / 16; i += 2) {
            uint32_t r[4];
            load_matrices_t(r, v0 + v_row.chunk(i, j));
#pragma unroll
            for (int x = 0; x < 2; ++x) {  // a word: channels 2g and 2g + 1 of two tokens
              if (i + x >= D / 16) break;
              const uint32_t y[4] = {widen_bf16(r[2 * x]), widen_bf16(r[2 * x] >> 8), widen_bf16(r[2 * x + 1]),
                                     widen_bf16(r[2 * x + 1] >> 8)};
              mma<V16>(o[i + x], y[0], y[1], y[2], y[3], hi[0], hi[1]);
              mma<V16>(o[i + x], y[0], y[1], y[2], y[3], rest[0], rest[1]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t r[4];
            load_matrices_t(r, v0 + v_row.chunk(2 * i, j));
            mma<V16>(o[i], r[0], r[1], r[2], r[3], hi[0], hi[1]);
            mma<V16>(o[i], r[0], r[1], r[2], r[3], rest[0], rest[1]);
          }
        }
      }
      __syncwarp();  // the stage has been read
      if (lane == 0) mbar_arrive(&empty[warp][stage]);
      if (++stage == stages) stage = 0, parity ^= 1;
    }
    if (broken) break;
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[0] += __shfl_xor_sync(kFull, l[0], x);
      l[1] += __shfl_xor_sync(kFull, l[1], x);
    }
    m[0] -= kLift, m[1] -= kLift;  // what the sums' weights are relative to
    if (first == 0 && last == tiles) {
      const float inv[2] = {rcp(l[0]), rcp(l[1])};
      const long row = static_cast<long>(b) * a.heads_q + q0;
      uint16_t* dst = static_cast<uint16_t*>(a.out) + (row + g) * D + (CODES ? 4 * t : 2 * t);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {  // transposed, a lane has neighbouring channels of head g
        const uint32_t x = transpose8(pack16<F16>(o[i][0] * inv[0], o[i][1] * inv[1]));
        const uint32_t y = transpose8(pack16<F16>(o[i][2] * inv[0], o[i][3] * inv[1]));
        if (g < nq) {
          if constexpr (CODES) {
            *reinterpret_cast<uint2*>(dst + 16 * i) = make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
          } else {
            *reinterpret_cast<uint32_t*>(dst + 16 * i) = x;
            *reinterpret_cast<uint32_t*>(dst + 16 * i + 8) = y;
          }
        }
      }
      if (g == 0) {
        if (2 * t < nq) a.lse[row + 2 * t] = (m[0] + lg2(l[0])) * kLn2;
        if (2 * t + 1 < nq) a.lse[row + 2 * t + 1] = (m[1] + lg2(l[1])) * kLn2;
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
          float* d = dst + part_head(n.cols) + col * D + (CODES ? 2 * g : g);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) d[16 * i] = o[i][x], d[16 * i + (CODES ? 1 : 8)] = o[i][2 + x];
        }
      }
    }
    at += last - first;
  }
  if (broken && warp < kWarps) {  // wait (with a limit) for what is still on its way, which must not outlive the CTA
    for (int s = 0; s < stages; ++s) {
      mbar_wait(&full[warp][stage], parity, a.status, kSite);
      if (++stage == stages) stage = 0, parity ^= 1;
    }
  }
  if (tid < 2 && a.record != nullptr) a.record[2 * blockIdx.x + tid] = make_int2(-1, 0);
  __syncthreads();

  // Parts of units that warps share. Lane i looks at segment i; neighbouring ones of one unit are a set: the first of them,
  // and those with which the runs of the warps behind it begin. The warps take the columns of all sets in turn.
  const int unit = lane < 2 * kWarps ? seg_unit[lane] : -1;
  const uint32_t used = __ballot_sync(kFull, unit >= 0), before = used & ((1u << lane) - 1);
  const int prev = __shfl_sync(kFull, unit, before ? 31 - __clz(before) : 0);
  uint32_t starts = __ballot_sync(kFull, unit >= 0 && (before == 0 || prev != unit));
  for (int col = warp; starts; starts &= starts - 1) {
    const int i0 = __ffs(starts) - 1;
    const uint32_t rest = starts & (starts - 1);
    const uint32_t members = used & ~((1u << i0) - 1) & (rest ? (1u << (__ffs(rest) - 1)) - 1 : kFull);
    const int id = seg_unit[i0], b = id / n.units, first = seg_first[i0], end = 31 - __clz(members);
    const Columns c(n, id - b * n.units);
    const bool whole = first == 0 && seg_last[end] == seg_tiles[i0];
    const int slot = 2 * blockIdx.x + (first == 0 ? 1 : 0);
    for (; col < c.nq; col += kWarps + S::kMovers) {
      if (col == 0 && lane == 0 && !whole) {
        // how many CTAs behind this one have a part of a unit that begins here
        const int left = seg_tiles[i0] - seg_last[end];
        int last_cta = blockIdx.x;
        if (left > 0) {
          const int tile = c1 + left - 1, each = total / busy, more = total - each * busy;  // who has this one
          last_cta = tile < more * (each + 1) ? tile / (each + 1) : (tile - more) / each;
        }
        a.record[slot] = make_int2(id, last_cta - blockIdx.x);
      }
      Join<D> j;
      j.run(__popc(members), n.cols, col, lane, [&](int i) { return part(i == 0 ? i0 : (i0 | 1) - 1 + 2 * i); });
      if (whole) j.template finish<F16>(a, static_cast<long>(b) * a.heads_q + c.q0 + col, lane);
      else j.keep(part_of<D>(a.part, slot, n.cols), n.cols, col, lane);
    }
    col -= c.nq;
  }
}

// Loads at this place in the program, not where the values are used.
template <int N>
__device__ __forceinline__ void ask(const float* at, float (&v)[N]) {
  if constexpr (N == 4)
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "l"(at) : "memory");
  else if constexpr (N == 2)
    asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "l"(at) : "memory");
  else
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v[0]) : "l"(at) : "memory");
}

// Joins the parts of the units that CTAs share. CTA (c, y): column y of the unit that begins in CTA c of the kernel above and does
// not end there, if any; its other parts are the first ones of the CTAs behind. WARPS > 1, for units of many parts: the
// warps take equal runs of them first.
//
// Most units have two parts, whose places are known without the record. So a warp asks for both along with it: one
// round trip to memory instead of three (61 x up to 1024 tokens 26.7 -> 25.7 us).
template <int D, bool F16, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) join_kernel(const DecodeArgs a) {
  const Heads n(a);
  const int col = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Join<D> j;
  constexpr int E = Join<D>::E;
  float m[2][1], l[2][1], v[2][E];
  if constexpr (WARPS == 1) {
    const int next = min(blockIdx.x + 1, gridDim.x - 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float* src = part_of<D>(a.part, i == 0 ? 2 * static_cast<int>(blockIdx.x) + 1 : 2 * next, n.cols);
      ask(src + col, m[i]), ask(src + n.cols + col, l[i]);
      ask(src + part_head(n.cols) + col * D + min(lane * E, D - E), v[i]);
    }
  }
  const int2 rec = a.record[2 * blockIdx.x + 1];
  if (rec.x < 0) return;
  const int b = rec.x / n.units, parts = rec.y + 1;
  const Columns c(n, rec.x - b * n.units);
  if (col >= c.nq) return;
  const int i0 = share(parts, warp, WARPS), i1 = share(parts, warp + 1, WARPS);
  if (WARPS == 1 && parts == 2) {
    j.top = fmaxf(m[0][0], m[1][0]);
    const float ref = j.top == -INFINITY ? 0.f : j.top, f0 = ex2(m[0][0] - ref), f1 = ex2(m[1][0] - ref);
    j.sum = l[0][0] * f0 + l[1][0] * f1;
#pragma unroll
    for (int k = 0; k < E; ++k) j.acc[k] = fmaf(v[0][k], f0, v[1][k] * f1);
    j.template finish<F16>(a, static_cast<long>(b) * a.heads_q + c.q0 + col, lane);
    return;
  }
  j.run(i1 - i0, n.cols, col, lane, [&](int i) {
    return part_of<D>(a.part, 2 * (static_cast<int>(blockIdx.x) + i0 + i) + (i0 + i == 0 ? 1 : 0), n.cols);
  });
  if constexpr (WARPS > 1) {
    __shared__ __align__(16) float own[WARPS * (part_head(1) + D)];
    j.keep(part_of<D>(own, warp, 1), 1, 0, lane);
    __syncthreads();
    if (warp > 0) return;
    j = Join<D>();
    j.run(WARPS, 1, 0, lane, [&](int i) { return part_of<D>(own, i, 1); });
  }
  j.template finish<F16>(a, static_cast<long>(b) * a.heads_q + c.q0 + col, lane);
}

// The cache as a tensor of (channel, slot, head, page) or, packed, of (byte of 128, row of 128 bytes, head, page).
template <int D, bool CODES>
CUtensorMap cache_map(const KvPool& p, const void* base, long page, long head, long slot, Boxes boxes) {
  using S = Shape<D, CODES>;
  const uint64_t es = S::kSize;
  const bool join = boxes.packed && S::kRow < 128;
  const uint32_t tokens = boxes.joint ? S::kTokens : 16;
  const uint64_t wide = join ? 128 / es : D, rows = join ? static_cast<uint64_t>(p.size) * S::kRow / 128 : p.size;
  const uint64_t sizes[4] = {wide, rows, static_cast<uint64_t>(p.heads), static_cast<uint64_t>(p.pages)};
  // (the stride of a dimension of one element is whatever it was given, and of no use)
  const uint64_t strides[3] = {join ? 128 : slot * es, p.heads > 1 ? head * es : 16, p.pages > 1 ? page * es : 16};
  const int line = join || S::kRow >= 128 ? 128 : S::kRow;
  const uint32_t box[4] = {line / static_cast<uint32_t>(es), join ? tokens * S::kRow / 128 : tokens, 1, 1};
  return make_tmap(CODES ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, sizes, strides, box,
                   line == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                   : line == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                   : line == 32 ? CU_TENSOR_MAP_SWIZZLE_32B
                                : CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int D, bool F16, bool CODES>
void launch(const DecodeArgs& a, int ctas, cudaStream_t s) {
  using S = Shape<D, CODES>;
  const auto parts_of = [](int cols) constexpr { return kWarps * (part_head(cols) + cols * D) * 4 + 1024; };
  constexpr int kRing = kWarps * (S::kStage + S::kExps);  // a stage of every warp
  const int parts = parts_of(std::min(a.heads_q / a.pool.heads, kCols));
  // 227 KB of an SM, less 1 KB a CTA and what the kernel declares
  constexpr int kRoom = (227 * 1024) / S::kCtas - 1024 - 9 * 1024;
  constexpr int kLeast = std::min(kMaxStages, (kRoom - parts_of(kCols)) / kRing);  // stages, with 8 query heads a K/V head
  static_assert(kLeast >= 1 && kLeast * S::kStage >= (part_head(kCols) + kCols * D) * 4, "a stage and a part have to fit");
  const int stages = std::min(kMaxStages, (kRoom - parts) / kRing);
  const size_t smem = static_cast<size_t>(stages) * kRing + parts;
  const auto kernel = decode_attn_kernel<D, F16, CODES>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may use that much shared memory
  const int dev = current_device();
  if (!(ready.load() >> dev & 1)) {
    HB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRoom));
    ready.fetch_or(1ull << dev);
  }
  const KvPool& p = a.pool;
  const Boxes boxes{p.ks == D && p.vs == D, p.size % S::kTokens == 0};
  CUtensorMap k_map{}, v_map{};  // a cache of no pages is not read
  if (p.pages > 0) {
    k_map = cache_map<D, CODES>(p, p.k, p.kp, p.kh, p.ks, boxes);
    v_map = cache_map<D, CODES>(p, p.v, p.vp, p.vh, p.vs, boxes);
  }
  kernel<<<ctas, S::kThreads, smem, s>>>(a, k_map, v_map, stages, boxes);
  HB_CUDA_CHECK(cudaGetLastError());
  if (a.record == nullptr) return;
  // Where a unit is spread over more than 16 CTAs on average, 8 warps join its parts (one sequence of 131072 tokens and one K/V
  // head: 24 us in all instead of 34); elsewhere one does, and a larger block would only start later (1 x 1024 tokens of 12 heads:
  // 10.8 us instead of 8.5).
  const int units = a.seqs * p.heads * ((a.heads_q / p.heads + kCols - 1) / kCols);
  const bool spread = ctas / 16 > units;
  cudaLaunchConfig_t cfg{};  // launched while the kernel above runs: it waits for its end by itself
  cfg.gridDim = dim3(ctas, std::min(a.heads_q / p.heads, kCols));
  cfg.blockDim = dim3(spread ? 8 * 32 : 32);
  cfg.stream = s;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = early;
  cfg.numAttrs = 1;
  HB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, spread ? join_kernel<D, F16, 8> : join_kernel<D, F16, 1>, a));
}
template <int D>
void launch_dim(const DecodeArgs& a, int ctas, cudaStream_t s) {
  if (a.pool.type == kKvCodes) a.f16 ? launch<D, true, true>(a, ctas, s) : launch<D, false, true>(a, ctas, s);
  else a.f16 ? launch<D, true, false>(a, ctas, s) : launch<D, false, false>(a, ctas, s);
}

// Tables of at most this many tokens, and of at most three times as many for each CTA that fits: CTAs take whole units, which
// saves the second kernel. When this was set, 12 heads of 64, bf16: 8 sequences of up to 256 tokens 6.4 us instead of 8.4,
// 64 of them 12.9 instead of 13.9 (664 tokens a CTA); but 128 of up to 200 19.2 instead of 18.1 (1038), 512 of up to 256 53
// instead of 45; and 8 of up to 512 8.0 instead of 9.4, but 1 of up to 512 8.3 instead of 7.3. (8 heads of 128, 4 query heads
// each, would gain beyond that: 128 of up to 200 19.7 instead of 22.3; 20 heads of 64 in codes would lose, 25 instead of
// 21.) The rule goes by the table's width, as the lengths are on the device: 8 sequences of 57 tokens take 6.0 us with a table of
// 64, 8.4 with one of 1024.
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
  const Fit f = p.dim == 16   ? fit_dim<16>(codes)
                : p.dim == 32 ? fit_dim<32>(codes)
                : p.dim == 64 ? fit_dim<64>(codes)
                              : fit_dim<128>(codes);
  DecodePlan d;
  const long tiles = (longest + f.tokens - 1) / f.tokens, most = (1l << 31) - 1;
  d.seqs = static_cast<int>(std::min<long>(std::min(seqs, kMaxSeqs), most / std::max(1l, units * tiles)));
  if (d.seqs == 0) return d;
  const long all = static_cast<long>(d.seqs) * units, sms = num_sms(current_device());
  const bool whole = longest <= kWholeTokens && all * longest <= 3l * kWholeTokens * f.ctas * sms;
  d.ctas = static_cast<int>(std::max(1l, std::min(f.ctas * sms, whole ? all : (all * tiles + kWarps - 1) / kWarps)));
  d.split = !whole && d.ctas > 1;
  return d;
}

void decode_attention_launch(const DecodeArgs& a, const DecodePlan& d, cudaStream_t s) {
  switch (a.pool.dim) {
    case 16: launch_dim<16>(a, d.ctas, s); break;
    case 32: launch_dim<32>(a, d.ctas, s); break;
    case 64: launch_dim<64>(a, d.ctas, s); break;
    default: launch_dim<128>(a, d.ctas, s); break;
  }
}

}  // namespace hb
