// Post-training losses: target log-probabilities of vocabulary logits, the clipped policy loss with a
// KL term, and the paired log-ratio (preference) loss, each with its gradient.
//
// For a row x of V logits with target t:
//   lse  = log sum_j exp(x_j),  logp = x_t - lse,  d logp / d x_j = [j == t] - exp(x_j - lse)
// Policy loss of a token, with d = logp - old, r = e^d, advantage A, u = ref - logp:
//   l = -min(r A, clip(r) A) + kl (e^u - u - 1)
//   dl / dlogp = (r A <= clip(r) A ? -r A : 0) + kl (1 - e^u)
// Rows whose target is `ignore_index` are not read: their log-probability is 0 and their gradient row zero.
// A target outside [0, V) gives NaN and the bad-argument status, as in the cross-entropy kernels.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "host_utils.h"
#include "post_args.h"

namespace hb {

namespace {

constexpr int kThreadsPerSm = 512;  // of the row kernel: 128 registers each
constexpr int kCtasPerSm = 2;  // where two CTAs' shares fit an SM's shared memory; else one has all the threads
constexpr int kUnroll = 4;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One 16-byte piece of a row: 8 elements of 16 bits, or 4 of 32.
template <int TYPE>
struct Piece {
  static constexpr int kElems = TYPE == kLogitF32 ? 4 : 8;
  static constexpr int kBytes = 16 / kElems;
  static constexpr bool kF16 = TYPE == kLogitF16;
  static constexpr uint32_t kMinusInf = TYPE == kLogitF32 ? 0xFF800000u : kF16 ? 0xFC00u : 0xFF80u;
  // elements at and behind `n` become `bits`
  static __device__ __forceinline__ void fill(uint4& r, int n, uint32_t bits) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == kLogitF32) {
        if (i >= n) w[i] = bits;
      } else {
        if (2 * i >= n) w[i] = bits | (bits << 16);
        else if (2 * i + 1 >= n) w[i] = (w[i] & 0xFFFFu) | (bits << 16);
      }
    }
  }
  static __device__ __forceinline__ void widen(const uint4& r, float (&v)[kElems]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == kLogitF32) {
        v[i] = __uint_as_float(w[i]);
      } else {
        v[2 * i] = lo16<kF16>(w[i]);
        v[2 * i + 1] = hi16<kF16>(w[i]);
      }
    }
  }
  // element e (known at run time) of a piece to element i of a row
  static __device__ __forceinline__ void store_at(const uint4& r, int e, void* base, long i) {
    const int k = TYPE == kLogitF32 ? e : e >> 1;
    const uint32_t w = k == 0 ? r.x : k == 1 ? r.y : k == 2 ? r.z : r.w;
    if constexpr (TYPE == kLogitF32) static_cast<uint32_t*>(base)[i] = w;
    else static_cast<uint16_t*>(base)[i] = static_cast<uint16_t>(e & 1 ? w >> 16 : w);
  }
  static __device__ __forceinline__ uint4 narrow(const float (&v)[kElems]) {
    uint4 r;
    if constexpr (TYPE == kLogitF32) {
      r = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    } else {
      r = make_uint4(pack16<kF16>(v[0], v[1]), pack16<kF16>(v[2], v[3]), pack16<kF16>(v[4], v[5]),
                     pack16<kF16>(v[6], v[7]));
    }
    return r;
  }
};

template <int TYPE>
__device__ __forceinline__ float load1(const void* base, long i) {
  if constexpr (TYPE == kLogitF32) return static_cast<const float*>(base)[i];
  else return to_f32<TYPE == kLogitF16>(static_cast<const uint16_t*>(base)[i]);
}
template <int TYPE>
__device__ __forceinline__ void store1(void* base, long i, float v) {
  if constexpr (TYPE == kLogitF32) static_cast<float*>(base)[i] = v;
  else static_cast<uint16_t*>(base)[i] = from_f32<TYPE == kLogitF16>(v);
}

// Asynchronous copy of one piece; the bytes behind `bytes` become 0.
__device__ __forceinline__ void copy_piece(uint32_t smem, const void* gmem, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_piece(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ uint4 read_piece(uint32_t smem) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(smem)
               : "memory");
  return r;
}
// Waits for all of this thread's copies.
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Running sum of exp(x - m) under the largest value so far; nothing, or only -inf, is s = 0 with any m; NaN and
// +inf make s NaN. x - m is taken before the factor log2 e, which alone would overflow for masks of the
// type's lowest value.
struct Sum {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ void add(float v) {
    if (v > m) {
      if (s != 0.f) s *= ex2((m - v) * kLog2e);
      m = v;
    }
    if (v != -INFINITY) s += ex2((v - m) * kLog2e);
  }
};

// Joins the sums of 2^k neighbouring lanes (k = log2 LANES): afterwards every lane holds the joint (m, s).
template <int LANES>
__device__ __forceinline__ void join_lanes(float& m, float& s) {
  float top = s == 0.f ? -INFINITY : m;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  s = s == 0.f ? 0.f : s * ex2((m - top) * kLog2e);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  m = top;
}

// What one row adds to the loss and its statistics, and the factor of its gradient.
struct RowTerm {
  float coef, loss, kl, clipped;
};
__device__ __forceinline__ RowTerm policy_term(const PolicyTerms& p, float logp, float old, float adv, float ref,
                                               float w) {
  RowTerm t{0.f, 0.f, 0.f, 0.f};
  const float r = expf(logp - old);
  const float c = fminf(fmaxf(r, p.clip_lo), p.clip_hi);
  // A ratio of infinity has overflowed 32 bits (log-ratios from 89) and stands for a finite one: an advantage, weight or
  // KL factor of 0 takes it out. NaN stays: nothing turns a NaN log-probability into a number.
  const float free = adv == 0.f && r == INFINITY ? 0.f : r * adv;
  const bool clipped = c * adv < free;  // false for a NaN ratio, which so reaches the loss and the gradient
  t.loss = clipped ? -c * adv : -free;
  t.coef = clipped ? 0.f : -free;
  t.clipped = clipped ? w : 0.f;
  if (p.ref_logp) {
    const float u = ref - logp;
    const float e = expm1f(u);
    t.kl = e - u;
    if (p.kl_coef != 0.f) {
      t.loss = fmaf(p.kl_coef, t.kl, t.loss);
      t.coef = fmaf(-p.kl_coef, e, t.coef);
    }
  }
  const auto weigh = [w](float v) { return w == 0.f && fabsf(v) == INFINITY ? 0.f : w * v; };
  t.loss = weigh(t.loss);
  t.kl = weigh(t.kl);
  t.coef = weigh(t.coef);
  return t;
}

enum Mode : int { kLogp = 0, kUnit = 1, kPolicy = 2 };

// How the rows are dealt out: clusters of `split` CTAs, each CTA holding `pieces` 16-byte pieces of a row.
struct Deal {
  int split, pieces, clusters, threads;
  int window, list;  // rows scanned at a time, and the entries of the list of a cluster's rows among them
  bool aligned;    // every row of the logits starts on a 16-byte boundary
  bool vec_store;  // rows of grad start at the same offset from a 16-byte boundary as those of the logits
};

// Row kernel. Clusters of `split` CTAs deal the counted rows, and apart from them the ignored ones, among themselves in
// turn (every CTA scans the targets and lists its own: equal work wherever the ignored rows are). CTA c holds pieces
// [c pieces, (c + 1) pieces) of the row in shared memory. Every thread copies, reads and refills its own 16-byte
// slots (asynchronous copies), so the copies need no barrier, and the next row's are issued slot by slot as the current
// row's gradient leaves (without a gradient: as its pieces are read), so they arrive during this row's arithmetic and
// that of the SM's other CTA.
//   pass 1: S = sum_j exp(x_j - x_t). The target's own logit is the reference of every
//          sum: its term is exactly 1, so S >= 1 cannot vanish, no running maximum is needed, sums of threads, CTAs
//          (one barrier) and the cluster (one exchange through shared memory) just add, and logp = -log S. Rows
//          where S passes 2^120 (a target more than 83 below the largest logit, or at -inf; NaN) are summed again
//          under a maximum.
//   pass 2 (gradient): coef ([j == t] - exp(x_j - x_t) / S) from the slots, in 16-byte pieces.
// The difference x_j - x_t is taken before the factor log2 e: it is exact or nearly so wherever the term matters,
// also for logits far from 0, and finite for masks of the type's lowest value.
// So a row crosses DRAM once each way. Rows may start at any element: the columns before the first 16-byte
// boundary (`head`, fewer than one piece) are read by single threads of the first CTA.
// Measured: 8192 x 50257 bf16 with a quarter of the rows ignored, 255 to 275 us by the run: 1.44 GB, 5.2 to 5.6 TB/s (a
// copy reaches 6.4); with none ignored 305 us, 5.4 TB/s; without a gradient 113 and 143 us (5.5, 5.8 TB/s). The
// arithmetic (8 instructions an element and pass) fills 56% of the issue slots and 62% of the transcendental unit. More
// warps, copies waited for in two or four groups and packed arithmetic do not change the time; the two CTAs of an SM
// overlap their phases.
template <int TYPE, int MODE, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreadsPerSm / kThreads)
    logit_rows_kernel(const LogitRows a, const PolicyTerms p, const Deal d, double* __restrict__ part) {
  using P = Piece<TYPE>;
  constexpr int E = P::kElems, kWarps = kThreads / 32;
  extern __shared__ uint4 slots[];
  __shared__ float sm_s[2][kWarps], xch[2][8], slow_m[kWarps], slow_s[kWarps], slow_x[8][2];
  __shared__ int sm_n[kWarps];
  int* const list = reinterpret_cast<int*>(slots + d.pieces);  // counted rows from the front, ignored from the back
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = d.split > 1 ? static_cast<int>(blockIdx.x) % d.split : 0;
  const int first = blockIdx.x / d.split;
  const int piece0 = rank * d.pieces;
  const int iters = (d.pieces + kThreads - 1) / kThreads;
  if constexpr (MODE == kPolicy) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (d.split > 1) cooperative_groups::this_cluster().sync();  // every CTA runs before its shared memory is written

  // A row as this CTA sees it: its address, the columns before the first 16-byte boundary, and how many of this
  // CTA's pieces lie wholly inside the V columns; `rest` elements more are in piece `full`.
  struct Row {
    const char* base;
    const char* body;  // address of this thread's first piece
    int head, full, rest;
  };
  const auto row_of = [&](int row) {
    Row r;
    r.base = static_cast<const char*>(a.x) + (long)row * a.ld * P::kBytes;
    r.head = static_cast<int>((16u - (reinterpret_cast<uintptr_t>(r.base) & 15u)) & 15u) / P::kBytes;
    const int cols = a.V - r.head - piece0 * E;  // from this CTA's first piece to the end of the row
    r.full = min(max(cols, 0) / E, d.pieces);
    r.rest = r.full < d.pieces ? max(cols, 0) - r.full * E : 0;
    r.body = r.base + (r.head + (long)piece0 * E) * P::kBytes + tid * 16;
    return r;
  };
  constexpr int kStep = kThreads * 16;  // bytes from one of a thread's slots to its next
  const uint32_t mine = smem_u32(slots) + tid * 16;
  // Iterations in which every thread has a whole piece, whatever the row's head; the uneven rest (fewer pieces than
  // threads, the last of them partial) is kept out of their loops.
  const int even = min(max(a.V - (d.aligned ? 0 : E - 1) - piece0 * E, 0) / E, d.pieces) / kThreads;
  const auto copy_rest = [&](const Row& r) {
#pragma unroll 1
    for (int k = even; k < iters; ++k) {
      const int i = k * kThreads + tid;
      const int n = i < r.full ? 16 : i == r.full ? r.rest * P::kBytes : 0;
      if (n > 0) copy_piece(mine + k * kStep, r.body + (long)k * kStep, n);
    }
  };
  const auto copy_row = [&](const Row& r) {
    const char* src = r.body;
#pragma unroll 4
    for (int k = 0; k < even; ++k) copy_piece(mine + k * kStep, src + (long)k * kStep);
    copy_rest(r);
  };

  // An ignored row: log-probability 0 and, with a gradient, zeros in this CTA's share of its columns.
  const auto zero_row = [&](int row) {
    if (rank == 0 && tid == 0) {
      a.logp[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
    }
    if constexpr (MODE != kLogp) {
      char* out = static_cast<char*>(a.grad) + (long)row * a.gld * P::kBytes;
      const int lo = min(piece0 * E, a.W), hi = min((piece0 + d.pieces) * E, a.W);
      const auto start = reinterpret_cast<uintptr_t>(out + (long)lo * P::kBytes);
      const int lead = static_cast<int>((16u - (start & 15u)) & 15u) / P::kBytes;
      const int body = min(lo + lead, hi), n = (hi - body) / E;
      if (tid < body - lo) store1<TYPE>(out, lo + tid, 0.f);
      uint4* to = reinterpret_cast<uint4*>(out + (long)body * P::kBytes);
#pragma unroll 4
      for (int i = tid; i < n; i += kThreads) to[i] = make_uint4(0u, 0u, 0u, 0u);
      if (tid < hi - body - n * E) store1<TYPE>(out, body + n * E + tid, 0.f);
    }
  };

  float unit_w = 0.f;
  double sum_loss = 0.0, sum_kl = 0.0, sum_clip = 0.0;
  int parity = 0;
  // Lists this cluster's rows of [w0, w0 + n): rank r of the counted (ignored) rows goes to cluster r % clusters.
  int mine_counted = 0, mine_ignored = 0;
  const auto scan = [&](int w0, int n) {
    constexpr int kBatch = 8;  // loads in flight
    const int seg = (n + kThreads * kBatch - 1) / (kThreads * kBatch) * (32 * kBatch);  // rows of one warp
    const int lo = min(warp * seg, n), hi = min(lo + seg, n);
    int c = 0;
    for (int i = lo; i < hi; i += 32 * kBatch) {
      int64_t t[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int at = i + 32 * k + lane;
        t[k] = at < hi ? a.targets[w0 + at] : a.ignore_index;
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) c += t[k] != a.ignore_index;
    }
    c = __reduce_add_sync(0xffffffffu, c);
    __syncthreads();  // the list's and sm_n's last readers are done
    if (lane == 0) sm_n[warp] = c;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sm_n[w];
      all += sm_n[w];
    }
    int counted = before, ignored = lo - before;
    for (int i = lo; i < hi; i += 32 * kBatch) {
      int64_t t[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int at = i + 32 * k + lane;
        t[k] = at < hi ? a.targets[w0 + at] : a.ignore_index;
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int at = i + 32 * k + lane;
        const bool in = at < hi, yes = in && t[k] != a.ignore_index, no = in && !yes;
        const uint32_t set = __ballot_sync(0xffffffffu, yes), out = __ballot_sync(0xffffffffu, no);
        const uint32_t below = (1u << lane) - 1u;
        const uint32_t r = yes ? counted + __popc(set & below) : ignored + __popc(out & below);
        const uint32_t q = r / static_cast<uint32_t>(d.clusters);
        if (in && r - q * d.clusters == static_cast<uint32_t>(first)) list[yes ? q : d.list - 1 - q] = w0 + at;
        counted += __popc(set);
        ignored += __popc(out);
      }
    }
    __syncthreads();
    mine_counted = (all - first + d.clusters - 1) / d.clusters;  // first < clusters: not negative
    mine_ignored = (n - all - first + d.clusters - 1) / d.clusters;
    return all;
  };
  // As many clusters as rows (`one_each`): nothing to list, and the row's copies need not wait for its target (an
  // ignored row is then read in vain, one per cluster).
  const bool one_each = a.M <= d.clusters;
  if (one_each) copy_row(row_of(first));
  const auto scan_one = [&] {
    if (tid == 0) list[0] = first;
    mine_counted = a.targets[first] != a.ignore_index;
    mine_ignored = 1 - mine_counted;
    int c = 0;
    if (MODE == kPolicy && !p.weights) {
      for (int i = tid; i < a.M; i += kThreads) c += a.targets[i] != a.ignore_index;
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) sm_n[warp] = c;
    }
    __syncthreads();
    if (MODE == kPolicy && !p.weights) {
      c = 0;
      for (int w = 0; w < kWarps; ++w) c += sm_n[w];
    }
    return c;
  };
  const int window = min(a.M, d.window);
  int all = 0;
  if (MODE == kPolicy && !p.weights && window < a.M) {  // 1 / (counted rows) of several windows
    for (int w0 = 0; w0 < a.M; w0 += window) all += scan(w0, min(window, a.M - w0));
    unit_w = 1.f / static_cast<float>(max(all, 1));
  }
  for (int w0 = 0; w0 < a.M; w0 += window) {
    all = one_each ? scan_one() : scan(w0, min(window, a.M - w0));
    if (MODE == kPolicy && window == a.M) unit_w = 1.f / static_cast<float>(max(all, 1));
    int zeros = 0;  // ignored rows done
    Row cur = row_of(mine_counted > 0 ? list[0] : 0);
    if (mine_counted > 0 && !one_each) copy_row(cur);
    for (int j = 0; j < mine_counted; ++j) {
      const int row = list[j];
      const bool more = j + 1 < mine_counted;  // there are copies to make
      const Row nxt = row_of(more ? list[j + 1] : row);
      const int64_t t = a.targets[row];
      const bool bad = t < 0 || t >= a.V;
      const int tc = bad ? -1 : static_cast<int>(t);
      const bool head_col = rank == 0 && tid < min(cur.head, a.V);
      // read here, used after pass 1
      const float xt = bad ? 0.f : load1<TYPE>(cur.base, tc), xh = head_col ? load1<TYPE>(cur.base, tid) : 0.f;
      float old = 0.f, adv = 0.f, ref = 0.f, w = unit_w;
      if constexpr (MODE == kPolicy) {
        old = p.old_logp[row];
        adv = p.adv[p.adv_rows == 1 ? row : row / p.adv_rows];
        if (p.ref_logp) ref = p.ref_logp[row];
        if (p.weights) w = p.weights[row];
      }
      // p_j = 2^((x_j - m) log2 e - log2s) with m = xt (or the row's maximum, `slow`)
      float logp = 0.f, lse = 0.f, log2s = 0.f, m = 0.f;
      bool slow = false;
      {
        float s0 = 0.f, s1 = 0.f;
        const auto add_piece = [&](const uint4& r) {
          float v[E];
          P::widen(r, v);
#pragma unroll
          for (int e = 0; e < E; e += 2) {
            s0 += ex2((v[e] - xt) * kLog2e);
            s1 += ex2((v[e + 1] - xt) * kLog2e);
          }
        };
        copies_wait();
        {
          uint32_t at = mine;
          const char* src = nxt.body;
#pragma unroll kUnroll
          for (int k = 0; k < even; ++k, at += kStep, src += kStep) {
            add_piece(read_piece(at));
            if (MODE == kLogp && more) copy_piece(at, src);  // the slot is free: the next row's piece
          }
        }
#pragma unroll 1
        for (int k = even; k < iters; ++k) {
          const int i = k * kThreads + tid;
          const int n = i < cur.full ? E : i == cur.full ? cur.rest : 0;
          if (n > 0) {
            uint4 r = read_piece(mine + k * kStep);
            if (n < E) P::fill(r, n, P::kMinusInf);
            add_piece(r);
          }
        }
        if (MODE == kLogp && more) copy_rest(nxt);
        float s = s0 + s1;
        if (head_col) s += ex2((xh - xt) * kLog2e);
        s = warp_sum(s);
        if (lane == 0) sm_s[parity][warp] = s;
        __syncthreads();
        s = sm_s[parity][lane % kWarps];
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (d.split > 1) {
          auto cl = cooperative_groups::this_cluster();
          if (tid < d.split) *cl.map_shared_rank(&xch[parity][rank], tid) = s;
          cl.sync();
          s = 0.f;
          for (int c = 0; c < d.split; ++c) s += xch[parity][c];
        }
        parity ^= 1;
        slow = bad || !(s < 1.329227995784916e36f);  // 2^120; also NaN
        if (!slow) {
          m = xt;
          const float ln = logf(s);
          log2s = ln * kLog2e;
          logp = -ln;
          lse = xt + ln;
        } else {
          // the same sum under a maximum, from global memory, one column at a time
          Sum z;
          const int lo = rank == 0 ? 0 : cur.head + piece0 * E;
          const int hi = min(a.V, cur.head + (piece0 + d.pieces) * E);
          for (int j = lo + tid; j < hi; j += kThreads) z.add(load1<TYPE>(cur.base, j));
          m = z.m;
          s = z.s;
          join_lanes<32>(m, s);
          if (lane == 0) {
            slow_m[warp] = m;
            slow_s[warp] = s;
          }
          __syncthreads();
          m = slow_m[lane % kWarps];
          s = slow_s[lane % kWarps];
          join_lanes<kWarps>(m, s);
          if (d.split > 1) {
            auto cl = cooperative_groups::this_cluster();
            if (tid < d.split) {
              float* to = cl.map_shared_rank(&slow_x[rank][0], tid);
              to[0] = m;
              to[1] = s;
            }
            cl.sync();
            m = slow_x[lane % d.split][0];
            s = lane < d.split ? slow_x[lane][1] : 0.f;
            join_lanes<32>(m, s);
            cl.sync();  // read before the next slow row writes it
          } else {
            __syncthreads();
          }
          log2s = log2f(s);
          const float ln = logf(s);
          lse = m + ln;
          logp = bad ? NAN : (xt - m) - ln;
        }
      }
      if (rank == 0 && tid == 0) {
        a.logp[row] = logp;
        if (a.lse) a.lse[row] = lse;
        if (bad) record_error(a.status, kBadArg, 410);
      }
      if constexpr (MODE != kLogp) {
        float coef = 1.f;
        if constexpr (MODE == kPolicy) {
          const RowTerm r = policy_term(p, logp, old, adv, ref, w);
          coef = r.coef * (p.grad_scale ? *p.grad_scale : 1.f);
          if (tid == 0) {
            sum_loss += r.loss;
            sum_kl += r.kl;
            sum_clip += r.clipped;
          }
        }
        if (bad) coef = NAN;
        char* out = static_cast<char*>(a.grad) + (long)row * a.gld * P::kBytes;
        char* out_body = out + (cur.head + (long)piece0 * E) * P::kBytes;
        char* out_mine = out_body + tid * 16;
        const bool zero = coef == 0.f;  // clipped tokens: nothing to evaluate
        const bool fast = d.vec_store && !slow;
        const auto grad_piece = [&](const uint4& r, float (&v)[E]) {
          P::widen(r, v);
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = -coef * ex2(fmaf(v[e] - xt, kLog2e, -log2s));
        };
        if (fast) {
          uint32_t at = mine;
          const char* src = nxt.body;
          if (!zero) {
#pragma unroll kUnroll
            for (int k = 0; k < even; ++k, at += kStep, src += kStep, out_mine += kStep) {
              float v[E];
              grad_piece(read_piece(at), v);
              *reinterpret_cast<uint4*>(out_mine) = P::narrow(v);
              if (more) copy_piece(at, src);  // the slot is free: the next row's piece
            }
          } else {
#pragma unroll 4
            for (int k = 0; k < even; ++k, at += kStep, src += kStep, out_mine += kStep) {
              *reinterpret_cast<uint4*>(out_mine) = make_uint4(0u, 0u, 0u, 0u);
              if (more) copy_piece(at, src);
            }
          }
        }
        // the uneven rest, the columns behind V, and rows that take single stores
        if (!slow) {
#pragma unroll 1
          for (int k = fast ? even : 0; k < iters; ++k) {
            const int i = k * kThreads + tid;
            const int c0 = cur.head + (piece0 + i) * E;
            if (i >= d.pieces || c0 >= a.W) break;
            const int n = zero ? 0 : i < cur.full ? E : i == cur.full ? cur.rest : 0;  // elements to evaluate
            float v[E];
            uint4 r = make_uint4(0u, 0u, 0u, 0u);
            if (n > 0) {
              grad_piece(read_piece(mine + k * kStep), v);
              r = P::narrow(v);
              if (n < E) P::fill(r, n, 0u);
            }
            if (fast && c0 + E <= a.W) {
              *reinterpret_cast<uint4*>(out_body + (long)i * 16) = r;
            } else {
#pragma unroll 1
              for (int e = 0; e < E && c0 + e < a.W; ++e) P::store_at(r, e, out_body, (long)i * E + e);
            }
          }
        }
        if (more) {
          if (fast) copy_rest(nxt);
          else copy_row(nxt);
        }
        if (rank == 0 && tid < min(cur.head, a.W) && !slow)
          store1<TYPE>(out, tid, head_col && !zero ? -coef * ex2(fmaf(xh - xt, kLog2e, -log2s)) : 0.f);
        if (slow) {
          const int lo = rank == 0 ? 0 : cur.head + piece0 * E;
          const int hi = min(a.W, cur.head + (piece0 + d.pieces) * E);
          for (int j = lo + tid; j < hi; j += kThreads) {
            float g = 0.f;
            if (j < a.V) {
              const float pj = ex2(fmaf(load1<TYPE>(cur.base, j) - m, kLog2e, -log2s));
              g = coef * ((j == tc ? 1.f : 0.f) - pj);
            }
            store1<TYPE>(out, j, g);
          }
        } else if (tc >= 0 && !zero) {
          // the target's element, by the thread that has just stored its piece (or head column)
          const int i = tc < cur.head ? -1 : (tc - cur.head) / E - piece0;
          const bool owner = i < 0 ? tc < cur.head && rank == 0 && tid == tc : i < d.pieces && tid == i % kThreads;
          // (1 - p_t from logp itself, which keeps its digits where p_t is near 1)
          if (owner) store1<TYPE>(out, tc, -coef * expm1f(logp));
        }
      }
      cur = nxt;
      // the ignored rows, spread over the counted ones: their stores go beside the next row's arithmetic
      for (; (long)zeros * mine_counted < (long)mine_ignored * (j + 1); ++zeros) zero_row(list[d.list - 1 - zeros]);
    }
    for (; zeros < mine_ignored; ++zeros) zero_row(one_each ? first : list[d.list - 1 - zeros]);
  }
  copies_wait();  // of a row read in vain
  if constexpr (MODE == kPolicy) {
    if (rank == 0 && tid == 0) {
      part[3L * first] = sum_loss;
      part[3L * first + 1] = sum_kl;
      part[3L * first + 2] = sum_clip;
    }
  }
}

// loss and statistics: the clusters' partial sums added in a fixed order, in 64 bits. Launched beside the row kernel
// (programmatic dependent launch), so that only its own few hundred nanoseconds follow the last row.
constexpr int kSumThreads = 128;
__global__ void __launch_bounds__(kSumThreads) policy_sum_kernel(const double* __restrict__ part, int n,
                                                                 float* __restrict__ loss, float* __restrict__ stats) {
  __shared__ double sh[kSumThreads / 32][3];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double s[3] = {0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < n; i += kSumThreads)
    for (int k = 0; k < 3; ++k) s[k] += __ldcg(part + 3L * i + k);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5][k] = s[k];
  }
  __syncthreads();
  if (threadIdx.x < 3) {
    double v = 0.0;
    for (int w = 0; w < kSumThreads / 32; ++w) v += sh[w][threadIdx.x];
    if (threadIdx.x == 0) loss[0] = static_cast<float>(v);
    else stats[threadIdx.x - 1] = static_cast<float>(v);
  }
}

// Preference loss. A group of G warps takes a pair: the sums of both sequences in 64 bits, the pair's factor, both
// gradient rows, and last the pair's loss (its logarithm is off the gradient's path). Batches whose pairs are one round of
// one CTA's groups run in it, and it also adds the losses; others spread over the SMs and leave each CTA's sum to
// preference_sum_kernel, launched beside them. The order of every sum is fixed. Measured in a graph, one CTA and two
// launches: one round, 1 x 57 tokens 4.5 and 5.6 us, 16 x 57 5.3 and 6.6, 1 x 4096 7.3 and 8.5; two rounds, 32 x 1 8.1
// and 5.8, 4 x 1024 9.9 and 7.1; more, 128 x 32 27 and 5.9, 4096 x 1 794 and 10.4 (3.1 us a round).
constexpr int kPrefThreads = 512;
constexpr int kPrefWarps = kPrefThreads / 32;
constexpr int kPrefMaxCtas = 1024;

struct Preference {
  const float *logp, *ref;  // ref may be nullptr
  const int64_t* targets;
  int64_t ignore_index;
  int P, T, G;
  double beta, smoothing;
  float *loss, *rewards, *dlogp;
  double* part;  // [gridDim.x]; nullptr: one CTA, which writes the loss
};

__global__ void __launch_bounds__(kPrefThreads) preference_kernel(const Preference a) {
  __shared__ double sums[2][kPrefWarps][2], losses[kPrefWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_cta = kPrefWarps / a.G, groups = per_cta * gridDim.x;
  const int group = blockIdx.x * per_cta + warp / a.G;
  const int gn = a.G * 32, gl = threadIdx.x & (gn - 1);  // threads of a group (a power of two), this one
  double loss = 0.0;
  int parity = 0;
  for (int p0 = 0; p0 < a.P; p0 += groups) {  // the same rounds for every thread of the CTA
    const int pair = p0 + group;
    const bool in = pair < a.P;
    double s[2] = {0.0, 0.0};
    uint32_t counted[2] = {0u, 0u};  // of this thread's first 32 tokens
    if (in) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long base = ((long)pair + (long)h * a.P) * a.T;
        constexpr int kBatch = 8;  // loads in flight
        for (int j0 = gl, n = 0; j0 < a.T; j0 += kBatch * gn, n += kBatch) {
          int64_t t[kBatch];
          float v[kBatch], r[kBatch];
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const int j = j0 + k * gn;
            const bool at = j < a.T;
            t[k] = at ? a.targets[base + j] : a.ignore_index;
            v[k] = at ? a.logp[base + j] : 0.f;
            r[k] = at && a.ref ? a.ref[base + j] : 0.f;
          }
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            if (t[k] != a.ignore_index) {
              s[h] += static_cast<double>(v[k]) - static_cast<double>(r[k]);
              if (n + k < 32) counted[h] |= 1u << (n + k);
            }
          }
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
      s[1] += __shfl_xor_sync(0xffffffffu, s[1], o);
    }
    if (a.G > 1) {
      if (lane == 0) {
        sums[parity][warp][0] = s[0];
        sums[parity][warp][1] = s[1];
      }
      __syncthreads();
      s[0] = s[1] = 0.0;
      const int w0 = warp & ~(a.G - 1);
      for (int w = w0; w < w0 + a.G; ++w) {
        s[0] += sums[parity][w][0];
        s[1] += sums[parity][w][1];
      }
      parity ^= 1;
    }
    if (in) {
      const double good = a.beta * s[0], poor = a.beta * s[1], z = good - poor;
      // sigmoid(|z|) and sigmoid(-|z|) from e = e^-|z|, which cannot overflow
      const double e = exp(-fabs(z)), big = 1.0 / (1.0 + e), small = e * big;
      const double sig = z >= 0.0 ? big : small, sig_neg = z >= 0.0 ? small : big;
      const double dz = a.smoothing * sig - (1.0 - a.smoothing) * sig_neg;  // dloss / dz
      const float c = static_cast<float>(z != z ? z : a.beta / a.P * dz);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long base = ((long)pair + (long)h * a.P) * a.T;
        const float g = h ? -c : c;
#pragma unroll 4
        for (int j = gl, n = 0; j < a.T; j += gn, ++n) {
          const bool yes = n < 32 ? (counted[h] >> n & 1u) != 0u : a.targets[base + j] != a.ignore_index;
          a.dlogp[base + j] = yes ? g : 0.f;
        }
      }
      if (gl == 0) {
        a.rewards[pair] = static_cast<float>(good);
        a.rewards[a.P + pair] = static_cast<float>(poor);
        const double l = log1p(e);  // log(1 + e^-z) = max(-z, 0) + l, log(1 + e^z) = max(z, 0) + l
        loss += z != z ? z : (1.0 - a.smoothing) * (fmax(-z, 0.0) + l) + a.smoothing * (fmax(z, 0.0) + l);
      }
    }
  }
  if (gl == 0) losses[warp] = loss;  // the first warp of each group holds its pairs' sum
  __syncthreads();
  if (threadIdx.x == 0) {
    double v = 0.0;
    for (int w = 0; w < kPrefWarps; w += a.G) v += losses[w];
    if (a.part) a.part[blockIdx.x] = v;
    else a.loss[0] = a.P > 0 ? static_cast<float>(v / a.P) : 0.f;
  }
}

__global__ void __launch_bounds__(32) preference_sum_kernel(const double* __restrict__ part, int n, int P,
                                                            float* __restrict__ loss) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double v = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 32) v += __ldcg(part + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x == 0) loss[0] = static_cast<float>(v / P);
}

// Launch of a kernel that starts with griddepcontrol.wait, beside the one before it on the stream.
template <class... Params, class... Args>
void launch_beside(void (*k)(Params...), int ctas, int threads, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  HB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, static_cast<Params>(args)...));
}

// Shared memory: 228 KB an SM, 227 KB a CTA; each CTA also takes 1 KB for the system and under 1 KB for the
// kernel's own arrays.
constexpr int kListRows = 510;  // rows of one window that a cluster takes, at most
constexpr int kListBytes = (kListRows + 2) * 4;
constexpr int kMaxPieces = (227 * 1024 - 1024 - kListBytes) / 16;                     // one CTA on the SM
constexpr int kMaxPiecesShared = (228 * 1024 / kCtasPerSm - 2048 - kListBytes) / 16;  // kCtasPerSm of them
constexpr int kMaxSplit = 8;

// Deals M rows of `row_pieces` pieces to clusters of 1, 2, 4 or 8 CTAs: the split with the least estimated
// time, rounds * (fixed cost of a row + its bytes, both ways, at an SM's share of the memory rate). It goes by the
// logits alone, with or without a gradient, so equal logits give equal bits in all three losses (the order of a
// row's sum goes by the split): a policy step on the tokens it has just scored starts at ratios of exactly 1.
// Measured (policy loss, 50257 columns, bf16; split 1 / 2 / 4 / 8): 16 rows 12.7 / 10.7 / 10.0 / 8.7 us, 61 rows 12.6 /
// 10.6 / 10.6 / 16.7, 500 rows 25 / 27 / 49 / 74, 4096 rows 135 / 156 / 354 / 571. A CTA that has an SM for itself gets the
// threads of two: 131072 columns, 4096 rows 393 us with 512 threads, 412 with 256.
Deal deal_rows(int M, long row_pieces, int sms) {
  Deal best{};
  double least = 0.0;
  for (int c = 1; c <= kMaxSplit; c *= 2) {
    const long pieces = (row_pieces + c - 1) / c;
    if (pieces > kMaxPieces) continue;
    const int resident = pieces <= kMaxPiecesShared ? kCtasPerSm : 1;
    const int most = sms * resident / c;
    const int clusters = std::max(1, std::min(M, most));
    const int rounds = (M + most - 1) / most;
    const double ns = rounds * ((c > 1 ? 2200.0 : 1500.0) + 32.0 * pieces * resident / 43.0);
    if (best.split == 0 || ns < least) {
      least = ns;
      best.split = c;
      best.pieces = static_cast<int>(pieces);
      best.clusters = clusters;
      best.threads = kThreadsPerSm / resident;
      best.window = static_cast<int>(std::min<long>(M, (long)clusters * kListRows));
      // ceil(counted / clusters) + ceil(ignored / clusters) entries at most
      best.list = (best.window + clusters - 1) / clusters + 1;
    }
  }
  return best;
}

template <int TYPE, int MODE, int THREADS>
void launch_typed(const LogitRows& a, const PolicyTerms& p, const Deal& d, double* part, cudaStream_t s) {
  auto* k = logit_rows_kernel<TYPE, MODE, THREADS>;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
  const int dev = current_device();
  if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    HB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPieces * 16 + kListBytes));
    ready.fetch_or(uint64_t{1} << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(d.clusters * d.split));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = static_cast<size_t>(d.pieces) * 16 + static_cast<size_t>(d.list) * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(d.split);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = d.split > 1 ? 1 : 0;
  HB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, a, p, d, part));
}

template <int MODE>
void launch_rows(const LogitRows& a, const PolicyTerms& p, const Deal& d, double* part, cudaStream_t s) {
  if (a.M == 0) return;
#define HB_ROWS(T)                                                      \
  (d.threads == kThreadsPerSm ? launch_typed<T, MODE, kThreadsPerSm>    \
                              : launch_typed<T, MODE, kThreadsPerSm / kCtasPerSm>)
  auto* launch = a.type == kLogitF32   ? HB_ROWS(kLogitF32)
                 : a.type == kLogitF16 ? HB_ROWS(kLogitF16)
                                       : HB_ROWS(kLogitBf16);
#undef HB_ROWS
  launch(a, p, d, part, s);
}

Deal deal_of(const LogitRows& a) {
  const int elems = a.type == kLogitF32 ? 4 : 8, bytes = 16 / elems;
  const long width = a.W > a.V ? a.W : a.V;
  Deal d = deal_rows(a.M, (width + elems - 1) / elems, num_sms(current_device()));
  if (d.split == 0) throw std::runtime_error("logit rows are too wide");  // the torch-facing checks refuse them first
  d.aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && (a.M <= 1 || a.ld * bytes % 16 == 0);
  d.vec_store = a.grad && reinterpret_cast<uintptr_t>(a.x) % 16 == reinterpret_cast<uintptr_t>(a.grad) % 16 &&
                (a.M <= 1 || (a.ld - a.gld) * bytes % 16 == 0);
  return d;
}

}  // namespace

long logit_row_limit(int type) { return static_cast<long>(kMaxPieces) * kMaxSplit * (type == kLogitF32 ? 4 : 8); }
long policy_scratch_doubles() { return 3L * kCtasPerSm * num_sms(current_device()); }
// Warps that take a pair of sequences of T tokens: 4 tokens of a sequence a thread, as far as a CTA's warps go.
static int preference_group(int T) {
  int g = 1;
  while (g < kPrefWarps && g * 128 < T) g *= 2;
  return g;
}
long preference_scratch_doubles(int P, int T) { return P <= kPrefWarps / preference_group(T) ? 0 : kPrefMaxCtas; }

void token_logprobs_launch(const LogitRows& a, cudaStream_t s) {
  const PolicyTerms none{};
  if (a.grad) launch_rows<kUnit>(a, none, deal_of(a), nullptr, s);
  else launch_rows<kLogp>(a, none, deal_of(a), nullptr, s);
}

void policy_loss_launch(const LogitRows& a, const PolicyTerms& p, double* scratch, float* loss, float* stats,
                        cudaStream_t s) {
  const Deal d = deal_of(a);
  launch_rows<kPolicy>(a, p, d, scratch, s);
  launch_beside(policy_sum_kernel, 1, kSumThreads, s, scratch, a.M > 0 ? d.clusters : 0, loss, stats);
}

void preference_loss_launch(const float* logp, const float* ref, const int64_t* targets, int64_t ignore_index, int P,
                            int T, double beta, double smoothing, float* loss, float* rewards, float* dlogp,
                            double* scratch, cudaStream_t s) {
  Preference a{logp, ref,       targets, ignore_index, P,     T, preference_group(T),
               beta, smoothing, loss,    rewards,      dlogp, nullptr};
  const int per_cta = kPrefWarps / a.G;
  const bool one = preference_scratch_doubles(P, T) == 0;
  const int ctas = one ? 1 : std::min((P + per_cta - 1) / per_cta, kPrefMaxCtas);
  if (!one) a.part = scratch;
  preference_kernel<<<ctas, kPrefThreads, 0, s>>>(a);
  HB_CUDA_CHECK(cudaGetLastError());
  if (!one) launch_beside(preference_sum_kernel, 1, 32, s, scratch, ctas, P, loss);
}

}  // namespace hb
