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

#include <atomic>

#include "common.cuh"
#include "host_utils.h"
#include "post_args.h"

namespace hb {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kCtasPerSm = 2;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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
  // elements at and behind `n` become -inf
  static __device__ __forceinline__ void mask(uint4& r, int n) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == kLogitF32) {
        if (i >= n) w[i] = 0xFF800000u;
      } else {
        constexpr uint32_t kInf = kF16 ? 0xFC00u : 0xFF80u;
        if (2 * i >= n) w[i] = kInf | (kInf << 16);
        else if (2 * i + 1 >= n) w[i] = (w[i] & 0xFFFFu) | (kInf << 16);
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
  static __device__ __forceinline__ float at(const uint4& r, int e) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
    if constexpr (TYPE == kLogitF32) return __uint_as_float(w[e]);
    else return e & 1 ? hi16<kF16>(w[e >> 1]) : lo16<kF16>(w[e >> 1]);
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

__device__ __forceinline__ void copy_piece(void* smem, const void* gmem, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Running sum of exp(x - m) against a reference m. The reference moves only when a value exceeds it by more
// than 6 (a term is then at most e^6, so 2^31 of them stay far below overflow), so almost no piece pays for a rescale.
// x - m is taken before the factor log2 e: the product alone would overflow for masks of the type's lowest
// value. An empty sum (nothing, or only -inf) has s = 0 and any m; NaN and +inf make s NaN.
struct Sum {
  float m = 0.f, limit = -INFINITY, s = 0.f;
  __device__ __forceinline__ void move(float to) {
    if (s != 0.f) s *= ex2((m - to) * kLog2e);
    m = to;
    limit = to + 6.f;
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N]) {
    float top = max3f(v[0], v[1], v[2]);
    if constexpr (N == 8) top = max3f(max3f(top, v[4], v[5]), v[6], v[7]);
    top = fmaxf(top, v[3]);
    if (top > limit) move(top);
    const uint64_t l2 = f2_pack(kLog2e, kLog2e), neg = f2_pack(-m, -m);
    uint64_t acc = f2_pack(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      float a, b;
      f2_unpack(f2_mul(f2_add(f2_pack(v[i], v[i + 1]), neg), l2), a, b);
      acc = f2_add(acc, f2_pack(ex2(a), ex2(b)));
    }
    float a, b;
    f2_unpack(acc, a, b);
    s += a + b;
  }
  __device__ __forceinline__ void add1(float v) {
    if (v > limit) move(v);
    s += ex2((v - m) * kLog2e);
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
  const bool clipped = c * adv < r * adv;  // false for a NaN ratio, which so reaches the loss and the gradient
  t.loss = clipped ? -c * adv : -r * adv;
  t.coef = clipped ? 0.f : -r * adv;
  t.clipped = clipped ? w : 0.f;
  if (p.ref_logp) {
    const float u = ref - logp;
    const float e = expm1f(u);
    t.kl = e - u;
    t.loss = fmaf(p.kl_coef, t.kl, t.loss);
    t.coef = fmaf(-p.kl_coef, e, t.coef);
  }
  t.loss *= w;
  t.kl *= w;
  t.coef *= w;
  return t;
}

enum Mode : int { kLogp = 0, kUnit = 1, kPolicy = 2 };

// How the rows are dealt out: clusters of `split` CTAs, each CTA holding `pieces` 16-byte pieces of a row.
struct Deal {
  int split, pieces, clusters;
  bool vec_store;  // rows of grad start at the same offset from a 16-byte boundary as those of the logits
};

constexpr int kStages = 4;  // copy groups of one row

// Row kernel. A cluster of `split` CTAs takes rows cluster, cluster + clusters, ...; CTA c holds pieces
// [c pieces, (c + 1) pieces) of the row in shared memory. Every thread copies, reads and refills its own 16-byte
// slots (asynchronous copies, waited for in four groups), so the copies need no barrier, and the next row's copies
// are issued slot by slot as the current row's gradient leaves: the memory pipe never drains.
//   pass 1 (while the copies arrive): per-thread running (m, s); joined over the warp, the CTA (one barrier) and,
//          where split > 1, the cluster (each CTA writes its (m, s, x_t) into every other's shared memory;
//          one cluster barrier);
//   pass 2 (gradient): coef ([j == t] - exp(x_j - lse)) from the slots, stored in 16-byte pieces.
// So a row crosses DRAM once each way. Rows may start at any element: the columns before the first 16-byte
// boundary (`head`, fewer than one piece) are read by single threads of the first CTA.
template <int TYPE, int MODE>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    logit_rows_kernel(const LogitRows a, const PolicyTerms p, const Deal d, double* __restrict__ part) {
  using P = Piece<TYPE>;
  constexpr int E = P::kElems;
  extern __shared__ uint4 slots[];
  __shared__ float sm_m[2][kWarps], sm_s[2][kWarps], sm_x[2], xch[2][8][3];
  __shared__ int sm_n[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = d.split > 1 ? static_cast<int>(blockIdx.x) % d.split : 0;
  const int first = blockIdx.x / d.split;
  const int piece0 = rank * d.pieces;
  const int iters = (d.pieces + kThreads - 1) / kThreads;
  if (d.split > 1) cooperative_groups::this_cluster().sync();  // every CTA runs before its shared memory is written

  const auto row_ptr = [&](int row) { return static_cast<const char*>(a.x) + (long)row * a.ld * P::kBytes; };
  // columns of a row before its first 16-byte boundary
  const auto head_of = [&](int row) {
    return static_cast<int>((16u - (reinterpret_cast<uintptr_t>(row_ptr(row)) & 15u)) & 15u) / P::kBytes;
  };
  const auto copy_slot = [&](const char* base, int head, int i) {
    const int n = a.V - head - (piece0 + i) * E;  // columns from here to the end
    if (i < d.pieces && n > 0) copy_piece(&slots[i], base + (head + (long)(piece0 + i) * E) * P::kBytes, min(n, E) * P::kBytes);
  };

  int64_t t = a.ignore_index;
  if (first < a.M) t = a.targets[first];
  if (first < a.M && t != a.ignore_index) {
    const char* base = row_ptr(first);
    const int head = head_of(first);
    for (int g = 0, k = 0; g < kStages; ++g) {
      for (; k < iters * (g + 1) / kStages; ++k) copy_slot(base, head, k * kThreads + tid);
      copies_commit();
    }
  } else {
    for (int g = 0; g < kStages; ++g) copies_commit();
  }

  float unit_w = 0.f;
  double sum_loss = 0.0, sum_kl = 0.0, sum_clip = 0.0;
  if constexpr (MODE == kPolicy) {
    if (!p.weights) {  // 1 / (counted rows): every CTA counts, while its first copies are in flight
      int n = 0;
#pragma unroll 4
      for (int i = tid; i < a.M; i += kThreads) n += a.targets[i] != a.ignore_index;
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) sm_n[warp] = n;
      __syncthreads();
      n = 0;
      for (int w = 0; w < kWarps; ++w) n += sm_n[w];
      unit_w = 1.f / static_cast<float>(max(n, 1));
    }
  }

  int parity = 0;
  for (int row = first; row < a.M; row += d.clusters) {
    const int next = row + d.clusters;
    const int64_t t_next = next < a.M ? a.targets[next] : a.ignore_index;
    const bool more = t_next != a.ignore_index;
    const char* next_base = row_ptr(more ? next : row);
    const int next_head = head_of(more ? next : row);
    const bool counted = t != a.ignore_index;
    const bool bad = counted && (t < 0 || t >= a.V);
    const char* base = row_ptr(row);
    const int head = head_of(row);
    float old = 0.f, adv = 0.f, ref = 0.f, w = unit_w;
    if constexpr (MODE == kPolicy) {  // read here, used after pass 1
      if (counted) {
        old = p.old_logp[row];
        adv = p.adv[row / p.adv_rows];
        if (p.ref_logp) ref = p.ref_logp[row];
        if (p.weights) w = p.weights[row];
      }
    }
    // the piece (of this CTA) and element that hold the target; head columns have piece -1
    const int tc = bad || !counted ? -1 : static_cast<int>(t);
    const bool head_col = rank == 0 && tid < min(head, a.V);
    float xh = 0.f;
    float logp = 0.f, lse = 0.f, m = 0.f, log2s = 0.f;
    if (counted) {
      if (head_col) xh = load1<TYPE>(base, tid);
      Sum sum;
#pragma unroll
      for (int g = 0, k = 0; g < kStages; ++g) {
        copies_wait<kStages - 1>();
        for (; k < iters * (g + 1) / kStages; ++k) {
          const int i = k * kThreads + tid;
          const int c0 = head + (piece0 + i) * E;
          if (i < d.pieces && c0 < a.V) {
            uint4 r = slots[i];
            if (c0 + E > a.V) P::mask(r, a.V - c0);
            float v[E];
            P::widen(r, v);
            if (static_cast<unsigned>(tc - c0) < static_cast<unsigned>(E)) {
              float x = v[0];
#pragma unroll
              for (int e = 1; e < E; ++e) x = e == tc - c0 ? v[e] : x;
              sm_x[parity] = x;
            }
            sum.add(v);
          }
          if constexpr (MODE == kLogp) {
            if (more) copy_slot(next_base, next_head, i);
          }
        }
        // pass 1 of a gradient row leaves its slots in place: an empty group keeps the count of groups
        copies_commit();
      }
      if (head_col) {
        sum.add1(xh);
        if (tid == tc) sm_x[parity] = xh;
      }
      float s = sum.s;
      m = sum.m;
      join_lanes<32>(m, s);
      if (lane == 0) {
        sm_m[parity][warp] = m;
        sm_s[parity][warp] = s;
      }
      __syncthreads();
      m = sm_m[parity][lane % kWarps];
      s = sm_s[parity][lane % kWarps];
      join_lanes<kWarps>(m, s);
      float xt = 0.f;
      const bool mine = tc >= 0 && (tc < head ? rank == 0 : (tc - head) / E / d.pieces == rank);
      if (mine) xt = sm_x[parity];
      if (d.split > 1) {
        auto cl = cooperative_groups::this_cluster();
        if (tid < d.split) {
          float* to = cl.map_shared_rank(&xch[parity][rank][0], tid);
          to[0] = m;
          to[1] = s;
          to[2] = mine ? xt : -INFINITY;
        }
        cl.sync();
        float top = -INFINITY;
        for (int c = 0; c < d.split; ++c)
          if (xch[parity][c][1] != 0.f) top = fmaxf(top, xch[parity][c][0]);
        s = 0.f;
        xt = -INFINITY;
        for (int c = 0; c < d.split; ++c) {
          const float sc = xch[parity][c][1], xc = xch[parity][c][2];
          if (sc != 0.f) s += sc * ex2((xch[parity][c][0] - top) * kLog2e);
          if (xc != -INFINITY) xt = xc;  // only the owner's is not -inf (NaN included)
        }
        m = top;
      }
      parity ^= 1;
      const float ln = logf(s);
      log2s = log2f(s);
      lse = m + ln;
      logp = bad ? NAN : (xt - m) - ln;
    } else {
#pragma unroll
      for (int g = 0, k = 0; g < kStages; ++g) {
        if constexpr (MODE == kLogp) {
          if (more)
            for (; k < iters * (g + 1) / kStages; ++k) copy_slot(next_base, next_head, k * kThreads + tid);
        }
        copies_commit();
      }
    }
    if (rank == 0 && tid == 0) {
      a.logp[row] = logp;
      if (a.lse) a.lse[row] = lse;
      if (bad) record_error(a.status, kBadArg, 410);
    }
    if constexpr (MODE != kLogp) {
      float coef = counted ? 1.f : 0.f;
      if constexpr (MODE == kPolicy) {
        if (counted) {
          const RowTerm r = policy_term(p, logp, old, adv, ref, w);
          coef = r.coef * (p.grad_scale ? *p.grad_scale : 1.f);
          sum_loss += r.loss;
          sum_kl += r.kl;
          sum_clip += r.clipped;
        }
      }
      if (bad) coef = NAN;
      const bool zero = coef == 0.f;  // ignored rows and clipped tokens: nothing to evaluate
      char* out = static_cast<char*>(a.grad) + (long)row * a.gld * P::kBytes;
      if (rank == 0 && tid < min(head, a.W)) {
        const float g = head_col && !zero ? coef * ((tid == tc ? 1.f : 0.f) - ex2(fmaf(xh - m, kLog2e, -log2s))) : 0.f;
        store1<TYPE>(out, tid, g);
      }
      const uint64_t l2 = f2_pack(kLog2e, kLog2e), neg = f2_pack(-m, -m), nl = f2_pack(-log2s, -log2s);
      const uint64_t nc = f2_pack(-coef, -coef);
#pragma unroll
      for (int g = 0, k = 0; g < kStages; ++g) {
        for (; k < iters * (g + 1) / kStages; ++k) {
          const int i = k * kThreads + tid;
          const int c0 = head + (piece0 + i) * E;
          if (i < d.pieces && c0 < a.W) {
            float v[E];
            if (zero || c0 >= a.V) {
#pragma unroll
              for (int e = 0; e < E; ++e) v[e] = 0.f;
            } else {
              P::widen(slots[i], v);
#pragma unroll
              for (int e = 0; e < E; e += 2) {
                float q0, q1;
                f2_unpack(f2_fma(f2_add(f2_pack(v[e], v[e + 1]), neg), l2, nl), q0, q1);
                f2_unpack(f2_mul(f2_pack(ex2(q0), ex2(q1)), nc), v[e], v[e + 1]);
              }
              if (static_cast<unsigned>(tc - c0) < static_cast<unsigned>(E)) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                  if (e == tc - c0) v[e] = fmaf(ex2(fmaf(P::at(slots[i], e) - m, kLog2e, -log2s)), -coef, coef);
              }
              if (c0 + E > a.V) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                  if (c0 + e >= a.V) v[e] = 0.f;
              }
            }
            if (d.vec_store && c0 + E <= a.W) {
              *reinterpret_cast<uint4*>(out + (long)c0 * P::kBytes) = P::narrow(v);
            } else {
#pragma unroll
              for (int e = 0; e < E; ++e)
                if (c0 + e < a.W) store1<TYPE>(out, c0 + e, v[e]);
            }
          }
          if (more) copy_slot(next_base, next_head, i);
        }
        copies_commit();
      }
    }
    t = t_next;
  }
  if constexpr (MODE == kPolicy) {
    if (rank == 0 && tid == 0) {
      part[3L * first] = sum_loss;
      part[3L * first + 1] = sum_kl;
      part[3L * first + 2] = sum_clip;
    }
  }
  copies_wait<0>();
}

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) v += sh[w];
  __syncthreads();
  return v;
}

// loss and statistics: the rows' terms added in a fixed order, in 64 bits.
__global__ void __launch_bounds__(1024) policy_sum_kernel(const double* __restrict__ part, int n,
                                                          float* __restrict__ loss, float* __restrict__ stats) {
  __shared__ double sh[32];
  double s[3] = {0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < n; i += 1024)
    for (int k = 0; k < 3; ++k) s[k] += part[3L * i + k];
  for (int k = 0; k < 3; ++k) s[k] = block_sum(s[k], sh);
  if (threadIdx.x == 0) {
    loss[0] = (float)s[0];
    stats[0] = (float)s[1];
    stats[1] = (float)s[2];
  }
}

// log(1 + e^t) without overflow.
__device__ __forceinline__ double softplus(double t) { return fmax(t, 0.0) + log1p(exp(-fabs(t))); }

// One CTA per pair: sums both sequences, then writes both gradient rows.
__global__ void __launch_bounds__(256) preference_kernel(const float* __restrict__ logp, const float* __restrict__ ref,
                                                         const int64_t* __restrict__ targets, int64_t ignore_index,
                                                         int P, int T, double beta, double smoothing,
                                                         float* __restrict__ rewards, float* __restrict__ dlogp,
                                                         double* __restrict__ part) {
  __shared__ double sh[32];
  const int i = blockIdx.x;
  double sum[2];
  for (int h = 0; h < 2; ++h) {
    const long base = (long)(i + h * P) * T;
    double v = 0.0;
    for (int j = threadIdx.x; j < T; j += blockDim.x)
      if (targets[base + j] != ignore_index) v += (double)logp[base + j] - (ref ? (double)ref[base + j] : 0.0);
    sum[h] = beta * block_sum(v, sh);
  }
  const double z = sum[0] - sum[1];
  const double c = beta / P * (smoothing / (1.0 + exp(-z)) - (1.0 - smoothing) / (1.0 + exp(z)));
  if (threadIdx.x == 0) {
    rewards[i] = (float)sum[0];
    rewards[P + i] = (float)sum[1];
    part[i] = (1.0 - smoothing) * softplus(-z) + smoothing * softplus(z);
  }
  for (int h = 0; h < 2; ++h) {
    const long base = (long)(i + h * P) * T;
    const float g = (float)(h ? -c : c);
    for (int j = threadIdx.x; j < T; j += blockDim.x) dlogp[base + j] = targets[base + j] != ignore_index ? g : 0.f;
  }
}

__global__ void __launch_bounds__(256) preference_sum_kernel(const double* __restrict__ part, int P,
                                                             float* __restrict__ loss) {
  __shared__ double sh[32];
  double v = 0.0;
  for (int i = threadIdx.x; i < P; i += 256) v += part[i];
  v = block_sum(v, sh);
  if (threadIdx.x == 0) loss[0] = P > 0 ? (float)(v / P) : 0.f;
}

// Shared memory: 228 KB an SM, 227 KB a CTA; each CTA also takes 1 KB for the system and under 1 KB for the
// kernel's own arrays.
constexpr int kMaxPieces = (227 * 1024 - 1024) / 16;                  // one CTA on the SM
constexpr int kMaxPiecesShared = (228 * 1024 / kCtasPerSm - 2048) / 16;  // kCtasPerSm of them
constexpr int kMaxSplit = 8;

// Deals M rows of `row_pieces` pieces to clusters of 1, 2, 4 or 8 CTAs: the split with the least estimated
// time, rounds * (fixed cost of a row + its bytes at an SM's share of the memory rate).
Deal deal_rows(int M, long row_pieces, int dirs, int sms) {
  Deal best{0, 0, 0, true};
  double least = 0.0;
  for (int c = 1; c <= kMaxSplit; c *= 2) {
    const long pieces = (row_pieces + c - 1) / c;
    if (pieces > kMaxPieces) continue;
    const int resident = pieces <= kMaxPiecesShared ? kCtasPerSm : 1;
    const int most = sms * resident / c;
    const int clusters = M < most ? M : most;
    const int rounds = (M + most - 1) / most;
    const double ns = rounds * ((c > 1 ? 2200.0 : 1500.0) + 16.0 * pieces * dirs * resident / 43.0);
    if (best.split == 0 || ns < least) {
      least = ns;
      best.split = c;
      best.pieces = static_cast<int>(pieces);
      best.clusters = clusters;
    }
  }
  return best;
}

template <int TYPE, int MODE>
void launch_typed(const LogitRows& a, const PolicyTerms& p, const Deal& d, double* part, cudaStream_t s) {
  auto* k = logit_rows_kernel<TYPE, MODE>;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
  const int dev = current_device();
  if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    HB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPieces * 16));
    ready.fetch_or(uint64_t{1} << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(d.clusters * d.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(d.pieces) * 16;
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
  if (a.type == kLogitF32) launch_typed<kLogitF32, MODE>(a, p, d, part, s);
  else if (a.type == kLogitF16) launch_typed<kLogitF16, MODE>(a, p, d, part, s);
  else launch_typed<kLogitBf16, MODE>(a, p, d, part, s);
}

Deal deal_of(const LogitRows& a) {
  const int elems = a.type == kLogitF32 ? 4 : 8, bytes = 16 / elems;
  const long width = a.grad && a.W > a.V ? a.W : a.V;
  Deal d = deal_rows(a.M, (width + elems - 1) / elems, a.grad ? 2 : 1, num_sms(current_device()));
  if (d.split == 0) throw std::runtime_error("logit rows are too wide");  // the torch-facing checks refuse them first
  d.vec_store = a.grad && reinterpret_cast<uintptr_t>(a.x) % 16 == reinterpret_cast<uintptr_t>(a.grad) % 16 &&
                (a.M <= 1 || (a.ld - a.gld) * bytes % 16 == 0);
  return d;
}

}  // namespace

long logit_row_limit(int type) { return static_cast<long>(kMaxPieces) * kMaxSplit * (type == kLogitF32 ? 4 : 8); }
long policy_scratch_doubles() { return 3L * kCtasPerSm * num_sms(current_device()); }
long preference_scratch_doubles(int P) { return P; }

void token_logprobs_launch(const LogitRows& a, cudaStream_t s) {
  const PolicyTerms none{};
  if (a.grad) launch_rows<kUnit>(a, none, deal_of(a), nullptr, s);
  else launch_rows<kLogp>(a, none, deal_of(a), nullptr, s);
}

void policy_loss_launch(const LogitRows& a, const PolicyTerms& p, double* scratch, float* loss, float* stats,
                        cudaStream_t s) {
  const Deal d = deal_of(a);
  launch_rows<kPolicy>(a, p, d, scratch, s);
  policy_sum_kernel<<<1, 1024, 0, s>>>(scratch, d.clusters, loss, stats);
  HB_CUDA_CHECK(cudaGetLastError());
}

void preference_loss_launch(const float* logp, const float* ref, const int64_t* targets, int64_t ignore_index, int P,
                            int T, double beta, double smoothing, float* loss, float* rewards, float* dlogp,
                            double* scratch, cudaStream_t s) {
  if (P > 0) {
    preference_kernel<<<P, 256, 0, s>>>(logp, ref, targets, ignore_index, P, T, beta, smoothing, rewards, dlogp,
                                        scratch);
    HB_CUDA_CHECK(cudaGetLastError());
  }
  preference_sum_kernel<<<1, 256, 0, s>>>(scratch, P, loss);
  HB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace hb
