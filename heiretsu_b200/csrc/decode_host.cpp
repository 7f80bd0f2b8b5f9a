// Torch-facing entry points of decoding (kv_cache.cu, decode_attn.cu, sample.cu): argument checks, stream
// selection, then the raw launchers. Refused calls raise before anything is launched; the device is looked at last, so
// every other refusal shows on a machine without one. Numbers go into the messages as strings: an extension whose
// linker brought its own static libstdc++ faults when it streams them.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <functional>
#include <limits>
#include <string>

#include "decode_args.h"
#include "host_utils.h"
#include "ops.h"

namespace hb {

void kv_write_launch(const KvTokens& t, const KvPool& p, int* status, cudaStream_t s);
void kv_read_launch(const int64_t* slots, const KvPool& p, void* k, void* v, int n, int out, int* status,
                    cudaStream_t s);
DecodePlan decode_attention_plan(const KvPool& p, int seqs, int units, int longest);
void decode_attention_launch(const DecodeArgs& a, const DecodePlan& d, cudaStream_t s);
void sample_tokens_launch(const SampleArgs& a, cudaStream_t s);

namespace {

using OptTensor = c10::optional<at::Tensor>;
constexpr int64_t kIntMax = std::numeric_limits<int>::max();
constexpr int64_t kLongest = 1 << 24;   // tokens of a sequence: the tiles of 1024 sequences are counted in 32 bits
constexpr int64_t kStride = int64_t{1} << 32;
constexpr int64_t kMaxVocab = 1 << 19;  // weights of 2^-44 then sum to less than 2^63

// An output, allocated without the dispatcher: a short call is bound by the host.
at::Tensor output(at::IntArrayRef sizes, at::ScalarType dt, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, dt, dev, c10::nullopt);
}

bool given(const OptTensor& t) { return t && t->defined(); }
bool half_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

std::string dims(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// Dimensions of more than one element, by stride.
struct Layout {
  int64_t stride[4], size[4], dim[4];
  int n = 0;
  explicit Layout(const at::Tensor& t) {
    for (int64_t i = 0; i < t.dim(); ++i) {
      if (t.size(i) <= 1) continue;
      int j = n++;
      for (; j > 0 && stride[j - 1] > t.stride(i); --j)
        stride[j] = stride[j - 1], size[j] = size[j - 1], dim[j] = dim[j - 1];
      stride[j] = t.stride(i), size[j] = t.size(i), dim[j] = i;
    }
  }
  int64_t reach(int inner) const {  // elements from the first to behind the last, of the first `inner` dimensions
    int64_t r = 1;
    for (int j = 0; j < inner; ++j) r += (size[j] - 1) * stride[j];
    return r;
  }
};
// No two elements at one address: each dimension steps over all that lies within the ones before.
bool disjoint(const at::Tensor& t) {
  const Layout x(t);
  for (int j = 0; j < x.n; ++j)
    if (x.stride[j] < (j > 0 ? x.stride[j - 1] * x.size[j - 1] : 1)) return false;
  return true;
}
// Whether two tensors of one type and the same sizes, each disjoint, reach into each other. The outer dimensions that both have
// with the same strides are told apart exactly, such as pages that hold K and V; what lies within them counts as a whole,
// so with the same strides throughout they do if they share an element.
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0) return false;
  const Layout x(a), y(b);
  int inner = x.n;
  while (inner > 0 && x.dim[inner - 1] == y.dim[inner - 1] && x.stride[inner - 1] == y.stride[inner - 1]) --inner;
  const int64_t bytes = reinterpret_cast<intptr_t>(b.data_ptr()) - reinterpret_cast<intptr_t>(a.data_ptr()), es = a.element_size();
  if (bytes % es != 0) return true;
  // the inner parts of two elements are less than a step of the next dimension apart: its share is the quotient or one more
  const std::function<bool(int64_t, int)> meet = [&](int64_t apart, int j) {
    if (j == inner) return apart < x.reach(inner) && -apart < y.reach(inner);
    const int64_t s = x.stride[j - 1], q = apart >= 0 ? apart / s : -((-apart + s - 1) / s);
    for (const int64_t i : {q, q + 1})
      if (std::abs(i) < x.size[j - 1] && meet(apart - i * s, j - 1)) return true;
    return false;
  };
  return meet(bytes / es, x.n);
}

void check_same_device(const at::Tensor& t, const at::Device& dev, const char* op, const char* name) {
  TORCH_CHECK(t.device() == dev, op, ": ", name, " must be on ", dev.str());
}

// A tensor of one type with exactly these sizes, contiguous.
void check_plain(const at::Tensor& t, at::ScalarType dt, at::IntArrayRef sizes, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == dt, op, ": ", name, " has the wrong dtype");
  TORCH_CHECK(t.sizes() == sizes && t.is_contiguous(), op, ": ", name, " must be contiguous, of the expected sizes; got ",
              dims(t));
}

// The cache's tensors. `half`: the 16-bit type of what is written, read or asked of it (Undefined: any).
KvPool check_pool(const at::Tensor& k, const at::Tensor& v, const OptTensor& ke, const OptTensor& ve, at::ScalarType half,
                  const char* op) {
  KvPool p{};
  TORCH_CHECK(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes(), op,
              ": k_pages and v_pages must both be [pages, heads, page size, head dim], got ", dims(k), " and ", dims(v));
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), op, ": k_pages and v_pages must have one dtype");
  const at::ScalarType dt = k.scalar_type();
  TORCH_CHECK(half_type(dt) || dt == at::kChar, op, ": a cache holds bf16, fp16 or, in 8 bits, int8 codes");
  TORCH_CHECK(dt == at::kChar || half == at::kByte || dt == half, op, ": a 16-bit cache must have the dtype of the tokens");
  const int64_t D = k.size(3), size = k.size(2);
  TORCH_CHECK(D == 16 || D == 32 || D == 64 || D == 128, op, ": head dim must be 16, 32, 64 or 128, got ", std::to_string(D));
  TORCH_CHECK(size >= 16 && size % 16 == 0 && size <= 65536, op,
              ": the page size must be a multiple of 16 in [16, 65536], got ", std::to_string(size));
  TORCH_CHECK(k.size(1) >= 1 && k.size(1) <= 65536, op, ": a cache needs 1 to 65536 heads");
  TORCH_CHECK(k.size(0) <= kIntMax, op, ": too many pages");
  for (const at::Tensor* t : {&k, &v}) {
    TORCH_CHECK(t->stride(3) == 1 && disjoint(*t), op, ": the cache's channels must be contiguous and no two slots overlap");
    const int64_t per = 16 / t->element_size();
    bool even = aligned16(*t);
    for (int i = 0; i < 3; ++i) even = even && (t->size(i) <= 1 || t->stride(i) % per == 0);
    TORCH_CHECK(even, op, ": the cache's slots must start on 16-byte boundaries");
    TORCH_CHECK(t->stride(0) < kStride && t->stride(1) < kStride && t->stride(2) < kStride, op,
                ": the cache's strides must be below 2^32 elements");
  }
  TORCH_CHECK(k.numel() == 0 || k.data_ptr() != v.data_ptr(), op, ": k_pages and v_pages must not be one buffer");
  p.k = k.data_ptr(), p.v = v.data_ptr();
  p.kp = k.stride(0), p.kh = k.stride(1), p.ks = k.stride(2);
  p.vp = v.stride(0), p.vh = v.stride(1), p.vs = v.stride(2);
  p.pages = static_cast<int>(k.size(0)), p.heads = static_cast<int>(k.size(1));
  p.size = static_cast<int>(size), p.dim = static_cast<int>(D);
  p.per_head = static_cast<uint32_t>(std::min((int64_t{1} << 32) / p.heads, (int64_t{1} << 32) - 1));
  p.per_slot = static_cast<uint32_t>((int64_t{1} << 32) / p.size);
  p.type = dt == at::kChar ? kKvCodes : dt == at::kHalf ? kKvF16 : kKvBf16;
  check_same_device(v, k.device(), op, "v_pages");
  TORCH_CHECK(given(ke) == (dt == at::kChar) && given(ve) == (dt == at::kChar), op,
              ": an int8 cache, and no other, has k_exp and v_exp");
  if (dt == at::kChar) {
    for (const at::Tensor* t : {&*ke, &*ve}) {
      TORCH_CHECK(t->scalar_type() == at::kByte && t->sizes() == k.sizes().slice(0, 3) &&
                      (t->stride(2) == 1) && disjoint(*t),
                  op, ": k_exp and v_exp must be uint8 [pages, heads, page size] with contiguous slots");
      TORCH_CHECK(t->stride(0) < kStride && t->stride(1) < kStride, op, ": the cache's strides must be below 2^32 elements");
      TORCH_CHECK(aligned16(*t) && (t->size(0) <= 1 || t->stride(0) % 16 == 0) && (t->size(1) <= 1 || t->stride(1) % 16 == 0),
                  op, ": the exponent bytes of a head of a page must start on a 16-byte boundary");
      check_same_device(*t, k.device(), op, "k_exp and v_exp");
    }
    TORCH_CHECK(ke->numel() == 0 || ke->data_ptr() != ve->data_ptr(), op, ": k_exp and v_exp must not be one buffer");
    p.ke = ke->data_ptr<uint8_t>(), p.ve = ve->data_ptr<uint8_t>();
    p.kep = ke->stride(0), p.keh = ke->stride(1), p.vep = ve->stride(0), p.veh = ve->stride(1);
  }
  return p;
}

void check_slots(const at::Tensor& slots, const char* op) {
  TORCH_CHECK(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous(), op,
              ": slots must be contiguous int64 [tokens]");
}
void check_rows(int64_t n, int64_t heads, const char* op) {
  TORCH_CHECK(n <= kIntMax / 16 / heads, op, ": too many tokens for one call");
}
// Whether every row of [n, heads, dim] starts on a 16-byte boundary.
bool rows_aligned(const at::Tensor& t) {
  return aligned16(t) && (t.size(0) <= 1 || t.stride(0) % 8 == 0) && (t.size(1) <= 1 || t.stride(1) % 8 == 0);
}

}  // namespace

void kv_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots, const at::Tensor& k_pages,
              const at::Tensor& v_pages, const OptTensor& k_exp, const OptTensor& v_exp) {
  const char* op = "kv_write";
  TORCH_CHECK(half_type(k.scalar_type()) && v.scalar_type() == k.scalar_type(), op, ": k and v must both be bf16 or fp16");
  const KvPool p = check_pool(k_pages, v_pages, k_exp, v_exp, k.scalar_type(), op);
  TORCH_CHECK(!overlap(k_pages, v_pages) && (p.type != kKvCodes || !overlap(*k_exp, *v_exp)), op,
              ": the cache's K and V must not overlap");
  check_slots(slots, op);
  TORCH_CHECK(k.dim() == 3 && k.sizes() == v.sizes() && k.size(0) == slots.size(0) && k.size(1) == p.heads &&
                  k.size(2) == p.dim,
              op, ": k and v must both be [tokens, heads, head dim] of the slots and the cache, got ", dims(k), " and ", dims(v));
  TORCH_CHECK(k.stride(2) == 1 && v.stride(2) == 1, op, ": the channels of k and v must be contiguous");
  for (const at::Tensor* x : {&k, &v})
    TORCH_CHECK(x->stride(0) < kStride && x->stride(1) < kStride, op, ": the strides of k and v must be below 2^32 elements");
  check_rows(k.size(0), p.heads, op);
  const at::Device dev = k_pages.device();
  check_same_device(k, dev, op, "k");
  check_same_device(v, dev, op, "v");
  check_same_device(slots, dev, op, "slots");
  TORCH_CHECK(k_pages.is_cuda(), op, ": the cache must be on a CUDA device");
  c10::cuda::CUDAGuard g(dev);
  KvTokens t{};
  t.k = k.data_ptr(), t.v = v.data_ptr();
  t.kt = k.stride(0), t.kh = k.stride(1), t.vt = v.stride(0), t.vh = v.stride(1);
  t.slots = slots.data_ptr<int64_t>();
  t.n = static_cast<int>(k.size(0));
  t.f16 = k.scalar_type() == at::kHalf;
  t.vec = rows_aligned(k) && rows_aligned(v);
  kv_write_launch(t, p, device_status_ptr(dev.index()), at::cuda::getCurrentCUDAStream());
}

std::tuple<at::Tensor, at::Tensor> kv_read(const at::Tensor& slots, const at::Tensor& k_pages, const at::Tensor& v_pages,
                                           const OptTensor& k_exp, const OptTensor& v_exp,
                                           const c10::optional<at::ScalarType>& dtype) {
  const char* op = "kv_read";
  const KvPool p = check_pool(k_pages, v_pages, k_exp, v_exp, at::kByte, op);
  check_slots(slots, op);
  const at::ScalarType dt = dtype ? *dtype : p.type == kKvCodes ? at::kBFloat16 : k_pages.scalar_type();
  TORCH_CHECK(half_type(dt) || dt == at::kFloat, op, ": dtype must be bf16, fp16 or fp32");
  TORCH_CHECK(p.type == kKvCodes || dt == k_pages.scalar_type(), op, ": a 16-bit cache is read in its own dtype");
  check_rows(slots.size(0), p.heads, op);
  const at::Device dev = k_pages.device();
  check_same_device(slots, dev, op, "slots");
  TORCH_CHECK(k_pages.is_cuda(), op, ": the cache must be on a CUDA device");
  c10::cuda::CUDAGuard g(dev);
  const int64_t n = slots.size(0);
  at::Tensor k = output({n, p.heads, p.dim}, dt, dev), v = output({n, p.heads, p.dim}, dt, dev);
  kv_read_launch(slots.data_ptr<int64_t>(), p, k.data_ptr(), v.data_ptr(), static_cast<int>(n),
                 dt == at::kFloat ? 2 : dt == at::kHalf ? 1 : 0, device_status_ptr(dev.index()),
                 at::cuda::getCurrentCUDAStream());
  return {k, v};
}

std::tuple<at::Tensor, at::Tensor> decode_attention(const at::Tensor& q, const at::Tensor& k_pages,
                                                    const at::Tensor& v_pages, const at::Tensor& table,
                                                    const at::Tensor& lengths, const OptTensor& k_exp,
                                                    const OptTensor& v_exp, const c10::optional<double>& scale) {
  const char* op = "decode_attention";
  TORCH_CHECK(half_type(q.scalar_type()), op, ": q must be bf16 or fp16");
  DecodeArgs a{};
  a.pool = check_pool(k_pages, v_pages, k_exp, v_exp, q.scalar_type(), op);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == a.pool.dim && q.stride(2) == 1, op,
              ": q must be [sequences, heads, head dim of the cache] with contiguous channels, got ", dims(q));
  TORCH_CHECK(q.size(1) >= 1 && q.size(1) % a.pool.heads == 0 && q.size(1) <= 65536, op,
              ": the query heads must be a multiple of the cache's ", std::to_string(a.pool.heads));
  const int64_t B = q.size(0);
  TORCH_CHECK(B <= kIntMax / q.size(1), op, ": too many sequences");
  TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == B &&
                  (table.size(1) <= 1 || table.stride(1) == 1) && table.stride(0) >= 0,
              op, ": table must be int32 [sequences, pages] with contiguous rows");
  TORCH_CHECK(table.size(1) <= kLongest / a.pool.size, op, ": table is too wide: at most ", std::to_string(kLongest), " tokens");
  check_plain(lengths, at::kInt, {B}, op, "lengths (int32 [sequences])");
  a.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(a.pool.dim)));
  TORCH_CHECK(std::isfinite(a.scale), op, ": scale must be finite");
  const at::Device dev = k_pages.device();
  check_same_device(q, dev, op, "q");
  check_same_device(table, dev, op, "table");
  check_same_device(lengths, dev, op, "lengths");
  TORCH_CHECK(k_pages.is_cuda(), op, ": the cache must be on a CUDA device");
  c10::cuda::CUDAGuard g(dev);
  at::Tensor out = output(q.sizes(), q.scalar_type(), dev), lse = output({B, q.size(1)}, at::kFloat, dev);
  a.qt = q.stride(0), a.qh = q.stride(1);
  a.q_vec = rows_aligned(q);
  a.f16 = q.scalar_type() == at::kHalf;
  a.tt = table.stride(0);
  a.longest = a.pool.pages == 0 ? 0 : static_cast<int>(table.size(1)) * a.pool.size;
  a.heads_q = static_cast<int>(q.size(1));
  a.status = device_status_ptr(dev.index());
  const int G = a.heads_q / a.pool.heads, cols = std::min(G, 8);
  DecodePlan plan;
  for (int64_t b = 0; b < B; b += plan.seqs) {
    plan = decode_attention_plan(a.pool, static_cast<int>(B - b), a.pool.heads * ((G + 7) / 8), a.longest);
    TORCH_CHECK(plan.seqs > 0, op, ": the table is too wide for so many heads");
    a.seqs = plan.seqs;
    a.q = static_cast<const uint16_t*>(q.data_ptr()) + b * a.qt;
    a.table = table.data_ptr<int>() + b * a.tt;
    a.lengths = lengths.data_ptr<int>() + b;
    a.out = static_cast<uint16_t*>(out.data_ptr()) + b * out.stride(0);
    a.lse = lse.data_ptr<float>() + b * a.heads_q;
    // Two parts and their records for each CTA. The next launch may be given the same memory: it begins when the join behind
    // this one has ended (only the join itself is launched early, beside the kernel that it waits for).
    at::Tensor part;
    a.record = nullptr;
    if (plan.split) {
      part = output({2l * plan.ctas * (2 + ((2 * cols + 3) & ~3) + static_cast<long>(cols) * a.pool.dim)}, at::kFloat, dev);
      a.record = reinterpret_cast<int2*>(part.data_ptr<float>());
      a.part = part.data_ptr<float>() + 4l * plan.ctas;
    }
    decode_attention_launch(a, plan, at::cuda::getCurrentCUDAStream());
  }
  return {out, lse};
}

at::Tensor sample_tokens(const at::Tensor& logits, int64_t V, const at::Tensor& u, const OptTensor& temperature,
                         double temperature0, const OptTensor& top_k, int64_t top_k0, const OptTensor& top_p,
                         double top_p0, const OptTensor& min_p, double min_p0) {
  const char* op = "sample_tokens";
  SampleArgs a{};
  switch (logits.scalar_type()) {
    case at::kBFloat16: a.type = 0; break;
    case at::kHalf: a.type = 1; break;
    case at::kFloat: a.type = 2; break;
    default: TORCH_CHECK(false, op, ": logits must be bf16, fp16 or fp32");
  }
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1) && logits.stride(0) >= 0, op,
              ": logits must be 2-D with contiguous rows");
  const int64_t M = logits.size(0);
  TORCH_CHECK(V >= 1 && V <= logits.size(1), op, ": V must be in [1, row width]");
  TORCH_CHECK(V <= kMaxVocab, op, ": V must be at most ", std::to_string(kMaxVocab));
  TORCH_CHECK(M <= kIntMax / 16, op, ": too many rows");
  check_plain(u, at::kFloat, {M}, op, "u (fp32 [rows])");
  const at::Device dev = logits.device();
  check_same_device(u, dev, op, "u");
  const auto setting = [&](const OptTensor& t, at::ScalarType dt, const char* name) -> const void* {
    if (!given(t)) return nullptr;
    check_plain(*t, dt, {M}, op, name);
    check_same_device(*t, dev, op, name);
    return t->data_ptr();
  };
  a.temperature = static_cast<const float*>(setting(temperature, at::kFloat, "temperature (fp32 [rows])"));
  a.top_k = static_cast<const int64_t*>(setting(top_k, at::kLong, "top_k (int64 [rows])"));
  a.top_p = static_cast<const float*>(setting(top_p, at::kFloat, "top_p (fp32 [rows])"));
  a.min_p = static_cast<const float*>(setting(min_p, at::kFloat, "min_p (fp32 [rows])"));
  TORCH_CHECK(!std::isnan(temperature0) && !std::isnan(top_p0) && !std::isnan(min_p0), op, ": a setting is not a number");
  TORCH_CHECK(logits.is_cuda(), op, ": logits must be on a CUDA device");
  c10::cuda::CUDAGuard g(dev);
  at::Tensor tokens = output({M}, at::kLong, dev);
  a.x = logits.data_ptr(), a.ld = logits.stride(0);
  a.rows = static_cast<int>(M), a.V = static_cast<int>(V);
  a.u = u.data_ptr<float>();
  a.temperature0 = temperature0, a.top_p0 = top_p0, a.min_p0 = min_p0, a.top_k0 = top_k0;
  a.tokens = tokens.data_ptr<int64_t>();
  sample_tokens_launch(a, at::cuda::getCurrentCUDAStream());
  return tokens;
}

}  // namespace hb
