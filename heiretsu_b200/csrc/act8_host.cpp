// Torch-facing entry points of the 8-bit activations (act8.cu): argument checks, stream selection,
// then the raw launchers. Refused calls raise before anything is launched. Numbers go into the messages as
// strings: an extension whose linker brought its own static libstdc++ faults when it streams them.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <limits>
#include <string>

#include "host_utils.h"
#include "ops.h"

namespace hb {

void act8_pack_launch(const void* x, long ld, int type, int8_t* q, uint8_t* e, long M, int N, cudaStream_t s);
void act8_unpack_launch(const int8_t* q, const uint8_t* e, int type, void* x, void* h, long M, int N, cudaStream_t s);
void ln_fwd_act8_launch(const float* x, const float* w, const float* b, void* y, int8_t* q, uint8_t* e, float* rstd,
                        int M, int H, float eps, bool f16, cudaStream_t s);
int ln_bwd_act8_ctas(int M, int H, int device);
void ln_bwd_act8_launch(const float* dy, const int8_t* q, const uint8_t* e, const float* rstd, const float* w,
                        const float* b, const float* dres_in, float* dres, void* dres16, void* y, float* part, int ctas,
                        float* dgamma, float* dbeta, int M, int H, bool f16, cudaStream_t s);

namespace {

constexpr int64_t kIntMax = std::numeric_limits<int>::max();
constexpr int64_t kBlock = 128;

// Element type as the kernels number it: 0 bf16, 1 fp16, 2 fp32.
int act_type(const at::Tensor& t, const char* op, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, op, ": ", name, " must be bf16, fp16 or fp32");
  }
}

void check_mat(const at::Tensor& t, at::ScalarType dt, int64_t M, int64_t N, const at::Device& dev, const char* op,
               const char* name) {
  TORCH_CHECK(t.device() == dev, op, ": ", name, " must be on ", dev.str());
  TORCH_CHECK(t.scalar_type() == dt, op, ": ", name, " has the wrong dtype");
  TORCH_CHECK(t.dim() == 2 && t.size(0) == M && t.size(1) == N && t.is_contiguous(), op, ": ", name,
              " must be contiguous [", std::to_string(M), ", ", std::to_string(N), "]");
}
void check_vec(const at::Tensor& t, int64_t n, const at::Device& dev, const char* op, const char* name) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == n, op, ": ", name,
              " must be ", std::to_string(n), " contiguous fp32 values on ", dev.str());
}
void check_codes(const at::Tensor& q, const at::Tensor& e, const char* op) {
  TORCH_CHECK(q.is_cuda(), op, ": q must be a CUDA tensor");
  TORCH_CHECK(q.dim() == 2 && q.size(1) <= kIntMax - kBlock, op, ": q must be [rows, columns]");
  check_mat(q, at::kChar, q.size(0), q.size(1), q.device(), op, "q");
  const int64_t nb = (q.size(1) + kBlock - 1) / kBlock;
  check_mat(e, at::kByte, q.size(0), nb, q.device(), op, "e");
  TORCH_CHECK(q.size(0) == 0 || nb <= (kIntMax - 64) / q.size(0), op, ": too many blocks");
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// The LayerNorm kernels read rows in 16-byte (fp32) pieces.
void check_width(int64_t M, int64_t H, const char* op) {
  TORCH_CHECK(H >= 4 && H % 4 == 0 && H <= 2048, op, ": the width must be a multiple of 4 in [4, 2048], got ",
              std::to_string(H));
  TORCH_CHECK(M <= kIntMax / 2, op, ": too many rows");
}

// Empty codes and exponent bytes of an [M, N] activation.
std::pair<at::Tensor, at::Tensor> codes_like(const at::Tensor& x) {
  const auto opts = x.options();
  return {at::empty(x.sizes(), opts.dtype(at::kChar)),
          at::empty({x.size(0), (x.size(1) + kBlock - 1) / kBlock}, opts.dtype(at::kByte))};
}
void check_out_type(at::ScalarType dt, const char* op) {
  TORCH_CHECK(dt == at::kBFloat16 || dt == at::kHalf || dt == at::kFloat, op, ": dtype must be bf16, fp16 or fp32");
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> act8_pack(const at::Tensor& x) {
  const char* op = "act8_pack";
  TORCH_CHECK(x.is_cuda(), op, ": x must be a CUDA tensor");
  TORCH_CHECK(x.dim() == 2 && (x.size(1) <= 1 || x.stride(1) == 1) && x.stride(0) >= 0, op,
              ": x must be 2-D with contiguous rows");
  const int type = act_type(x, op, "x");
  c10::cuda::CUDAGuard g(x.device());
  auto [q, e] = codes_like(x);
  check_codes(q, e, op);
  act8_pack_launch(x.data_ptr(), x.stride(0), type, q.data_ptr<int8_t>(), e.data_ptr<uint8_t>(), x.size(0),
                   static_cast<int>(x.size(1)), at::cuda::getCurrentCUDAStream());
  return {q, e};
}

std::tuple<at::Tensor, at::Tensor> act8_unpack(const at::Tensor& q, const at::Tensor& e, at::ScalarType dtype,
                                               bool gelu) {
  const char* op = gelu ? "act8_unpack_gelu" : "act8_unpack";
  check_codes(q, e, op);
  check_out_type(dtype, op);
  c10::cuda::CUDAGuard g(q.device());
  at::Tensor x = at::empty(q.sizes(), q.options().dtype(dtype)), h;
  if (gelu) h = at::empty_like(x);
  act8_unpack_launch(q.data_ptr<int8_t>(), e.data_ptr<uint8_t>(), act_type(x, op, "x"), x.data_ptr(),
                     gelu ? h.data_ptr() : nullptr, q.size(0), static_cast<int>(q.size(1)),
                     at::cuda::getCurrentCUDAStream());
  return {x, h};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> layernorm_fwd_act8(const at::Tensor& x, const at::Tensor& w,
                                                                              const at::Tensor& b, double eps,
                                                                              at::ScalarType dtype) {
  const char* op = "layernorm_fwd_act8";
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, op, ": x must be a CUDA matrix");
  c10::cuda::CUDAGuard g(x.device());
  const at::Device dev = x.device();
  const int64_t M = x.size(0), H = x.size(1);
  check_width(M, H, op);
  check_mat(x, at::kFloat, M, H, dev, op, "x");
  check_vec(w, H, dev, op, "w");
  check_vec(b, H, dev, op, "b");
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kHalf, op, ": dtype must be bf16 or fp16");
  TORCH_CHECK(aligned16(x) && aligned16(w) && aligned16(b), op, ": x, w and b must start on 16-byte boundaries");
  auto [q, e] = codes_like(x);
  at::Tensor y = at::empty({M, H}, x.options().dtype(dtype)), rstd = at::empty({M}, x.options());
  ln_fwd_act8_launch(x.data_ptr<float>(), w.data_ptr<float>(), b.data_ptr<float>(), y.data_ptr(), q.data_ptr<int8_t>(),
                     e.data_ptr<uint8_t>(), rstd.data_ptr<float>(), static_cast<int>(M), static_cast<int>(H),
                     static_cast<float>(eps), dtype == at::kHalf, at::cuda::getCurrentCUDAStream());
  return {y, q, e, rstd};
}

at::Tensor layernorm_bwd_act8(const at::Tensor& dy, const at::Tensor& q, const at::Tensor& e, const at::Tensor& rstd,
                              const at::Tensor& w, const at::Tensor& b, const at::Tensor& dres_in, at::Tensor& dres,
                              at::Tensor& dres16, at::Tensor& dgamma, at::Tensor& dbeta) {
  const char* op = "layernorm_bwd_act8";
  check_codes(q, e, op);
  c10::cuda::CUDAGuard g(q.device());
  const at::Device dev = q.device();
  const int64_t M = q.size(0), H = q.size(1);
  check_width(M, H, op);
  check_mat(dy, at::kFloat, M, H, dev, op, "dy");
  check_vec(rstd, M, dev, op, "rstd");
  check_vec(w, H, dev, op, "w");
  check_vec(b, H, dev, op, "b");
  check_mat(dres_in, at::kFloat, M, H, dev, op, "dres_in");
  check_mat(dres, at::kFloat, M, H, dev, op, "dres");
  const auto from = reinterpret_cast<uintptr_t>(dres_in.data_ptr()), to = reinterpret_cast<uintptr_t>(dres.data_ptr());
  const auto bytes = static_cast<uintptr_t>(M * H * 4);
  TORCH_CHECK(from == to || from + bytes <= to || to + bytes <= from, op,
              ": dres must be dres_in itself or not overlap it");
  TORCH_CHECK(act_type(dres16, op, "dres16") != 2, op, ": dres16 must be bf16 or fp16");
  check_mat(dres16, dres16.scalar_type(), M, H, dev, op, "dres16");
  check_vec(dgamma, H, dev, op, "dgamma");
  check_vec(dbeta, H, dev, op, "dbeta");
  const int ctas = ln_bwd_act8_ctas(static_cast<int>(M), static_cast<int>(H), q.get_device());
  TORCH_CHECK(aligned16(dy) && aligned16(q) && aligned16(w) && aligned16(b) && aligned16(dres_in) && aligned16(dres) &&
                  aligned16(dres16),
              op, ": every matrix must start on a 16-byte boundary");
  const auto gamma = reinterpret_cast<uintptr_t>(dgamma.data_ptr()), beta = reinterpret_cast<uintptr_t>(dbeta.data_ptr());
  TORCH_CHECK(gamma + H * 4 <= beta || beta + H * 4 <= gamma, op, ": dgamma and dbeta must not overlap");
  at::Tensor y = at::empty({M, H}, dres16.options()), scratch = at::empty({ctas * 2 * H}, dy.options());
  ln_bwd_act8_launch(dy.data_ptr<float>(), q.data_ptr<int8_t>(), e.data_ptr<uint8_t>(), rstd.data_ptr<float>(),
                     w.data_ptr<float>(), b.data_ptr<float>(), dres_in.data_ptr<float>(), dres.data_ptr<float>(),
                     dres16.data_ptr(), y.data_ptr(), scratch.data_ptr<float>(), ctas, dgamma.data_ptr<float>(),
                     dbeta.data_ptr<float>(), static_cast<int>(M), static_cast<int>(H),
                     dres16.scalar_type() == at::kHalf, at::cuda::getCurrentCUDAStream());
  return y;
}

}  // namespace hb
