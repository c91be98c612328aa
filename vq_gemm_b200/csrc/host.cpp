// Host side of the 4-bit products, their quantiser, the expert router and the experts' layer for Python: argument checks,
// allocation and the call into the C ABI (include/vqg.h) in one native call.  These operators are called once per layer and
// token; checked and marshalled in Python, a call took 11 us, twice what its kernel does for one token.
//
// Module vq_gemm_b200._host; vq_gemm_b200/ops.py and quantize.py are its only callers and document the operators.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>

#include "../../include/vqg.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void check_status(int st, const char* what) {
  TORCH_CHECK(st == VQG_OK, what, ": ", vqg_status_string(st), " (status ", st, ")");
}

void check_cuda(const Tensor& first, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "vq_gemm_b200 has no CPU path: all tensors must be CUDA tensors");
  TORCH_CHECK(t.device() == first.device(), "all tensors must be on the same CUDA device");
  TORCH_CHECK(t.is_contiguous(), "tensors must be contiguous");
}

const void* ptr(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }

// dtype code of the C ABI, or -1
int float_code(const Tensor& t) { return t.scalar_type() == at::kHalf ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1; }

struct Weight {
  int64_t N, group, experts;
};
// A 4-bit weight with K input features, after checking that its tensors fit one another (ops._int4_weight is the same rule).
Weight check_weight(const Tensor& packed, const Tensor& scales, const OptTensor& zeros, int64_t K, bool experts) {
  TORCH_CHECK(packed.scalar_type() == at::kByte && float_code(scales) >= 0,
              "4-bit weights need packed uint8 and scales float16 or bfloat16");
  const int64_t lead = experts ? 1 : 0;
  TORCH_CHECK(packed.dim() == 3 + lead && scales.dim() == 2 + lead && packed.size(-1) == 512,
              "4-bit weights need packed [ceil(N/16), ceil(K/64), 512] and scales [K/group, N]",
              experts ? ", each with a leading dimension of experts" : "");
  const int64_t G = scales.size(-2), N = scales.size(-1);
  TORCH_CHECK(G >= 1 && K >= 1 && K % G == 0 && packed.size(-3) == (N + 15) / 16 && packed.size(-2) == (K + 63) / 64 &&
                  (!experts || packed.size(0) == scales.size(0)),
              "packed ", packed.sizes(), " and scales ", scales.sizes(), " do not match K=", K);
  const int64_t group = K / G;
  TORCH_CHECK(K % 32 == 0 && (group == 32 || group % 64 == 0 || G == 1), "K=", K, " in groups of ", group,
              ": K must be a multiple of 32 and a group 32, a multiple of 64, or K");
  TORCH_CHECK(N < (int64_t(1) << 31) && K < (int64_t(1) << 31), "weight too large");
  if (zeros) TORCH_CHECK(zeros->scalar_type() == at::kByte && zeros->sizes() == scales.sizes(), "zeros must be uint8 and of the shape of scales");
  return {N, group, experts ? packed.size(0) : 1};
}

Tensor output(const OptTensor& out, at::IntArrayRef shape, const Tensor& like, const char* what) {
  if (!out) return at::empty(shape, like.options());
  TORCH_CHECK(out->sizes() == shape && out->scalar_type() == like.scalar_type() && out->is_contiguous() && out->device() == like.device(),
              "out must be a contiguous ", what);
  return *out;
}

Tensor int4_gemm(const Tensor& x, const Tensor& packed, const Tensor& scales, const OptTensor& zeros, const OptTensor& out) {
  check_cuda(x, x); check_cuda(x, packed); check_cuda(x, scales);
  if (zeros) check_cuda(x, *zeros);
  TORCH_CHECK(x.dim() == 2 && x.scalar_type() == scales.scalar_type(), "x must be [M, K] and of the type of scales");
  const int64_t M = x.size(0), K = x.size(1);
  const Weight w = check_weight(packed, scales, zeros, K, false);
  TORCH_CHECK(M < (int64_t(1) << 31), "too many rows");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = output(out, {M, w.N}, x, "[M, N] tensor of x's type on the inputs' device");
  // Scratch belongs to the call: graphs captured on one stream may be replayed on two.
  const size_t need = vqg_int4_workspace_bytes(static_cast<int>(M), w.N, static_cast<int>(K));
  Tensor ws;
  if (need) ws = at::empty({static_cast<int64_t>(need)}, x.options().dtype(at::kByte));
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = vqg_int4_gemm(x.const_data_ptr(), packed.const_data_ptr(), scales.const_data_ptr(), ptr(zeros), y.mutable_data_ptr(),
                       M, w.N, K, w.group, float_code(x), need ? ws.mutable_data_ptr() : nullptr,
                       need, s);
  }
  check_status(st, "int4_gemm");
  return y;
}

Tensor int4_dequant(const Tensor& packed, const Tensor& scales, const OptTensor& zeros, int64_t K, const OptTensor& out) {
  check_cuda(packed, packed); check_cuda(packed, scales);
  if (zeros) check_cuda(packed, *zeros);
  const bool experts = packed.dim() == 4;
  TORCH_CHECK(packed.dim() >= 3, "4-bit weights need packed [ceil(N/16), ceil(K/64), 512] and scales [K/group, N]");
  if (K < 0) K = packed.size(-2) * 64;
  const Weight w = check_weight(packed, scales, zeros, K, experts);
  c10::cuda::CUDAGuard guard(packed.device());
  Tensor y = experts ? output(out, {w.experts, w.N, K}, scales, "[E, N, K] tensor of the type of scales on the inputs' device")
                     : output(out, {w.N, K}, scales, "[N, K] tensor of the type of scales on the inputs' device");
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = vqg_int4_dequant(packed.const_data_ptr(), scales.const_data_ptr(), ptr(zeros), y.mutable_data_ptr(), w.experts, w.N, K,
                          w.group, float_code(scales), s);
  }
  check_status(st, "int4_dequant");
  return y;
}

std::tuple<Tensor, Tensor, OptTensor> int4_quantize(const Tensor& weight, int64_t group, bool symmetric) {
  check_cuda(weight, weight);
  TORCH_CHECK((weight.dim() == 2 || weight.dim() == 3) && float_code(weight) >= 0,
              "weight must be a float16 or bfloat16 [N, K] or [E, N, K] tensor");
  const int64_t N = weight.size(-2), K = weight.size(-1), E = weight.dim() == 3 ? weight.size(0) : 1;
  if (group == 0) group = K;
  TORCH_CHECK(N >= 1 && K >= 1 && K % 32 == 0 && group >= 1 && K % group == 0 && (group == 32 || group % 64 == 0 || group == K),
              "K=", K, " in groups of ", group, ": K must be a multiple of 32 and a group 32, a multiple of 64, or K");
  TORCH_CHECK(N < (int64_t(1) << 31) && K < (int64_t(1) << 31), "weight too large");
  c10::cuda::CUDAGuard guard(weight.device());
  c10::SmallVector<int64_t, 4> packed_shape{(N + 15) / 16, (K + 63) / 64, 512}, scale_shape{K / group, N};
  if (weight.dim() == 3) {
    packed_shape.insert(packed_shape.begin(), E);
    scale_shape.insert(scale_shape.begin(), E);
  }
  Tensor packed = at::empty(packed_shape, weight.options().dtype(at::kByte)), scales = at::empty(scale_shape, weight.options());
  OptTensor zeros;
  if (!symmetric) zeros = at::empty(scale_shape, weight.options().dtype(at::kByte));
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = vqg_int4_quantize(weight.const_data_ptr(), packed.mutable_data_ptr(), scales.mutable_data_ptr(),
                           zeros ? zeros->mutable_data_ptr() : nullptr, E, N, K, group, float_code(weight), s);
  }
  check_status(st, "quantize.int4_quantize");
  return {packed, scales, zeros};
}

std::tuple<Tensor, Tensor> route_experts(const Tensor& logits, int64_t top_k, const std::string& scoring, const OptTensor& bias,
                                         int64_t groups, std::optional<int64_t> top, const std::string& group_score,
                                         bool renormalize, double scale) {
  check_cuda(logits, logits);
  if (bias) check_cuda(logits, *bias);
  const int type = logits.scalar_type() == at::kFloat ? 2 : float_code(logits);
  TORCH_CHECK(logits.dim() == 2 && type >= 0, "logits must be [T, E], float16, bfloat16 or float32");
  const int64_t T = logits.size(0), E = logits.size(1), top_groups = top.value_or(groups);
  const bool sigmoid = scoring == "sigmoid", largest = group_score == "max";
  TORCH_CHECK((sigmoid || scoring == "softmax") && (largest || group_score == "top2"),
              "scoring must be softmax or sigmoid, group_score top2 or max");
  if (bias) TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == E, "bias must be a float32 [E] tensor");
  TORCH_CHECK(E >= 1 && top_k >= 1 && top_k <= E && groups >= 1 && E % groups == 0 && top_groups >= 1 && top_groups <= groups,
              "cannot choose ", top_k, " of ", E, " experts in ", top_groups, " of ", groups, " groups");
  TORCH_CHECK(T < (int64_t(1) << 31) && E < (int64_t(1) << 31), "too many rows");
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor weights = at::empty({T, top_k}, logits.options().dtype(at::kFloat)), ids = at::empty({T, top_k}, logits.options().dtype(at::kInt));
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = vqg_route_experts(logits.const_data_ptr(), ptr(bias), weights.mutable_data_ptr(), ids.mutable_data_ptr(), T, E, top_k,
                           sigmoid, groups, top_groups, largest, renormalize, static_cast<float>(scale), type, s);
  }
  check_status(st, "route_experts");
  return {weights, ids};
}

Tensor int4_experts(const Tensor& x, const Tensor& experts, const Tensor& weights, const Tensor& up_packed, const Tensor& up_scales,
                    const OptTensor& up_zeros, const Tensor& down_packed, const Tensor& down_scales, const OptTensor& down_zeros,
                    const OptTensor& out) {
  for (const Tensor* t : {&x, &experts, &weights, &up_packed, &up_scales, &down_packed, &down_scales}) check_cuda(x, *t);
  if (up_zeros) check_cuda(x, *up_zeros);
  if (down_zeros) check_cuda(x, *down_zeros);
  TORCH_CHECK(x.dim() == 2 && x.scalar_type() == up_scales.scalar_type() && x.scalar_type() == down_scales.scalar_type(),
              "x must be [T, hidden] and of the type of both weights' scales");
  const int64_t T = x.size(0), hidden = x.size(1);
  TORCH_CHECK(experts.dim() == 2 && experts.size(0) == T && experts.scalar_type() == at::kInt && experts.size(1) >= 1,
              "experts must be an int32 [T, top_k] tensor");
  TORCH_CHECK(weights.sizes() == experts.sizes() && weights.scalar_type() == at::kFloat,
              "weights must be a float32 tensor of the shape of experts");
  const Weight up = check_weight(up_packed, up_scales, up_zeros, hidden, true);
  TORCH_CHECK(up.N >= 2 && up.N % 2 == 0, "gate_up needs an even number of rows (gate, up pairs)");
  const int64_t inner = up.N / 2, E = up.experts, top_k = experts.size(1);
  const Weight down = check_weight(down_packed, down_scales, down_zeros, inner, true);
  TORCH_CHECK(down.N == hidden && down.experts == E, "down must be [", E, ", ", hidden, ", ", inner, "] to follow gate_up");
  TORCH_CHECK(T < (int64_t(1) << 31) && top_k < (int64_t(1) << 31) && T * top_k < (int64_t(1) << 31), "too many rows");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = output(out, {T, hidden}, x, "[T, hidden] tensor of x's type on the inputs' device");
  const size_t need = vqg_int4_experts_workspace_bytes(T, top_k, E, hidden, inner);
  Tensor ws = at::empty({static_cast<int64_t>(need)}, x.options().dtype(at::kByte));
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = vqg_int4_experts(x.const_data_ptr(), experts.const_data_ptr(), weights.const_data_ptr(), up_packed.const_data_ptr(),
                          up_scales.const_data_ptr(), ptr(up_zeros), down_packed.const_data_ptr(), down_scales.const_data_ptr(),
                          ptr(down_zeros), y.mutable_data_ptr(), T, top_k, E, hidden, inner, up.group, down.group, float_code(x),
                          ws.mutable_data_ptr(), need, s);
  }
  check_status(st, "int4_experts");
  return y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("int4_gemm", &int4_gemm);
  m.def("int4_dequant", &int4_dequant);
  m.def("int4_quantize", &int4_quantize);
  m.def("route_experts", &route_experts);
  m.def("int4_experts", &int4_experts);
}
