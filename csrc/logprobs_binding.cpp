// Torch-facing wrapper of csrc/logprobs.cu.  What a call looks at on the host is checked before the device, so that a refused call is
// refused anywhere.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/pybind11.h>
#include <torch/extension.h>

#include "logprobs.h"

namespace py = pybind11;
using namespace penny;

namespace {
void need(bool ok, const char* msg) { TORCH_CHECK(ok, "penny: ", msg); }
}  // namespace

void bind_logprobs(py::module_& m) {
  m.attr("LOGPROBS_MAX_TOP") = kLogprobsMaxTop;
  // logits [rows, vocab]; returns (logprobs [rows], entropy [rows], top_logprobs [rows, top] fp32, top_ids [rows, top] int64).
  m.def("token_logprobs", [](at::Tensor logits, at::Tensor tokens, int64_t top) {
    const at::ScalarType t = logits.scalar_type();
    need(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, "token_logprobs: bf16, fp16 or fp32 logits");
    need(logits.dim() == 2 && logits.size(1) >= 1 && logits.size(1) <= (1 << 30) && logits.size(0) < (1ll << 28), "token_logprobs: logits [rows, vocab]");
    const int64_t R = logits.size(0), V = logits.size(1);
    need((V == 1 || logits.stride(1) == 1) && (R <= 1 || logits.stride(0) >= 0), "token_logprobs: logits with contiguous rows");
    need(tokens.scalar_type() == at::kLong && tokens.is_contiguous() && tokens.dim() == 1 && tokens.numel() == R, "token_logprobs: tokens [rows] int64");
    need(top >= 0 && top <= kLogprobsMaxTop && top <= V, "token_logprobs: a top of LOGPROBS_MAX_TOP tokens at most, and of the vocabulary");
    need(!logits.requires_grad() || !at::GradMode::is_enabled(), "token_logprobs: no gradients");
    need(logits.is_cuda() && tokens.device() == logits.device(), "token_logprobs expects tensors on one CUDA device");
    const at::cuda::OptionalCUDAGuard guard(logits.device());
    const at::Tensor both = at::detail::empty_cuda({2, R}, at::kFloat, logits.device(), c10::nullopt);
    const at::Tensor top_logprobs = at::detail::empty_cuda({R, top}, at::kFloat, logits.device(), c10::nullopt);
    const at::Tensor top_ids = at::detail::empty_cuda({R, top}, at::kLong, logits.device(), c10::nullopt);
    const TokenLogprobs a = {logits.data_ptr(), logits.stride(0), (const long long*)tokens.data_ptr<int64_t>(), both.data_ptr<float>(),
                             both.data_ptr<float>() + R, top_logprobs.data_ptr<float>(), (long long*)top_ids.data_ptr<int64_t>(), (int)R, (int)V, (int)top};
    int sms = 0;
    cudaError_t rc = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, logits.get_device());
    if (rc == cudaSuccess)
      rc = launch_token_logprobs(a, t == at::kBFloat16 ? LOGITS_BF16 : t == at::kHalf ? LOGITS_FP16 : LOGITS_FP32, sms,
                                 at::cuda::getCurrentCUDAStream().stream());
    TORCH_CHECK(rc == cudaSuccess, "penny: token_logprobs: ", cudaGetErrorString(rc));
    return std::make_tuple(both[0], both[1], top_logprobs, top_ids);
  }, py::arg("logits"), py::arg("tokens"), py::arg("top") = 0);
}
