// Weight gradient of a projection whose input was kept in 8 bits:
//   grad_w[n, k] = sum_m grad[m, n] * (q[m, k] * scale[m])
#include "quant_common.cuh"

namespace hlm {

template <typename T>
__global__ void __launch_bounds__(256) weight_grad_q8_simple_kernel(
    const T* __restrict__ grad, const int8_t* __restrict__ q, const float* __restrict__ scale,
    T* __restrict__ grad_w, int64_t tokens, int64_t N, int64_t K) {
  const int64_t total = N * K;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t n = i / K, k = i - n * K;
    float acc = 0.0f;
    for (int64_t m = 0; m < tokens; ++m)
      acc += to_f32(grad[m * N + n]) * (static_cast<float>(q[m * K + k]) * scale[m]);
    grad_w[i] = from_f32<T>(acc);
  }
}

}  // namespace hlm

using namespace hlm;

extern "C" size_t hlm_weight_grad_q8_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int hlm_weight_grad_q8(const void* grad, const void* q, const float* scale, void* grad_w,
                                  void* workspace, size_t workspace_bytes, int64_t tokens, int64_t N,
                                  int64_t K, int dtype, void* stream) {
  if (tokens < 0 || N < 0 || K < 0) return HLM_ERR_INVALID_ARG;
  if (dtype != HLM_BF16 && dtype != HLM_F16) return HLM_ERR_UNSUPPORTED;
  if (N == 0 || K == 0) return HLM_OK;
  if (grad_w == nullptr) return HLM_ERR_INVALID_ARG;
  if (N % 8 != 0 || K % 16 != 0 || tokens > (1ll << 31) - 512 || N > (1ll << 30) || K > (1ll << 30))
    return HLM_ERR_UNSUPPORTED;
  if (!host_aligned16(grad_w)) return HLM_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tokens == 0) {  // an empty sum
    return cudaMemsetAsync(grad_w, 0, static_cast<size_t>(N) * static_cast<size_t>(K) * 2, s) == cudaSuccess
               ? HLM_OK
               : HLM_ERR_LAUNCH;
  }
  if (grad == nullptr || q == nullptr || scale == nullptr) return HLM_ERR_INVALID_ARG;
  if (!host_aligned16(grad) || !host_aligned16(q)) return HLM_ERR_UNSUPPORTED;
  const size_t need = hlm_weight_grad_q8_workspace_bytes(tokens, N, K);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return HLM_ERR_WORKSPACE;
  const int64_t blocks64 = (N * K + 255) / 256;
  const int64_t cap = static_cast<int64_t>(num_sms_of_current_device()) * 64;
  const int blocks = static_cast<int>(blocks64 < cap ? blocks64 : cap);
  LaunchScope scope(HLM_KERNEL_WEIGHT_GRAD_Q8, s);
  if (dtype == HLM_BF16)
    weight_grad_q8_simple_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(
        static_cast<const __nv_bfloat16*>(grad), static_cast<const int8_t*>(q), scale,
        static_cast<__nv_bfloat16*>(grad_w), tokens, N, K);
  else
    weight_grad_q8_simple_kernel<__half><<<blocks, 256, 0, s>>>(
        static_cast<const __half*>(grad), static_cast<const int8_t*>(q), scale,
        static_cast<__half*>(grad_w), tokens, N, K);
  return launch_status();
}
