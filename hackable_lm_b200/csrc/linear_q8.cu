// 8-bit integer projection: y[m, n] = (sum_k q[m, k] w[n, k]) * scale[m] * w_scale[n],
// q and w int8 (K contiguous), exact int32 sums.
#include "quant_common.cuh"

namespace hlm {

template <typename T>
__global__ void __launch_bounds__(256) linear_q8_simple_kernel(
    const int8_t* __restrict__ q, const float* __restrict__ scale, const int8_t* __restrict__ w,
    const float* __restrict__ w_scale, T* __restrict__ out, int64_t M, int64_t N, int64_t K) {
  const int64_t total = M * N;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t m = i / N, n = i - m * N;
    const int8_t* a = q + m * K;
    const int8_t* b = w + n * K;
    int acc = 0;
    for (int64_t k = 0; k < K; k += 16) {
      const uint4 x = ld_global_v4(a + k), y = ld_global_v4(b + k);
      acc = __dp4a(static_cast<int>(x.x), static_cast<int>(y.x), acc);
      acc = __dp4a(static_cast<int>(x.y), static_cast<int>(y.y), acc);
      acc = __dp4a(static_cast<int>(x.z), static_cast<int>(y.z), acc);
      acc = __dp4a(static_cast<int>(x.w), static_cast<int>(y.w), acc);
    }
    out[i] = from_f32<T>(static_cast<float>(acc) * scale[m] * w_scale[n]);
  }
}

}  // namespace hlm

using namespace hlm;

extern "C" int hlm_linear_q8(const void* q, const float* scale, const void* w, const float* w_scale,
                             void* out, int64_t M, int64_t N, int64_t K, int out_dtype, void* stream) {
  if (M < 0 || N < 0 || K < 0) return HLM_ERR_INVALID_ARG;
  if (out_dtype != HLM_F32 && out_dtype != HLM_BF16 && out_dtype != HLM_F16)
    return HLM_ERR_UNSUPPORTED;
  if (M == 0 || N == 0) return HLM_OK;
  if (q == nullptr || scale == nullptr || w == nullptr || w_scale == nullptr || out == nullptr)
    return HLM_ERR_INVALID_ARG;
  // 128 * 128 * K stays within int32 up to K = 131056; TMA rows are 16-byte multiples
  if (K == 0 || K % 16 != 0 || K > HLM_LINEAR_Q8_MAX_K) return HLM_ERR_UNSUPPORTED;
  if (M > (1ll << 31) - 512 || N > (1ll << 31) - 512) return HLM_ERR_UNSUPPORTED;
  if (!host_aligned16(q) || !host_aligned16(w)) return HLM_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t blocks64 = (M * N + 255) / 256;
  const int64_t cap = static_cast<int64_t>(num_sms_of_current_device()) * 64;
  const int blocks = static_cast<int>(blocks64 < cap ? blocks64 : cap);
  LaunchScope scope(HLM_KERNEL_LINEAR_Q8, s);
  const int8_t* qp = static_cast<const int8_t*>(q);
  const int8_t* wp = static_cast<const int8_t*>(w);
  if (out_dtype == HLM_BF16)
    linear_q8_simple_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(
        qp, scale, wp, w_scale, static_cast<__nv_bfloat16*>(out), M, N, K);
  else if (out_dtype == HLM_F16)
    linear_q8_simple_kernel<__half><<<blocks, 256, 0, s>>>(qp, scale, wp, w_scale,
                                                           static_cast<__half*>(out), M, N, K);
  else
    linear_q8_simple_kernel<float><<<blocks, 256, 0, s>>>(qp, scale, wp, w_scale,
                                                          static_cast<float*>(out), M, N, K);
  return launch_status();
}
