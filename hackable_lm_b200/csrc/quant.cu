// Operators that write or read the 8-bit format of quant_common.cuh: rows
// quantised and read back, residual-add + RMSNorm with an 8-bit output, and
// SwiGLU that keeps its input in 8 bits for the backward pass.
#include "quant_common.cuh"

namespace hlm {

#define HLM_QUANT_DISPATCH(dtype, T, ...) \
  switch (dtype) {                        \
    case HLM_F32: {                       \
      using T = float;                    \
      __VA_ARGS__;                        \
      break;                              \
    }                                     \
    case HLM_BF16: {                      \
      using T = __nv_bfloat16;            \
      __VA_ARGS__;                        \
      break;                              \
    }                                     \
    case HLM_F16: {                       \
      using T = __half;                   \
      __VA_ARGS__;                        \
      break;                              \
    }                                     \
    default:                              \
      return HLM_ERR_UNSUPPORTED;         \
  }

// Blocks for one warp (or thread group) per item, capped for tall inputs (the
// kernels stride over the rest).
static inline int quant_grid(int64_t items, int per_block) {
  const int64_t cap = static_cast<int64_t>(num_sms_of_current_device()) * 64;
  int64_t blocks = (items + per_block - 1) / per_block;
  if (blocks > cap) blocks = cap;
  if (blocks < 1) blocks = 1;
  return static_cast<int>(blocks);
}

// One warp per row, two passes over it (the second one hits L1/L2).
// NORM: v = round(residual + branch) [* weight], written to `out` when there is
// a residual, and the scale is multiplied by 1/rms of the sum: 1/rms is common
// to the row, so it cancels from the codes and scales the step alone.
template <typename T, bool NORM>
__global__ void __launch_bounds__(256) quant_rows_scalar_kernel(
    const T* __restrict__ residual, const T* __restrict__ x, const T* __restrict__ weight,
    T* __restrict__ out, int8_t* __restrict__ q, float* __restrict__ scale, int64_t rows, int cols,
    float eps) {
  const int lane = threadIdx.x & 31;
  const int wpb = blockDim.x >> 5;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * wpb + (threadIdx.x >> 5); row < rows;
       row += static_cast<int64_t>(gridDim.x) * wpb) {
    const int64_t base = row * cols;
    float ss = 0.0f;
    uint32_t m = 0;
    for (int c = lane; c < cols; c += 32) {
      float v = to_f32(x[base + c]);
      if constexpr (NORM) {
        if (residual != nullptr) {
          const T o = from_f32<T>(v + to_f32(residual[base + c]));
          out[base + c] = o;
          v = to_f32(o);
        }
        ss += v * v;
        if (weight != nullptr) v = __fmul_rn(v, to_f32(weight[c]));
      }
      m = max(m, mag_bits(v));
    }
    const QuantStep st = quant_step(warp_max_u32(m));
    if constexpr (NORM) ss = warp_sum(ss);
    __syncwarp();
    for (int c = lane; c < cols; c += 32) {
      float v;
      if constexpr (NORM) {
        v = residual != nullptr ? to_f32(out[base + c]) : to_f32(x[base + c]);
        if (weight != nullptr) v = __fmul_rn(v, to_f32(weight[c]));
      } else {
        v = to_f32(x[base + c]);
      }
      q[base + c] = quant_code(v, st);
    }
    if (lane == 0)
      scale[row] = NORM ? st.scale * rsqrtf(ss / static_cast<float>(cols) + eps) : st.scale;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) dequant_rows_scalar_kernel(const int8_t* __restrict__ q,
                                                                 const float* __restrict__ scale,
                                                                 T* __restrict__ out, int64_t rows,
                                                                 int cols) {
  const int lane = threadIdx.x & 31;
  const int wpb = blockDim.x >> 5;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * wpb + (threadIdx.x >> 5); row < rows;
       row += static_cast<int64_t>(gridDim.x) * wpb) {
    const float s = scale[row];
    for (int c = lane; c < cols; c += 32)
      out[row * cols + c] = from_f32<T>(static_cast<float>(q[row * cols + c]) * s);
  }
}

// SwiGLU checkpoint, one warp per row and group of 128 hidden units: the gate
// group and the up group each get their own scale.
template <typename T>
__global__ void __launch_bounds__(256) swiglu_ckpt8_fwd_scalar_kernel(
    const T* __restrict__ gate_up, T* __restrict__ h, int8_t* __restrict__ q,
    float* __restrict__ scale, int64_t rows, int64_t hidden, int groups) {
  const int lane = threadIdx.x & 31;
  const int wpb = blockDim.x >> 5;
  const int64_t items = rows * groups;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * wpb + (threadIdx.x >> 5); it < items;
       it += static_cast<int64_t>(gridDim.x) * wpb) {
    const int64_t row = it / groups;
    const int grp = static_cast<int>(it - row * groups);
    const int64_t gbase = row * 2 * hidden;
    float g[4], u[4];
    uint32_t mg = 0, mu = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t c = static_cast<int64_t>(grp) * kCkptGroup + lane + 32 * i;
      g[i] = u[i] = 0.0f;
      if (c < hidden) {
        g[i] = to_f32(gate_up[gbase + c]);
        u[i] = to_f32(gate_up[gbase + hidden + c]);
        h[row * hidden + c] = from_f32<T>(g[i] * sigmoid_fast(g[i]) * u[i]);
      }
      mg = max(mg, mag_bits(g[i]));
      mu = max(mu, mag_bits(u[i]));
    }
    const QuantStep sg = quant_step(warp_max_u32(mg));
    const QuantStep su = quant_step(warp_max_u32(mu));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t c = static_cast<int64_t>(grp) * kCkptGroup + lane + 32 * i;
      if (c < hidden) {
        q[gbase + c] = quant_code(g[i], sg);
        q[gbase + hidden + c] = quant_code(u[i], su);
      }
    }
    if (lane == 0) {
      scale[row * 2 * groups + grp] = sg.scale;
      scale[row * 2 * groups + groups + grp] = su.scale;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) swiglu_ckpt8_bwd_scalar_kernel(
    const int8_t* __restrict__ q, const float* __restrict__ scale, const T* __restrict__ grad_h,
    T* __restrict__ grad_gate_up, int64_t rows, int64_t hidden, int groups) {
  const int lane = threadIdx.x & 31;
  const int wpb = blockDim.x >> 5;
  const int64_t items = rows * groups;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * wpb + (threadIdx.x >> 5); it < items;
       it += static_cast<int64_t>(gridDim.x) * wpb) {
    const int64_t row = it / groups;
    const int grp = static_cast<int>(it - row * groups);
    const int64_t gbase = row * 2 * hidden;
    const float sg = scale[row * 2 * groups + grp];
    const float su = scale[row * 2 * groups + groups + grp];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t c = static_cast<int64_t>(grp) * kCkptGroup + lane + 32 * i;
      if (c >= hidden) continue;
      const float g = static_cast<float>(q[gbase + c]) * sg;
      const float u = static_cast<float>(q[gbase + hidden + c]) * su;
      const float d = to_f32(grad_h[row * hidden + c]);
      const float s = sigmoid_fast(g);
      grad_gate_up[gbase + c] = from_f32<T>(d * u * (s * (1.0f + g * (1.0f - s))));
      grad_gate_up[gbase + hidden + c] = from_f32<T>(d * (g * s));
    }
  }
}

}  // namespace hlm

using namespace hlm;

extern "C" int hlm_quantize_rows(const void* x, void* q, float* scale, int64_t rows, int64_t cols,
                                 int dtype, void* stream) {
  if (rows < 0 || cols < 1 || cols > (1ll << 30)) return HLM_ERR_INVALID_ARG;
  if (rows == 0) return HLM_OK;
  if (x == nullptr || q == nullptr || scale == nullptr) return HLM_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  HLM_QUANT_DISPATCH(dtype, T, {
    LaunchScope scope(HLM_KERNEL_QUANT_ROWS, s);
    quant_rows_scalar_kernel<T, false><<<quant_grid(rows, 8), 256, 0, s>>>(
        nullptr, static_cast<const T*>(x), nullptr, nullptr, static_cast<int8_t*>(q), scale, rows,
        static_cast<int>(cols), 0.0f);
  });
  return launch_status();
}

extern "C" int hlm_dequantize_rows(const void* q, const float* scale, void* out, int64_t rows,
                                   int64_t cols, int dtype, void* stream) {
  if (rows < 0 || cols < 1 || cols > (1ll << 30)) return HLM_ERR_INVALID_ARG;
  if (rows == 0) return HLM_OK;
  if (q == nullptr || scale == nullptr || out == nullptr) return HLM_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  HLM_QUANT_DISPATCH(dtype, T, {
    LaunchScope scope(HLM_KERNEL_DEQUANT_ROWS, s);
    dequant_rows_scalar_kernel<T><<<quant_grid(rows, 8), 256, 0, s>>>(
        static_cast<const int8_t*>(q), scale, static_cast<T*>(out), rows, static_cast<int>(cols));
  });
  return launch_status();
}

extern "C" int hlm_residual_rms_norm_q8(const void* residual, const void* branch, const void* weight,
                                        void* out, void* q, float* scale, int64_t rows, int64_t cols,
                                        float eps, int dtype, void* stream) {
  if (rows < 0 || cols < 1 || cols > (1ll << 30)) return HLM_ERR_INVALID_ARG;
  if (rows == 0) return HLM_OK;
  if (branch == nullptr || q == nullptr || scale == nullptr) return HLM_ERR_INVALID_ARG;
  if (residual != nullptr && out == nullptr) return HLM_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  HLM_QUANT_DISPATCH(dtype, T, {
    LaunchScope scope(HLM_KERNEL_NORM_Q8, s);
    quant_rows_scalar_kernel<T, true><<<quant_grid(rows, 8), 256, 0, s>>>(
        static_cast<const T*>(residual), static_cast<const T*>(branch),
        static_cast<const T*>(weight), static_cast<T*>(out), static_cast<int8_t*>(q), scale, rows,
        static_cast<int>(cols), eps);
  });
  return launch_status();
}

extern "C" int hlm_swiglu_ckpt8_fwd(const void* gate_up, void* h, void* q, float* scale,
                                    int64_t rows, int64_t hidden, int dtype, void* stream) {
  if (rows < 0 || hidden < 0 || hidden > (1ll << 30)) return HLM_ERR_INVALID_ARG;
  if (rows == 0 || hidden == 0) return HLM_OK;
  if (gate_up == nullptr || h == nullptr || q == nullptr || scale == nullptr)
    return HLM_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int groups = static_cast<int>((hidden + kCkptGroup - 1) / kCkptGroup);
  HLM_QUANT_DISPATCH(dtype, T, {
    LaunchScope scope(HLM_KERNEL_SWIGLU_CKPT8_FWD, s);
    swiglu_ckpt8_fwd_scalar_kernel<T><<<quant_grid(rows * groups, 8), 256, 0, s>>>(
        static_cast<const T*>(gate_up), static_cast<T*>(h), static_cast<int8_t*>(q), scale, rows,
        hidden, groups);
  });
  return launch_status();
}

extern "C" int hlm_swiglu_ckpt8_bwd(const void* q, const float* scale, const void* grad_h,
                                    void* grad_gate_up, int64_t rows, int64_t hidden, int dtype,
                                    void* stream) {
  if (rows < 0 || hidden < 0 || hidden > (1ll << 30)) return HLM_ERR_INVALID_ARG;
  if (rows == 0 || hidden == 0) return HLM_OK;
  if (q == nullptr || scale == nullptr || grad_h == nullptr || grad_gate_up == nullptr)
    return HLM_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int groups = static_cast<int>((hidden + kCkptGroup - 1) / kCkptGroup);
  HLM_QUANT_DISPATCH(dtype, T, {
    LaunchScope scope(HLM_KERNEL_SWIGLU_CKPT8_BWD, s);
    swiglu_ckpt8_bwd_scalar_kernel<T><<<quant_grid(rows * groups, 8), 256, 0, s>>>(
        static_cast<const int8_t*>(q), scale, static_cast<const T*>(grad_h),
        static_cast<T*>(grad_gate_up), rows, hidden, groups);
  });
  return launch_status();
}
