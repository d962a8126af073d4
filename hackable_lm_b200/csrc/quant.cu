// Operators that write or read the 8-bit format of quant_common.cuh: rows
// quantised and read back, residual-add + RMSNorm with an 8-bit output, and
// SwiGLU that keeps its input in 8 bits for the backward pass.
//
// All bound by HBM: each reads its inputs once (16-byte vectors, kept in registers
// between the maximum and the codes) and writes its outputs once.  Measured with the
// inputs out of L2, share of the measured copy rate (6.55 TB/s):
//   quantise   [32768, 2048] bf16 32.1 us (96%), fp32 50.6 us (101%)
//   read back  [32768, 2048] bf16 31.5 us (97%), fp32 52.4 us (98%)
//   norm       [32768, 768] bf16 27.0 us (100%), [32768, 2048] 73 us (98%)
//   SwiGLU     [32768, 2 x 2048] bf16 82 us forward and backward (100%)
// A few rows: 1.4 to 2 us, a launch.  Arithmetic on packed fp32 pairs: under the power cap
// the clock falls to 1.4 GHz and the SwiGLU kernels come near their issue rate (0.78
// instructions a cycle at full clock before).  Launched as dependents of the kernel before:
// quantise and read back, one after the other, 69.6 -> 65.6 us.
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

// Launch as a dependent of the kernel before (a failure shows in launch_status()).
template <class... Params, class... Args>
static inline void launch_quant(void (*kern)(Params...), int grid, int block, cudaStream_t s, Args... args) {
  (void)launch_dependent(kern, dim3(static_cast<unsigned>(grid)), dim3(static_cast<unsigned>(block)), 0, s, 1, args...);
}

// Rows wider than 16,384 16-bit or 8,192 fp32 columns, and tensors that are aligned
// differently: one warp per row, two passes over it (the second one hits L1/L2).
// NORM: v = round(residual + branch) [* weight], written to `out` when there is
// a residual, and the scale is multiplied by 1/rms of the sum: 1/rms is common
// to the row, so it cancels from the codes and scales the step alone.
template <typename T, bool NORM>
__global__ void __launch_bounds__(256) quant_rows_scalar_kernel(
    const T* residual, const T* x, const T* weight,
    T* out, int8_t* q, float* scale, int64_t rows, int cols,
    float eps) {
  grid_launch_next();
  grid_wait();
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
__global__ void __launch_bounds__(256) dequant_rows_scalar_kernel(const int8_t* q,
                                                                 const float* scale,
                                                                 T* out, int64_t rows,
                                                                 int cols) {
  grid_launch_next();
  grid_wait();
  const int lane = threadIdx.x & 31;
  const int wpb = blockDim.x >> 5;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * wpb + (threadIdx.x >> 5); row < rows;
       row += static_cast<int64_t>(gridDim.x) * wpb) {
    const float s = scale[row];
    for (int c = lane; c < cols; c += 32)
      out[row * cols + c] = from_f32<T>(static_cast<float>(q[row * cols + c]) * s);
  }
}

// SwiGLU checkpoint for halves that are not 16-byte multiples: a block per row, a warp per
// group of 128 hidden units (four elements of each half per lane), of which the gate part
// and the up part each get their own scale.  Bound by instructions, not by memory (16-bit
// elements one by one); two and four rows a warp at once measured slower (fewer warps fit).
template <typename T>
__global__ void __launch_bounds__(256) swiglu_ckpt8_fwd_scalar_kernel(
    const T* gate_up, T* h, int8_t* q,
    float* scale, int64_t rows, int hidden, int groups) {
  grid_launch_next();
  grid_wait();
  const int lane = threadIdx.x & 31;
  const int wpb = blockDim.x >> 5;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* gp = gate_up + row * 2 * hidden;
    T* hp = h + row * hidden;
    int8_t* qp = q + row * 2 * hidden;
    float* sp = scale + row * 2 * groups;
    for (int grp = threadIdx.x >> 5; grp < groups; grp += wpb) {
      const int c0 = grp * kCkptGroup + lane;
      float g[4], u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g[i] = u[i] = 0.0f;
        if (c0 + 32 * i < hidden) {
          g[i] = to_f32(gp[c0 + 32 * i]);
          u[i] = to_f32(gp[hidden + c0 + 32 * i]);
        }
      }
      uint32_t mg = 0, mu = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mg = max(mg, mag_bits(g[i]));
        mu = max(mu, mag_bits(u[i]));
      }
      const QuantStep sg = quant_step(warp_max_u32(mg));
      const QuantStep su = quant_step(warp_max_u32(mu));
      const uint32_t cg = quant_pack4(f2(g[0], g[1]), f2(g[2], g[3]), sg.inv);
      const uint32_t cu = quant_pack4(f2(u[0], u[1]), f2(u[2], u[3]), su.inv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + 32 * i;
        if (c < hidden) {
          hp[c] = from_f32<T>(g[i] * sigmoidf_(g[i]) * u[i]);
          qp[c] = static_cast<int8_t>(cg >> (8 * i));
          qp[hidden + c] = static_cast<int8_t>(cu >> (8 * i));
        }
      }
      if (lane == 0) {
        sp[grp] = sg.scale;
        sp[groups + grp] = su.scale;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) swiglu_ckpt8_bwd_scalar_kernel(
    const int8_t* q, const float* scale, const T* grad_h,
    T* grad_gate_up, int64_t rows, int hidden, int groups) {
  grid_launch_next();
  grid_wait();
  const int lane = threadIdx.x & 31;
  const int wpb = blockDim.x >> 5;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int8_t* qp = q + row * 2 * hidden;
    const T* dp = grad_h + row * hidden;
    T* gp = grad_gate_up + row * 2 * hidden;
    const float* sp = scale + row * 2 * groups;
    for (int grp = threadIdx.x >> 5; grp < groups; grp += wpb) {
      const float sg = sp[grp], su = sp[groups + grp];
      const int c0 = grp * kCkptGroup + lane;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + 32 * i;
        if (c >= hidden) continue;
        const float g = static_cast<float>(qp[c]) * sg;
        const float u = static_cast<float>(qp[hidden + c]) * su;
        const float d = to_f32(dp[c]);
        float s, rest;
        if constexpr (sizeof(T) == 4) {
          sigmoid_exact(g, s, rest);
        } else {
          s = sigmoid_fast(g);
          rest = 1.0f - s;
        }
        gp[c] = from_f32<T>(d * u * (s * (1.0f + g * rest)));
        gp[hidden + c] = from_f32<T>(d * (g * s));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Rows, vectorised: TPR threads per row, up to NV 16-byte vectors per thread, the row
// kept in registers between the maximum (and the sum of squares) and the codes.
//
// A row starts anywhere in its 16-byte vector when cols is not a multiple of the
// vector (SHIFT; [16384, 2047] bf16 26 us, 60% of the copy rate): threads then load the aligned vectors that cover the row, elements
// outside the row count as zeros, and the codes go through shared memory so that
// they too leave in 16-byte stores.  Only the row's first and last vectors, whose
// other elements belong to the neighbouring rows, are read and written by elements.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

// Barrier of one row's threads (a block holds several rows; they do not wait for each other).
template <int TPR>
HLM_DEVICE void row_sync() {
  if constexpr (TPR == 32)
    __syncwarp();
  else if constexpr (TPR == kRowThreads)
    __syncthreads();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / TPR), "n"(TPR) : "memory");
}

template <int TPR>
HLM_DEVICE uint32_t row_max(uint32_t v, uint32_t* sh, int t) {
  v = warp_max_u32(v);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int w0 = (threadIdx.x / TPR) * W;
    if ((t & 31) == 0) sh[w0 + (t >> 5)] = v;
    row_sync<TPR>();
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) m = max(m, sh[w0 + i]);
    v = m;
  }
  return v;
}

// Weights of the VEC columns from c on; columns outside the row (SHIFT) count as zeros.
template <typename T, bool SHIFT>
HLM_DEVICE void load_weight(const T* weight, int c, int cols, F2 (&w)[8 / sizeof(T)]) {
  if constexpr (!SHIFT) {
    f2_load<T>(ld_global_v4(weight + c), w);
  } else {
#pragma unroll
    for (int i = 0; i < static_cast<int>(8 / sizeof(T)); ++i) {
      const int k = c + 2 * i;
      w[i] = f2(k >= 0 && k < cols ? to_f32(weight[k]) : 0.0f,
                k + 1 >= 0 && k + 1 < cols ? to_f32(weight[k + 1]) : 0.0f);
    }
  }
}

template <typename T, int TPR, int NV, bool NORM, bool SHIFT>
__global__ void __launch_bounds__(kRowThreads) quant_rows_vec_kernel(
    const T* residual, const T* x, const T* weight,
    T* out, int8_t* q, float* scale, int64_t rows, int cols,
    float eps) {
  grid_launch_next();
  grid_wait();
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  constexpr int RPB = kRowThreads / TPR;
  constexpr int kStage = SHIFT ? TPR * NV * VEC + 16 : 16;  // bytes of one row's codes
  __shared__ uint32_t sh_max[kRowThreads / 32];
  __shared__ float sh_sum[kRowThreads / 32];
  __shared__ alignas(16) int8_t stage[SHIFT ? RPB * kStage : 16];
  const int t = threadIdx.x % TPR;
  const int64_t total = rows * cols;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * RPB; r0 < rows; r0 += static_cast<int64_t>(gridDim.x) * RPB) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool row_ok = row < rows;  // the same for the row's threads
    const int64_t base = row * cols;
    // elements of x that lie before the row in its first vector
    const int head = SHIFT ? static_cast<int>((reinterpret_cast<uintptr_t>(x + base) & 15) / sizeof(T)) : 0;
    uint4 v[NV], rr[NORM ? NV : 1];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      v[j] = make_uint4(0, 0, 0, 0);
      if constexpr (NORM) rr[j] = make_uint4(0, 0, 0, 0);
      const int c = (t + TPR * j) * VEC - head;  // column of the vector's first element
      if (!row_ok || c >= cols) continue;
      if (!SHIFT || (base + c >= 0 && base + c + VEC <= total)) {
        v[j] = ld_global_stream_v4(x + base + c);
        if (NORM && residual != nullptr) rr[j] = ld_global_stream_v4(residual + base + c);
      } else {  // the tensor's own first or last vector
        T* e = reinterpret_cast<T*>(&v[j]);
        T* f = reinterpret_cast<T*>(&rr[NORM ? j : 0]);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (c + i >= 0 && c + i < cols) {
            e[i] = x[base + c + i];
            if (NORM && residual != nullptr) f[i] = residual[base + c + i];
          }
      }
    }
    // elements of the neighbouring rows (after every load has been issued)
#pragma unroll
    for (int j = 0; j < (SHIFT ? NV : 0); ++j) {
      const int c = (t + TPR * j) * VEC - head;
      if (row_ok && c < cols && (c < 0 || c + VEC > cols)) {
        T* e = reinterpret_cast<T*>(&v[j]);
        T* f = reinterpret_cast<T*>(&rr[NORM ? j : 0]);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (c + i < 0 || c + i >= cols) {
            e[i] = from_f32<T>(0.0f);
            if (NORM) f[i] = from_f32<T>(0.0f);
          }
      }
    }
    // the sum, rounded to T once, back in v; squares and magnitudes of it
    F2 ss2 = f2(0.0f);
    uint32_t mp = 0;
    uint32_t mw = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (t + TPR * j) * VEC - head;
      if constexpr (NORM) {
        F2 f[VEC / 2];
        f2_load<T>(v[j], f);
        if (residual != nullptr) {
          F2 g[VEC / 2];
          f2_load<T>(rr[j], g);
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) f[i] = f[i] + g[i];
          v[j] = f2_store<T>(f);
          f2_load<T>(v[j], f);
          if (row_ok && c < cols) {
            if (!SHIFT || (c >= 0 && c + VEC <= cols)) {
              st_global_v4(out + base + c, v[j]);
            } else {
              const T* e = reinterpret_cast<const T*>(&v[j]);
#pragma unroll
              for (int i = 0; i < VEC; ++i)
                if (c + i >= 0 && c + i < cols) out[base + c + i] = e[i];
            }
          }
        }
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) ss2 = f2_fma(f[i], f[i], ss2);
        if (weight != nullptr && row_ok && c < cols) {
          F2 w[VEC / 2];
          load_weight<T, SHIFT>(weight, c, cols, w);
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            float a, b;
            f2_split(f[i] * w[i], a, b);
            mw = max(mw, max(mag_bits(a), mag_bits(b)));
          }
        }
      }
      mp = max_packed<T>(mp, max16_packed<T>(v[j]));
    }
    uint32_t m = unpack_max<T>(mp);
    if (NORM && weight != nullptr) m = mw;
    m = row_max<TPR>(m, sh_max, t);
    const QuantStep st = quant_step(m);
    float ss = 0.0f;
    if constexpr (NORM) {
      float lo, hi;
      f2_split(ss2, lo, hi);
      ss = warp_sum(lo + hi);
      if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int w0 = (threadIdx.x / TPR) * W;
        if ((t & 31) == 0) sh_sum[w0 + (t >> 5)] = ss;
        row_sync<TPR>();
        ss = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) ss += sh_sum[w0 + i];
      }
    }
    int8_t* row_stage = stage + (SHIFT ? (threadIdx.x / TPR) * kStage : 0);
    // the row's first code lies `qhead` bytes into its word of q; the stage holds the codes of
    // the row's vectors one after the other, so its first code is at byte `head`
    const int qhead = SHIFT ? static_cast<int>(reinterpret_cast<uintptr_t>(q + base) & 3) : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (t + TPR * j) * VEC - head;
      if (!row_ok || c >= cols) continue;
      F2 f[VEC / 2];
      f2_load<T>(v[j], f);
      if (NORM && weight != nullptr) {
        F2 w[VEC / 2];
        load_weight<T, SHIFT>(weight, c, cols, w);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) f[i] = f[i] * w[i];
      }
      int8_t* dst = SHIFT ? row_stage + c + head : q + base + c;
      if constexpr (VEC == 8)
        *reinterpret_cast<uint2*>(dst) = make_uint2(quant_pack4(f[0], f[1], st.inv), quant_pack4(f[2], f[3], st.inv));
      else
        *reinterpret_cast<uint32_t*>(dst) = quant_pack4(f[0], f[1], st.inv);
    }
    if constexpr (SHIFT) {
      row_sync<TPR>();
      if (row_ok) {
        // aligned words of q: word b holds columns b - qhead ..., staged from byte head + b - qhead on
        const int delta = head - qhead;
        for (int b = t * 4; b < qhead + cols; b += TPR * 4) {
          int8_t* dst = q + base - qhead + b;
          if (b >= qhead && b + 4 <= qhead + cols) {
            const int o = b + delta;
            const uint32_t* w = reinterpret_cast<const uint32_t*>(row_stage) + (o >> 2);
            *reinterpret_cast<uint32_t*>(dst) = __funnelshift_r(w[0], w[1], (o & 3) * 8);
          } else {
            for (int i = 0; i < 4; ++i)
              if (b + i >= qhead && b + i < qhead + cols) dst[i] = row_stage[b + delta + i];
          }
        }
      }
    }
    if (row_ok && t == 0) {
      if constexpr (NORM)
        scale[row] = st.scale * rsqrtf(ss / static_cast<float>(cols) + eps);
      else
        scale[row] = st.scale;
    }
    // shared memory is rewritten by the block's next rows
    if constexpr (TPR > 32 || SHIFT) row_sync<TPR>();
  }
}

// Launch of the vector kernel that holds a row of `cols`, or false when the row is too
// wide (or its tensors are aligned differently): the scalar kernel takes those.
template <typename T, bool NORM>
static bool launch_quant_rows_vec(const T* residual, const T* x, const T* weight, T* out, int8_t* q,
                                  float* scale, int64_t rows, int cols, float eps, cudaStream_t s) {
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  auto mod16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) & 15u; };
  const bool same = residual == nullptr || (mod16(residual) == mod16(x) && mod16(out) == mod16(x));
  if (!same || mod16(x) % sizeof(T) != 0) return false;
  const bool aligned = cols % VEC == 0 && mod16(x) == 0 && reinterpret_cast<uintptr_t>(q) % VEC == 0 &&
                       (weight == nullptr || mod16(weight) == 0);
  // vectors that cover a row, at most
  const int64_t nv = aligned ? cols / VEC : (cols + VEC - 1) / VEC + 1;
#define HLM_ROWS_LAUNCH(TPR, NV, SHIFT)                                                                     \
  do {                                                                                                      \
    launch_quant(quant_rows_vec_kernel<T, TPR, NV, NORM, SHIFT>, quant_grid(rows, kRowThreads / TPR), kRowThreads, s, \
                 residual, x, weight, out, q, scale, rows, cols, eps);                                       \
    return true;                                                                                            \
  } while (0)
  if (aligned) {
    if (nv <= 32) HLM_ROWS_LAUNCH(32, 1, false);
    if (nv <= 64) HLM_ROWS_LAUNCH(32, 2, false);
    if (nv <= 96) HLM_ROWS_LAUNCH(32, 3, false);
    if (nv <= 128) HLM_ROWS_LAUNCH(32, 4, false);
    if (nv <= 256) HLM_ROWS_LAUNCH(64, 4, false);
    if (nv <= 512) HLM_ROWS_LAUNCH(128, 4, false);
    if (nv <= 1024) HLM_ROWS_LAUNCH(256, 4, false);
    if (nv <= 2048) HLM_ROWS_LAUNCH(256, 8, false);
    return false;
  }
  // five vectors, since a row of a power of two plus or minus a few columns spans one more
  if (nv <= 64) HLM_ROWS_LAUNCH(32, 2, true);
  if (nv <= 160) HLM_ROWS_LAUNCH(32, 5, true);
  if (nv <= 320) HLM_ROWS_LAUNCH(64, 5, true);
  if (nv <= 640) HLM_ROWS_LAUNCH(128, 5, true);
  if (nv <= 1280) HLM_ROWS_LAUNCH(256, 5, true);
  if (nv <= 2304) HLM_ROWS_LAUNCH(256, 9, true);
#undef HLM_ROWS_LAUNCH
  return false;
}

// Read back, over the flat tensor: a thread takes VEC consecutive codes (one 16-byte
// store) whatever the row length, since so few lie in at most two rows of 16 or more
// columns; one division finds the row.  Four such steps of a block in flight.
template <typename T, typename I>
__global__ void __launch_bounds__(256) dequant_flat_kernel(const int8_t* q,
                                                          const float* scale,
                                                          T* out, I total, I cols) {
  grid_launch_next();
  grid_wait();
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  constexpr int U = 4;
  constexpr I kSpan = 256 * VEC;  // codes of one step of the block
  for (I e0 = static_cast<I>(blockIdx.x) * (U * kSpan) + threadIdx.x * VEC; e0 < total;
       e0 += static_cast<I>(gridDim.x) * (U * kSpan)) {
    uint32_t w[U][VEC / 4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const I e = e0 + u * kSpan;
      if (e + VEC <= total) {
        if constexpr (VEC == 8) {
          const uint2 a = *reinterpret_cast<const uint2*>(q + e);
          w[u][0] = a.x;
          w[u][1] = a.y;
        } else {
          w[u][0] = *reinterpret_cast<const uint32_t*>(q + e);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const I e = e0 + u * kSpan;
      if (e >= total) break;
      const I row = e / cols;
      const I next = (row + 1) * cols - e;  // codes from here on belong to the next row
      const float s0 = scale[row];
      if (e + VEC <= total) {
        F2 f[VEC / 2];
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) codes_to_f2(w[u][k], f[2 * k], f[2 * k + 1]);
        if (next >= VEC) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) f[i] = f[i] * f2(s0);
        } else {  // a row ends among these codes
          const float s1 = scale[row + 1];
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i)
            f[i] = f[i] * f2(static_cast<I>(2 * i) < next ? s0 : s1, static_cast<I>(2 * i + 1) < next ? s0 : s1);
        }
        st_global_v4(out + e, f2_store<T>(f));
      } else {
        for (I i = 0; e + i < total; ++i)
          out[e + i] = from_f32<T>(static_cast<float>(q[e + i]) * (i < next ? s0 : scale[row + 1]));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// SwiGLU checkpoint, vectorised: a thread owns one 16-byte vector of gate and the
// matching one of up in R consecutive rows; the 128 / VEC threads of a group (half a
// warp for 16-bit types, a warp for fp32) find its two maxima by shuffles, both in
// one packed word for the 16-bit types.
// ---------------------------------------------------------------------------
template <typename T>
HLM_DEVICE void group_maxima(uint4 g, uint4 u, uint32_t& mg, uint32_t& mu) {
  if constexpr (sizeof(T) == 4) {
    mg = warp_max_u32(max16_packed<T>(g));
    mu = warp_max_u32(max16_packed<T>(u));
  } else {
    const uint32_t a = max16_packed<T>(g), b = max16_packed<T>(u);
    // one 16-bit maximum of each, gate low and up high
    uint32_t m = __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    mg = unpack_max<T>(m & 0xffffu);
    mu = unpack_max<T>(m >> 16);
  }
}

// Threads of a block that walks rows of `n` vectors: the fewest steps of at most 256, evenly filled.
static inline int row_block(int64_t n) {
  const int64_t steps = (n + 255) / 256;
  return static_cast<int>(((n + steps - 1) / steps + 31) / 32 * 32);
}

template <typename T, int R>
__global__ void __launch_bounds__(256) swiglu_ckpt8_fwd_vec_kernel(
    const T* gate_up, T* h, int8_t* q,
    float* scale, int64_t rows, int hv, int groups) {
  grid_launch_next();
  grid_wait();
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  constexpr int GT = kCkptGroup / VEC;  // threads of a group
  const int64_t hidden = static_cast<int64_t>(hv) * VEC;
  const int hv_pad = groups * GT;  // a group's threads stay together past the last vector
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * R; r0 < rows;
       r0 += static_cast<int64_t>(gridDim.x) * R) {
    for (int c0 = 0; c0 < hv_pad; c0 += blockDim.x) {
      const int cv = c0 + threadIdx.x;
      uint4 gr[R], ur[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        gr[r] = ur[r] = make_uint4(0, 0, 0, 0);
        if (r0 + r < rows && cv < hv) {
          const T* src = gate_up + (r0 + r) * 2 * hidden + static_cast<int64_t>(cv) * VEC;
          gr[r] = ld_global_stream_v4(src);
          ur[r] = ld_global_stream_v4(src + hidden);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        uint32_t mg, mu;
        group_maxima<T>(gr[r], ur[r], mg, mu);  // all threads: shuffles
        // one division per lane: of a group's threads, 0 and 1 make the gate and up scales (which
        // they write), 2 and 3 the inverses
        const float quot = quant_quotient((threadIdx.x & 1) ? mu : mg, threadIdx.x & 2);
        const float inv_g = __shfl_sync(0xffffffffu, quot, (threadIdx.x & (32 - GT)) + 2);
        const float inv_u = __shfl_sync(0xffffffffu, quot, (threadIdx.x & (32 - GT)) + 3);
        if (r0 + r >= rows || cv >= hv_pad) continue;
        if (cv % GT < 2) scale[(r0 + r) * 2 * groups + (cv & 1) * groups + cv / GT] = quot;
        if (cv >= hv) continue;
        F2 g[VEC / 2], u[VEC / 2], o[VEC / 2];
        f2_load<T>(gr[r], g);
        f2_load<T>(ur[r], u);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) o[i] = g[i] * f2_sigmoid(g[i]) * u[i];
        st_global_v4(h + (r0 + r) * hidden + static_cast<int64_t>(cv) * VEC, f2_store<T>(o));
        int8_t* qg = q + (r0 + r) * 2 * hidden + static_cast<int64_t>(cv) * VEC;
        if constexpr (VEC == 8) {
          *reinterpret_cast<uint2*>(qg) = make_uint2(quant_pack4(g[0], g[1], inv_g), quant_pack4(g[2], g[3], inv_g));
          *reinterpret_cast<uint2*>(qg + hidden) =
              make_uint2(quant_pack4(u[0], u[1], inv_u), quant_pack4(u[2], u[3], inv_u));
        } else {
          *reinterpret_cast<uint32_t*>(qg) = quant_pack4(g[0], g[1], inv_g);
          *reinterpret_cast<uint32_t*>(qg + hidden) = quant_pack4(u[0], u[1], inv_u);
        }
      }
    }
  }
}

template <typename T, int R>
__global__ void __launch_bounds__(256) swiglu_ckpt8_bwd_vec_kernel(
    const int8_t* q, const float* scale, const T* grad_h,
    T* grad_gate_up, int64_t rows, int hv, int groups) {
  grid_launch_next();
  grid_wait();
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  constexpr int GT = kCkptGroup / VEC;
  const int64_t hidden = static_cast<int64_t>(hv) * VEC;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * R; r0 < rows;
       r0 += static_cast<int64_t>(gridDim.x) * R) {
    for (int cv = threadIdx.x; cv < hv; cv += blockDim.x) {
      uint32_t qg[R][VEC / 4], qu[R][VEC / 4];
      uint4 dr[R];
      float sg[R], su[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r0 + r < rows) {
          const int8_t* src = q + (r0 + r) * 2 * hidden + static_cast<int64_t>(cv) * VEC;
          if constexpr (VEC == 8) {
            const uint2 a = *reinterpret_cast<const uint2*>(src);
            const uint2 b = *reinterpret_cast<const uint2*>(src + hidden);
            qg[r][0] = a.x;
            qg[r][1] = a.y;
            qu[r][0] = b.x;
            qu[r][1] = b.y;
          } else {
            qg[r][0] = *reinterpret_cast<const uint32_t*>(src);
            qu[r][0] = *reinterpret_cast<const uint32_t*>(src + hidden);
          }
          dr[r] = ld_global_stream_v4(grad_h + (r0 + r) * hidden + static_cast<int64_t>(cv) * VEC);
          const float* sp = scale + (r0 + r) * 2 * groups + cv / GT;
          sg[r] = sp[0];
          su[r] = sp[groups];
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r0 + r >= rows) continue;
        F2 d[VEC / 2], rg[VEC / 2], ru[VEC / 2];
        f2_load<T>(dr[r], d);
        const F2 one = f2(1.0f), minus = f2(-1.0f), sg2 = f2(sg[r]), su2 = f2(su[r]);
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) {
          F2 g[2], u[2];
          codes_to_f2(qg[r][k], g[0], g[1]);
          codes_to_f2(qu[r][k], u[0], u[1]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const F2 gv = g[i] * sg2, uv = u[i] * su2, dd = d[2 * k + i];
            F2 s, rest;  // sigmoid(g) and 1 - sigmoid(g)
            if constexpr (sizeof(T) == 4) {
              float g0, g1, s0, s1, r0, r1;
              f2_split(gv, g0, g1);
              sigmoid_exact(g0, s0, r0);
              sigmoid_exact(g1, s1, r1);
              s = f2(s0, s1);
              rest = f2(r0, r1);
            } else {
              s = f2_sigmoid(gv);
              rest = f2_fma(s, minus, one);
            }
            // d u s (1 + g (1 - s)) and d (g s)
            rg[2 * k + i] = dd * uv * (s * f2_fma(gv, rest, one));
            ru[2 * k + i] = dd * (gv * s);
          }
        }
        T* dst = grad_gate_up + (r0 + r) * 2 * hidden + static_cast<int64_t>(cv) * VEC;
        st_global_v4(dst, f2_store<T>(rg));
        st_global_v4(dst + hidden, f2_store<T>(ru));
      }
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
    if (!launch_quant_rows_vec<T, false>(nullptr, static_cast<const T*>(x), nullptr, nullptr,
                                         static_cast<int8_t*>(q), scale, rows, static_cast<int>(cols), 0.0f, s))
      launch_quant(quant_rows_scalar_kernel<T, false>, quant_grid(rows, 8), 256, s, 
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
    const int64_t total = rows * cols;
    const int grid = quant_grid((total + 16 / sizeof(T) - 1) / (16 / sizeof(T)), 4 * 256);
    if (cols >= 16 && host_aligned16(q) && host_aligned16(out)) {
      if (total < (1ll << 31))  // 32-bit division; a step past the end stays below 2^32
        launch_quant(dequant_flat_kernel<T, uint32_t>, grid, 256, s, static_cast<const int8_t*>(q), scale,
                                                              static_cast<T*>(out), static_cast<uint32_t>(total),
                                                              static_cast<uint32_t>(cols));
      else
        launch_quant(dequant_flat_kernel<T, uint64_t>, grid, 256, s, static_cast<const int8_t*>(q), scale,
                                                              static_cast<T*>(out), static_cast<uint64_t>(total),
                                                              static_cast<uint64_t>(cols));
    } else
      launch_quant(dequant_rows_scalar_kernel<T>, quant_grid(rows, 8), 256, s, 
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
    if (!launch_quant_rows_vec<T, true>(static_cast<const T*>(residual), static_cast<const T*>(branch),
                                        static_cast<const T*>(weight), static_cast<T*>(out),
                                        static_cast<int8_t*>(q), scale, rows, static_cast<int>(cols), eps, s))
      launch_quant(quant_rows_scalar_kernel<T, true>, quant_grid(rows, 8), 256, s, 
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
    constexpr int VEC = 16 / sizeof(T);
    if (hidden % VEC == 0 && host_aligned16(gate_up) && host_aligned16(h) && host_aligned16(q)) {
      constexpr int R = 2;
      launch_quant(swiglu_ckpt8_fwd_vec_kernel<T, R>, quant_grid(rows, R), row_block(hidden / VEC), s, 
          static_cast<const T*>(gate_up), static_cast<T*>(h), static_cast<int8_t*>(q), scale, rows,
          static_cast<int>(hidden / VEC), groups);
    } else
      launch_quant(swiglu_ckpt8_fwd_scalar_kernel<T>, quant_grid(rows, 1), row_block(32 * static_cast<int64_t>(groups)), s, 
        static_cast<const T*>(gate_up), static_cast<T*>(h), static_cast<int8_t*>(q), scale, rows,
        static_cast<int>(hidden), groups);
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
    constexpr int VEC = 16 / sizeof(T);
    if (hidden % VEC == 0 && host_aligned16(grad_h) && host_aligned16(grad_gate_up) && host_aligned16(q)) {
      constexpr int R = 2;
      launch_quant(swiglu_ckpt8_bwd_vec_kernel<T, R>, quant_grid(rows, R), row_block(hidden / VEC), s, 
          static_cast<const int8_t*>(q), scale, static_cast<const T*>(grad_h),
          static_cast<T*>(grad_gate_up), rows, static_cast<int>(hidden / VEC), groups);
    } else
      launch_quant(swiglu_ckpt8_bwd_scalar_kernel<T>, quant_grid(rows, 1), row_block(32 * static_cast<int64_t>(groups)), s, 
        static_cast<const int8_t*>(q), scale, static_cast<const T*>(grad_h),
        static_cast<T*>(grad_gate_up), rows, static_cast<int>(hidden), groups);
  });
  return launch_status();
}
