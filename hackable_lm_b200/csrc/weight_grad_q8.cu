// Weight gradient of a projection whose input was kept in 8 bits:
//
//   grad_w[n, k] = sum_m grad[m, n] * (q[m, k] * scale[m])
//
// Two passes: the codes are read back once to the workspace, as two values of the gradient's
// type (the tensor cores take one 16-bit type for both operands): x = q * scale in fp32 is cut
// into hi, its leading 8 or 11 bits, and lo, the rest rounded, so that hi + lo is x to within
// 2^-15 (bf16) or 2^-21 (fp16) of it.  A CTA-pair tcgen05 GEMM (256 x 256 or 256 x 128 tiles of
// grad_w, both operands MN-major, tokens as the reduction) multiplies each block of the gradient
// by both.  One rounded value in place of the two halves the products, but rounds as coarsely
// as the result itself: the error against 64 bits is then 1.4 times that of the exact result
// rounded once, with the two it is that.
// Making the operand inside the GEMM, by converter warps from codes in shared memory, was built
// first (with one value: 206 us at [32768 tokens, 4096, 768] against 165): every row of tiles
// then converts the codes again, and the converters' shared-memory traffic (their reads and
// writes beside the MMA's) holds the tensor cores back.
//
// Bound by the tensor cores (4 * tokens * N * K operations): [32768, 4096, 768] bf16 277 us a call
// at full clock (1.49 PFLOP/s over the whole call), 333 at the power cap; small gradients
// ([1003, 520, 272] 11.2 us, [64, 1024, 1024] 8.6) are their launches' latency.  Few tiles: the
// tokens are split and each split writes an fp32 partial to the workspace; a third kernel adds
// the partials in the order of the splits (the same bits every time) and rounds.
#include "gemm_sm100.cuh"
#include "quant_common.cuh"

namespace hlm {

constexpr int kWgEpiWarps = 8;

// Write every `parts`-th 32-column group, from `part` on, of a warp's 32 accumulator rows as
// O (fp32 partial, or the 16-bit result, times `up`): staged in a 32 x 64-byte box (16-byte chunks swizzled by row
// pairs), out in 16-byte stores, eight 64-byte row segments per instruction.
template <typename O, int GROUPS>
HLM_DEVICE void wg_store_tile(O* dst, int64_t ld, int row0, int rows, int col0, int cols, uint32_t taddr,
                              uint32_t buf, int lane, int part, int parts, float up) {
  constexpr int kCols = 64 / static_cast<int>(sizeof(O));  // columns of a box: 16 fp32 or 32 16-bit
  constexpr int kPerChunk = 16 / static_cast<int>(sizeof(O));
  if (row0 >= rows) return;
  const uint32_t sw = static_cast<uint32_t>(lane >> 1) & 3u;
#pragma unroll 1
  for (int g = part; g < GROUPS; g += parts) {
    if (col0 + 32 * g >= cols) break;
    uint32_t a[32];
    tmem_ld_32x32b_x32(taddr + static_cast<uint32_t>(g * 32), a);
    tmem_ld_wait();
#pragma unroll
    for (int hs = 0; hs < 32 / kCols; ++hs) {
      __syncwarp();  // the box's last columns have been read
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint4 v;
        if constexpr (sizeof(O) == 4) {
          v = make_uint4(a[16 * hs + 4 * c], a[16 * hs + 4 * c + 1], a[16 * hs + 4 * c + 2], a[16 * hs + 4 * c + 3]);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = pack2<O>(__uint_as_float(a[8 * c + 2 * i]) * up, __uint_as_float(a[8 * c + 2 * i + 1]) * up);
          v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        st_shared_v4(buf + static_cast<uint32_t>(lane * 64) + ((static_cast<uint32_t>(c) ^ sw) << 4), v);
      }
      __syncwarp();
      const int chunk = lane & 3;
      const int c0 = col0 + 32 * g + hs * kCols + chunk * kPerChunk;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        const uint4 v = ld_shared_v4(buf + static_cast<uint32_t>(r * 64 + ((chunk ^ ((r >> 1) & 3)) << 4)));
        if (row0 + r < rows && c0 < cols) st_global_v4(dst + static_cast<int64_t>(row0 + r) * ld + c0, v);
      }
    }
  }
}

// x as two values of type T: hi, x cut towards zero, and lo, the rest.  The rest is exact in
// fp32 and rounded to T.  Both have the sign of x, and lo is not zero unless x is (a rest of
// zero becomes 2^-24 of x, or fp16's smallest value), so that an infinite gradient times
// either is the same infinity.
template <typename T>
HLM_DEVICE void split_value(float x, float& hi, float& lo);
template <>
HLM_DEVICE void split_value<__nv_bfloat16>(float x, float& hi, float& lo) {
  hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  lo = x - hi;
  if (lo == 0.0f) lo = x * 5.9604644775390625e-8f;
  if (!isfinite(x)) hi = lo = x;
}
template <>
HLM_DEVICE void split_value<__half>(float x, float& hi, float& lo) {
  hi = __half2float(__float2half_rz(x));
  lo = __half2float(__float2half_rn(x - hi));
  if (lo == 0.0f && x != 0.0f) lo = copysignf(5.9604644775390625e-8f, x);
  if (!isfinite(x)) hi = lo = x;
}

// fp16 holds less than the scales' range (the codes may be those of wider values: fp32 rows,
// whole tensors of tiny ones).  Its values read back are therefore held times a power of two
// that puts the largest scale into [2^7, 2^8), their largest magnitude below 2^15, and the
// sums are multiplied by its inverse in fp32.  What is off by its subnormal steps is then off
// by at most 2^-39 of the largest value that the scales allow.

// The largest finite magnitude among n floats, by the block's 256 threads.
HLM_DEVICE float block_max_finite(const float* v, int64_t n) {
  __shared__ uint32_t sh[8];
  uint32_t m = 0;
  for (int64_t i = threadIdx.x; i < n; i += 256) {
    const uint32_t b = mag_bits(v[i]);
    if (b < kInfBits) m = max(m, b);
  }
  m = warp_max_u32(m);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, sh[i]);
  return __uint_as_float(m);
}
constexpr int kScalePart = 1024;  // scales that every block of the next kernel may read itself
constexpr int kScaleBlocks = 128;

// Partial maxima of more of them.
__global__ void __launch_bounds__(256) weight_grad_q8_scale_max_kernel(const float* scale, int64_t tokens, int64_t per,
                                                                      float* maxima) {
  grid_launch_next();
  grid_wait();
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * per;
  const float m = block_max_finite(scale + i0, min(per, tokens - i0));
  if (threadIdx.x == 0) maxima[blockIdx.x] = m;
}

// The codes read back as hi and lo; a thread takes eight consecutive codes (of one row: K is
// a multiple of 16), four such steps of a block in flight.  fp16: `maxima` holds the scales or
// maxima of them, and *up gets the factor of the sums.
template <typename T, typename I>
__global__ void __launch_bounds__(256) weight_grad_q8_split_kernel(const int8_t* q, const float* scale,
                                                                  const float* maxima, int n_maxima, float* up, T* hi,
                                                                  T* lo, I total, I cols) {
  grid_launch_next();
  grid_wait();
  float down = 1.0f;
  if constexpr (std::is_same_v<T, __half>) {
    const uint32_t e = max(__float_as_uint(block_max_finite(maxima, n_maxima)) >> 23, 8u);  // biased exponent
    down = __uint_as_float((127u + 7u + 127u - e) << 23);
    if (blockIdx.x == 0 && threadIdx.x == 0) *up = __uint_as_float((e - 7u) << 23);
  }
  constexpr int U = 4;
  constexpr I kSpan = 256 * 8;
  for (I e0 = static_cast<I>(blockIdx.x) * (U * kSpan) + threadIdx.x * 8; e0 < total;
       e0 += static_cast<I>(gridDim.x) * (U * kSpan)) {
    uint2 w[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const I e = e0 + u * kSpan;
      if (e < total) {
        w[u] = *reinterpret_cast<const uint2*>(q + e);
        s[u] = scale[e / cols] * down;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const I e = e0 + u * kSpan;
      if (e >= total) break;
      F2 f[4], a[4], b[4];
      codes_to_f2(w[u].x, f[0], f[1]);
      codes_to_f2(w[u].y, f[2], f[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x0, x1, h0, h1, l0, l1;
        f2_split(f[i] * f2(s[u]), x0, x1);
        split_value<T>(x0, h0, l0);
        split_value<T>(x1, h1, l1);
        a[i] = f2(h0, h1);
        b[i] = f2(l0, l1);
      }
      st_global_v4(hi + e, f2_store<T>(a));
      st_global_v4(lo + e, f2_store<T>(b));
    }
  }
}

struct EpiWeightGrad {
  struct Params {
    void* out;       // grad_w [N][K], 16-bit
    float* partial;  // or fp32 partials [splits][N][K]
    const float* up;  // the sums' factor (fp16)
    int fp16;
  };
  static constexpr bool kRelaxedRelease = true;
  static constexpr bool kDependentLaunch = true;
  static constexpr bool kSplitB = true;
  template <int EPI_WARPS>
  static constexpr int smem_bytes() {
    return EPI_WARPS * 2048;
  }
  template <int BN, int kParts>
  static HLM_DEVICE void run(const Params& ep, const GemmParams& p, uint8_t* smem, uint32_t taddr, int m_tile,
                             int n_tile, int split, int quad, int part, int lane) {
    constexpr int kGroups = BN / 32;
    const uint32_t buf = smem_u32(smem) + static_cast<uint32_t>(part * 4 + quad) * 2048u;
    const int row0 = m_tile * kBM + quad * 32;
    if (ep.partial != nullptr)
      wg_store_tile<float, kGroups>(ep.partial + static_cast<int64_t>(split) * p.M * p.N, p.N, row0, p.M, n_tile * BN,
                                    p.N, taddr, buf, lane, part, kParts, 1.0f);
    else if (ep.fp16)
      wg_store_tile<__half, kGroups>(static_cast<__half*>(ep.out), p.N, row0, p.M, n_tile * BN, p.N, taddr, buf, lane,
                                     part, kParts, *ep.up);
    else
      wg_store_tile<__nv_bfloat16, kGroups>(static_cast<__nv_bfloat16*>(ep.out), p.N, row0, p.M, n_tile * BN, p.N,
                                            taddr, buf, lane, part, kParts, 1.0f);
  }
};

// Sum of the splits' partials in their order, times *up (fp16), rounded to T; eight elements per thread.
template <typename T>
__global__ void __launch_bounds__(256) weight_grad_q8_reduce_kernel(const float* partial,
                                                                   T* grad_w, int64_t n, int splits,
                                                                   const float* up) {
  grid_launch_next();
  grid_wait();
  const float factor = std::is_same_v<T, __half> ? *up : 1.0f;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 8; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x * 8) {
    float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const float4 a = __ldcs(reinterpret_cast<const float4*>(partial + s * n + i));
      const float4 b = __ldcs(reinterpret_cast<const float4*>(partial + s * n + i + 4));
      f[0] += a.x;
      f[1] += a.y;
      f[2] += a.z;
      f[3] += a.w;
      f[4] += b.x;
      f[5] += b.y;
      f[6] += b.z;
      f[7] += b.w;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] *= factor;
    Vec16<T> o;
    o.from_float(f);
    st_global_v4(grad_w + i, o.raw);
  }
}

// Tile width and splits of the tokens: the pair that the cost in microseconds is least for,
// of rounds of pair tiles at 0.47 us (256 x 128) or 0.70 us (256 x 256) per 64 tokens and 1 us to fill
// and drain, and, with partials, 2 us of another launch (less than its 3.5 us alone, since it
// overlaps) and 8 bytes per partial element at 7 TB/s (most of it L2).  Within 6% of the best of
// all pairs at fifteen sizes measured, [1003, 520, 272] apart (128 columns x 8 splits 11.5 to
// 14 us, x 4 11.2, x 1 16.4): [4096, 768, 768] 128 x 4 20.7, 256 x 8 21.7; [8192, 2304, 768] 256 x 5 52.4,
// 128 x 4 60.5; [2048, 2304, 768] 128 x 1 22.3, 128 x 4 27.9.
struct WgPlan {
  int bn;  // 256 x bn tiles
  int splits;
};
static WgPlan weight_grad_q8_plan(int64_t tokens, int64_t N, int64_t K) {
  const int64_t pairs = num_sms_of_current_device() / 2;
  const int kb = static_cast<int>((tokens + kBK - 1) / kBK);
  const double part_us = static_cast<double>(N) * static_cast<double>(K) * 8.0 / 7.0e6;
  WgPlan best = {256, 1};
  double best_us = 1e30;
  for (int bn = 128; bn <= 256; bn += 128) {
    const int64_t tiles = ((N + 255) / 256) * ((K + bn - 1) / bn);
    const double block = bn == 256 ? 0.70 : 0.47;
    for (int s = 1; s <= 32 && s <= kb; ++s) {
      const double extra = s > 1 ? 2.0 + s * part_us : 0.0;
      if (extra >= best_us) break;
      const int per = (kb + s - 1) / s;
      if ((kb + per - 1) / per != s) continue;  // the same blocks with fewer splits
      const double us = static_cast<double>((tiles * s + pairs - 1) / pairs) * (block * per + 1.0) + extra;
      if (us < best_us) {
        best_us = us;
        best = {bn, s};
      }
    }
  }
  return best;
}

// Workspace: the sums' factor and the scales' maxima, the input read back, hi and lo (each of
// this many bytes), then the partials.
constexpr size_t kWgHeadBytes = (1 + kScaleBlocks) * sizeof(float) + 252;
static_assert(kWgHeadBytes % 256 == 0, "what follows stays aligned");
static size_t weight_grad_q8_back_bytes(int64_t tokens, int64_t K) {
  return (static_cast<size_t>(tokens) * static_cast<size_t>(K) * 2 + 255) / 256 * 256;
}

template <class Kind, int BN>
static int weight_grad_q8_gemm(const void* grad, const void* hi, const void* lo, void* grad_w, float* partial,
                               const float* up, int fp16,
                               int64_t tokens, int64_t N, int64_t K, int splits, cudaStream_t s) {
  CUtensorMap ma, mh, ml;  // all [tokens][features]: boxes of 64 features x 64 tokens
  if (!encode_map(&ma, grad, 2, N, tokens, N, 64) || !encode_map(&mh, hi, 2, K, tokens, K, 64) ||
      !encode_map(&ml, lo, 2, K, tokens, K, 64))
    return HLM_ERR_DRIVER;
  GemmParams p;
  gemm_tiling_pair(p, static_cast<int>(N), static_cast<int>(K), static_cast<int>(tokens), BN, splits);
  if (static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.splits > (1ll << 30)) return HLM_ERR_UNSUPPORTED;
  p.err = device_error_ptr();
  if (p.err == nullptr) return HLM_ERR_LAUNCH;
  EpiWeightGrad::Params ep;
  ep.out = grad_w;
  ep.partial = p.splits > 1 ? partial : nullptr;
  ep.up = up;
  ep.fp16 = fp16;
  constexpr int kStages = BN == 256 ? 4 : 6;  // of 48 and 32 KB
  return launch_gemm_pair<BN, kStages, true, true, EpiWeightGrad, kWgEpiWarps, Kind>(
      ma, ml, ma, mh, p, ep, s, HLM_KERNEL_WEIGHT_GRAD_Q8);
}

template <typename T>
static int weight_grad_q8_split(const void* q, const float* scale, float* head, void* hi, void* lo, int64_t tokens,
                                int64_t K, cudaStream_t s) {
  const float* maxima = scale;
  int64_t n_maxima = tokens;
  if (std::is_same_v<T, __half> && tokens > kScalePart) {
    const int64_t least = (tokens + kScaleBlocks - 1) / kScaleBlocks, per = least > kScalePart ? least : kScalePart;
    n_maxima = (tokens + per - 1) / per;
    LaunchScope scope(0, s);
    (void)launch_dependent(weight_grad_q8_scale_max_kernel, dim3(static_cast<unsigned>(n_maxima)), dim3(256), 0, s, 1,
                           scale, tokens, per, head + 1);
    maxima = head + 1;
  }
  const int64_t total = tokens * K;
  const int64_t blocks = (total + 4 * 2048 - 1) / (4 * 2048);
  const int64_t cap = static_cast<int64_t>(num_sms_of_current_device()) * 64;
  const dim3 grid(static_cast<unsigned>(blocks < cap ? blocks : cap));
  const int8_t* qp = static_cast<const int8_t*>(q);
  T *hp = static_cast<T*>(hi), *lp = static_cast<T*>(lo);
  LaunchScope scope(HLM_KERNEL_DEQUANT_ROWS, s);
  if (total < (1ll << 31))  // 32-bit division; a step past the end stays below 2^32
    (void)launch_dependent(weight_grad_q8_split_kernel<T, uint32_t>, grid, dim3(256), 0, s, 1, qp, scale,
                           maxima, static_cast<int>(n_maxima), head, hp, lp,
                           static_cast<uint32_t>(total), static_cast<uint32_t>(K));
  else
    (void)launch_dependent(weight_grad_q8_split_kernel<T, uint64_t>, grid, dim3(256), 0, s, 1, qp, scale,
                           maxima, static_cast<int>(n_maxima), head, hp, lp,
                           static_cast<uint64_t>(total), static_cast<uint64_t>(K));
  return launch_status();
}

template <typename T>
static int weight_grad_q8_reduce(const float* partial, void* grad_w, int64_t n, int splits, const float* up,
                                 cudaStream_t s) {
  const int64_t blocks = (n / 8 + 255) / 256, cap = static_cast<int64_t>(num_sms_of_current_device()) * 16;
  LaunchScope scope(0, s);
  (void)launch_dependent(weight_grad_q8_reduce_kernel<T>, dim3(static_cast<unsigned>(blocks < cap ? blocks : cap)),
                         dim3(256), 0, s, 1, partial, static_cast<T*>(grad_w), n, splits, up);
  return launch_status();
}

}  // namespace hlm

using namespace hlm;

static size_t weight_grad_q8_bytes(const WgPlan& plan, int64_t tokens, int64_t N, int64_t K) {
  const size_t part =
      plan.splits > 1 ? static_cast<size_t>(plan.splits) * static_cast<size_t>(N) * static_cast<size_t>(K) * 4 : 0;
  return kWgHeadBytes + 2 * weight_grad_q8_back_bytes(tokens, K) + part;
}

extern "C" size_t hlm_weight_grad_q8_workspace_bytes(int64_t tokens, int64_t N, int64_t K) {
  if (tokens <= 0 || N <= 0 || K <= 0) return 0;
  return weight_grad_q8_bytes(weight_grad_q8_plan(tokens, N, K), tokens, N, K);
}

extern "C" int hlm_weight_grad_q8_plan(int64_t tokens, int64_t N, int64_t K, int* columns, int* splits) {
  if (tokens <= 0 || N <= 0 || K <= 0 || columns == nullptr || splits == nullptr) return HLM_ERR_INVALID_ARG;
  const WgPlan plan = weight_grad_q8_plan(tokens, N, K);
  *columns = plan.bn;
  *splits = plan.splits;
  return HLM_OK;
}

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
  const WgPlan plan = weight_grad_q8_plan(tokens, N, K);
  if (workspace == nullptr || workspace_bytes < weight_grad_q8_bytes(plan, tokens, N, K)) return HLM_ERR_WORKSPACE;
  if (!host_aligned16(workspace)) return HLM_ERR_UNSUPPORTED;
  const int splits = plan.splits;
  float* head = static_cast<float*>(workspace);
  uint8_t* hi = static_cast<uint8_t*>(workspace) + kWgHeadBytes;
  uint8_t* lo = hi + weight_grad_q8_back_bytes(tokens, K);
  float* partial = reinterpret_cast<float*>(lo + weight_grad_q8_back_bytes(tokens, K));
  const int fp16 = dtype == HLM_F16;
  int rc = fp16 ? weight_grad_q8_split<__half>(q, scale, head, hi, lo, tokens, K, s)
                : weight_grad_q8_split<__nv_bfloat16>(q, scale, head, hi, lo, tokens, K, s);
  if (rc != HLM_OK) return rc;
  auto gemm = plan.bn == 128 ? (fp16 ? weight_grad_q8_gemm<KindF16, 128> : weight_grad_q8_gemm<KindBf16, 128>)
                             : (fp16 ? weight_grad_q8_gemm<KindF16, 256> : weight_grad_q8_gemm<KindBf16, 256>);
  rc = gemm(grad, hi, lo, grad_w, partial, head, fp16, tokens, N, K, splits, s);
  if (rc != HLM_OK || splits == 1) return rc;
  return fp16 ? weight_grad_q8_reduce<__half>(partial, grad_w, N * K, splits, head, s)
              : weight_grad_q8_reduce<__nv_bfloat16>(partial, grad_w, N * K, splits, head, s);
}
