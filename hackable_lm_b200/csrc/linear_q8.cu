// 8-bit integer projection:
//
//   y[m, n] = (sum_k q[m, k] w[n, k]) * scale[m] * w_scale[n]
//
// q [M, K] and w [N, K] int8 with K contiguous, exact int32 sums (any order gives
// the same bits), the two scales applied in fp32, one rounding to the output type.
// Three kernels, by M and the number of output tiles:
//
//  - rows kernel, one token, or up to 8 and few weights: one pass over the weights with
//    dp4a; bound by reading w (and by launch latency at small sizes).
//  - split kernel, few output tiles: weights as the 128-row MMA operand, tokens as
//    the 16..128-column one, K split over a thread-block cluster whose CTAs add
//    their int32 partial tiles through distributed shared memory (no workspace,
//    one launch).
//  - pair kernel, many: the persistent CTA-pair GEMM of gemm_sm100.cuh with
//    kind::i8 (256 x 128 or 256 x 256 tiles) and the scales in its epilogue.
//
// Measured (bf16 out, weights out of L2): one token [4096, 768] 2.0 us, [8192, 8192]
// 12.7 us (5.3 TB/s of weights); [24, 768, 2048] 3.0 us; [777, 1111, 1360] 7.9 us;
// [32768, 4096, 768] 94 us, 2.2 POP/s and 2.9 TB/s of output (110 us once the power cap
// holds the clock at 1.4 GHz).  That case takes 66 us without its epilogue (3.1 POP/s), 79
// with it but for the stores, 94 to 96 whole: the output's way out holds it, not the tensor
// cores, which reach 2.9 POP/s at [8192, 8192, 8192].  Launched as
// dependents of the kernel before: [24, 768, 2048] 3.7 -> 3.0 us, [1024, 4096, 768]
// 8.1 -> 7.0.
#include <atomic>

#include "gemm_sm100.cuh"
#include "quant_common.cuh"

namespace hlm {

template <typename T>
HLM_DEVICE T scaled(int acc, float row_scale, float col_scale) {
  return from_f32<T>(static_cast<float>(acc) * row_scale * col_scale);
}

// ---------------------------------------------------------------------------
// M <= 8: R output channels per KS warps, lanes (and the KS warps) along K.
// ---------------------------------------------------------------------------
constexpr int kRowsWarps = 4;  // warps of a block

template <typename T, int MR, int R, int KS>
__global__ void __launch_bounds__(32 * kRowsWarps) linear_q8_rows_kernel(
    const int8_t* q, const float* scale, const int8_t* w,
    const float* w_scale, T* out, int M, int N, int K) {
  static_assert(KS == 1 || KS == kRowsWarps, "a warp's own channels, or a block's");
  grid_launch_next();
  grid_wait();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t n0 = (KS == 1 ? static_cast<int64_t>(blockIdx.x) * kRowsWarps + warp : blockIdx.x) * R;
  if (n0 >= N) return;  // KS > 1: the same for the whole block
  int acc[R][MR];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[r][m] = 0;
#pragma unroll 4
  for (int k = ((KS == 1 ? 0 : warp) * 32 + lane) * 16; k < K; k += 512 * KS) {
    uint4 wv[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t n = n0 + r < N ? n0 + r : N - 1;  // the last warp's spare rows repeat a row
      wv[r] = ld_global_stream_v4(w + n * K + k);
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const int mm = m < M ? m : M - 1;
      const uint4 x = ld_global_v4(q + static_cast<int64_t>(mm) * K + k);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        acc[r][m] = __dp4a(static_cast<int>(wv[r].x), static_cast<int>(x.x), acc[r][m]);
        acc[r][m] = __dp4a(static_cast<int>(wv[r].y), static_cast<int>(x.y), acc[r][m]);
        acc[r][m] = __dp4a(static_cast<int>(wv[r].z), static_cast<int>(x.z), acc[r][m]);
        acc[r][m] = __dp4a(static_cast<int>(wv[r].w), static_cast<int>(x.w), acc[r][m]);
      }
    }
  }
  // lane r * MR + m writes output (m, n0 + r)
  const int r_out = lane / MR, m_out = lane - r_out * MR;
  const bool writes = r_out < R && m_out < M && n0 + r_out < N && (KS == 1 || warp == 0);
  float rs = 0.0f, cs = 0.0f;
  if (writes) {  // on their way while the lanes' sums are added
    rs = scale[m_out];
    cs = w_scale[n0 + r_out];
  }
  int mine = 0;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const int sum = __reduce_add_sync(0xffffffffu, acc[r][m]);
      if (lane == r * MR + m) mine = sum;
    }
  if constexpr (KS > 1) {
    __shared__ int part[kRowsWarps][32];
    part[warp][lane] = mine;
    __syncthreads();
    if (warp != 0) return;
    mine = 0;
#pragma unroll
    for (int i = 0; i < kRowsWarps; ++i) mine += part[i][lane];
  }
  if (writes) out[static_cast<int64_t>(m_out) * N + n0 + r_out] = scaled<T>(mine, rs, cs);
}

// ---------------------------------------------------------------------------
// Few output tiles: K split over a cluster.
// ---------------------------------------------------------------------------
constexpr int kSplitThreads = 192;  // TMA warp, MMA warp, 4 epilogue warps
constexpr int kMaxSplits = 8;       // portable cluster size

template <int MT>
struct SplitSmem {
  static constexpr int kStages = MT <= 64 ? 6 : 4;
  static constexpr int kABytes = 128 * 128;  // 128 output channels x 128 bytes of K
  static constexpr int kBBytes = MT * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // partial sums from every CTA of the cluster for the token columns that this one
  // owns: [CTA][owned column][channel] int32; at most MT + 7 columns in all
  static constexpr int kPartOffset = kStages * kStageBytes;
  static constexpr int kPartBytes = (MT + kMaxSplits) * 128 * 4;
  static constexpr int kBarOffset = kPartOffset + kPartBytes;
  static constexpr int kTmemSlotOffset = kBarOffset + (2 * kStages + 1) * 8;
  static constexpr int kBytes = kTmemSlotOffset + 16 + 1024;
  static constexpr int kTmemCols = MT < 32 ? 32 : MT;
  static_assert(kBytes <= 232448, "shared memory budget exceeded");
};

HLM_DEVICE void st_shared_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
HLM_DEVICE int ld_shared_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// The two halves of a cluster barrier that hands over no memory.
HLM_DEVICE void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
HLM_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
HLM_DEVICE uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// One output tile (128 channels x MT tokens) per cluster; CTA `rank` sums K blocks
// [rank * kb_per, ...).  Token column c belongs to CTA c mod S: every CTA writes its
// int32 partial of that column (128 channels) into the owner's shared memory, and
// after one cluster barrier the owner adds the S partials, scales and writes them.
// Nothing is read remotely (such loads, one latency after the other, cost 16 us at
// 128 tokens), and no CTA touches a peer's memory after the barrier.
template <typename T, int MT>
__global__ void __launch_bounds__(kSplitThreads, 1)
    linear_q8_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_q,
                           const float* scale, const float* w_scale,
                           T* out, int M, int N, int k_blocks, int kb_per, int vec, int* err) {
  using L = SplitSmem<MT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw_addr);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t bar0 = base + L::kBarOffset;
  const uint32_t done_bar = bar0 + 8u * (2 * L::kStages);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + L::kTmemSlotOffset);
  const int rank = static_cast<int>(cluster_ctarank());
  const int splits = static_cast<int>(cluster_nctarank());
  const int n0 = static_cast<int>(cluster_id_x()) * 128;
  const int m0 = static_cast<int>(blockIdx.y) * MT;
  const int kb0 = rank * kb_per;
  const int kb1 = min(kb0 + kb_per, k_blocks);
  const int tokens = min(MT, M - m0);
  const int per = (tokens + splits - 1) / splits;  // columns that one CTA owns, at most

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(bar0 + 8u * s, 1);
      mbar_init(bar0 + 8u * (L::kStages + s), 1);
    }
    mbar_init(done_bar, 1);
    fence_mbar_init();
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_q);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_arrive_relaxed();  // this CTA runs: its memory may be written from now on
  grid_launch_next();
  grid_wait();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  // What the last step needs from global memory, fetched now.  A warp then takes the owned
  // columns warp, warp + 6, ...: lane l keeps the token scale of the l-th of them (at most
  // 128 / 6 = 22), and every lane the scales of its four channels: consecutive ones where
  // four outputs are one store (vec), else 32 apart (coalesced single stores).
  constexpr int kWarps = kSplitThreads / 32;
  const int my_col = rank + (warp + kWarps * lane) * splits;
  const float my_scale = my_col < tokens ? scale[m0 + my_col] : 0.0f;
  const int ch0 = vec ? 4 * lane : lane, ch_step = vec ? 1 : 32;
  float cs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) cs[i] = n0 + ch0 + i * ch_step < N ? w_scale[n0 + ch0 + i * ch_step] : 0.0f;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, armed_mask = 0, armed_par = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(bar0 + 8u * (L::kStages + stage), phase ^ 1u, err, kDevErrTimeoutEmpty)) break;
        const uint32_t full = bar0 + 8u * stage;
        mbar_arrive_expect_tx(full, L::kStageBytes);
        armed_mask |= 1u << stage;
        armed_par = (armed_par & ~(1u << stage)) | (phase << stage);
        const uint32_t sa = base + stage * L::kStageBytes;
        tma_load_2d(sa, &tm_w, kb * KindS8::kBlockK, n0, full);
        tma_load_2d(sa + L::kABytes, &tm_q, kb * KindS8::kBlockK, m0, full);
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      for (int s = 0; s < L::kStages; ++s)
        if (armed_mask & (1u << s)) mbar_wait_drain(bar0 + 8u * s, (armed_par >> s) & 1u, err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_s8_s32(128, MT);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(bar0 + 8u * stage, phase, err, kDevErrTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sa = base + stage * L::kStageBytes;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          tc_mma_i8(tmem_base, make_sw128_desc(sa + kk * 32u, 16u, 1024u),
                    make_sw128_desc(sa + L::kABytes + kk * 32u, 16u, 1024u), idesc,
                    (kb > kb0 || kk > 0) ? 1u : 0u);
        tc_commit(bar0 + 8u * (L::kStages + stage));
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) tc_commit(done_bar);
    }
  } else {
    const int quad = warp & 3;
    const bool ok = warp_wait(done_bar, 0, err, kDevErrTimeoutTmemFull, lane);
    cluster_wait();  // the owners run
    if (ok) {
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
      // slot of column c: CTA c % splits, row rank * per + c / splits
      const uint32_t mine = base + L::kPartOffset + static_cast<uint32_t>((rank * per * 128 + quad * 32 + lane) * 4);
      int owner = 0;
      uint32_t slot = 0;
#pragma unroll 1
      for (int c = 0; c < tokens; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(taddr + static_cast<uint32_t>(c), r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          if (c + j < tokens) st_shared_cluster_u32(mapa_shared(mine + slot, static_cast<uint32_t>(owner)), r[j]);
          if (++owner == splits) {
            owner = 0;
            slot += 512u;
          }
        }
      }
      tc_fence_before();
    }
  }
  __syncwarp();
  if (warp < 2) cluster_wait();  // pairs with the first arrive, like the epilogue warps' above
  cluster_sync_all();            // every partial of this CTA's columns has arrived
#pragma unroll 2
  for (int j = 0; j < (128 + kWarps - 1) / kWarps; ++j) {
    const int i = warp + kWarps * j;
    if (rank + i * splits >= tokens) break;
    const int m = m0 + rank + i * splits;
    const float rs = __shfl_sync(0xffffffffu, my_scale, j);
    const uint32_t col = base + L::kPartOffset + static_cast<uint32_t>(i * 512);
    int sum[4] = {0, 0, 0, 0};
    if (vec) {
      for (int s = 0; s < splits; ++s) {
        const uint4 v = ld_shared_v4(col + static_cast<uint32_t>(s * per * 512 + lane * 16));
        sum[0] += static_cast<int>(v.x);
        sum[1] += static_cast<int>(v.y);
        sum[2] += static_cast<int>(v.z);
        sum[3] += static_cast<int>(v.w);
      }
    } else {
      for (int s = 0; s < splits; ++s) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          sum[k] += ld_shared_s32(col + static_cast<uint32_t>(s * per * 512 + (lane + 32 * k) * 4));
      }
    }
    alignas(16) T y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = scaled<T>(sum[k], rs, cs[k]);
    T* dst = out + static_cast<int64_t>(m) * N + n0;
    if (vec) {
      if (n0 + ch0 < N) {  // N % 4 == 0: all four or none
        if constexpr (sizeof(T) == 4)
          *reinterpret_cast<uint4*>(dst + ch0) = *reinterpret_cast<const uint4*>(y);
        else
          *reinterpret_cast<uint2*>(dst + ch0) = *reinterpret_cast<const uint2*>(y);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n0 + lane + 32 * k < N) dst[lane + 32 * k] = y[k];
    }
  }
  __syncwarp();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Many output tiles: CTA-pair GEMM with the scales in the epilogue.
// ---------------------------------------------------------------------------
// Per warp (32 rows) and group of 128 output bytes (64 or 32 columns): int32
// columns from TMEM (one row per lane), scaled, staged as a 32 x 128-byte box
// (16-byte chunks swizzled by row) and written out with 16-byte stores, four
// whole 128-byte row segments per instruction.  Plain stores and not TMA: nothing
// waits for them ([32768, 4096, 768] 113 us against 121 with TMA stores of two boxes a
// warp, and 99 once the accumulator goes back without a release).  Outputs whose rows are not 16-byte multiples leave the box
// element by element, a row segment per step.
template <typename T>
struct EpiScaleQ8 {
  struct Params {
    T* out;
    const float* row_scale;
    const float* col_scale;
    int vec;  // rows of the output are 16-byte aligned
  };
  static constexpr bool kRelaxedRelease = true;
  static constexpr bool kDependentLaunch = true;
  static constexpr int kCols = 128 / static_cast<int>(sizeof(T));  // columns of a group
  static constexpr int kPerChunk = 16 / static_cast<int>(sizeof(T));
  static constexpr int kBoxBytes = 32 * 128;
  static constexpr int kWarpBytes = kBoxBytes + 256;  // box, then the group's column scales
  template <int EPI_WARPS>
  static constexpr int smem_bytes() {
    return EPI_WARPS * kWarpBytes;
  }

  // This lane's row scale and its column scales of every group the warp takes, loaded
  // before the wait for the accumulator.
  struct Early {
    float rs;
    float cs[4][2];
  };
  template <int BN, int kParts>
  static HLM_DEVICE void load_early(const Params& ep, const GemmParams& p, Early& e, int m_tile, int n_tile,
                                    int quad, int part, int lane) {
    const int row = m_tile * kBM + quad * 32 + lane;
    e.rs = row < p.M ? ep.row_scale[row] : 0.0f;
    static_assert(BN / kCols <= 4 * kParts, "groups of a warp");
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) {
        const int g = part + k * kParts;
        const int col = n_tile * BN + g * kCols + 32 * i + lane;
        e.cs[k][i] = g < BN / kCols && col < p.N ? ep.col_scale[col] : 0.0f;
      }
  }

  template <int BN, int kParts>
  static HLM_DEVICE void run(const Params& ep, const GemmParams& p, uint8_t* smem, uint32_t taddr,
                             int m_tile, int n_tile, int, int quad, int part, int lane, const Early& e) {
    uint8_t* box = smem + (part * 4 + quad) * kWarpBytes;
    const uint32_t buf = smem_u32(box);
    float* cs_ptr = reinterpret_cast<float*>(box + kBoxBytes);
    const uint32_t cs_addr = buf + kBoxBytes;
    const int row0 = m_tile * kBM + quad * 32;
    const float rs = e.rs;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int g = part + k * kParts;
      if (g >= BN / kCols) break;
      const int col0 = n_tile * BN + g * kCols;
      if (col0 >= p.N) break;  // the same for the whole warp
      __syncwarp();            // the box's last group has been read
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) cs_ptr[32 * i + lane] = e.cs[k][i];
      __syncwarp();
#pragma unroll
      for (int hs = 0; hs < kCols / 32; ++hs) {
        uint32_t a[32];
        tmem_ld_32x32b_x32(taddr + static_cast<uint32_t>(g * kCols + hs * 32), a);
        tmem_ld_wait();
        float f[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint4 c4 = ld_shared_v4(cs_addr + static_cast<uint32_t>(hs * 128 + j * 16));
          f[4 * j] = static_cast<float>(static_cast<int>(a[4 * j])) * rs * __uint_as_float(c4.x);
          f[4 * j + 1] = static_cast<float>(static_cast<int>(a[4 * j + 1])) * rs * __uint_as_float(c4.y);
          f[4 * j + 2] = static_cast<float>(static_cast<int>(a[4 * j + 2])) * rs * __uint_as_float(c4.z);
          f[4 * j + 3] = static_cast<float>(static_cast<int>(a[4 * j + 3])) * rs * __uint_as_float(c4.w);
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            st_shared_v4(buf + static_cast<uint32_t>(lane * 128 + ((c ^ (lane & 7)) << 4)),
                         make_uint4(__float_as_uint(f[4 * c]), __float_as_uint(f[4 * c + 1]),
                                    __float_as_uint(f[4 * c + 2]), __float_as_uint(f[4 * c + 3])));
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int cc = hs * 4 + c;
            st_shared_v4(buf + static_cast<uint32_t>(lane * 128 + ((cc ^ (lane & 7)) << 4)),
                         make_uint4(pack2<T>(f[8 * c], f[8 * c + 1]), pack2<T>(f[8 * c + 2], f[8 * c + 3]),
                                    pack2<T>(f[8 * c + 4], f[8 * c + 5]), pack2<T>(f[8 * c + 6], f[8 * c + 7])));
          }
        }
      }
      __syncwarp();
      if (ep.vec) {
        const int chunk = lane & 7;
        const bool col_ok = col0 + chunk * kPerChunk < p.N;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + (lane >> 3);
          const uint4 v = ld_shared_v4(buf + static_cast<uint32_t>(r * 128 + ((chunk ^ (r & 7)) << 4)));
          if (col_ok && row0 + r < p.M)
            st_global_v4(ep.out + static_cast<int64_t>(row0 + r) * p.N + col0 + chunk * kPerChunk, v);
        }
      } else {
        const int rows = min(32, p.M - row0);
        for (int r = 0; r < rows; ++r) {
#pragma unroll
          for (int i = 0; i < kCols / 32; ++i) {
            const int c = 32 * i + lane;
            const T v = *reinterpret_cast<const T*>(box + r * 128 + (((c / kPerChunk) ^ (r & 7)) << 4) +
                                                    (c % kPerChunk) * static_cast<int>(sizeof(T)));
            if (col0 + c < p.N) ep.out[static_cast<int64_t>(row0 + r) * p.N + col0 + c] = v;
          }
        }
      }
    }
  }
};

constexpr int kQ8EpiWarps = 8;

template <typename T, int BN>
static int linear_q8_pair(const void* q, const float* scale, const void* w, const float* w_scale, T* out,
                          int64_t M, int64_t N, int64_t K, int* err, cudaStream_t s) {
  CUtensorMap ma, mb;
  if (!encode_map(&ma, q, 1, K, M, K, kBM) || !encode_map(&mb, w, 1, K, N, K, 64)) return HLM_ERR_DRIVER;
  typename EpiScaleQ8<T>::Params ep;
  ep.out = out;
  ep.row_scale = scale;
  ep.col_scale = w_scale;
  ep.vec = (N * static_cast<int64_t>(sizeof(T))) % 16 == 0 && host_aligned16(out);
  GemmParams p;
  gemm_tiling_pair(p, static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), BN, 1, KindS8::kBlockK);
  p.err = err;
  return launch_gemm_pair<BN, BN == 256 ? 5 : 7, false, false, EpiScaleQ8<T>, kQ8EpiWarps, KindS8>(
      ma, ma, ma, mb, p, ep, s, HLM_KERNEL_LINEAR_Q8);
}

// Clusters of `size` CTAs, one to an SM, that the current device holds at once: fewer than
// SMs / size, since a cluster lies within one GPC (of 148 SMs, 16 clusters of eight).
// Asked of the runtime once per device and size.
static int max_clusters(int size) {
  static std::atomic<int> cache[64][kMaxSplits + 1];
  int dev = 0;
  if (size <= 1 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return num_sms_of_current_device();
  int n = cache[dev][size].load(std::memory_order_relaxed);
  if (n > 0) return n;
  using L = SplitSmem<64>;
  auto kern = linear_q8_split_kernel<__nv_bfloat16, 64>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(size);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(size), 1, 1);
  cfg.blockDim = dim3(kSplitThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    n = 1;
  }
  cache[dev][size].store(n, std::memory_order_relaxed);
  return n;
}

// K blocks of a CTA of the split kernel: the most splits whose clusters run at once.
static int blocks_per_split(int64_t tiles, int k_blocks) {
  int64_t splits = num_sms_of_current_device() / tiles;
  if (splits > kMaxSplits) splits = kMaxSplits;
  if (splits > k_blocks) splits = k_blocks;
  while (splits > 1 && max_clusters(static_cast<int>(splits)) < tiles) --splits;
  if (splits < 1) splits = 1;
  return static_cast<int>((k_blocks + splits - 1) / splits);
}

template <typename T, int MT>
static int linear_q8_split(const void* q, const float* scale, const void* w, const float* w_scale, T* out,
                           int64_t M, int64_t N, int64_t K, int* err, cudaStream_t s) {
  using L = SplitSmem<MT>;
  CUtensorMap mw, mq;
  if (!encode_map(&mw, w, 1, K, N, K, 128) || !encode_map(&mq, q, 1, K, M, K, MT)) return HLM_ERR_DRIVER;
  const int n_tiles = static_cast<int>((N + 127) / 128), m_tiles = static_cast<int>((M + MT - 1) / MT);
  const int k_blocks = static_cast<int>((K + KindS8::kBlockK - 1) / KindS8::kBlockK);
  const int kb_per = blocks_per_split(static_cast<int64_t>(n_tiles) * m_tiles, k_blocks);
  const int splits = (k_blocks + kb_per - 1) / kb_per;
  auto kern = linear_q8_split_kernel<T, MT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes) != cudaSuccess)
    return launch_status();
  // four outputs of a lane as one store
  const int vec = N % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0;
  {
    LaunchScope scope(HLM_KERNEL_LINEAR_Q8, s);
    (void)launch_dependent(kern, dim3(static_cast<unsigned>(n_tiles * splits), static_cast<unsigned>(m_tiles)),
                           dim3(kSplitThreads), L::kBytes, s, splits, mw, mq, scale, w_scale, out, static_cast<int>(M),
                           static_cast<int>(N), k_blocks, kb_per, vec, err);
  }
  return launch_status();
}

// A block's warps share a pair of channels where rows are long and the warps of single
// pairs few or their tokens one: [1, 4096, 4096] 5.1 us against 6.7 with a warp a pair,
// [8, 768, 2048] 2.4 against 3.3; but [1, 4096, 1024] 2.8 against 2.6, and
// [8, 4096, 2048], where the adding of 16 sums weighs, 6.7 against 4.8.
template <typename T, int MR>
static int linear_q8_rows(const void* q, const float* scale, const void* w, const float* w_scale, T* out,
                          int64_t M, int64_t N, int64_t K, cudaStream_t s) {
  constexpr int R = 2;
  const int8_t* qp = static_cast<const int8_t*>(q);
  const int8_t* wp = static_cast<const int8_t*>(w);
  LaunchScope scope(HLM_KERNEL_LINEAR_Q8, s);
  const bool shared = K >= 2048 && (M == 1 || N <= 2048);
  const int64_t blocks = shared ? (N + R - 1) / R : (N + R * kRowsWarps - 1) / (R * kRowsWarps);
  (void)launch_dependent(shared ? linear_q8_rows_kernel<T, MR, R, kRowsWarps> : linear_q8_rows_kernel<T, MR, R, 1>,
                         dim3(static_cast<unsigned>(blocks)), dim3(32 * kRowsWarps), 0, s, 1, qp, scale, wp, w_scale, out,
                         static_cast<int>(M), static_cast<int>(N), static_cast<int>(K));
  return launch_status();
}

// The tensor-core kernel that takes least time, in microseconds as measured with K blocks
// of 128: the split kernel with 16, 32, 64 or 128 tokens a tile (while its tiles fit the
// SMs at once), or the pair kernel with 256 x 128 (-128) or 256 x 256 (-256) tiles, whose
// pairs take further tiles in rounds.  Measured either way:
//   [64, 4096, 768]    32 tokens 4.5 us, 64 tokens 4.9
//   [128, 768, 2048]   64 tokens 5.2, 128 tokens 6.0;  [128, 8192, 8192] 128 tokens 20, 64 tokens 25
//   [300, 1000, 4096]  64 tokens 7.7, 256 x 128 14.0;  [512, 2304, 768] 7.3 and 6.5
//   [1024, 2304, 768]  256 x 128 6.9, 256 x 256 7.7;   [1024, 4096, 768] 9.5 and 8.3
//   [777, 1111, 1360] to fp32 (rows of 4444 bytes)  64 tokens 8.9, 256 x 128 10.3
static int choose_tile(int64_t M, int64_t N, int64_t K, bool aligned_rows) {
  const int64_t sms = num_sms_of_current_device(), pairs = sms / 2 > 0 ? sms / 2 : 1;
  const int kb = static_cast<int>((K + KindS8::kBlockK - 1) / KindS8::kBlockK);
  struct {
    int tokens;
    double fixed, block;
  } const split[4] = {{16, 3.4, 0.30}, {32, 3.9, 0.31}, {64, 4.5, 0.34}, {128, 5.5, 0.48}};
  auto rounds = [&](int64_t bn) {
    return static_cast<double>((((M + 255) / 256) * ((N + bn - 1) / bn) + pairs - 1) / pairs);
  };
  const double r128 = rounds(128), r256 = rounds(256);
  const double next256 = 0.45 * kb > 3.0 ? 0.45 * kb : 3.0;
  const double ragged = aligned_rows ? 0.0 : 1.7;  // its epilogue by elements, a round
  const double pair128 = 4.7 + r128 * (0.29 * kb + ragged) + (r128 - 1.0) * 1.2;
  const double pair256 = 5.5 + 0.33 * kb + (r256 - 1.0) * next256 + r256 * 2.0 * ragged;
  int best = pair128 < pair256 ? -128 : -256;
  double best_us = pair128 < pair256 ? pair128 : pair256;
  for (const auto& t : split) {
    const int64_t tiles = ((M + t.tokens - 1) / t.tokens) * ((N + 127) / 128);
    if (tiles > sms && M > 128) continue;  // (up to 128 tokens a tile is mostly weights: further waves stream on)
    const double waves = static_cast<double>((tiles + sms - 1) / sms);
    const double us = t.fixed + waves * t.block * blocks_per_split(tiles, kb);
    if (us < best_us) {
      best_us = us;
      best = t.tokens;
    }
  }
  return best;
}

// dp4a for a few tokens of small weights: with M tokens it needs M instructions for four
// weights, and falls behind the tensor cores from about 8 M weights on ([8, 4096, 2048]
// 4.8 us against 5.6, [8, 4096, 4096] 7.8 against 7.0, [8, 8192, 8192] 25 against 15)
static bool rows_kernel(int64_t M, int64_t N, int64_t K) { return M == 1 || (M <= 8 && N * K <= (1ll << 23)); }

template <typename T>
static int linear_q8(const void* q, const float* scale, const void* w, const float* w_scale, T* out, int64_t M,
                     int64_t N, int64_t K, cudaStream_t s) {
  if (rows_kernel(M, N, K)) {
    if (M == 1) return linear_q8_rows<T, 1>(q, scale, w, w_scale, out, M, N, K, s);
    if (M <= 4) return linear_q8_rows<T, 4>(q, scale, w, w_scale, out, M, N, K, s);
    return linear_q8_rows<T, 8>(q, scale, w, w_scale, out, M, N, K, s);
  }
  int* err = device_error_ptr();
  if (err == nullptr) return HLM_ERR_LAUNCH;
  switch (choose_tile(M, N, K, N * static_cast<int64_t>(sizeof(T)) % 16 == 0 && host_aligned16(out))) {
    case 16:
      return linear_q8_split<T, 16>(q, scale, w, w_scale, out, M, N, K, err, s);
    case 32:
      return linear_q8_split<T, 32>(q, scale, w, w_scale, out, M, N, K, err, s);
    case 64:
      return linear_q8_split<T, 64>(q, scale, w, w_scale, out, M, N, K, err, s);
    case 128:
      return linear_q8_split<T, 128>(q, scale, w, w_scale, out, M, N, K, err, s);
    case -128:
      return linear_q8_pair<T, 128>(q, scale, w, w_scale, out, M, N, K, err, s);
    default:
      return linear_q8_pair<T, 256>(q, scale, w, w_scale, out, M, N, K, err, s);
  }
}

}  // namespace hlm

using namespace hlm;

static bool linear_q8_supported(int64_t M, int64_t N, int64_t K) {
  // 128 * 128 * K stays within int32 up to K = 131056; TMA rows are 16-byte multiples
  return K > 0 && K % 16 == 0 && K <= HLM_LINEAR_Q8_MAX_K && M <= (1ll << 31) - 512 && N <= (1ll << 31) - 512;
}

extern "C" int hlm_linear_q8_plan(int64_t M, int64_t N, int64_t K, int out_dtype, int* tile) {
  if (M <= 0 || N <= 0 || K < 0 || tile == nullptr) return HLM_ERR_INVALID_ARG;
  if (out_dtype != HLM_F32 && out_dtype != HLM_BF16 && out_dtype != HLM_F16) return HLM_ERR_UNSUPPORTED;
  if (!linear_q8_supported(M, N, K)) return HLM_ERR_UNSUPPORTED;
  *tile = rows_kernel(M, N, K) ? 0 : choose_tile(M, N, K, N * (out_dtype == HLM_F32 ? 4 : 2) % 16 == 0);
  return HLM_OK;
}

extern "C" int hlm_linear_q8(const void* q, const float* scale, const void* w, const float* w_scale,
                             void* out, int64_t M, int64_t N, int64_t K, int out_dtype, void* stream) {
  if (M < 0 || N < 0 || K < 0) return HLM_ERR_INVALID_ARG;
  if (out_dtype != HLM_F32 && out_dtype != HLM_BF16 && out_dtype != HLM_F16)
    return HLM_ERR_UNSUPPORTED;
  if (M == 0 || N == 0) return HLM_OK;
  if (q == nullptr || scale == nullptr || w == nullptr || w_scale == nullptr || out == nullptr)
    return HLM_ERR_INVALID_ARG;
  if (!linear_q8_supported(M, N, K)) return HLM_ERR_UNSUPPORTED;
  if (!host_aligned16(q) || !host_aligned16(w)) return HLM_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (out_dtype) {
    case HLM_BF16:
      return linear_q8<__nv_bfloat16>(q, scale, w, w_scale, static_cast<__nv_bfloat16*>(out), M, N, K, s);
    case HLM_F16:
      return linear_q8<__half>(q, scale, w, w_scale, static_cast<__half*>(out), M, N, K, s);
    default:
      return linear_q8<float>(q, scale, w, w_scale, static_cast<float*>(out), M, N, K, s);
  }
}
