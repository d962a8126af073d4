// Weight gradient of a projection whose input was kept in 8 bits:
//
//   grad_w[n, k] = sum_m grad[m, n] * (q[m, k] * scale[m])
//
// One CTA-pair tcgen05 GEMM (512 x 256 tiles of grad_w, tokens as the reduction),
// whose B operand is made in the kernel: TMA brings the int8 codes of 64 tokens x
// 128 input features per CTA, eight converter warps read them back to the gradient's
// type (q * scale in fp32, rounded once: the MMA takes one 16-bit type for both
// operands) and write the swizzled MN-major tile that the MMA reads.  The codes are
// half the bytes of the activations, and no read-back tensor goes to memory.
//
// A tile is two 256-row MMAs on the same B: each converted value feeds 512 rows.
// With one 256-row MMA (two accumulators instead, the epilogue overlapped) the
// converters' shared-memory traffic and latency held the tensor cores to 990
// TFLOP/s at [2048 tokens, 8192, 8192].
//
// Few tiles: the tokens are split and each split writes an fp32 partial to the
// workspace; a second kernel adds the partials in the order of the splits (the same
// bits every time) and rounds.
#include "gemm_sm100.cuh"
#include "quant_common.cuh"

namespace hlm {

constexpr int kWgStages = 4;     // A tiles
constexpr int kWgRawStages = 4;  // codes: their own ring and producer, so that they run ahead of A
constexpr int kWgBStages = 3;    // read-back tiles
constexpr int kWgGroups = 2;     // converter groups, which take turns on the token blocks
constexpr int kWgGroupWarps = 4;
// A group skips the barrier phases of the other groups' blocks, and a parity wait tells
// a phase only from its neighbours, so the phase before the awaited one must be known
// to be over.  Read-back tiles: the group's last block n waited for the MMAs of block
// n - kWgBStages, and n + kWgGroups - 2 kWgBStages is not after it.  Codes: block
// n - kWgRawStages was the group's own.
static_assert(kWgBStages >= kWgGroups && kWgRawStages % kWgGroups == 0, "unambiguous phases");
constexpr int kWgConvWarps = kWgGroups * kWgGroupWarps;
constexpr int kWgEpiWarps = 8;  // two per TMEM lane quadrant, one for each half of the tile's rows
constexpr int kWgConvWarp0 = kEpiWarp0 + kWgEpiWarps;
constexpr int kWgRawWarp = kWgConvWarp0 + kWgConvWarps;
constexpr int kWgBM = 512;       // rows (output features) of a pair's tile
constexpr int kWgThreads = 32 * (kWgRawWarp + 1);

struct WgSmem {
  static constexpr int kSubBytes = kBM * kBK * 2;  // 128 output features x 64 tokens, 16-bit
  static constexpr int kABytes = 2 * kSubBytes;  // this CTA's rows of the two MMAs
  static constexpr int kRawBytes = 128 * kBK;    // 128 input features x 64 tokens, codes
  static constexpr int kBBytes = 128 * kBK * 2;  // the same, read back
  static constexpr int kRawOffset = kWgStages * kABytes;
  static constexpr int kBOffset = kRawOffset + kWgRawStages * kRawBytes;
  static constexpr int kBoxOffset = kBOffset + kWgBStages * kBBytes;  // epilogue boxes, 2 KB per warp
  static constexpr int kBarOffset = kBoxOffset + kWgEpiWarps * 2048;
  static constexpr int kNumBars = 2 * kWgStages + 2 * kWgRawStages + 2 * kWgBStages + 3;
  static constexpr int kTmemSlotOffset = kBarOffset + kNumBars * 8;
  static constexpr int kBytes = kTmemSlotOffset + 16 + 1024;
  static_assert(kBytes <= 232448, "shared memory budget exceeded");
};

template <typename T>
HLM_DEVICE uint32_t pack2_16(float a, float b);
template <>
HLM_DEVICE uint32_t pack2_16<__nv_bfloat16>(float a, float b) {
  return pack_bf16x2(a, b);
}
template <>
HLM_DEVICE uint32_t pack2_16<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Instruction descriptor for kind::f16 with MN-major operands of type T and fp32 D.
template <typename T>
constexpr uint32_t wg_idesc() {
  constexpr uint32_t type = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;  // bf16 or f16
  return (1u << 4) | (type << 7) | (type << 10) | (1u << 15) | (1u << 16) | ((256u >> 3) << 17) | ((256u >> 4) << 24);
}

// Write a warp's 32 rows x 256 columns of the accumulator as O (fp32 partial or the
// 16-bit result): staged in a 32 x 64-byte box (16-byte chunks swizzled by row pairs),
// out in 16-byte stores, eight 64-byte row segments per instruction.
template <typename O>
HLM_DEVICE void wg_store_tile(O* dst, int64_t ld, int row0, int rows, int col0, int cols, uint32_t taddr,
                              uint32_t buf, int lane) {
  constexpr int kCols = 64 / static_cast<int>(sizeof(O));  // columns of a box: 16 fp32 or 32 16-bit
  constexpr int kPerChunk = 16 / static_cast<int>(sizeof(O));
  if (row0 >= rows) return;
  const uint32_t sw = static_cast<uint32_t>(lane >> 1) & 3u;
#pragma unroll 1
  for (int g = 0; g < 8; ++g) {
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
            w[i] = pack2_16<O>(__uint_as_float(a[8 * c + 2 * i]), __uint_as_float(a[8 * c + 2 * i + 1]));
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

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWgThreads, 1)
    weight_grad_q8_kernel(const __grid_constant__ CUtensorMap tm_g, const __grid_constant__ CUtensorMap tm_q,
                          const float* __restrict__ scale, T* __restrict__ grad_w, float* __restrict__ partial,
                          int tokens, const GemmParams p) {
  using L = WgSmem;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw_addr);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t bar0 = base + L::kBarOffset;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + L::kTmemSlotOffset);
  int* err = p.err;
#define FULL_BAR(s) (bar0 + 8u * (s))                                // even CTA: both halves of A landed
#define EMPTY_BAR(s) (bar0 + 8u * (kWgStages + (s)))                 // pair MMAs done with A
#define RAWF_BAR(r) (bar0 + 8u * (2 * kWgStages + (r)))              // this CTA's codes landed
#define RAWE_BAR(r) (bar0 + 8u * (2 * kWgStages + kWgRawStages + (r)))  // converters have read them
#define BAR_B0 (2 * kWgStages + 2 * kWgRawStages)
#define BRDY_BAR(b) (bar0 + 8u * (BAR_B0 + (b)))                     // even CTA: both CTAs' B tiles written
#define BEMP_BAR(b) (bar0 + 8u * (BAR_B0 + kWgBStages + (b)))        // pair MMAs done with B
#define TFULL_BAR (bar0 + 8u * (BAR_B0 + 2 * kWgBStages))
#define TEMPTY_BAR(h) (bar0 + 8u * (BAR_B0 + 2 * kWgBStages + 1 + (h)))  // even CTA: half h of the tile drained

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < kWgStages; ++s) {
      mbar_init(FULL_BAR(s), 1);
      mbar_init(EMPTY_BAR(s), 1);
    }
    for (int r = 0; r < kWgRawStages; ++r) {
      mbar_init(RAWF_BAR(r), 1);
      mbar_init(RAWE_BAR(r), kWgGroupWarps);
    }
    for (int b = 0; b < kWgBStages; ++b) {
      mbar_init(BRDY_BAR(b), 2 * kWgGroupWarps);
      mbar_init(BEMP_BAR(b), 1);
    }
    mbar_init(TFULL_BAR, 1);
    for (int h = 0; h < 2; ++h) mbar_init(TEMPTY_BAR(h), kWgEpiWarps);  // four warps of each CTA
    fence_mbar_init();
    prefetch_tensormap(&tm_g);
    prefetch_tensormap(&tm_q);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();  // both CTAs' barriers initialised before any cross-CTA signal
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const int total = p.m_tiles * p.n_tiles * p.splits;
  const int w_first = static_cast<int>(cluster_id_x());
  const int w_step = static_cast<int>(num_clusters_x());

  if (warp == 0) {
    // ------------------------------------------------------------ producer of A
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t armed = 0, armed_par = 0;  // stages whose loads are in flight, and their parity
      bool ok = true;
      for (int w = w_first; w < total && ok; w += w_step) {
        int m_pair, n_tile, split;
        decode_work(w, p, m_pair, n_tile, split);
        const int n0 = m_pair * kWgBM + static_cast<int>(rank) * kBM;
        const int subs = m_pair * kWgBM + 256 < p.M ? 2 : 1;  // 256-row MMAs with rows in them
        const int kb0 = split * p.kb_per_split;
        const int kb1 = min(kb0 + p.kb_per_split, p.k_blocks);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(EMPTY_BAR(stage), phase ^ 1u, err, kDevErrTimeoutEmpty)) {
            ok = false;
            break;
          }
          if (rank == 0) {
            mbar_arrive_expect_tx(FULL_BAR(stage), static_cast<uint32_t>(subs) * 2 * L::kSubBytes);
            armed |= 1u << stage;
            armed_par = (armed_par & ~(1u << stage)) | (phase << stage);
          }
          const uint32_t full = mapa_shared(FULL_BAR(stage), 0);
          const uint32_t sa = base + stage * L::kABytes;
          for (int h = 0; h < subs; ++h) {
            tma_load_2d_pair(sa + h * L::kSubBytes, &tm_g, n0 + 256 * h, kb * kBK, full);
            tma_load_2d_pair(sa + h * L::kSubBytes + 8192u, &tm_g, n0 + 256 * h + 64, kb * kBK, full);
          }
          if (++stage == kWgStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // Drain (even CTA): every armed stage, including the peer's half, has landed before
      // either CTA releases its shared memory.
      for (int s = 0; s < kWgStages; ++s)
        if (armed & (1u << s)) mbar_wait_drain(FULL_BAR(s), (armed_par >> s) & 1u, err);
    }
  } else if (warp == kWgRawWarp) {
    // ------------------------------------------------------------ producer of the codes
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t armed = 0, armed_par = 0;
      bool ok = true;
      for (int w = w_first; w < total && ok; w += w_step) {
        int m_pair, n_tile, split;
        decode_work(w, p, m_pair, n_tile, split);
        const int k0 = n_tile * 256 + static_cast<int>(rank) * 128;
        const int kb0 = split * p.kb_per_split;
        const int kb1 = min(kb0 + p.kb_per_split, p.k_blocks);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(RAWE_BAR(stage), phase ^ 1u, err, kDevErrTimeoutEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(RAWF_BAR(stage), L::kRawBytes);
          armed |= 1u << stage;
          armed_par = (armed_par & ~(1u << stage)) | (phase << stage);
          tma_load_2d(base + L::kRawOffset + stage * L::kRawBytes, &tm_q, k0, kb * kBK, RAWF_BAR(stage));
          if (++stage == kWgRawStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      for (int s = 0; s < kWgRawStages; ++s)
        if (armed & (1u << s)) mbar_wait_drain(RAWF_BAR(s), (armed_par >> s) & 1u, err);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ pair MMA issuer (even CTA)
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = wg_idesc<T>();
      int stage = 0, bs = 0;
      uint32_t phase = 0, bphase = 0;
      int it = 0;
      bool ok = true;
      for (int w = w_first; w < total && ok; w += w_step, ++it) {
        int m_pair, n_tile, split;
        decode_work(w, p, m_pair, n_tile, split);
        const int kb0 = split * p.kb_per_split;
        const int kb1 = min(kb0 + p.kb_per_split, p.k_blocks);
        const int subs = m_pair * kWgBM + 256 < p.M ? 2 : 1;
        const uint32_t free_par = (static_cast<uint32_t>(it) & 1u) ^ 1u;
        if (!mbar_wait_cluster(TEMPTY_BAR(0), free_par, err, kDevErrTimeoutTmemEmpty) ||
            !mbar_wait_cluster(TEMPTY_BAR(1), free_par, err, kDevErrTimeoutTmemEmpty)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_cluster(FULL_BAR(stage), phase, err, kDevErrTimeoutFull) ||
              !mbar_wait_cluster(BRDY_BAR(bs), bphase, err, kDevErrTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = base + stage * L::kABytes;
          const uint32_t sb = base + L::kBOffset + bs * L::kBBytes;
#pragma unroll
          for (int kk = 0; kk < kBK / kUmmaK; ++kk)
            tc_mma_f16_pair(tmem_base, make_sw128_desc(sa + kk * 2048u, 8192u, 1024u),
                            make_sw128_desc(sb + kk * 2048u, 8192u, 1024u), idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
          if (subs == 2) {
#pragma unroll
            for (int kk = 0; kk < kBK / kUmmaK; ++kk)
              tc_mma_f16_pair(tmem_base + 256u, make_sw128_desc(sa + L::kSubBytes + kk * 2048u, 8192u, 1024u),
                              make_sw128_desc(sb + kk * 2048u, 8192u, 1024u), idesc,
                              (kb > kb0 || kk > 0) ? 1u : 0u);
          }
          tc_commit_pair(EMPTY_BAR(stage));
          tc_commit_pair(mapa_shared(EMPTY_BAR(stage), 1));
          tc_commit_pair(BEMP_BAR(bs));
          tc_commit_pair(mapa_shared(BEMP_BAR(bs), 1));
          if (++stage == kWgStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (++bs == kWgBStages) {
            bs = 0;
            bphase ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit_pair(TFULL_BAR);
        tc_commit_pair(mapa_shared(TFULL_BAR, 1));
      }
    }
  } else if (warp < kWgConvWarp0) {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int quad = warp & 3;
    const int half = (warp - kEpiWarp0) >> 2;
    const uint32_t buf = base + L::kBoxOffset + static_cast<uint32_t>(warp - kEpiWarp0) * 2048u;
    int it = 0;
    for (int w = w_first; w < total; w += w_step, ++it) {
      int m_pair, n_tile, split;
      decode_work(w, p, m_pair, n_tile, split);
      if (!warp_wait(TFULL_BAR, static_cast<uint32_t>(it) & 1u, err, kDevErrTimeoutTmemFull, lane)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(half * 256);
      const int row0 = m_pair * kWgBM + half * 256 + static_cast<int>(rank) * kBM + quad * 32;
      if (partial != nullptr)
        wg_store_tile<float>(partial + static_cast<int64_t>(split) * p.M * p.N, p.N, row0, p.M, n_tile * 256, p.N,
                             taddr, buf, lane);
      else
        wg_store_tile<T>(grad_w, p.N, row0, p.M, n_tile * 256, p.N, taddr, buf, lane);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(TEMPTY_BAR(half), 0));
    }
  } else {
    // ------------------------------------------------------------ converters (both CTAs)
    // A group's four warps make one block's tile (two groups: the waits, the proxy fence and
    // the arrive of a block are latency, which they overlap).  A warp makes 32 tokens of one
    // box (64 features): in each of four steps its lanes take eight tokens x four 16-byte
    // pieces of codes, and a piece becomes two 16-byte chunks of the read-back box.  The
    // eight lanes that access shared memory together hold tokens m and m ^ 5: under the
    // 128-byte swizzle both their reads (bit 2 differs) and their writes (bit 0 differs)
    // fall on eight different chunks.
    const int group = (warp - kWgConvWarp0) / kWgGroupWarps;
    const int box = (warp - kWgConvWarp0) & 1;
    const int tok0 = ((warp - kWgConvWarp0) & 2) * 16;  // the warp's first token of a block
    const int piece = lane & 3;
    const int m7 = (lane >> 3) ^ ((lane & 4) ? 5 : 0);  // token within a step's eight
    const uint32_t rd = static_cast<uint32_t>((tok0 + m7) * 128 + (((4 * box + piece) ^ m7) << 4));
    const uint32_t wr0 = static_cast<uint32_t>(box * 8192 + (tok0 + m7) * 128 + (((2 * piece) ^ m7) << 4));
    const uint32_t wr1 = static_cast<uint32_t>(box * 8192 + (tok0 + m7) * 128 + (((2 * piece + 1) ^ m7) << 4));
    float sc[4];     // scales of this lane's tokens in block sc_kb
    int sc_kb = -1;
    auto load_scales = [&](int kb) {
      const int tok = kb * kBK + tok0 + m7;
      sc_kb = kb;
#pragma unroll
      for (int j = 0; j < 4; ++j)  // tokens past the end: their codes and gradients arrive as zeros
        sc[j] = tok + 8 * j < tokens ? __ldg(scale + tok + 8 * j) : 0.0f;
    };
    int stage = 0, bs = 0, turn = 0;
    uint32_t phase = 0, bphase = 0;
    bool ok = true;
    for (int w = w_first; w < total && ok; w += w_step) {
      int m_pair, n_tile, split;
      decode_work(w, p, m_pair, n_tile, split);
      const int kb0 = split * p.kb_per_split;
      const int kb1 = min(kb0 + p.kb_per_split, p.k_blocks);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (turn == group) {
          if (sc_kb != kb) load_scales(kb);
          if (!warp_wait(RAWF_BAR(stage), phase, err, kDevErrTimeoutFull, lane)) {
            ok = false;
            break;
          }
          const uint32_t raw = base + L::kRawOffset + stage * L::kRawBytes + rd;
          const uint32_t sb = base + L::kBOffset + bs * L::kBBytes;
          if (!warp_wait(BEMP_BAR(bs), bphase ^ 1u, err, kDevErrTimeoutEmpty, lane)) {
            ok = false;
            break;
          }
          uint4 v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = ld_shared_v4(raw + j * 1024u);
          __syncwarp();
          if (lane == 0) mbar_arrive(RAWE_BAR(stage));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t words[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
            uint32_t h[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float f[4];
              codes_to_float_dp4a(words[k], f);
              h[2 * k] = pack2_16<T>(f[0] * sc[j], f[1] * sc[j]);
              h[2 * k + 1] = pack2_16<T>(f[2] * sc[j], f[3] * sc[j]);
            }
            st_shared_v4(sb + wr0 + j * 1024u, make_uint4(h[0], h[1], h[2], h[3]));
            st_shared_v4(sb + wr1 + j * 1024u, make_uint4(h[4], h[5], h[6], h[7]));
          }
          // the group's next block in this split: its scales, a global load away
          if (kb + kWgGroups < kb1) load_scales(kb + kWgGroups);
          fence_proxy_async_smem();  // the tensor cores read the tile
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(BRDY_BAR(bs), 0));
        }
        if (++turn == kWgGroups) turn = 0;
        if (++stage == kWgRawStages) {
          stage = 0;
          phase ^= 1u;
        }
        if (++bs == kWgBStages) {
          bs = 0;
          bphase ^= 1u;
        }
      }
    }
  }

  // Neither CTA may leave while the other can still signal its barriers or the
  // pair MMAs can still read its shared memory.
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
#undef FULL_BAR
#undef EMPTY_BAR
#undef RAWF_BAR
#undef RAWE_BAR
#undef BRDY_BAR
#undef BEMP_BAR
#undef BAR_B0
#undef TFULL_BAR
#undef TEMPTY_BAR
}

// Sum of the splits' partials in their order, rounded to T; eight elements per thread.
template <typename T>
__global__ void __launch_bounds__(256) weight_grad_q8_reduce_kernel(const float* __restrict__ partial,
                                                                   T* __restrict__ grad_w, int64_t n, int splits) {
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
    Vec16<T> o;
    o.from_float(f);
    st_global_v4(grad_w + i, o.raw);
  }
}

// Splits of the tokens: the number that the cost in microseconds is least for, of
// rounds of pair tiles at 0.8 us per 64 tokens (0.45 with one 256-row MMA) and 6 us for
// an epilogue, and, with partials, a second launch (3 us) and 8 bytes per partial
// element at 6 TB/s.
static int weight_grad_q8_splits(int64_t tokens, int64_t N, int64_t K) {
  const int64_t tiles = ((N + kWgBM - 1) / kWgBM) * ((K + 255) / 256);
  const double block_us = N > 256 ? 0.8 : 0.45;
  const int64_t pairs = num_sms_of_current_device() / 2;
  const int64_t kb = (tokens + kBK - 1) / kBK;
  int best = 1;
  double best_us = 1e30;
  for (int s = 1; s <= 32 && s <= kb; ++s) {
    const int64_t per = (kb + s - 1) / s;
    if ((kb + per - 1) / per != s) continue;  // the same blocks with fewer splits
    double us = static_cast<double>((tiles * s + pairs - 1) / pairs) * (block_us * static_cast<double>(per) + 6.0);
    if (s > 1) us += 3.0 + static_cast<double>(s) * static_cast<double>(N) * static_cast<double>(K) * 8.0 / 6.0e6;
    if (us < best_us) {
      best_us = us;
      best = s;
    }
  }
  return best;
}

template <typename T>
static int weight_grad_q8(const void* grad, const void* q, const float* scale, T* grad_w, float* partial,
                          int64_t tokens, int64_t N, int64_t K, int splits, cudaStream_t s) {
  CUtensorMap mg, mq;
  // g [tokens][N]: boxes of 64 output features x 64 tokens; q [tokens][K]: 128 features x 64 tokens
  if (!encode_map(&mg, grad, 2, N, tokens, N, kBK) || !encode_map(&mq, q, 1, K, tokens, K, kBK))
    return HLM_ERR_DRIVER;
  GemmParams p;
  gemm_tiling(p, static_cast<int>(N), static_cast<int>(K), static_cast<int>(tokens), 256, splits);
  p.m_tiles = static_cast<int>((N + kWgBM - 1) / kWgBM);
  p.err = device_error_ptr();
  if (p.err == nullptr) return HLM_ERR_LAUNCH;
  auto kern = weight_grad_q8_kernel<T>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WgSmem::kBytes) != cudaSuccess)
    return HLM_ERR_LAUNCH;
  const int64_t total = static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.splits;
  if (total > (1ll << 30)) return HLM_ERR_UNSUPPORTED;
  int pairs = num_sms_of_current_device() / 2;
  if (pairs > total) pairs = static_cast<int>(total);
  {
    LaunchScope scope(HLM_KERNEL_WEIGHT_GRAD_Q8, s);
    kern<<<2 * pairs, kWgThreads, WgSmem::kBytes, s>>>(mg, mq, scale, grad_w, p.splits > 1 ? partial : nullptr,
                                                       static_cast<int>(tokens), p);
  }
  const int rc = launch_status();
  if (rc != HLM_OK || p.splits == 1) return rc;
  const int64_t n = N * K;
  const int64_t blocks = (n / 8 + 255) / 256, cap = static_cast<int64_t>(num_sms_of_current_device()) * 16;
  {
    LaunchScope scope(0, s);
    weight_grad_q8_reduce_kernel<T><<<static_cast<int>(blocks < cap ? blocks : cap), 256, 0, s>>>(partial, grad_w, n,
                                                                                               p.splits);
  }
  return launch_status();
}

}  // namespace hlm

using namespace hlm;

extern "C" size_t hlm_weight_grad_q8_workspace_bytes(int64_t tokens, int64_t N, int64_t K) {
  if (tokens <= 0 || N <= 0 || K <= 0) return 0;
  const int splits = weight_grad_q8_splits(tokens, N, K);
  return splits > 1 ? static_cast<size_t>(splits) * static_cast<size_t>(N) * static_cast<size_t>(K) * sizeof(float) : 0;
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
  const int splits = weight_grad_q8_splits(tokens, N, K);
  const size_t need = hlm_weight_grad_q8_workspace_bytes(tokens, N, K);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return HLM_ERR_WORKSPACE;
  if (need > 0 && !host_aligned16(workspace)) return HLM_ERR_UNSUPPORTED;
  if (dtype == HLM_BF16)
    return weight_grad_q8<__nv_bfloat16>(grad, q, scale, static_cast<__nv_bfloat16*>(grad_w),
                                         static_cast<float*>(workspace), tokens, N, K, splits, s);
  return weight_grad_q8<__half>(grad, q, scale, static_cast<__half*>(grad_w), static_cast<float*>(workspace), tokens,
                                N, K, splits, s);
}
