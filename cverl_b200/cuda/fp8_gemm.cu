// Block-scaled 8-bit matrix product for sm_100a:
//
//   C[M,N] (+)= sum_k 2^(ea[m, k/128] + eb[n, k/128]) * A[m,k] * B[n,k]        fp32 accumulation in TMEM
//
// Codes are K-major bytes staged by TMA (a 128-byte swizzle row holds one scale block of 128 elements), the scales
// travel with them as 512-byte images of tensor-memory cells and are applied by the tensor core itself
// (tcgen05.mma kind::mxf8f6f4.block_scale).  The instruction takes one scale per 32 elements of K; a block of 128 is
// four instructions that name the same scale byte.  Nothing is rescaled outside the tensor core, so the accumulator
// stays in TMEM over all of K.
#include "fp8_common.cuh"
#include "gemm_tcgen05.h"

namespace cvb {

enum : int { FP8_OUT_BF16 = 0, FP8_OUT_F32 = 1, FP8_OUT_F32_ACC = 2 };

struct Fp8GemmParams {
  const uint8_t *a_sf, *b_sf;
  void* C;
  long long ldc;
  int M, N, kblocks, kgroups;
  int a_fmt, b_fmt, out_kind;
  int vec;                 // C and its row stride are 16-byte aligned
  int m_tiles, n_tiles;
  int split, kb_per_split; // small kernel: CTAs of a cluster that share a tile's K, and K blocks of each
  int group_m, total;      // pair kernel: M tiles walked per N tile, tiles in all
  int* status;
};

constexpr int F8_THREADS = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue

// 16 bytes or more, both sides 16-byte aligned, global to this CTA's shared memory
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// `n` (1 to 4) consecutive results of one row
__device__ __forceinline__ void fp8_store4(const Fp8GemmParams& p, long long off, float4 v, int n) {
  const float f[4] = {v.x, v.y, v.z, v.w};
  if (p.out_kind == FP8_OUT_BF16) {
    __nv_bfloat16* c = reinterpret_cast<__nv_bfloat16*>(p.C) + off;
    if (p.vec && n == 4) {
      *reinterpret_cast<uint2*>(c) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) c[i] = __float2bfloat16_rn(f[i]);
    return;
  }
  float* c = reinterpret_cast<float*>(p.C) + off;
  const bool acc = p.out_kind == FP8_OUT_F32_ACC;
  if (p.vec && n == 4) {
    if (acc) {
      const float4 o = *reinterpret_cast<const float4*>(c);
      v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
    }
    *reinterpret_cast<float4*>(c) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) c[i] = acc ? c[i] + f[i] : f[i];
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// ---------------------------------------------------------------------------------------------------
// Few rows: 128 columns of C (rows of B, the M side of the MMA) by TN rows of C (rows of A, its N side).
//
// Such a product reads the weights once and is bound by HBM, or, where they are a few MB, by the latency of one pass
// through an SM.  Weights take the MMA's M side, so that a single token costs an MMA 16 wide, not 128 rows of padding.
// The CTAs of a cluster share a tile's K, which fills the SMs where the tiles alone would not; their fp32 partial
// tiles meet in shared memory, where each CTA sums a share of the rows in the order of the ranks.  No atomics, no
// workspace: the result is the same from run to run.
// ---------------------------------------------------------------------------------------------------
template <int TN>
struct F8SmallCfg {
  static constexpr int B_BYTES = 128 * 128;
  static constexpr int A_BYTES = TN * 128;
  static constexpr int SF_BYTES = 1024;                     // 512 for B, 512 for A
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SF_BYTES;
  static constexpr int STAGES = 5;
  static constexpr int SF_SLOTS = 3;                        // TMEM copies of the scales of four K blocks
  static constexpr int TMEM_USED = TN + SF_SLOTS * 8;
  static constexpr int TMEM_COLS = TMEM_USED <= 64 ? 64 : TMEM_USED <= 128 ? 128 : 256;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256;
};

template <int TN>
__global__ void __launch_bounds__(F8_THREADS)
fp8_gemm_small_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                      const Fp8GemmParams p) {
  using Cfg = F8SmallCfg<TN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_smem = smem + Cfg::STAGES * (Cfg::A_BYTES + Cfg::B_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::STAGES * Cfg::STAGE_BYTES);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + Cfg::STAGES;
  uint64_t* done_bar = bars + 2 * Cfg::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / p.split;
  const int m0 = (tile % p.m_tiles) * TN;
  const int n0 = (tile / p.m_tiles) * 128;
  const int kb0 = rank * p.kb_per_split, kb1 = min(p.kblocks, kb0 + p.kb_per_split);   // never empty

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, armed = 0, armed_parity = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, abort_flag)) {
          if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_EMPTY);
          *abort_flag = 1;
          ok = false;
          break;
        }
        uint8_t* sb = smem + stage * (Cfg::A_BYTES + Cfg::B_BYTES);
        const bool scales = kb == kb0 || (kb & 3) == 0;
        mbar_arrive_expect_tx(&full_bar[stage], Cfg::A_BYTES + Cfg::B_BYTES + (scales ? Cfg::SF_BYTES : 0));
        tma_load_2d(sb, &tmB, &full_bar[stage], kb * 128, n0);
        tma_load_2d(sb + Cfg::B_BYTES, &tmA, &full_bar[stage], kb * 128, m0);
        if (scales) {
          uint8_t* sf = sf_smem + stage * Cfg::SF_BYTES;
          bulk_load(sf, p.b_sf + (static_cast<long long>(n0 >> 7) * p.kgroups + (kb >> 2)) * 512, 512, &full_bar[stage]);
          bulk_load(sf + 512, p.a_sf + (static_cast<long long>(m0 >> 7) * p.kgroups + (kb >> 2)) * 512, 512,
                    &full_bar[stage]);
        }
        armed |= 1u << stage;
        armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == Cfg::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok || *abort_flag) {
        for (int s = 0; s < Cfg::STAGES; ++s) {
          if (armed & (1u << s)) {
            int dummy = 0;
            mbar_wait_bounded(&full_bar[s], (armed_parity >> s) & 1, &dummy);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_mxf8(128, TN, p.b_fmt, p.a_fmt);
      int stage = 0;
      uint32_t phase = 0;
      int slot = -1;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&full_bar[stage], phase, abort_flag)) {
          if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_FULL);
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sb = smem_u32(smem + stage * (Cfg::A_BYTES + Cfg::B_BYTES));
        const uint32_t sa = sb + Cfg::B_BYTES;
        if (kb == kb0 || (kb & 3) == 0) {
          // A slot is written again SF_SLOTS groups later.  This stage was filled after the MMAs STAGES blocks back
          // had retired, and the slot's last reader is at least 4 * (SF_SLOTS - 1) + 1 >= STAGES blocks back.
          static_assert(4 * (Cfg::SF_SLOTS - 1) + 1 >= Cfg::STAGES, "scale slot reused before its readers retired");
          slot = slot + 1 == Cfg::SF_SLOTS ? 0 : slot + 1;
          const uint32_t sf = smem_u32(sf_smem + stage * Cfg::SF_BYTES);
          tmem_cp_scales(tmem + TN + slot * 8, umma_scale_desc(sf));
          tmem_cp_scales(tmem + TN + slot * 8 + 4, umma_scale_desc(sf + 512));
        }
        const uint32_t id = umma_idesc_scale_id(idesc, kb & 3);
        const uint32_t sfb = tmem + TN + slot * 8, sfa = sfb + 4;   // m0 is a multiple of 128: TN < 128 has one tile
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_mxf8(tmem, umma_smem_desc(sb + k * 32, 16, 1024), umma_smem_desc(sa + k * 32, 16, 1024), id, sfb, sfa,
                    (kb > kb0 || k > 0) ? 1u : 0u);
        umma_commit(&empty_bar[stage]);
        if (++stage == Cfg::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (ok) umma_commit(done_bar);
    }
  } else {
    const int q = warp & 3;
    bool ok = mbar_wait_bounded(done_bar, 0, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) {
      if (lane == 0) {
        if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_TMEM_FULL);
        *abort_flag = 1;
      }
    } else {
      tc_fence_after();
      // this CTA's partial tile as [row of C][128 columns]: the stages are free, every copy into them has been read
      float* part = reinterpret_cast<float*>(smem) + q * 32 + lane;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < TN; c += 16) {
        uint32_t r[16];
        __syncwarp();
        tmem_ld_32x16(taddr + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c + i) * 128] = __uint_as_float(r[i]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
  // rows rank, rank + split, ... of the tile: one warp a row, four columns a lane
  const int n = n0 + lane * 4, nn = min(4, p.N - n);
  const uint32_t part = smem_u32(smem) + lane * 16;
  for (int r = rank + warp * p.split; r < min(TN, p.M - m0); r += (F8_THREADS / 32) * p.split) {
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.split; ++s) {
      const float4 v = ld_cluster4(mapa_cluster(part + r * 512, s));
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    if (nn > 0) fp8_store4(p, static_cast<long long>(m0 + r) * p.ldc + n, sum, nn);
  }
  cluster_sync_all();   // nobody leaves while a peer reads its tile
}

// ---------------------------------------------------------------------------------------------------
// Many rows: 256 x 256 tiles over a CTA pair (cta_group::2), persistent.
//
// Bound by the tensor cores; per K block of 128 an SM moves 32 KB through shared memory for 128 x 256 x 128 products,
// the most an accumulator of 256 columns allows.  CTA r of a pair stages rows [128 r, + 128) of A and of B, holds the
// scales of its own rows of A and of all 256 of B, and owns 128 rows of the accumulator.
//
// Tensor memory: two accumulators of 256 columns and the scales do not fit 512 columns side by side, so the
// accumulators overlap: columns 0-255 and 192-447, scales in 448-479.  The epilogue reads the shared 64 columns
// first and then lets the next tile's MMAs start; the rest of its work runs under them.
// ---------------------------------------------------------------------------------------------------
struct F8PairCfg {
  static constexpr int A_BYTES = 128 * 128, B_BYTES = 128 * 128;
  static constexpr int TILE_BYTES = A_BYTES + B_BYTES;
  static constexpr int SF_BYTES = 3 * 512;                  // A's rows of this CTA, B's two groups of 128 rows
  static constexpr int STAGES = 5;
  static constexpr int ACC1 = 192, SF_COL = 448;            // second accumulator, scales (two slots of 16 columns)
  static constexpr int EPI_WARPS = 8;                       // two to a lane quarter, each with every other 64 columns
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int STG_BUFS = 8 / EPI_WARPS;            // 4 KB store buffers of an epilogue warp
  static constexpr int STG_OFF = STAGES * TILE_BYTES;
  static constexpr int SF_OFF = STG_OFF + EPI_WARPS * STG_BUFS * 4096;
  static constexpr int BAR_OFF = SF_OFF + STAGES * SF_BYTES;
  static constexpr int SMEM_BYTES = BAR_OFF + 256 + 1024;
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* m, const void* smem_src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void tma_add_2d(const CUtensorMap* m, const void* smem_src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y)
               : "memory");
}
// the stores committed by this thread before its last one have read their shared memory
__device__ __forceinline__ void tma_store_wait_read1() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }

// 32 rows x 64 columns of one epilogue warp, lane = row, out of registers.  Where C allows it, as boxes of 32 rows of
// 128 bytes (128-byte swizzle, two buffers a warp) that TMA stores, or adds for accumulation (one addition an
// element: the result does not depend on the order); TMA drops what lies outside C.  Else value by value.
__device__ __forceinline__ void fp8_pair_store(const Fp8GemmParams& p, const CUtensorMap* tmC, const uint32_t (&r)[64],
                                               uint8_t* stg, int* buf, int row0, int col0, int lane) {
  if (p.vec) {
    const int boxes = p.out_kind == FP8_OUT_BF16 ? 1 : 2;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half == boxes) break;
      if (lane == 0) {     // this buffer's last store has read it; with two, the other's may still be reading
        if (F8PairCfg::STG_BUFS == 2) tma_store_wait_read1();
        else tma_store_wait_read();
      }
      __syncwarp();
      uint8_t* row = stg + *buf * 4096 + lane * 128;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        uint4 o;
        if (p.out_kind == FP8_OUT_BF16)
          o = make_uint4(pack_bf16x2(__uint_as_float(r[g * 8]), __uint_as_float(r[g * 8 + 1])),
                         pack_bf16x2(__uint_as_float(r[g * 8 + 2]), __uint_as_float(r[g * 8 + 3])),
                         pack_bf16x2(__uint_as_float(r[g * 8 + 4]), __uint_as_float(r[g * 8 + 5])),
                         pack_bf16x2(__uint_as_float(r[g * 8 + 6]), __uint_as_float(r[g * 8 + 7])));
        else
          o = make_uint4(r[half * 32 + g * 4], r[half * 32 + g * 4 + 1], r[half * 32 + g * 4 + 2], r[half * 32 + g * 4 + 3]);
        *reinterpret_cast<uint4*>(row + ((g ^ (lane & 7)) << 4)) = o;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        const void* src = stg + *buf * 4096;
        if (row0 < p.M && col0 + half * 32 < p.N) {
          if (p.out_kind == FP8_OUT_F32_ACC) tma_add_2d(tmC, src, col0 + half * 32, row0);
          else tma_store_2d(tmC, src, col0 + half * 32, row0);
        }
        tma_store_commit();
      }
      *buf ^= F8PairCfg::STG_BUFS - 1;
    }
    return;
  }
  if (row0 + lane >= p.M) return;
  const long long off = static_cast<long long>(row0 + lane) * p.ldc + col0;
#pragma unroll
  for (int g = 0; g < 16; ++g)
    fp8_store4(p, off + g * 4, make_float4(__uint_as_float(r[g * 4]), __uint_as_float(r[g * 4 + 1]),
                                           __uint_as_float(r[g * 4 + 2]), __uint_as_float(r[g * 4 + 3])),
               p.N - col0 - g * 4);
}

__device__ __forceinline__ void fp8_pair_tile(const Fp8GemmParams& p, int t, int* mb, int* nb) {
  const int per = p.group_m * p.n_tiles;
  const int g = t / per, r = t - g * per;
  const int first = g * p.group_m, size = min(p.group_m, p.m_tiles - first);
  *mb = first + r % size;
  *nb = r / size;
}

__global__ void __launch_bounds__(F8PairCfg::THREADS, 1)
fp8_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                     const __grid_constant__ CUtensorMap tmC, const Fp8GemmParams p) {
  using Cfg = F8PairCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFF);   // even CTA's: bytes of both CTAs
  uint64_t* empty_bar = full_bar + Cfg::STAGES;                            // each CTA's, committed to both
  uint64_t* tfull_bar = empty_bar + Cfg::STAGES;                           // each CTA's: a tile is complete
  uint64_t* tfree_bar = tfull_bar + 1;                                     // even CTA's: the shared columns are read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfree_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(tfull_bar, 1);
    mbar_init(tfree_bar, 2 * Cfg::EPI_WARPS);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
    if (p.vec) tma_prefetch_desc(&tmC);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; ok && t < p.total; t += pairs) {
        int mb, nb;
        fp8_pair_tile(p, t, &mb, &nb);
        const int ra = mb * 2 + rank, rb = nb * 2;              // groups of 128 rows
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, abort_flag)) {
            if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_EMPTY);
            *abort_flag = 1;
            ok = false;
            break;
          }
          uint8_t* sa = smem + stage * Cfg::TILE_BYTES;
          uint8_t* sf = smem + Cfg::SF_OFF + stage * Cfg::SF_BYTES;
          const bool scales = (kb & 3) == 0;
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * (Cfg::TILE_BYTES + (scales ? Cfg::SF_BYTES : 0)));
          const uint32_t fb = mapa_cluster(smem_u32(&full_bar[stage]), 0);
          tma_load_2d_pair(sa, &tmA, fb, kb * 128, ra * 128);
          tma_load_2d_pair(sa + Cfg::A_BYTES, &tmB, fb, kb * 128, (rb + rank) * 128);
          if (scales) {   // rows of scale cells past the last read as zero: they belong to rows that are not stored
            tma_load_2d_pair(sf, &tmSA, fb, 0, ra * p.kgroups + (kb >> 2));
            tma_load_2d_pair(sf + 512, &tmSB, fb, 0, rb * p.kgroups + (kb >> 2));
            tma_load_2d_pair(sf + 1024, &tmSB, fb, 0, (rb + 1) * p.kgroups + (kb >> 2));
          }
          if (++stage == Cfg::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok || *abort_flag) {
        // This CTA's copies report to the even CTA's barriers, so it cannot wait on them itself: give those in
        // flight a bounded time to land before the CTA ends.
        const long long t0 = clock64();
        while (clock64() - t0 < (1ll << 21)) {
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = umma_idesc_mxf8(256, 256, p.a_fmt, p.b_fmt);
      int stage = 0, local = 0, slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; ok && t < p.total; t += pairs, ++local) {
        // the tile before has been read where the accumulators overlap; the one before that was read entirely then
        if (local > 0 && !mbar_wait_bounded(tfree_bar, (local - 1) & 1, abort_flag)) {
          if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_TMEM_EMPTY);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t acc = tmem + (local & 1 ? Cfg::ACC1 : 0);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!mbar_wait_bounded(&full_bar[stage], phase, abort_flag)) {
            if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_FULL);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * Cfg::TILE_BYTES), sb = sa + Cfg::A_BYTES;
          if ((kb & 3) == 0) {
            // The slot's last readers are at least five K blocks back in this tile, or in a tile whose MMAs have
            // retired; this stage was filled after the MMAs five blocks back had.
            static_assert(Cfg::STAGES <= 5, "scale slot reused before its readers retired");
            slot ^= 1;
            const uint32_t sf = smem_u32(smem + Cfg::SF_OFF + stage * Cfg::SF_BYTES);
            const uint32_t col = tmem + Cfg::SF_COL + slot * 16;
            tmem_cp_scales_pair(col, umma_scale_desc(sf));
            tmem_cp_scales_pair(col + 4, umma_scale_desc(sf + 512));
            tmem_cp_scales_pair(col + 8, umma_scale_desc(sf + 1024));
          }
          const uint32_t id = umma_idesc_scale_id(idesc, kb & 3);
          const uint32_t sfa = tmem + Cfg::SF_COL + slot * 16;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_mxf8_pair(acc, umma_smem_desc(sa + k * 32, 16, 1024), umma_smem_desc(sb + k * 32, 16, 1024), id, sfa,
                           sfa + 4, (kb > 0 || k > 0) ? 1u : 0u);
          umma_commit_pair(&empty_bar[stage], 3);
          if (++stage == Cfg::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok) umma_commit_pair(tfull_bar, 3);
      }
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;
    constexpr int PARTS = Cfg::EPI_WARPS / 4;
    uint8_t* stg = smem + Cfg::STG_OFF + (warp - 2) * Cfg::STG_BUFS * 4096;
    int buf = 0;
    int local = 0;
    for (int t = pair; t < p.total; t += pairs, ++local) {
      int mb, nb;
      fp8_pair_tile(p, t, &mb, &nb);
      bool ok = mbar_wait_bounded(tfull_bar, local & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) {
          if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_TMEM_FULL);
          *abort_flag = 1;
        }
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + (local & 1 ? Cfg::ACC1 : 0);
      const int row0 = mb * 256 + rank * 128 + q * 32, n0 = nb * 256;
#pragma unroll 1
      for (int i = part; i < 4; i += PARTS) {
        const int c = ((i + (local & 1 ? 0 : 3)) & 3) * 64;     // the shared columns first: 192-255, or 0-63
        uint32_t r[64];
        __syncwarp();
        tmem_ld_32x32(taddr + c, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
        tmem_ld_32x32(taddr + c + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
        tmem_ld_wait();
        if (i == part) {   // the shared columns are in registers, and the tile before has been read by this warp
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_cluster(smem_u32(tfree_bar), 0));
        }
        if (n0 + c < p.N) fp8_pair_store(p, &tmC, r, stg, &buf, row0, n0 + c, lane);
      }
    }
    if (lane == 0) tma_store_wait_read();
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

struct Fp8Operands {
  const void *a, *b;
  long long lda, ldb;
  int M, N, K;
};

static cudaLaunchConfig_t cluster_config(cudaLaunchAttribute* at, unsigned grid, int threads, int cluster, size_t smem,
                                         cudaStream_t stream) {
  at->id = cudaLaunchAttributeClusterDimension;
  at->val.clusterDim.x = cluster;
  at->val.clusterDim.y = 1;
  at->val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cfg;
}

template <int TN>
static int launch_small(const Fp8Operands& o, Fp8GemmParams p, cudaStream_t stream) {
  using Cfg = F8SmallCfg<TN>;
  static_assert(TN * 512 <= Cfg::STAGES * (Cfg::A_BYTES + Cfg::B_BYTES), "the partial tile fits the stages");
  CUtensorMap ta, tb;
  if (encode_tensor_map(&ta, o.a, 1, o.K, o.M, 0, o.lda, 0, 128, TN) ||
      encode_tensor_map(&tb, o.b, 1, o.K, o.N, 0, o.ldb, 0, 128, 128))
    return -10;
  auto kern = fp8_gemm_small_kernel<TN>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
  if (e != cudaSuccess) return static_cast<int>(e);
  p.m_tiles = (p.M + TN - 1) / TN;
  p.n_tiles = (p.N + 127) / 128;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  p.split = 1;
  while (p.split < 8 && tiles * p.split * 2 <= 148 && p.split * 2 <= p.kblocks) p.split *= 2;
  p.kb_per_split = (p.kblocks + p.split - 1) / p.split;
  p.split = (p.kblocks + p.kb_per_split - 1) / p.kb_per_split;
  if (tiles * p.split > 0x7fffffffll) return -11;
  cudaLaunchAttribute at;
  const cudaLaunchConfig_t cfg =
      cluster_config(&at, static_cast<unsigned>(tiles * p.split), F8_THREADS, p.split, Cfg::SMEM_BYTES, stream);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, ta, tb, p));
}

// CTA pairs that can be resident at once
static int fp8_pair_capacity() {
  static const int cached = [] {
    if (cudaFuncSetAttribute(fp8_gemm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F8PairCfg::SMEM_BYTES) !=
        cudaSuccess)
      return 0;
    cudaLaunchAttribute at;
    cudaLaunchConfig_t cfg = cluster_config(&at, 2 * 148, F8PairCfg::THREADS, 2, F8PairCfg::SMEM_BYTES, nullptr);
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, fp8_gemm_pair_kernel, &cfg) != cudaSuccess) n = 0;
    return n;
  }();
  return cached;
}

static int launch_pair(const Fp8Operands& o, Fp8GemmParams p, int pairs, cudaStream_t stream) {
  CUtensorMap ta, tb, sa, sb, tc = {};
  const uint64_t ra = static_cast<uint64_t>((o.M + 127) / 128) * p.kgroups;
  const uint64_t rb = static_cast<uint64_t>((o.N + 127) / 128) * p.kgroups;
  if (encode_tensor_map(&ta, o.a, 1, o.K, o.M, 0, o.lda, 0, 128, 128) ||
      encode_tensor_map(&tb, o.b, 1, o.K, o.N, 0, o.ldb, 0, 128, 128) ||
      encode_tensor_map(&sa, p.a_sf, TMAP_U32_PLAIN, 128, ra, 0, 512, 0, 128, 1) ||
      encode_tensor_map(&sb, p.b_sf, TMAP_U32_PLAIN, 128, rb, 0, 512, 0, 128, 1))
    return -10;
  const int elem = p.out_kind == FP8_OUT_BF16 ? 2 : 4;
  if (p.vec && encode_tensor_map(&tc, p.C, elem, p.N, p.M, 0, p.ldc * elem, 0, 128 / elem, 32)) return -10;
  const cudaError_t e =
      cudaFuncSetAttribute(fp8_gemm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F8PairCfg::SMEM_BYTES);
  if (e != cudaSuccess) return static_cast<int>(e);
  p.m_tiles = (p.M + 255) / 256;
  p.n_tiles = (p.N + 255) / 256;
  if (static_cast<long long>(p.m_tiles) * p.n_tiles > 0x3fffffffll) return -11;
  p.total = p.m_tiles * p.n_tiles;
  p.group_m = p.m_tiles < 16 ? p.m_tiles : 16;
  const int n = p.total < pairs ? p.total : pairs;
  cudaLaunchAttribute at;
  const cudaLaunchConfig_t cfg = cluster_config(&at, 2u * n, F8PairCfg::THREADS, 2, F8PairCfg::SMEM_BYTES, stream);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, fp8_gemm_pair_kernel, ta, tb, sa, sb, tc, p));
}

}  // namespace cvb

using namespace cvb;

extern "C" int cvb_fp8_gemm(const void* a, const void* a_sf, long long lda, int a_fmt, const void* b, const void* b_sf,
                            long long ldb, int b_fmt, int M, int N, int K, void* c, long long ldc, int out_kind,
                            int* status, void* stream_v) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (a_fmt < 0 || a_fmt > 1 || b_fmt < 0 || b_fmt > 1 || out_kind < 0 || out_kind > 2) return -1;
  if (!status || !a || !b || !a_sf || !b_sf || !c) return -2;
  // TMA and bulk copies start on 16-byte boundaries
  if (((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(a_sf) |
        reinterpret_cast<uintptr_t>(b_sf)) & 15) || lda % 16 || ldb % 16 || lda < K || ldb < K || ldc < N)
    return -3;
  Fp8GemmParams p = {};
  p.a_sf = static_cast<const uint8_t*>(a_sf), p.b_sf = static_cast<const uint8_t*>(b_sf);
  p.C = c, p.ldc = ldc, p.M = M, p.N = N;
  p.kblocks = (K + 127) / 128, p.kgroups = (p.kblocks + 3) / 4;
  p.a_fmt = a_fmt, p.b_fmt = b_fmt, p.out_kind = out_kind, p.status = status;
  const int elem = out_kind == FP8_OUT_BF16 ? 2 : 4;
  p.vec = (reinterpret_cast<uintptr_t>(c) & 15) == 0 && (ldc * elem) % 16 == 0;
  const Fp8Operands o = {a, b, lda, ldb, M, N, K};
  // Pairs where their tiles fill at least half of the SMs: 8 tiles (512 x 1024, K 1024) take 12.3 us against 10.2 us
  // with the other kernel, 64 (2048 x 2048, K 2048) 16.4 against 30.7.
  const long long pair_tiles = static_cast<long long>((M + 255) / 256) * ((N + 255) / 256);
  const int pairs = M > 128 && N > 128 && pair_tiles >= 37 ? fp8_pair_capacity() : 0;
  if (pairs > 0) return launch_pair(o, p, pairs, stream);
  if (M <= 16) return launch_small<16>(o, p, stream);
  if (M <= 32) return launch_small<32>(o, p, stream);
  if (M <= 64) return launch_small<64>(o, p, stream);
  return launch_small<128>(o, p, stream);
}
