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
  int m_tiles;
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

__device__ __forceinline__ void fp8_store(const Fp8GemmParams& p, long long off, float v) {
  if (p.out_kind == FP8_OUT_BF16) reinterpret_cast<__nv_bfloat16*>(p.C)[off] = __float2bfloat16_rn(v);
  else if (p.out_kind == FP8_OUT_F32) reinterpret_cast<float*>(p.C)[off] = v;
  else reinterpret_cast<float*>(p.C)[off] += v;
}

// ---------------------------------------------------------------------------------------------------
// One CTA, 128 columns of C (rows of B, the M side of the MMA) by TN rows of C (rows of A, its N side).
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
  const int m0 = (blockIdx.x % p.m_tiles) * TN;
  const int n0 = (blockIdx.x / p.m_tiles) * 128;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, armed = 0, armed_parity = 0;
      bool ok = true;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, abort_flag)) {
          if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_EMPTY);
          *abort_flag = 1;
          ok = false;
          break;
        }
        uint8_t* sb = smem + stage * (Cfg::A_BYTES + Cfg::B_BYTES);
        const bool scales = (kb & 3) == 0;
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
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_bounded(&full_bar[stage], phase, abort_flag)) {
          if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_FULL);
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sb = smem_u32(smem + stage * (Cfg::A_BYTES + Cfg::B_BYTES));
        const uint32_t sa = sb + Cfg::B_BYTES;
        if ((kb & 3) == 0) {
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
                    (kb > 0 || k > 0) ? 1u : 0u);
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
      const int n = n0 + q * 32 + lane;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < TN; c += 16) {
        uint32_t r[16];
        __syncwarp();
        tmem_ld_32x16(taddr + c, r);
        tmem_ld_wait();
        if (n < p.N) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (m0 + c + i < p.M) fp8_store(p, static_cast<long long>(m0 + c + i) * p.ldc + n, __uint_as_float(r[i]));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

struct Fp8Operands {
  const void *a, *b;
  long long lda, ldb;
  int M, N, K;
};

template <int TN>
static int launch_small(const Fp8Operands& o, Fp8GemmParams p, cudaStream_t stream) {
  using Cfg = F8SmallCfg<TN>;
  CUtensorMap ta, tb;
  if (encode_tensor_map(&ta, o.a, 1, o.K, o.M, 0, o.lda, 0, 128, TN) ||
      encode_tensor_map(&tb, o.b, 1, o.K, o.N, 0, o.ldb, 0, 128, 128))
    return -10;
  auto kern = fp8_gemm_small_kernel<TN>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
  if (e != cudaSuccess) return static_cast<int>(e);
  p.m_tiles = (p.M + TN - 1) / TN;
  const long long grid = static_cast<long long>(p.m_tiles) * ((p.N + 127) / 128);
  if (grid > 0x7fffffffll) return -11;
  kern<<<static_cast<unsigned>(grid), F8_THREADS, Cfg::SMEM_BYTES, stream>>>(ta, tb, p);
  return static_cast<int>(cudaGetLastError());
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
  const Fp8Operands o = {a, b, lda, ldb, M, N, K};
  if (M <= 16) return launch_small<16>(o, p, stream);
  if (M <= 32) return launch_small<32>(o, p, stream);
  if (M <= 64) return launch_small<64>(o, p, stream);
  return launch_small<128>(o, p, stream);
}
