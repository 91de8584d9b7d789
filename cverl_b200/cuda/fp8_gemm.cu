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
#include "fp8_launch.h"
#include "gemm_tcgen05.h"
#include <atomic>

namespace cvb {

enum : int { FP8_OUT_BF16 = 0, FP8_OUT_F32 = 1, FP8_OUT_F32_ACC = 2 };

// Products, like the quantisations and the norm's forward pass, are launched so that they may be placed while the kernel
// before them in the stream still runs (programmatic dependent launch).  A product sets up its barriers and tensor memory
// meanwhile, loads B where the caller says that nobody writes it, and touches no other global memory before that kernel
// has ended.  128 rows, N = 1024, K = 3584, quantised and multiplied: 7.5 us, 8.6 one after the other; 16 rows, N = 7168,
// K = 1024 after a norm: 6.0, 7.9.
struct Fp8GemmParams {
  const uint8_t *a_sf, *b_sf;
  const __nv_bfloat16* x;  // small kernel, FUSE: A as bf16 rows, quantised on the way
  long long x_stride;
  int x_vec, K;
  void* C;
  long long ldc;
  int M, N, kblocks, kgroups;
  int a_fmt, b_fmt, out_kind;
  int vec;                 // bytes that C and its row stride are aligned to: 32, 16 or less
  int m_tiles, n_tiles;
  int split, kb_per_split; // CTAs (or CTA pairs) of a cluster that share a tile's K, and K blocks of each
  int group_m, total;      // pair kernel: M tiles walked per N tile, tiles in all
  int b_ready;             // B was complete before the kernel before this one started
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

// The warp that issues MMAs walks its loop with all lanes and one elected lane issues: loop state and descriptors are
// then the same in every lane as far as the compiler can tell, and stay in uniform registers.  With the loop inside
// `if (lane == 0)` the issue took 600 cycles for the four MMAs of a K block, whatever their width: more than the
// tensor cores take for 256 columns.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t"
      ".reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}\n"
      : "=r"(p));
  return p != 0;
}
// Barrier over the cluster after which nobody reads this CTA's shared memory any more.  It orders no memory accesses
// (with release semantics it would wait for the result stores before it): every value that was read from a peer has to
// have been used, in an instruction before this one.
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t warp_uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag));
  if (!ok) {
    if (elect_one()) {
      if (!*abort_flag) atomicCAS(status, 0, code);
      *abort_flag = 1;
    }
    __syncwarp();
  }
  return ok;
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

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
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
//
// FUSE: A comes as bf16 rows.  The four epilogue warps, idle until the MMAs end, read 128 columns at a time, find each
// row's scale and write codes and scale bytes where TMA would have put them; every column of tiles does so for itself,
// which for up to 16 rows costs less than a launch and a pass through memory (one token, N = 7168, K = 1024: 5.0 us back
// to back against 5.4 for two kernels that overlap; 24 rows 6.9 against 5.8).  A stage's scale cells hold this block's
// byte only, so they move to tensor memory once a block.
// ---------------------------------------------------------------------------------------------------
template <int TN>
struct F8SmallCfg {
  static constexpr int B_BYTES = 128 * 128;
  static constexpr int A_BYTES = TN * 128;
  static constexpr int SF_BYTES = 1024;                     // 512 for B, 512 for A
  static constexpr int TILE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = TN == 128 ? 3 : TN == 64 ? 4 : 5;   // two CTAs fit an SM
  static constexpr int SF_SLOTS = 3;                        // TMEM copies of the scales of four K blocks
  // as in the pair kernel below; a CTA's first group may be shorter than four blocks, its later ones are not
  static_assert(4 * (SF_SLOTS - 1) + 1 >= STAGES, "scale slot reused before its readers retired");
  static constexpr int SFB_COL = TN, SFA_COL = TN + 4 * SF_SLOTS;   // scales of B by slot; of A by slot, or by stage (FUSE)
  static constexpr int TMEM_USED = SFA_COL + 4 * (STAGES > SF_SLOTS ? STAGES : SF_SLOTS);
  static constexpr int TMEM_COLS = TMEM_USED <= 64 ? 64 : TMEM_USED <= 128 ? 128 : 256;
  static constexpr int SMEM_BYTES = STAGES * (TILE_BYTES + SF_BYTES) + 1024 + 256;
};

template <int TN, bool FUSE>
__global__ void __launch_bounds__(F8_THREADS, 2)
fp8_gemm_small_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                      const Fp8GemmParams p) {
  using Cfg = F8SmallCfg<TN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_smem = smem + Cfg::STAGES * Cfg::TILE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sf_smem + Cfg::STAGES * Cfg::SF_BYTES);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + Cfg::STAGES;
  uint64_t* done_bar = bars + 2 * Cfg::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = static_cast<int>(warp_uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full_bar[s], FUSE ? 5 : 1);     // the producer, and each of the quantising warps
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    mbar_fence_init();
    if (!FUSE) tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  launch_dependents();       // there is room for a quantisation or a norm beside these CTAs, to wait for their end
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_uniform(*tmem_slot);
  const int rank = static_cast<int>(warp_uniform(cluster_ctarank()));
  const int tile = blockIdx.x / p.split;
  const int m0 = (tile % p.m_tiles) * TN;
  const int n0 = (tile / p.m_tiles) * 128;
  const int kb0 = rank * p.kb_per_split, kb1 = min(p.kblocks, kb0 + p.kb_per_split);   // never empty

  if (warp == 0) {
    const bool leader = elect_one();
    const uint8_t* b_sf = p.b_sf + static_cast<long long>(n0 >> 7) * p.kgroups * 512;
    const uint8_t* a_sf = FUSE ? nullptr : p.a_sf + static_cast<long long>(m0 >> 7) * p.kgroups * 512;
    constexpr uint32_t BYTES = FUSE ? Cfg::B_BYTES : Cfg::TILE_BYTES, SF = FUSE ? 512 : 1024;
    auto fill_b = [&](int kb, int stage) {
      const bool scales = kb == kb0 || (kb & 3) == 0;
      mbar_arrive_expect_tx(&full_bar[stage], BYTES + (scales ? SF : 0));
      tma_load_2d(smem + stage * Cfg::TILE_BYTES, &tmB, &full_bar[stage], kb * 128, n0);
      if (scales)
        bulk_load(sf_smem + stage * Cfg::SF_BYTES, b_sf + static_cast<long long>(kb >> 2) * 512, 512, &full_bar[stage]);
    };
    auto fill_a = [&](int kb, int stage) {
      if (FUSE) return;
      tma_load_2d(smem + stage * Cfg::TILE_BYTES + Cfg::B_BYTES, &tmA, &full_bar[stage], kb * 128, m0);
      if (kb == kb0 || (kb & 3) == 0)
        bulk_load(sf_smem + stage * Cfg::SF_BYTES + 512, a_sf + static_cast<long long>(kb >> 2) * 512, 512, &full_bar[stage]);
    };
    // The first fill of every stage waits for nothing: one lane a stage.  One after the other they took 560 cycles each
    // (one row, N = K = 1024: 3.7 us against 3.4).
    const bool first = lane < Cfg::STAGES && kb0 + lane < kb1;
    if (!p.b_ready) wait_for_previous_kernel();
    if (first) fill_b(kb0 + lane, lane);
    if (p.b_ready) wait_for_previous_kernel();
    if (first) fill_a(kb0 + lane, lane);
    __syncwarp();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int kb = kb0 + Cfg::STAGES; kb < kb1; ++kb) {
      if (!warp_wait(&empty_bar[stage], phase, abort_flag, p.status, ERR_WAIT_EMPTY)) {
        ok = false;
        break;
      }
      if (leader) {
        fill_b(kb, stage);
        fill_a(kb, stage);
      }
      __syncwarp();
      if (++stage == Cfg::STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!ok || *abort_flag) {
      // leave no copy in flight: give those that are a bounded time to land before the CTA ends
      const long long t0 = clock64();
      while (clock64() - t0 < (1ll << 21)) {
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = umma_idesc_mxf8(128, TN, p.b_fmt, p.a_fmt);
    // where the tile's rows begin in their group's scales (copied whole): 0, or 2 columns for the second 64 of 128 rows.
    // Narrower tiles are the only one of their group: the operand may not begin at an odd column.
    const uint32_t a_col = TN == 64 ? (m0 & 127) >> 5 : 0;
    const bool leader = elect_one();
    const uint64_t db0 = umma_smem_desc(smem_u32(smem), 16, 1024);
    const uint64_t da0 = umma_smem_desc(smem_u32(smem) + Cfg::B_BYTES, 16, 1024);
    const uint64_t ds0 = umma_scale_desc(smem_u32(sf_smem));
    int stage = 0, slot = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_wait(&full_bar[stage], phase, abort_flag, p.status, ERR_WAIT_FULL)) break;
      tc_fence_after();
      const bool scales = kb == kb0 || (kb & 3) == 0, last = kb + 1 == kb1;
      if (scales) slot = slot + 1 == Cfg::SF_SLOTS ? 0 : slot + 1;
      const uint64_t db = db0 + stage * (Cfg::TILE_BYTES >> 4), da = da0 + stage * (Cfg::TILE_BYTES >> 4);
      const uint64_t ds = ds0 + stage * (Cfg::SF_BYTES >> 4);
      const uint32_t id = umma_idesc_scale_id(idesc, kb & 3);
      const uint32_t sfb = tmem + Cfg::SFB_COL + slot * 4, sfa = tmem + Cfg::SFA_COL + (FUSE ? stage : slot) * 4;
      const uint32_t rows_a = sfa + a_col;
      if (leader) {
        if (scales) tmem_cp_scales(sfb, ds);
        if (scales || FUSE) tmem_cp_scales(sfa, ds + 32);
        umma_mxf8(tmem, db, da, id, sfb, rows_a, kb > kb0 ? 1u : 0u);
#pragma unroll
        for (int k = 1; k < 4; ++k) umma_mxf8(tmem, db + 2 * k, da + 2 * k, id, sfb, rows_a, 1u);
        umma_commit(&empty_bar[stage]);
        if (last) umma_commit(done_bar);
      }
      __syncwarp();
      if (++stage == Cfg::STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
  } else {
    const int q = warp & 3;
    if constexpr (FUSE) {
      static_assert(TN == 16, "eight threads a row, 16 columns each");
      const int r = (threadIdx.x - 64) >> 3, j = threadIdx.x & 7, row = m0 + r;
      uint4 raw[2], next[2];                            // this block's values and the next one's
      auto load = [&](int kb, uint4(&out)[2]) {
        const int c = kb * 128 + j * 16;
        const __nv_bfloat16* src = p.x + row * p.x_stride + c;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = row < p.M ? max(0, min(8, p.K - c - h * 8)) : 0;
          out[h] = p.x_vec ? load_raw8<true>(src + h * 8, n) : load_raw8<false>(src + h * 8, n);
        }
      };
      wait_for_previous_kernel();
      load(kb0, raw);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (kb + 1 < kb1) load(kb + 1, next);
        if (!warp_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, ERR_WAIT_EMPTY)) break;
        float lo[8], hi[8];
        widen8(raw[0], lo);
        widen8(raw[1], hi);
        bool odd = false;
        uint32_t m = fp8_max16(max(fp8_finite_max(lo, &odd), fp8_finite_max(hi, &odd)));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const uint32_t byte = fp8_scale_bytes<FP8_E4M3>(m) & 0xFFu;
        const float inv = fp8_low(fp8_inverse_scales(byte));
        const uint2 a = fp8_pack8<FP8_E4M3>(lo, inv), b = fp8_pack8<FP8_E4M3>(hi, inv);
        uint8_t* dst = smem + stage * Cfg::TILE_BYTES + Cfg::B_BYTES + r * 128 + ((j ^ (r & 7)) << 4);   // 128-byte swizzle
        *reinterpret_cast<uint4*>(dst) = make_uint4(a.x, a.y, b.x, b.y);
        if (odd) {
          fp8_fix_inf<FP8_E4M3>(lo, dst, 8);
          fp8_fix_inf<FP8_E4M3>(hi, dst + 8, 8);
        }
        if (j == 0) sf_smem[stage * Cfg::SF_BYTES + 512 + r * 16 + (kb & 3)] = static_cast<uint8_t>(byte);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full_bar[stage]);
        if (++stage == Cfg::STAGES) {
          stage = 0;
          phase ^= 1;
        }
        raw[0] = next[0], raw[1] = next[1];
      }
    }
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
      constexpr int COLS = TN < 32 ? TN : 32;
#pragma unroll 1
      for (int c = 0; c < TN; c += COLS) {
        uint32_t r[COLS];
        __syncwarp();
        if constexpr (COLS == 16) tmem_ld_32x16(taddr + c, r);
        else tmem_ld_32x32(taddr + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < COLS; ++i) part[(c + i) * 128] = __uint_as_float(r[i]);
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
    // all of a row's loads are under way before the first is used (128 rows, N = 1024, K = 3584: 7.7 us against 8.1)
    float4 v[8];
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (nn > 0 && s < p.split) v[s] = ld_cluster4(mapa_cluster(part + r * 512, s));
    if (nn <= 0) continue;     // nothing was read that is not stored below: see cluster_sync_relaxed
    float4 sum = v[0];
#pragma unroll
    for (int s = 1; s < 8; ++s)
      if (s < p.split) sum.x += v[s].x, sum.y += v[s].y, sum.z += v[s].z, sum.w += v[s].w;
    fp8_store4(p, static_cast<long long>(m0 + r) * p.ldc + n, sum, nn);
  }
  __syncwarp();
  cluster_sync_relaxed();   // nobody leaves while a peer reads its tile
}

// ---------------------------------------------------------------------------------------------------
// Many rows: 256 x BN tiles over a CTA pair (cta_group::2), persistent.
//
// Bound by the tensor cores; per K block of 128 an SM moves 16 KB + BN / 2 * 128 bytes through shared memory for
// 128 x BN x 128 products.  CTA r of a pair stages rows [128 r, + 128) of A and [BN / 2 * r, + BN / 2) of B, holds
// the scales of its own rows of A and of all BN of B, and owns 128 rows of the accumulator.
//
// Tensor memory: two accumulators, so that a tile's results leave under the next tile's MMAs, and the scales.  At
// BN = 256 they do not fit 512 columns side by side: the accumulators overlap (columns 0-255 and 192-447), the
// epilogue reads the shared 64 columns first and then lets the next tile begin.  That hand-over costs about 500
// cycles a tile; BN = 192 has none, but loads more for a product and pads other widths.
// Four epilogue warps belong to each accumulator, so they have two tiles' time for one.
//
// SPLIT: few tiles and a long K (weight gradients).  `split` pairs of a cluster share a tile's K, one tile a cluster;
// their partial tiles meet in shared memory as in the kernel above.
//
// PRODUCTS = 2: the two gradients of a layer, of which the weight's has few tiles with a long K and leaves SMs idle alone:
// 20480 x 3584 x 1024 110 us for both, 122 one after the other; 1301 x 1000 x 520 8.1 and 14.7.
// ---------------------------------------------------------------------------------------------------
template <int BN>
struct F8PairCfg {
  static constexpr bool OVERLAP = BN == 256;
  static constexpr int HALF = BN / 2;                       // rows of B that each CTA stages
  static constexpr int A_BYTES = 128 * 128, B_BYTES = HALF * 128;
  static constexpr int TILE_BYTES = A_BYTES + B_BYTES;
  static constexpr int SF_GROUPS = BN == 128 ? 1 : 2;       // groups of 128 rows of B whose scales a tile reads
  static constexpr int SF_BYTES = (1 + SF_GROUPS) * 512;    // and those of A's rows of this CTA
  static constexpr int STAGES = OVERLAP ? 6 : BN == 192 ? 7 : 8;
  static constexpr int SF_SLOTS = 4;                        // TMEM copies of the scales of four K blocks
  static constexpr int ACC1 = OVERLAP ? 192 : BN;
  static constexpr int SF_COL = ACC1 + BN;                  // 16 columns a slot
  static constexpr int THREADS = 64 + 32 * 8;
  static constexpr int SF_OFF = STAGES * TILE_BYTES;
  static constexpr int BAR_OFF = SF_OFF + STAGES * SF_BYTES;
  static constexpr int SMEM_BYTES = BAR_OFF + 256 + 1024;
  static_assert(SF_COL + 16 * SF_SLOTS <= 512, "tensor memory");
  // A slot is written again SF_SLOTS groups of up to four K blocks later, when its readers have retired: either they
  // belong to the tile before the last (its accumulator has been read), or at most one of the groups between is the
  // short one that ends a tile, so the last reader is at least 4 (SF_SLOTS - 2) + 1 + 1 blocks back, and the stage that
  // brings the new scales was filled after the MMAs STAGES blocks back had retired.
  static_assert(4 * (SF_SLOTS - 2) + 2 >= STAGES, "scale slot reused before its readers retired");
};

// Arrival that orders nothing but tensor memory (its reads are complete, tcgen05.fence::before_thread_sync precedes):
// a releasing one would first wait for the result stores of the chunk before.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void st_global_32b(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e,
                                              uint32_t f, uint32_t g, uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d),
               "r"(e), "r"(f), "r"(g), "r"(h)
               : "memory");
}

// C += a lane's 16 columns of its row, columns and rows of whole vectors: four lanes exchange vectors of four, so that
// an instruction adds 64 bytes of a row from four lanes.
__device__ __forceinline__ void fp8_quad_add(const Fp8GemmParams& p, const uint32_t* r, int row, int col) {
  const int j = threadIdx.x & 3;
  uint32_t x[4][4];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i >> 2][i & 3] = r[i];
#pragma unroll
  for (int m = 1; m <= 2; m <<= 1)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      if (v & m) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, j & m ? x[v][i] : x[v | m][i], m);
        if (j & m) x[v][i] = got;
        else x[v | m][i] = got;
      }
    }
  row &= ~3;                    // lane j has vector j of rows row + 0 ... 3
  float* dst = reinterpret_cast<float*>(p.C) + static_cast<long long>(row) * p.ldc + col + j * 4;
#pragma unroll
  for (int k = 0; k < 4; ++k, dst += p.ldc)
    if (row + k < p.M)
      red_add_v4_f32(dst, __uint_as_float(x[k][0]), __uint_as_float(x[k][1]), __uint_as_float(x[k][2]), __uint_as_float(x[k][3]));
}

// 32 rows x 64 columns of one epilogue warp, lane = row, straight from registers: a lane's 64 results are 128 (or
// 256) bytes of its row, stored as whole 32-byte sectors.  An accumulating product adds by reduction, one addition an
// element: the result does not depend on the order.  Value by value where C is not aligned or the columns end.
__device__ __forceinline__ void fp8_pair_store(const Fp8GemmParams& p, const uint32_t (&r)[64], int row, int col) {
  if (p.out_kind == FP8_OUT_F32_ACC && p.vec >= 16 && col + 64 <= p.N) {
#pragma unroll
    for (int g = 0; g < 64; g += 16) fp8_quad_add(p, r + g, row, col + g);
    return;
  }
  if (row >= p.M) return;
  const long long off = static_cast<long long>(row) * p.ldc + col;
  const int n = p.N - col;
  if (p.out_kind == FP8_OUT_BF16) {
    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.C) + off;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = pack_bf16x2(__uint_as_float(r[g * 16 + 2 * i]), __uint_as_float(r[g * 16 + 2 * i + 1]));
      if (p.vec == 32 && g * 16 + 16 <= n) {
        st_global_32b(dst + g * 16, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
      } else if (p.vec >= 16 && g * 16 + 16 <= n) {
        *reinterpret_cast<uint4*>(dst + g * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(dst + g * 16 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (g * 16 + i < n)
            reinterpret_cast<uint16_t*>(dst)[g * 16 + i] = static_cast<uint16_t>(w[i >> 1] >> ((i & 1) * 16));
      }
    }
    return;
  }
  float* dst = reinterpret_cast<float*>(p.C) + off;
  const bool acc = p.out_kind == FP8_OUT_F32_ACC;
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    const uint32_t* w = r + g * 8;
    if (p.vec >= 16 && g * 8 + 8 <= n) {
      if (acc) {
        red_add_v4_f32(dst + g * 8, __uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
        red_add_v4_f32(dst + g * 8 + 4, __uint_as_float(w[4]), __uint_as_float(w[5]), __uint_as_float(w[6]),
                       __uint_as_float(w[7]));
      } else if (p.vec == 32) {
        st_global_32b(dst + g * 8, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
      } else {
        *reinterpret_cast<uint4*>(dst + g * 8) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(dst + g * 8 + 4) = make_uint4(w[4], w[5], w[6], w[7]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (g * 8 + i < n) {
          if (acc) atomicAdd(dst + g * 8 + i, __uint_as_float(w[i]));
          else dst[g * 8 + i] = __uint_as_float(w[i]);
        }
    }
  }
}

__device__ __forceinline__ void fp8_pair_tile(const Fp8GemmParams& p, int t, int* mb, int* nb) {
  const int per = p.group_m * p.n_tiles;
  const int g = t / per, r = t - g * per;
  const int first = g * p.group_m, size = min(p.group_m, p.m_tiles - first);
  *mb = first + r % size;
  *nb = r / size;
}

// One product, or two that a launch computes together: the first has the longer K.
template <int PRODUCTS>
struct Fp8PairArgs {
  CUtensorMap a[PRODUCTS], b[PRODUCTS], sa[PRODUCTS], sb[PRODUCTS];
  Fp8GemmParams p[PRODUCTS];
  int head;                // two products: rounds of the second's tiles beside the last of the first's
};

// The tile that a pair computes as its l-th; false past its last.  Two products: the first's tiles in turn, as for one.
// The pairs that get none in its last round take `head` tiles of the second meanwhile, then all pairs take the rest in
// turn, so pairs that run at the same time work on neighbouring tiles all along.
template <int PRODUCTS>
__device__ __forceinline__ bool fp8_pair_next(const Fp8PairArgs<PRODUCTS>& g, int pair, int pairs, int l, int* which, int* t) {
  *which = 0;
  *t = pair + l * pairs;
  if (*t < g.p[0].total) return true;
  if (PRODUCTS == 1) return false;
  constexpr int W = PRODUCTS - 1;
  const int rest = g.p[0].total % pairs, m = l - (g.p[0].total / pairs + (pair < rest));
  *which = W;
  if (rest == 0) *t = pair + m * pairs;
  else if (pair < rest) *t = g.head * (pairs - rest) + m * pairs + pair;
  else if (m < g.head) *t = m * (pairs - rest) + pair - rest;
  else *t = g.head * (pairs - rest) + (m - g.head) * pairs + pair;
  return *t < g.p[W].total;
}

template <int BN, bool SPLIT, int PRODUCTS>
__global__ void __launch_bounds__(F8PairCfg<BN>::THREADS, 1)
fp8_gemm_pair_kernel(const __grid_constant__ Fp8PairArgs<PRODUCTS> g) {
  static_assert(!SPLIT || PRODUCTS == 1, "a split is of one product");
  using Cfg = F8PairCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFF);   // even CTA's: bytes of both CTAs
  uint64_t* empty_bar = full_bar + Cfg::STAGES;                            // each CTA's, committed to both
  uint64_t* tfull_bar = empty_bar + Cfg::STAGES;                           // [2] each CTA's: an accumulator is complete
  uint64_t* tdone_bar = tfull_bar + 2;                                     // [2] even CTA's: it has been read
  uint64_t* tfree_bar = tdone_bar + 2;                                     // [2] even CTA's: its shared columns have
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfree_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = static_cast<int>(warp_uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int crank = static_cast<int>(warp_uniform(cluster_ctarank()));
  const int rank = crank & 1, even = crank & ~1;                // within the pair; the pair's CTA that issues
  // first tile and stride of this pair's walk; SPLIT: the cluster's only tile, this pair's range of its K
  const int pair = SPLIT ? blockIdx.x / (2 * g.p[0].split) : blockIdx.x >> 1;
  const int pairs = SPLIT ? g.p[0].total : gridDim.x >> 1;
  const int kb0 = SPLIT ? (crank >> 1) * g.p[0].kb_per_split : 0;
  const uint16_t both = static_cast<uint16_t>(3 << even);

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tdone_bar[a], 8);     // an accumulator's four epilogue warps in each CTA
      mbar_init(&tfree_bar[a], 8);
    }
    *abort_flag = 0;
    mbar_fence_init();
    for (int w = 0; w < PRODUCTS; ++w) {
      tma_prefetch_desc(&g.a[w]);
      tma_prefetch_desc(&g.b[w]);
      tma_prefetch_desc(&g.sa[w]);
      tma_prefetch_desc(&g.sb[w]);
    }
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = warp_uniform(*tmem_slot);

  if (warp == 0) {
    const bool leader = elect_one();
    const uint32_t full0 = mapa_cluster(smem_u32(full_bar), even);
    wait_for_previous_kernel();          // the stores of this pair follow on its loads
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    int w, t;
    for (int l = 0; ok && fp8_pair_next(g, pair, pairs, l, &w, &t); ++l) {
      const Fp8GemmParams& p = g.p[w];
      const int kb1 = SPLIT ? min(p.kblocks, kb0 + p.kb_per_split) : p.kblocks;
      int mb, nb;
      fp8_pair_tile(p, t, &mb, &nb);
      const int ra = mb * 2 + rank, rb = nb * BN / 128;         // groups of 128 rows
      const int row_a = ra * 128, row_b = nb * BN + rank * Cfg::HALF;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!warp_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, ERR_WAIT_EMPTY)) {
          ok = false;
          break;
        }
        const bool scales = kb == kb0 || (kb & 3) == 0;
        uint8_t* sa = smem + stage * Cfg::TILE_BYTES;
        uint8_t* sf = smem + Cfg::SF_OFF + stage * Cfg::SF_BYTES;
        const uint32_t fb = full0 + stage * 8;
        const int kg = kb >> 2;
        if (leader) {
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * (Cfg::TILE_BYTES + (scales ? Cfg::SF_BYTES : 0)));
          tma_load_2d_pair(sa, &g.a[w], fb, kb * 128, row_a);
          tma_load_2d_pair(sa + Cfg::A_BYTES, &g.b[w], fb, kb * 128, row_b);
          if (scales) {   // rows of scale cells past the last read as zero: they belong to rows that are not stored
            tma_load_2d_pair(sf, &g.sa[w], fb, 0, ra * p.kgroups + kg);
            tma_load_2d_pair(sf + 512, &g.sb[w], fb, 0, rb * p.kgroups + kg);
            if (Cfg::SF_GROUPS == 2) tma_load_2d_pair(sf + 1024, &g.sb[w], fb, 0, (rb + 1) * p.kgroups + kg);
          }
        }
        __syncwarp();
        if (++stage == Cfg::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok || *abort_flag) {
      // This CTA's copies report to the even CTA's barriers, so it cannot wait on them itself: give those in flight a
      // bounded time to land before the CTA ends.
      const long long t0 = clock64();
      while (clock64() - t0 < (1ll << 21)) {
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = elect_one();
      // descriptors of stage 0: a stage adds TILE_BYTES / 16 to the address field, 32 elements of K two
      const uint64_t da0 = umma_smem_desc(smem_u32(smem), 16, 1024);
      const uint64_t db0 = umma_smem_desc(smem_u32(smem) + Cfg::A_BYTES, 16, 1024);
      const uint64_t ds0 = umma_scale_desc(smem_u32(smem) + Cfg::SF_OFF);
      int stage = 0, slot = 0, w, t;
      uint32_t phase = 0;
      bool ok = true;
      for (int local = 0; ok && fp8_pair_next(g, pair, pairs, local, &w, &t); ++local) {
        const Fp8GemmParams& p = g.p[w];
        const int kb1 = SPLIT ? min(p.kblocks, kb0 + p.kb_per_split) : p.kblocks;
        const uint32_t idesc = umma_idesc_mxf8(256, BN, p.a_fmt, p.b_fmt);
        const int a = local & 1, use = local >> 1;
        // this accumulator's last tile has been read, and the other's where the two overlap
        if (use > 0 && !warp_wait(&tdone_bar[a], (use - 1) & 1, abort_flag, p.status, ERR_WAIT_TMEM_EMPTY)) break;
        if (Cfg::OVERLAP && local > 0 &&
            !warp_wait(&tfree_bar[a ^ 1], ((local - 1) >> 1) & 1, abort_flag, p.status, ERR_WAIT_TMEM_EMPTY))
          break;
        tc_fence_after();
        const uint32_t acc = tmem + (a ? Cfg::ACC1 : 0);
        uint32_t sfb_col = 0;                                   // the tile's first row in its group's scale cells
        if (BN % 128 != 0) {
          int mb, nb;
          fp8_pair_tile(p, t, &mb, &nb);
          sfb_col = ((nb * BN) & 127) >> 5;
        }
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!warp_wait(&full_bar[stage], phase, abort_flag, p.status, ERR_WAIT_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const bool scales = kb == kb0 || (kb & 3) == 0;
          if (scales) slot = slot + 1 == Cfg::SF_SLOTS ? 0 : slot + 1;
          const uint32_t sfa = tmem + Cfg::SF_COL + slot * 16, sfb = sfa + 4 + sfb_col;
          const uint64_t ds = ds0 + stage * (Cfg::SF_BYTES >> 4);
          const uint64_t da = da0 + stage * (Cfg::TILE_BYTES >> 4), db = db0 + stage * (Cfg::TILE_BYTES >> 4);
          const uint32_t id = umma_idesc_scale_id(idesc, kb & 3);
          const bool last = kb + 1 == kb1;
          if (leader) {
            if (scales) {
              tmem_cp_scales_pair(sfa, ds);
              tmem_cp_scales_pair(sfa + 4, ds + 32);
              if (Cfg::SF_GROUPS == 2) tmem_cp_scales_pair(sfa + 8, ds + 64);
            }
            umma_mxf8_pair(acc, da, db, id, sfa, sfb, kb > kb0 ? 1u : 0u);
#pragma unroll
            for (int k = 1; k < 4; ++k) umma_mxf8_pair(acc, da + 2 * k, db + 2 * k, id, sfa, sfb, 1u);
            umma_commit_pair(&empty_bar[stage], both);
            if (last) umma_commit_pair(&tfull_bar[a], both);
          }
          __syncwarp();
          if (++stage == Cfg::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else {
    const int q = warp & 3, a = (warp - 2) >> 2;             // lane quarter, accumulator
    const uint32_t tfree = mapa_cluster(smem_u32(&tfree_bar[a]), even), tdone = mapa_cluster(smem_u32(&tdone_bar[a]), even);
    uint32_t use = 0;
    if (SPLIT) {
      const Fp8GemmParams& p = g.p[0];
      const bool ok = warp_wait(&tfull_bar[0], 0, abort_flag, p.status, ERR_WAIT_TMEM_FULL);
      tc_fence_after();
      // this pair's partial tile as [column][128 rows of this CTA]: the stages are free, every copy has been read.
      // The two sets of warps take half of the columns each.
      float* part = reinterpret_cast<float*>(smem) + q * 32 + lane;
#pragma unroll 1
      for (int c = a * Cfg::HALF; ok && c < (a + 1) * Cfg::HALF; c += 32) {
        uint32_t r[32];
        __syncwarp();
        tmem_ld_32x32(tmem + (static_cast<uint32_t>(q * 32) << 16) + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) part[(c + i) * 128] = __uint_as_float(r[i]);
      }
    }
    int w, t;
    for (int l = a; !SPLIT && fp8_pair_next(g, pair, pairs, l, &w, &t); l += 2, ++use) {
      const Fp8GemmParams& p = g.p[w];
      int mb, nb;
      fp8_pair_tile(p, t, &mb, &nb);
      bool ok = mbar_wait_bounded(&tfull_bar[a], use & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) {
          if (!*abort_flag) atomicCAS(p.status, 0, ERR_WAIT_TMEM_FULL);
          *abort_flag = 1;
        }
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + (a ? Cfg::ACC1 : 0);
      const int row0 = mb * 256 + rank * 128 + q * 32, n0 = nb * BN;
#pragma unroll 1
      for (int i = 0; i < BN / 64; ++i) {
        // the shared columns first: 192-255 of the first accumulator, 0-63 of the second
        const int c = (Cfg::OVERLAP && a == 0 ? (i + 3) & 3 : i) * 64;
        uint32_t r[64];
        __syncwarp();
        tmem_ld_32x32(taddr + c, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
        tmem_ld_32x32(taddr + c + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
        tmem_ld_wait();
        if ((Cfg::OVERLAP && i == 0) || i == BN / 64 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(i == 0 ? tfree : tdone);
        }
        if (n0 + c < p.N) fp8_pair_store(p, r, row0 + lane, n0 + c);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
  if (SPLIT) {
    // 64 columns at a time: chunk i belongs to pair i % split, there to the set of warps i / split
    if (warp >= 2) {
      const Fp8GemmParams& p = g.p[0];
      const int q = warp & 3, a = (warp - 2) >> 2;
      int mb, nb;
      fp8_pair_tile(p, pair, &mb, &nb);
      for (int i = (crank >> 1) + a * p.split; i < BN / 64; i += 2 * p.split) {
        uint32_t r[64];
#pragma unroll
        for (int c = 0; c < 64; ++c) r[c] = 0u;
        for (int z = 0; z < p.split; ++z) {       // in the order of the ranks
          const uint32_t src = mapa_cluster(smem_u32(smem) + (i * 64 * 128 + q * 32 + lane) * 4, 2 * z + rank);
#pragma unroll
          for (int c = 0; c < 64; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) + ld_cluster(src + c * 512));
        }
        if (nb * BN + i * 64 < p.N) fp8_pair_store(p, r, mb * 256 + rank * 128 + q * 32 + lane, nb * BN + i * 64);
      }
    }
    __syncwarp();
    cluster_sync_all();   // nobody leaves while a peer reads its tile
  }
}

struct Fp8Product {
  const void *a, *b;
  long long lda, ldb;
  Fp8GemmParams p;
};

// The shared-memory opt-in of a kernel, made once per device: a call costs as much as an eighth of a small product.
template <auto KERN>
static int opt_in_smem(int bytes) {
  static std::atomic<uint64_t> done{0};       // one bit a device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return 0;
  e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return static_cast<int>(e);
}

static cudaLaunchConfig_t cluster_config(cudaLaunchAttribute (&at)[2], unsigned grid, int threads, int cluster,
                                         size_t smem, cudaStream_t stream) {
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cfg;
}

template <int TN, bool FUSE>
static int launch_small(const Fp8Product& o, cudaStream_t stream) {
  using Cfg = F8SmallCfg<TN>;
  static_assert(TN * 512 <= Cfg::STAGES * Cfg::TILE_BYTES, "the partial tile fits the stages");
  CUtensorMap ta = {}, tb;
  Fp8GemmParams p = o.p;
  if ((!FUSE && encode_tensor_map(&ta, o.a, 1, p.K, p.M, 0, o.lda, 0, 128, TN)) ||
      encode_tensor_map(&tb, o.b, 1, p.K, p.N, 0, o.ldb, 0, 128, 128))
    return -10;
  auto kern = fp8_gemm_small_kernel<TN, FUSE>;
  if (const int e = opt_in_smem<fp8_gemm_small_kernel<TN, FUSE>>(Cfg::SMEM_BYTES)) return e;
  p.m_tiles = (p.M + TN - 1) / TN;
  p.n_tiles = (p.N + 127) / 128;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  // Fill the SMs: one CTA each (two where each still has 8 K blocks), clusters of eight only where there are few of them
  // or each CTA still has 6 K blocks.  One token, N = 1024, K = 3584: 10.2 us with one CTA a tile, 4.3 with eight; 128
  // rows, N = 1024, K = 3584: 6.5 with four, 6.8 with eight; 16 rows, N = 2048, K = 8192: 7.4 with four, 6.2 with eight;
  // 128 rows, N = K = 8192, weights in L2: 27.0 with one, 17.6 with two, 14.6 with four (19.2 with weights from HBM).
  p.split = 1;
  while (p.split < 8) {
    const int next = p.split * 2, per = p.kblocks / next;
    const long long room = next == 8 ? (per >= 6 ? 128 : 74) : per >= 8 ? 296 : 148;
    if (per < 1 || tiles * next > room) break;
    p.split = next;
  }
  p.kb_per_split = (p.kblocks + p.split - 1) / p.split;
  p.split = (p.kblocks + p.kb_per_split - 1) / p.kb_per_split;
  if (tiles * p.split > 0x7fffffffll) return -11;
  cudaLaunchAttribute at[2];
  const cudaLaunchConfig_t cfg =
      cluster_config(at, static_cast<unsigned>(tiles * p.split), F8_THREADS, p.split, Cfg::SMEM_BYTES, stream);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, ta, tb, p));
}

// CTA pairs that can be resident at once
template <int BN>
static int fp8_pair_capacity() {
  static const int cached = [] {
    using Cfg = F8PairCfg<BN>;
    auto kern = fp8_gemm_pair_kernel<BN, false, 1>;
    if (opt_in_smem<fp8_gemm_pair_kernel<BN, false, 1>>(Cfg::SMEM_BYTES)) return 0;
    cudaLaunchAttribute at[2];
    cudaLaunchConfig_t cfg = cluster_config(at, 2 * 148, Cfg::THREADS, 2, Cfg::SMEM_BYTES, nullptr);
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) n = 0;
    return n;
  }();
  return cached;
}

// product w of a launch
template <int BN, int PRODUCTS>
static int pair_product(Fp8PairArgs<PRODUCTS>* g, int w, const Fp8Product& o) {
  Fp8GemmParams& p = g->p[w];
  p = o.p;
  const uint64_t ra = static_cast<uint64_t>((p.M + 127) / 128) * p.kgroups;
  const uint64_t rb = static_cast<uint64_t>((p.N + 127) / 128) * p.kgroups;
  if (encode_tensor_map(&g->a[w], o.a, 1, p.K, p.M, 0, o.lda, 0, 128, 128) ||
      encode_tensor_map(&g->b[w], o.b, 1, p.K, p.N, 0, o.ldb, 0, 128, F8PairCfg<BN>::HALF) ||
      encode_tensor_map(&g->sa[w], p.a_sf, TMAP_U32_PLAIN, 128, ra, 0, 512, 0, 128, 1) ||
      encode_tensor_map(&g->sb[w], p.b_sf, TMAP_U32_PLAIN, 128, rb, 0, 512, 0, 128, 1))
    return -10;
  p.m_tiles = (p.M + 255) / 256;
  p.n_tiles = (p.N + BN - 1) / BN;
  if (static_cast<long long>(p.m_tiles) * p.n_tiles > 0x0fffffffll || ra > 0x7fffffffull || rb > 0x7fffffffull) return -11;
  p.total = p.m_tiles * p.n_tiles;
  p.group_m = p.m_tiles < 16 ? p.m_tiles : 16;
  return 0;
}

template <int BN, bool SPLIT, int PRODUCTS>
static int launch_pairs(const Fp8PairArgs<PRODUCTS>& g, int clusters, int split, cudaStream_t stream) {
  using Cfg = F8PairCfg<BN>;
  static_assert(BN * 512 <= Cfg::STAGES * Cfg::TILE_BYTES, "the partial tile fits the stages");
  if (const int e = opt_in_smem<fp8_gemm_pair_kernel<BN, SPLIT, PRODUCTS>>(Cfg::SMEM_BYTES)) return e;
  cudaLaunchAttribute at[2];
  const cudaLaunchConfig_t cfg =
      cluster_config(at, 2u * split * clusters, Cfg::THREADS, 2 * split, Cfg::SMEM_BYTES, stream);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, fp8_gemm_pair_kernel<BN, SPLIT, PRODUCTS>, g));
}

template <int BN, bool SPLIT>
static int launch_pair(const Fp8Product& o, int split, cudaStream_t stream) {
  const int pairs = fp8_pair_capacity<BN>();
  if (pairs <= 0) return -12;
  Fp8PairArgs<1> g = {};
  if (const int e = pair_product<BN>(&g, 0, o)) return e;
  Fp8GemmParams& p = g.p[0];
  p.kb_per_split = (p.kblocks + split - 1) / split;
  p.split = (p.kblocks + p.kb_per_split - 1) / p.kb_per_split;
  return launch_pairs<BN, SPLIT>(g, SPLIT ? p.total : p.total < pairs ? p.total : pairs, p.split, stream);
}

// Tile width and split for the pair kernel: the least of waves * (K blocks * c + o), in cycles.  c is what a K block
// takes once the pipeline runs and o what a tile adds, both from timing the variants over K = 1024 ... 20480 at one and
// at many waves; a split halves K and adds the meeting of the partial tiles.  Two pairs sharing K pay only while all
// clusters are resident: [1024, 20480] x [2048, 20480]^T takes 53 us in 32 tiles of 256 columns, 36 with two pairs each.
struct PairCost {
  int bn, split, c, o;
};
static constexpr PairCost PAIR_COSTS[] = {
    {256, 1, 530, 1250}, {192, 1, 418, 750}, {128, 1, 408, 650}, {256, 2, 530, 5250}, {128, 2, 408, 3150}};
static long long pair_tiles(const Fp8GemmParams& p, int bn) {
  return static_cast<long long>((p.M + 255) / 256) * ((p.N + bn - 1) / bn);
}
static PairCost choose_pair(const Fp8GemmParams& p, long long* least) {
  PairCost best = PAIR_COSTS[0];
  *least = -1;
  for (const PairCost& w : PAIR_COSTS) {
    const long long tiles = pair_tiles(p, w.bn);
    if (w.split > 1 && (tiles * w.split > 74 || p.kblocks < 2 * w.split)) continue;
    const long long waves = (tiles * w.split + 73) / 74;
    const long long cost = waves * (static_cast<long long>((p.kblocks + w.split - 1) / w.split) * w.c + w.o);
    if (*least < 0 || cost < *least) *least = cost, best = w;
  }
  return best;
}
// Above 128 rows always pairs; from 65 where tiles of 128 columns fill half of the SMs and K is short (128 rows,
// N = 7168, K = 1024: 6.6 us against 8.8 with the other kernel; N = 1024, K = 3584: 9.3 against 6.6; N = K = 8192:
// 19.2 against 14.6).
static bool fills_pairs(const Fp8GemmParams& p) {
  return p.M > 128 || (p.M > 64 && p.N >= 37 * 128 && p.kblocks <= 12);
}
// But tiles of 64 x 128 while four CTAs of a cluster each find an SM: 256 rows, N = 1024, K = 3584: 6.9 us against 9.3
// in pairs; 512 rows, N = 512, K = 4096: 7.4 against 9.9; 512 rows, N = K = 1024 (64 tiles): 6.9 against 6.4.
static bool takes_pairs(const Fp8GemmParams& p) {
  const long long tiles = static_cast<long long>((p.M + 63) / 64) * ((p.N + 127) / 128);
  return fills_pairs(p) && (p.M <= 128 || tiles > 37);
}

static int launch_product(const Fp8Product& o, cudaStream_t stream) {
  const Fp8GemmParams& p = o.p;
  if (takes_pairs(p)) {
    long long cost;
    const PairCost pick = choose_pair(p, &cost);
    if (pick.split == 2)
      return pick.bn == 256 ? launch_pair<256, true>(o, 2, stream) : launch_pair<128, true>(o, 2, stream);
    if (pick.bn == 256) return launch_pair<256, false>(o, 1, stream);
    if (pick.bn == 192) return launch_pair<192, false>(o, 1, stream);
    return launch_pair<128, false>(o, 1, stream);
  }
  if (p.M <= 16) return launch_small<16, false>(o, stream);
  if (p.M <= 32) return launch_small<32, false>(o, stream);
  // two tiles of 64 rows instead of one of 128 while their CTAs find an SM each: half as much to meet and to store
  // (128 rows, N = 1024, K = 3584: 6.6 us against 7.1; N = K = 2048: 6.3 against 7.5; N = K = 8192: 17.3 against 14.5)
  if (p.M <= 64 || p.N <= 37 * 128) return launch_small<64, false>(o, stream);
  return launch_small<128, false>(o, stream);
}

// Cycles of two products in one launch, by the same model, and the rounds `head` that make them fewest.
static long long together_cost(const Fp8GemmParams& first, const Fp8GemmParams& second, const PairCost& w, int* head) {
  const long long n1 = pair_tiles(first, w.bn), n2 = pair_tiles(second, w.bn), pairs = n1 + n2 < 74 ? n1 + n2 : 74;
  const long long c1 = static_cast<long long>(first.kblocks) * w.c + w.o, c2 = static_cast<long long>(second.kblocks) * w.c + w.o;
  const long long rest = n1 % pairs;
  *head = 0;
  if (rest == 0) return n1 / pairs * c1 + (n2 + pairs - 1) / pairs * c2;
  long long least = -1;
  for (long long h = c1 / c2; h <= c1 / c2 + 1; ++h) {
    const long long left = n2 - h * (pairs - rest), more = left > 0 ? (left + pairs - 1) / pairs : 0;
    const long long cost = n1 / pairs * c1 + (c1 > h * c2 ? c1 : h * c2) + more * c2;
    if (least < 0 || cost < least) least = cost, *head = static_cast<int>(h < 0x0fffffff ? h : 0x0fffffff);
  }
  return least;
}

// How the two gradients of a layer [M, K] x [N, K] are computed: bn of one launch for both, 0 for a launch each.  A
// launch costs the host and the drain of the one before about 4000 cycles.
struct GradsPlan {
  int bn, head;
  bool x_first;
};
static GradsPlan plan_grads(int M, int N, int K) {
  Fp8GemmParams x = {}, w = {};
  x.M = M, x.N = K, x.kblocks = (N + 127) / 128;
  w.M = N, w.N = K, w.kblocks = (M + 127) / 128;
  GradsPlan plan = {0, 0, x.kblocks > w.kblocks};
  if (!fills_pairs(x) || !fills_pairs(w)) return plan;
  long long least, apart;
  choose_pair(x, &least);
  choose_pair(w, &apart);
  least += apart + 4000;
  for (const PairCost& way : PAIR_COSTS) {
    if (way.split > 1 || way.bn == 192) continue;
    int head;
    const long long cost = plan.x_first ? together_cost(x, w, way, &head) : together_cost(w, x, way, &head);
    if (cost <= least) least = cost, plan.bn = way.bn, plan.head = head;
  }
  return plan;
}

template <int BN>
static int launch_together(const Fp8Product& first, const Fp8Product& second, int head, cudaStream_t stream) {
  const int pairs = fp8_pair_capacity<BN>();
  if (pairs <= 0) return -12;
  Fp8PairArgs<2> g = {};
  if (const int e = pair_product<BN>(&g, 0, first)) return e;
  if (const int e = pair_product<BN>(&g, 1, second)) return e;
  g.p[0].split = g.p[1].split = 1;
  g.head = head;
  const long long total = static_cast<long long>(g.p[0].total) + g.p[1].total;
  return launch_pairs<BN, false>(g, total < pairs ? static_cast<int>(total) : pairs, 1, stream);
}

}  // namespace cvb

using namespace cvb;

static void output_params(Fp8GemmParams& p, void* c, long long ldc, int out_kind, int* status) {
  p.C = c, p.ldc = ldc, p.out_kind = out_kind, p.status = status;
  const uintptr_t at = reinterpret_cast<uintptr_t>(c) | static_cast<uintptr_t>(ldc * (out_kind == FP8_OUT_BF16 ? 2 : 4));
  p.vec = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : 0;
}

static int product_params(Fp8Product* o, const void* a, const void* a_sf, long long lda, int a_fmt, const void* b,
                          const void* b_sf, long long ldb, int b_fmt, int M, int N, int K, void* c, long long ldc,
                          int out_kind, int b_ready, int* status) {
  if (a_fmt < 0 || a_fmt > 1 || b_fmt < 0 || b_fmt > 1 || out_kind < 0 || out_kind > 2) return -1;
  if (!status || !a || !b || !a_sf || !b_sf || !c) return -2;
  // TMA and bulk copies start on 16-byte boundaries
  if (((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(a_sf) |
        reinterpret_cast<uintptr_t>(b_sf)) & 15) || lda % 16 || ldb % 16 || lda < K || ldb < K || ldc < N)
    return -3;
  *o = {a, b, lda, ldb, {}};
  Fp8GemmParams& p = o->p;
  p.a_sf = static_cast<const uint8_t*>(a_sf), p.b_sf = static_cast<const uint8_t*>(b_sf);
  p.M = M, p.N = N, p.K = K;
  p.kblocks = (K + 127) / 128, p.kgroups = (p.kblocks + 3) / 4;
  p.a_fmt = a_fmt, p.b_fmt = b_fmt, p.b_ready = b_ready;
  output_params(p, c, ldc, out_kind, status);
  return 0;
}

// C = Q(x) B^T for up to 16 bf16 rows x, quantised to e4m3 within the product
extern "C" int cvb_fp8_gemm_rows(const void* x, long long x_stride, const void* b, const void* b_sf, long long ldb,
                                 int b_fmt, int M, int N, int K, void* c, long long ldc, int out_kind, int* status,
                                 void* stream_v) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (M > 16 || b_fmt < 0 || b_fmt > 1 || out_kind < 0 || out_kind > 2) return -1;
  if (!status || !x || !b || !b_sf || !c) return -2;
  if (((reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(b_sf)) & 15) || ldb % 16 || ldb < K || ldc < N) return -3;
  Fp8GemmParams p = {};
  p.b_sf = static_cast<const uint8_t*>(b_sf);
  p.x = static_cast<const __nv_bfloat16*>(x), p.x_stride = x_stride, p.K = K;
  p.x_vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && x_stride % 8 == 0 && K % 8 == 0;
  p.M = M, p.N = N, p.kblocks = (K + 127) / 128, p.kgroups = (p.kblocks + 3) / 4;
  p.a_fmt = FP8_E4M3, p.b_fmt = b_fmt;
  output_params(p, c, ldc, out_kind, status);
  const Fp8Product o = {nullptr, b, 0, ldb, p};
  return launch_small<16, true>(o, stream);
}

// b_ready: B is not written by the kernel before this one, and was complete before that started
extern "C" int cvb_fp8_gemm(const void* a, const void* a_sf, long long lda, int a_fmt, const void* b, const void* b_sf,
                            long long ldb, int b_fmt, int M, int N, int K, void* c, long long ldc, int out_kind,
                            int b_ready, int* status, void* stream_v) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  Fp8Product o;
  const int e = product_params(&o, a, a_sf, lda, a_fmt, b, b_sf, ldb, b_fmt, M, N, K, c, ldc, out_kind, b_ready, status);
  return e ? e : launch_product(o, static_cast<cudaStream_t>(stream_v));
}

// The two gradients of a linear layer, dx [M, K] = dy [M, N] wt [K, N]^T and dw [N, K] (+)= dyt [N, M] xt [K, M]^T, in
// one launch where that fills the SMs better than one after the other.
extern "C" int cvb_fp8_gemm_grads(const void* dy, const void* dy_sf, long long ld_dy, const void* wt, const void* wt_sf,
                                  long long ld_wt, const void* dyt, const void* dyt_sf, long long ld_dyt,
                                  const void* xt, const void* xt_sf, long long ld_xt, int grad_fmt, int M, int N, int K,
                                  void* dx, long long lddx, int dx_kind, void* dw, long long lddw, int dw_kind,
                                  int* status, void* stream_v) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  Fp8Product x, w;
  int e = product_params(&x, dy, dy_sf, ld_dy, grad_fmt, wt, wt_sf, ld_wt, FP8_E4M3, M, K, N, dx, lddx, dx_kind,
                         0, status);
  if (!e)
    e = product_params(&w, dyt, dyt_sf, ld_dyt, grad_fmt, xt, xt_sf, ld_xt, FP8_E4M3, N, K, M, dw, lddw, dw_kind,
                       0, status);
  if (e) return e;
  const GradsPlan plan = plan_grads(M, N, K);
  if (plan.bn == 256) return launch_together<256>(plan.x_first ? x : w, plan.x_first ? w : x, plan.head, stream);
  if (plan.bn == 128) return launch_together<128>(plan.x_first ? x : w, plan.x_first ? w : x, plan.head, stream);
  if ((e = launch_product(x, stream))) return e;
  return launch_product(w, stream);
}

// launches of cvb_fp8_gemm_grads
extern "C" int cvb_fp8_gemm_grads_launches(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return plan_grads(M, N, K).bn ? 1 : 2;
}
