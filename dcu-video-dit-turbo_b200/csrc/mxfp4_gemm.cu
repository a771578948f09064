// Product of two MXFP4 matrices: out bf16 [M, N] = bf16(A [M, K] . W [N, K]^T + bias), fp32
// accumulation, one rounding.
//
// tcgen05.mma kind::mxf4 multiplies packed 4-bit operands (64 columns per instruction) and applies
// the two power-of-two scales of every 32 columns inside the tensor core, so neither operand is
// ever expanded.  Elements go from global memory to shared memory by TMA (128-byte swizzle, 256
// columns per stage); the scale tiles, already in tensor-memory order (mxfp4.cuh), by TMA without a
// swizzle, and from there into tensor memory by tcgen05.cp.
//
//   warp 0     loads: per stage A, W, A's scales, W's scales
//   warp 1     one lane copies a stage's scales into tensor memory and issues its MMAs
//   warps 2-5  epilogue: accumulators -> bias -> bf16 -> staging tile -> TMA store
//
// PAIR: two CTAs of a cluster (two SMs) make one 256 x 256 tile with cta_group::2 MMAs, each loading
// its own 128 rows of A and its own half of W's rows (32 KB per stage and SM against 48 KB for a
// 128 x 256 tile of one CTA): at 4 bits the tensor core eats a stage in 512 clocks, and what an SM
// can draw from L2 in that time is what bounds the product.  The leader issues for both; W's scales
// are needed whole in both tensor memories.  TMA loads are plain per-CTA ones.
// Measured, 23638 x 9216 x 3072: 266 us, 5.03 PFLOP/s (18944 x 2048 x 8192: 107 us, 5.96 PFLOP/s); the
// loads alone take 221 us and the MMAs alone 217.  One CTA per tile took 458 us, pairs 403; the rest was
// the issuing warp: with a lane-divergent region around the MMAs and a second commit per stage a stage
// took 1260 clocks, with the whole warp in step and one commit 730.
//
// Tensor memory (512 columns): a tile's 256 accumulator columns, twice, leave no room for scales,
// so the two accumulators overlap by 64 columns (0-255 and 192-447) and the scales have the last
// 64, two stages of 24.  The epilogue reads the shared 64 columns first and then lets the next
// tile's MMAs begin, so the main loop stands still for two tensor-memory loads per tile and not for
// a whole epilogue.  A stage's scales may replace those of two stages before only when that stage's
// MMAs are complete (their commit is waited for): the order of an MMA and a later copy into its
// scales is not promised.
// Calls whose 128 x 128 tiles do not fill the GPU once (few rows, above all) are bound by how many SMs
// pull on the weights: mxfp4_gemm_split_kernel gives each such tile to a cluster of 1, 2, 4 or 8
// CTAs that take a share of K each; their fp32 sums meet in shared memory, where every CTA adds up
// its share of the columns (in rank order: the same bits every time) and stores it.  8 x 9216 x 3072
// between two events: 14.3 us where the kernel for many tiles took 20.5 (an empty kernel 6).
// Every wait is bounded; on a timeout the kernel records a status word and returns.
#include "b2_common.cuh"
#include "b2_launch.h"
#include "gemm_epilogue.cuh"
#include "mxfp4.cuh"
#include "sm100_pair.cuh"
#include "sm100_ptx.cuh"

namespace b2 {

unsigned int read_clear_status_mxfp4() { return read_and_clear_device_status(); }

namespace {

constexpr int BM = 128;                    // rows per CTA
constexpr int BN = 256;                    // columns per tile
constexpr int BKE = 256;                   // columns of K per stage
constexpr int BKB = BKE / 2;               // ... in bytes: one 128-byte swizzled line
constexpr int UMMA_K = 64;
constexpr int NUM_THREADS = 192;
constexpr int EPI_THREADS = 128;
constexpr int TMEM_COLS = 512;
constexpr int ACC1 = 192;                  // first column of the second accumulator
constexpr int SHARED_COLS = 64;            // columns the two accumulators have in common
constexpr int SF_COL = 448;                // scales: two buffers of 32 columns
constexpr int SF_STRIDE = 32;
constexpr int SFB_COL = 8;                 // within a buffer: A's 2 x 4 columns, then W's 2 x 8

constexpr int A_BYTES = BM * BKB;          // 16 KB
constexpr int SFA_BYTES = 2 * kMxTileBytes;
constexpr int SFB_BYTES = 4 * kMxTileBytes;
constexpr int SF_STAGE = SFA_BYTES + SFB_BYTES;
constexpr int SMEM_LIMIT = 227 * 1024;

template <bool PAIR>
struct Layout {
  static constexpr int STAGES = PAIR ? 5 : 4;
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;        // rows of W that one CTA loads
  static constexpr int STAGE_BYTES = A_BYTES + B_ROWS * BKB;
  static constexpr int SF = STAGES * STAGE_BYTES;
  static constexpr int OUT = SF + STAGES * SF_STAGE;
  static constexpr int BIAS = OUT + (EPI_THREADS / 32) * kEpiStageBytes;
  static constexpr int BARS = BIAS + 2 * BN * 4;
  static constexpr int NUM_BARS = 2 * STAGES + 2 + 1;
  static constexpr int TOTAL = 1024 + BARS + NUM_BARS * 8 + 16;
  static_assert(TOTAL <= SMEM_LIMIT, "shared memory budget");
  static_assert(OUT % 1024 == 0, "staging tiles are 1024-byte aligned");
};

struct MxGemmArgs {
  int M, N, K;
  int tiles_m, tiles_n, num_tiles, k_blocks, group_m;
  const void* bias;
  int bias_kind;
};

__device__ __forceinline__ void decode_tile(int tile, const MxGemmArgs& a, int& m_idx, int& n_idx) {
  const int per_group = a.group_m * a.tiles_n;
  const int group = tile / per_group;
  const int first_m = group * a.group_m;
  const int rows = min(a.group_m, a.tiles_m - first_m);
  const int in_group = tile - group * per_group;
  m_idx = first_m + in_group % rows;
  n_idx = in_group / rows;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// One scale tile: 32 lines of 16 bytes -> 32 lanes x 4 columns, repeated in all four lane quarters
// (PAIR: in each CTA, from its own shared memory).
template <bool PAIR>
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t smem_addr) {
  // no swizzle; 8 lines of 16 bytes are contiguous, the next 8 follow 128 bytes on
  const uint64_t desc = (uint64_t)((smem_addr >> 4) & 0x3fffu) | (1ull << 16) | (8ull << 32) | (1ull << 46);
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
#define B2_MXF4(group)                                                                                     \
  asm volatile(                                                                                            \
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                  \
      "tcgen05.mma.cta_group::" group                                                                      \
      ".kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),          \
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                              \
      : "memory")
template <bool PAIR>
__device__ __forceinline__ void mma_mxf4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (PAIR)
    B2_MXF4("2");
  else
    B2_MXF4("1");
}
#undef B2_MXF4
// Arrive on the CTA's barrier (on both CTAs' when PAIR) once all MMAs and copies so far completed.
template <bool PAIR>
__device__ __forceinline__ void commit_all(uint32_t bar) {
  if constexpr (PAIR)
    tc_commit_pair(bar);
  else
    tc_commit(bar);
}
// Instruction descriptor of kind::mxf4: scale word halves 4-5 (W) and 29-30 (A), formats 7-9 and
// 10-11 (1 = E2M1), N >> 3 in 17-22, scale format bit 23 (1 = E8M0), M >> 4 from bit 24.
__host__ __device__ constexpr uint32_t mx_idesc(uint32_t m, uint32_t n, uint32_t half) {
  return ((half * 2) << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24) | ((half * 2) << 29);
}

template <bool PAIR>
__device__ __forceinline__ void mxfp4_gemm_body(const CUtensorMap& tmap_a, const CUtensorMap& tmap_b,
                                                const CUtensorMap& tmap_sa, const CUtensorMap& tmap_sb,
                                                const CUtensorMap& tmap_out, const MxGemmArgs& args) {
  using L = Layout<PAIR>;
  constexpr int STAGES = L::STAGES;
  constexpr int TILE_M = PAIR ? 2 * BM : BM;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* bias_s = reinterpret_cast<float*>(smem + L::BIAS);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::NUM_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t ring = smem_u32(smem);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + STAGES * 8;
  const uint32_t tfull0 = empty0 + STAGES * 8;   // accumulator complete (2)
  const uint32_t tfree = tfull0 + 2 * 8;         // the shared columns of the tile before are read
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;   // 0 = leader
  const int first_tile = PAIR ? blockIdx.x >> 1 : blockIdx.x;
  const int tile_step = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + s * 8, 1);
      mbar_init(empty0 + s * 8, 1);
    }
    mbar_init(tfull0, 1);
    mbar_init(tfull0 + 8, 1);
    mbar_init(tfree, (PAIR ? 2 : 1) * EPI_THREADS / 32);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    tma_prefetch_desc(&tmap_sa);
    tma_prefetch_desc(&tmap_sb);
    tma_prefetch_desc(&tmap_out);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();   // both CTAs' barriers are initialised before any remote access
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < args.num_tiles; tile += tile_step) {
        int m_idx, n_idx;
        decode_tile(tile, args, m_idx, n_idx);
        const int a_row = m_idx * TILE_M + (int)rank * BM;
        const int b_row = n_idx * BN + (int)rank * L::B_ROWS;
        for (int kb = 0; kb < args.k_blocks; ++kb) {
          if (!(ok = mbar_wait(empty0 + stage * 8, phase ^ 1, abort_flag, kStatusGemmTimeout))) break;
          const uint32_t dst = ring + stage * L::STAGE_BYTES;
          const uint32_t sf = ring + L::SF + stage * SF_STAGE;
          // scale tiles [row tile][k tile]: one row tile of A, two of W, two k tiles each (zeros where
          // there are none)
          if constexpr (PAIR) {
            const uint32_t bar = map_to_cta(full0 + stage * 8, 0);
            if (rank == 0) mbar_expect_tx(full0 + stage * 8, 2 * (L::STAGE_BYTES + SF_STAGE));   // both CTAs' bytes
            tma_load_2d_pair(dst, &tmap_a, bar, kb * BKB, a_row);
            tma_load_2d_pair(dst + A_BYTES, &tmap_b, bar, kb * BKB, b_row);
            tma_load_3d_pair(sf, &tmap_sa, bar, 0, kb * 2, a_row / kMxTileRows);
            tma_load_3d_pair(sf + SFA_BYTES, &tmap_sb, bar, 0, kb * 2, n_idx * (BN / kMxTileRows));
          } else {
            const uint32_t bar = full0 + stage * 8;
            mbar_expect_tx(bar, L::STAGE_BYTES + SF_STAGE);
            tma_load_2d(dst, &tmap_a, bar, kb * BKB, a_row);
            tma_load_2d(dst + A_BYTES, &tmap_b, bar, kb * BKB, b_row);
            tma_load_3d(sf, &tmap_sa, bar, 0, kb * 2, a_row / kMxTileRows);
            tma_load_3d(sf + SFA_BYTES, &tmap_sb, bar, 0, kb * 2, n_idx * (BN / kMxTileRows));
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // The whole warp walks the loop and one elected lane issues: without a lane-divergent region
      // around them, addresses and descriptors stay warp-uniform.  A lane whose wait gave up walks on
      // without waiting: every lane meets the others after each stage, or none would get past it.
      const bool leader = elect_one() != 0;
      int stage = 0;
      uint32_t phase = 0;
      int sbuf = 0;
      int buf = 0;
      uint32_t fphase = 0;
      bool first = true, ok = true;
      int back = STAGES - 2;   // ring position of two stages ago, and the parity of its release
      uint32_t back_phase = 1;
      for (int tile = first_tile; tile < args.num_tiles; tile += tile_step) {
        // the tile before must have left the columns that this one's accumulator shares with it
        if (!first) {
          if (ok) ok = mbar_wait(tfree, fphase, abort_flag, kStatusGemmTimeout);
          fphase ^= 1;
          tc_fence_after();
        }
        first = false;
        const uint32_t d_tmem = tmem_base + (buf ? ACC1 : 0);
        for (int kb = 0; kb < args.k_blocks; ++kb) {
          // the stage is filled, and the MMAs that used this scale buffer (two stages ago) are done
          if (ok) ok = mbar_wait(full0 + stage * 8, phase, abort_flag, kStatusGemmTimeout);
          if (ok) ok = mbar_wait(empty0 + back * 8, back_phase, abort_flag, kStatusGemmTimeout);
          tc_fence_after();
          const int steps = min(BKE / UMMA_K, (args.K - kb * BKE + UMMA_K - 1) / UMMA_K);
          const uint32_t sf = ring + L::SF + stage * SF_STAGE;
          const uint32_t sf_tmem = tmem_base + SF_COL + sbuf * SF_STRIDE;
          const uint32_t a_addr = ring + stage * L::STAGE_BYTES;
          const uint64_t adesc = make_smem_desc_sw128(a_addr, 16, 1024);
          const uint64_t bdesc = make_smem_desc_sw128(a_addr + A_BYTES, 16, 1024);
          if (leader && ok) {
            // [k tile][row group of 32]: 4 columns of A per k tile, 8 of W
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
              scales_to_tmem<PAIR>(sf_tmem + kt * 4, sf + kt * kMxTileBytes);
#pragma unroll
              for (int t = 0; t < 2; ++t)
                scales_to_tmem<PAIR>(sf_tmem + SFB_COL + kt * 8 + t * 4, sf + SFA_BYTES + (t * 2 + kt) * kMxTileBytes);
            }
#pragma unroll
            for (int k = 0; k < BKE / UMMA_K; ++k)
              if (k < steps)
                mma_mxf4<PAIR>(d_tmem, adesc + 2 * k, bdesc + 2 * k, mx_idesc(TILE_M, BN, k & 1), sf_tmem + (k >> 1) * 4,
                               sf_tmem + SFB_COL + (k >> 1) * 8, (kb | k) != 0);
            commit_all<PAIR>(empty0 + stage * 8);
          }
          __syncwarp();   // no lane falls a phase of a barrier behind the one that issues
          sbuf ^= 1;
          if (++back == STAGES) {
            back = 0;
            back_phase ^= 1;
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (leader && ok) commit_all<PAIR>(tfull0 + buf * 8);
        buf ^= 1;
      }
    }
  } else {
    const int quarter = warp & 3;
    const int et = threadIdx.x - 64;
    int buf = 0;
    uint32_t buf_phase = 0;
    const uint32_t stage = ring + L::OUT + quarter * kEpiStageBytes;
    const uint32_t tfree_leader = PAIR ? map_to_cta(tfree, 0) : tfree;
    bool ok = true;   // after a timeout a warp still walks its tiles (and meets the others), without waiting
    for (int tile = first_tile; tile < args.num_tiles; tile += tile_step, buf ^= 1, buf_phase ^= buf ^ 1) {
      int m_idx, n_idx;
      decode_tile(tile, args, m_idx, n_idx);
      const int col0 = n_idx * BN;
      const int row_warp = m_idx * TILE_M + (int)rank * BM + quarter * 32;
      float* bias = bias_s + buf * BN;
      for (int c = et; c < BN; c += EPI_THREADS) {
        float b = 0.f;
        if (col0 + c < args.N) {
          if (args.bias_kind == B2_BIAS_BF16) b = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(args.bias)[col0 + c]);
          if (args.bias_kind == B2_BIAS_FP32) b = reinterpret_cast<const float*>(args.bias)[col0 + c];
        }
        bias[c] = b;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (ok) ok = mbar_wait_warp(tfull0 + buf * 8, buf_phase, abort_flag, kStatusGemmTimeout);
      if (!ok) continue;
      tc_fence_after();
      const uint32_t taddr = tmem_base + (buf ? ACC1 : 0) + ((uint32_t)(quarter * 32) << 16);
      // the columns shared with the other accumulator come first: the last 64 of the first one,
      // the first 64 of the second
#pragma unroll 1
      for (int i = 0; i < BN / 64; ++i) {
        const int c = buf ? 64 * i : (64 * i + BN - SHARED_COLS) % BN;
        uint32_t v[2][32];
        tmem_ld_32x32b_x32(taddr + c, v[0]);
        tmem_ld_32x32b_x32(taddr + c + 32, v[1]);
        tmem_wait_ld();
        if (i == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR)
              mbar_arrive_cluster(tfree_leader);
            else
              mbar_arrive(tfree);
          }
        }
        if (col0 + c >= args.N) continue;
        if (lane == 0) bulk_wait_group_read<0>();   // the previous store has read the tile
        __syncwarp();
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t o[16];
          const float* bc = bias + c + 32 * hh;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            o[j] = pack_bf16x2_rn(__uint_as_float(v[hh][2 * j]) + bc[2 * j], __uint_as_float(v[hh][2 * j + 1]) + bc[2 * j + 1]);
          epilogue_stage_write(stage, lane, hh, o);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && row_warp < args.M) {
          tma_store_2d(&tmap_out, stage, col0 + c, row_warp);
          bulk_commit_group();
        }
      }
    }
    if (lane == 0) bulk_wait_group<0>();   // this warp's stores are complete before the CTA may retire
  }

  __syncwarp();
  if (*abort_flag != 0) {
    const long long t0 = clock64();
    while (clock64() - t0 < 200000) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();   // neither CTA retires (or frees tensor memory) before both are done
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else
      tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

__global__ void __launch_bounds__(NUM_THREADS, 1)
mxfp4_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                  const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb,
                  const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ MxGemmArgs args) {
  mxfp4_gemm_body<false>(tmap_a, tmap_b, tmap_sa, tmap_sb, tmap_out, args);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NUM_THREADS, 1)
mxfp4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                       const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb,
                       const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ MxGemmArgs args) {
  mxfp4_gemm_body<true>(tmap_a, tmap_b, tmap_sa, tmap_sb, tmap_out, args);
}

// ---- few tiles: a cluster of CTAs shares K ----------------------------------------------------

constexpr int SBN = 128;                   // columns per tile
constexpr int S_STAGES = 5;
constexpr int S_STAGE_BYTES = A_BYTES + SBN * BKB;
constexpr int S_SF_STAGE = 4 * kMxTileBytes;             // two k tiles of A, two of W
constexpr int S_SF = S_STAGES * S_STAGE_BYTES;
constexpr int S_BARS = S_SF + S_STAGES * S_SF_STAGE;
constexpr int S_NUM_BARS = 2 * S_STAGES + 1;
constexpr int S_TOTAL = 1024 + S_BARS + S_NUM_BARS * 8 + 16;
constexpr int S_TMEM_COLS = 256;           // 128 of accumulator, scales from column 128: two buffers of 16 in 32
constexpr int S_SF_COL = 128;
constexpr int S_PITCH = SBN + 4;           // floats per row of a CTA's sums: rows start 4 banks apart
static_assert(BM * S_PITCH * 4 <= S_SF, "the sums take the place of the operand ring");
static_assert(S_TOTAL <= SMEM_LIMIT, "shared memory budget");

__global__ void __launch_bounds__(NUM_THREADS, 1)
mxfp4_gemm_split_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                        const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb,
                        __nv_bfloat16* __restrict__ out, int splits, const __grid_constant__ MxGemmArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S_BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S_NUM_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t ring = smem_u32(smem);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + S_STAGES * 8, tfull = empty0 + S_STAGES * 8;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int m_idx = tile % args.tiles_m, n_idx = tile / args.tiles_m;
  const int kb0 = (int)((int64_t)args.k_blocks * rank / splits);
  const int kb1 = (int)((int64_t)args.k_blocks * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int i = 0; i < S_NUM_BARS; ++i) mbar_init(full0 + i * 8, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    tma_prefetch_desc(&tmap_sa);
    tma_prefetch_desc(&tmap_sb);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), S_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(empty0 + stage * 8, phase ^ 1, abort_flag, kStatusGemmTimeout)) break;
        const uint32_t bar = full0 + stage * 8;
        const uint32_t dst = ring + stage * S_STAGE_BYTES;
        const uint32_t sf = ring + S_SF + stage * S_SF_STAGE;
        mbar_expect_tx(bar, S_STAGE_BYTES + S_SF_STAGE);
        tma_load_2d(dst + A_BYTES, &tmap_b, bar, kb * BKB, n_idx * SBN);
        tma_load_3d(sf + SFA_BYTES, &tmap_sb, bar, 0, kb * 2, n_idx);
        tma_load_2d(dst, &tmap_a, bar, kb * BKB, m_idx * BM);
        tma_load_3d(sf, &tmap_sa, bar, 0, kb * 2, m_idx);
        if (++stage == S_STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one() != 0;
    int stage = 0, sbuf = 0;
    uint32_t phase = 0;
    int back = S_STAGES - 2;
    uint32_t back_phase = 1;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (ok) ok = mbar_wait(full0 + stage * 8, phase, abort_flag, kStatusGemmTimeout);
      if (ok) ok = mbar_wait(empty0 + back * 8, back_phase, abort_flag, kStatusGemmTimeout);
      tc_fence_after();
      const int steps = min(BKE / UMMA_K, (args.K - kb * BKE + UMMA_K - 1) / UMMA_K);
      const uint32_t sf = ring + S_SF + stage * S_SF_STAGE;
      const uint32_t sf_tmem = tmem_base + S_SF_COL + sbuf * SF_STRIDE;
      const uint32_t a_addr = ring + stage * S_STAGE_BYTES;
      const uint64_t adesc = make_smem_desc_sw128(a_addr, 16, 1024);
      const uint64_t bdesc = make_smem_desc_sw128(a_addr + A_BYTES, 16, 1024);
      if (leader && ok) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          scales_to_tmem<false>(sf_tmem + kt * 4, sf + kt * kMxTileBytes);
          scales_to_tmem<false>(sf_tmem + SFB_COL + kt * 4, sf + SFA_BYTES + kt * kMxTileBytes);
        }
#pragma unroll
        for (int k = 0; k < BKE / UMMA_K; ++k)
          if (k < steps)
            mma_mxf4<false>(tmem_base, adesc + 2 * k, bdesc + 2 * k, mx_idesc(BM, SBN, k & 1), sf_tmem + (k >> 1) * 4,
                            sf_tmem + SFB_COL + (k >> 1) * 4, (kb > kb0 || k > 0) ? 1u : 0u);
        tc_commit(empty0 + stage * 8);
      }
      __syncwarp();   // no lane falls a phase of a barrier behind the one that issues
      sbuf ^= 1;
      if (++back == S_STAGES) {
        back = 0;
        back_phase ^= 1;
      }
      if (++stage == S_STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (ok && leader) tc_commit(tfull);
  } else {
    // every MMA is complete and every load has been used: the sums go where the ring was
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    if (mbar_wait_warp(tfull, 0, abort_flag, kStatusGemmTimeout) && m_idx * BM + quarter * 32 < args.M) {
      tc_fence_after();
      float* dst = reinterpret_cast<float*>(smem) + row * S_PITCH;
#pragma unroll 1
      for (int c = 0; c < SBN; c += 32) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tmem_base + c + ((uint32_t)(quarter * 32) << 16), v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<uint4*>(dst + c)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  if (splits > 1)
    cluster_sync_all();
  else
    __syncthreads();
  // this CTA's share of the columns, eight per thread and step
  const int share = SBN / splits;
  const int groups = share / 8;
  const int rows = min(BM, args.M - m_idx * BM);
  if (*abort_flag == 0) {
    for (int i = threadIdx.x; i < rows * groups; i += NUM_THREADS) {
      const int row = i / groups;
      const int c = rank * share + (i - row * groups) * 8;
      const int col = n_idx * SBN + c;
      if (col >= args.N) continue;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = 0.f;
        if (args.bias_kind == B2_BIAS_BF16) f[j] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(args.bias)[col + j]);
        if (args.bias_kind == B2_BIAS_FP32) f[j] = reinterpret_cast<const float*>(args.bias)[col + j];
      }
      const uint32_t at = ring + (row * S_PITCH + c) * 4;
      float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
      for (int r = 0; r < splits; ++r) {
        const uint32_t src = splits > 1 ? map_to_cta(at, r) : at;
        const float4 x = ld_cluster_f4(src), y = ld_cluster_f4(src + 16);
        lo = make_float4(lo.x + x.x, lo.y + x.y, lo.z + x.z, lo.w + x.w);
        hi = make_float4(hi.x + y.x, hi.y + y.y, hi.z + y.z, hi.w + y.w);
      }
      uint4 o;
      o.x = pack_bf16x2_rn(lo.x + f[0], lo.y + f[1]);
      o.y = pack_bf16x2_rn(lo.z + f[2], lo.w + f[3]);
      o.z = pack_bf16x2_rn(hi.x + f[4], hi.y + f[5]);
      o.w = pack_bf16x2_rn(hi.z + f[6], hi.w + f[7]);
      *reinterpret_cast<uint4*>(out + (int64_t)(m_idx * BM + row) * args.N + col) = o;
    }
  } else {
    const long long t0 = clock64();
    while (clock64() - t0 < 200000) {
    }
  }
  if (splits > 1)
    cluster_sync_all();   // no CTA retires while another reads its sums
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S_TMEM_COLS);
  }
}

int encode_operand(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int box_rows) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)(k / 2), (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(k / 2)};
  const cuuint32_t box[2] = {BKB, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: tensor map encode failed (%d)", (int)r);
  return B2_OK;
}

// Scale bytes as [row tile][k tile][128 words]; a box is two k tiles of `row_tiles` row tiles.
int encode_scales(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int row_tiles) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t k_tiles = (cuuint64_t)((k + kMxTileCols - 1) / kMxTileCols);
  const cuuint64_t dims[3] = {kMxTileBytes / 4, k_tiles, (cuuint64_t)((rows + kMxTileRows - 1) / kMxTileRows)};
  const cuuint64_t strides[2] = {kMxTileBytes, kMxTileBytes * k_tiles};
  const cuuint32_t box[3] = {kMxTileBytes / 4, 2, (cuuint32_t)row_tiles};
  const cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: scale tensor map encode failed (%d)", (int)r);
  return B2_OK;
}

int encode_out(CUtensorMap* map, void* base, int64_t M, int64_t N) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
  const cuuint64_t strides[1] = {(cuuint64_t)N * 2};
  const cuuint32_t box[2] = {64, 32};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: output tensor map encode failed (%d)", (int)r);
  return B2_OK;
}

}  // namespace

int launch_mxfp4_gemm(const uint8_t* A, const uint8_t* a_scale, const uint8_t* W, const uint8_t* w_scale,
                      const void* bias, int bias_kind, void* out, int64_t M, int64_t N, int64_t K,
                      cudaStream_t stream) {
  // slot.a = SMs, slot.b = CTA pairs that run at once (0: none)
  static PerDeviceSetup per_device;
  const DeviceSlot* slot = nullptr;
  const int setup_status = per_device.get("mxfp4_gemm", [](int dev, DeviceSlot& s) -> int {
    cudaError_t e = cudaFuncSetAttribute(mxfp4_gemm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         Layout<false>::TOTAL);
    if (e != cudaSuccess) return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: smem attribute: %s", cudaGetErrorString(e));
    e = cudaFuncSetAttribute(mxfp4_gemm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<true>::TOTAL);
    if (e != cudaSuccess) return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: smem attribute: %s", cudaGetErrorString(e));
    e = cudaFuncSetAttribute(mxfp4_gemm_split_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S_TOTAL);
    if (e != cudaSuccess) return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: smem attribute: %s", cudaGetErrorString(e));
    s.a = kNumSMsB200;
    cudaDeviceGetAttribute(&s.a, cudaDevAttrMultiProcessorCount, dev);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(s.a / 2 * 2));
    cfg.blockDim = dim3(NUM_THREADS);
    cfg.dynamicSmemBytes = Layout<true>::TOTAL;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&s.b, mxfp4_gemm_pair_kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      s.b = 0;
    }
    return B2_OK;
  }, &slot);
  if (setup_status != B2_OK) return setup_status;
  CUtensorMap ta, tb, tsa, tsb, tout;
  MxGemmArgs a;
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.k_blocks = (int)((K + BKE - 1) / BKE);
  a.bias = bias;
  a.bias_kind = bias_kind;
  a.group_m = 1;
  // one 128 x 128 tile (or a share of its K) per SM, while there are SMs
  const int64_t small_tiles = ((M + BM - 1) / BM) * ((N + SBN - 1) / SBN);
  if (small_tiles <= slot->a) {
    // clusters of four and eight leave SMs without a place (132 and 120 of 148 can be used)
    int splits = 1;
    for (int s = 2; s <= 8 && s <= a.k_blocks; s *= 2)
      if (small_tiles * s <= (s == 2 ? slot->a : s == 4 ? 132 : 120)) splits = s;
    int st = encode_operand(&ta, A, M, K, BM);
    if (st == B2_OK) st = encode_operand(&tb, W, N, K, SBN);
    if (st == B2_OK) st = encode_scales(&tsa, a_scale, M, K, 1);
    if (st == B2_OK) st = encode_scales(&tsb, w_scale, N, K, 1);
    if (st != B2_OK) return st;
    a.tiles_m = (int)((M + BM - 1) / BM);
    a.tiles_n = (int)((N + SBN - 1) / SBN);
    a.num_tiles = (int)small_tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(small_tiles * splits));
    cfg.blockDim = dim3(NUM_THREADS);
    cfg.dynamicSmemBytes = S_TOTAL;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)splits;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, mxfp4_gemm_split_kernel, ta, tb, tsa, tsb, (__nv_bfloat16*)out, splits, a);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(B2_LAUNCH_FAILED, "mxfp4_gemm: launch failed: %s", cudaGetErrorString(e));
    }
    return B2_OK;
  }
  const bool pair = slot->b > 0 && M > BM;
  const int tile_m = pair ? 2 * BM : BM;
  int st = encode_operand(&ta, A, M, K, BM);
  if (st != B2_OK) return st;
  st = encode_operand(&tb, W, N, K, pair ? Layout<true>::B_ROWS : Layout<false>::B_ROWS);
  if (st != B2_OK) return st;
  st = encode_scales(&tsa, a_scale, M, K, 1);
  if (st != B2_OK) return st;
  st = encode_scales(&tsb, w_scale, N, K, BN / kMxTileRows);
  if (st != B2_OK) return st;
  st = encode_out(&tout, out, M, N);
  if (st != B2_OK) return st;
  a.tiles_m = (int)((M + tile_m - 1) / tile_m);
  a.tiles_n = (int)((N + BN - 1) / BN);
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
  if (tiles > 0x7fffffffLL) return fail(B2_TOO_LARGE, "mxfp4_gemm: too many tiles");
  a.num_tiles = (int)tiles;
  a.group_m = pair ? 8 : 16;
  if (pair) {
    const int clusters = a.num_tiles < slot->b ? a.num_tiles : slot->b;
    mxfp4_gemm_pair_kernel<<<clusters * 2, NUM_THREADS, Layout<true>::TOTAL, stream>>>(ta, tb, tsa, tsb, tout, a);
  } else {
    const int grid = a.num_tiles < slot->a ? a.num_tiles : slot->a;
    mxfp4_gemm_kernel<<<grid, NUM_THREADS, Layout<false>::TOTAL, stream>>>(ta, tb, tsa, tsb, tout, a);
  }
  return check_launch("mxfp4_gemm");
}

}  // namespace b2
