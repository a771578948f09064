// bf16 -> MXFP4 quantiser (plain, or of the SwiGLU product) and the way back, for sm_100a; and
// the values of rowwise int8.
//
// All are bound by memory: quantising K columns of a row moves 2K (4K with SwiGLU) bytes in and
// K/2 + K/32 out.  The unit is one scale tile, 128 rows x 128 columns: 16 lanes hold a row's 128
// columns, 16 bytes each (four lanes per block of 32, so the block's maximum is two shuffles).  The
// tile's 512 scale bytes meet in shared memory and leave as full lines; written row by row they
// would be 4-byte pieces of eight lines each.
#include "b2_common.cuh"
#include "b2_launch.h"
#include "mxfp4.cuh"
#include "sm100_ptx.cuh"

namespace b2 {

unsigned int read_clear_status_mxfp4_quantize() { return read_and_clear_device_status(); }

namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerPass = kThreads / 16;                 // 16
constexpr int kPasses = kMxTileRows / kRowsPerPass;         // 8

// silu(g) * u = g / (1 + 2^(-g log2 e)) * u of a pair, in fp32 with the fast exponential and
// reciprocal (a few units in the last place, five decimal digits below the step of the 4-bit
// elements).  Holds for g >= kFarGate: below -87 the reciprocal is flushed to zero.
__device__ __forceinline__ uint64_t silu_mul2(uint64_t g, uint64_t u) {
  float x0, x1;
  unpack2(mul2(g, pack2(-1.4426950408889634f, -1.4426950408889634f)), x0, x1);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x0));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x1));
  unpack2(add2(pack2(x0, x1), pack2(1.0f, 1.0f)), x0, x1);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x1));
  return mul2(mul2(g, pack2(x0, x1)), u);
}

// Gates below it are rare (silu there is above -1.5e-33), but their product with a large `up` is not
// zero: 2^-129, half the smallest element, is reached down to g = -183.  e^g = (e^(g/4))^4 times g and u one
// after another, so no factor is flushed before the product is (1 + e^g is 1 here).
constexpr float kFarGate = -80.0f;
constexpr uint32_t kFarGateBits = 0xc2a0u;                  // in bf16; larger ones are further, -infinity or NaN
__device__ __forceinline__ float silu_mul_far(float g, float u) {
  const float e = expf(0.25f * g);
  return g * e * u * e * e * e;
}

// A stage is 32 KB: a whole tile's rows, or with SwiGLU half of them, gate and up.
constexpr int kStages = 2;
constexpr int kBoxBytes = 64 * kMxTileCols * 2;             // 64 rows x 128 columns
constexpr int kStageBytes = 2 * kBoxBytes;
constexpr int kTileBuf = kStages * kStageBytes;             // scale bytes of the tile in hand, twice
constexpr int kBarOffset = kTileBuf + 2 * kMxTileBytes;
constexpr int kQuantSmem = 128 + kBarOffset + 2 * kStages * 8 + 16;

// Persistent: three CTAs per SM walk the tiles, one more warp keeps the ring of TMA loads full, so what
// is in flight does not depend on how many loads the compiler keeps together.  109099 x 3072 takes
// 141 us, 6.0 TB/s (254 us with SwiGLU, 6.0 TB/s); a thread per 16-byte load and row 154 and 293
// us, two CTAs with three stages 154 and 272, six with one 158 and 260.  Rows and columns outside
// the matrix arrive as zeros.
template <bool SWIGLU>
__global__ void __launch_bounds__(kThreads + 32, 3)
quantize_mxfp4_kernel(const __grid_constant__ CUtensorMap tmap, uint32_t* __restrict__ q, uint8_t* __restrict__ scales,
                      int M, int K, int col_tiles, int tiles) {
  constexpr int PARTS = SWIGLU ? 2 : 1;                     // stages per tile
  constexpr int PART_PASSES = kPasses / PARTS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  const uint32_t full0 = smem_u32(smem + kBarOffset), empty0 = full0 + kStages * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kBarOffset + 2 * kStages * 8);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full0 + i * 8, 1);
      mbar_init(empty0 + i * 8, kThreads / 32);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmap);
  }
  __syncthreads();
  int stage = 0;
  uint32_t phase = 0;
  auto advance = [&]() {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  };
  if (threadIdx.x >= kThreads) {
    if (threadIdx.x == kThreads) {
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
        const int col = (t % col_tiles) * kMxTileCols, row = (t / col_tiles) * kMxTileRows;
        for (int part = 0; part < PARTS; ++part) {
          if (!(ok = mbar_wait(empty0 + stage * 8, phase ^ 1, abort_flag, kStatusGemmTimeout))) break;
          const uint32_t dst = smem_u32(smem + stage * kStageBytes);
          mbar_expect_tx(full0 + stage * 8, kStageBytes);
          tma_load_2d(dst, &tmap, full0 + stage * 8, col, row + part * 64);
          // the tile's other rows, or the up columns of these
          tma_load_2d(dst + kBoxBytes, &tmap, full0 + stage * 8, SWIGLU ? K + col : col, SWIGLU ? row + part * 64 : row + 64);
          advance();
        }
      }
    }
    return;
  }
  const int lane16 = threadIdx.x & 15;
  const int row_in_pass = threadIdx.x >> 4;
  int turn = 0;
  bool ok = true;
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int col = (t % col_tiles) * kMxTileCols + lane16 * 8;
    const int first = (t / col_tiles) * kMxTileRows + row_in_pass;
    const int rows_left = col < K ? M - first : 0;          // pass p is stored for p * 16 < rows_left
    uint32_t* dst = q + (int64_t)first * (K / 8) + col / 8;
    uint32_t* tile = reinterpret_cast<uint32_t*>(smem + kTileBuf + turn * kMxTileBytes);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      // after a timeout every thread still walks its tiles (and meets the barriers), without waiting
      if (ok) ok = mbar_wait(full0 + stage * 8, phase, abort_flag, kStatusGemmTimeout);
      const uint4* src = reinterpret_cast<const uint4*>(smem + stage * kStageBytes) + row_in_pass * 16 + lane16;
      uint32_t gates = 0;                                   // the furthest gate's bits, in halves
      // pass pp: this lane's eight columns of a row; `far` where some gates of the warp's rows are
      auto pass = [&](int pp, bool far) {
        const int p = part * PART_PASSES + pp;
        const uint4 v = src[pp * kRowsPerPass * 16];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        float f[8];
        uint32_t m;
        if constexpr (SWIGLU) {
          const uint4 u = src[kBoxBytes / 16 + pp * kRowsPerPass * 16];
          const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            unpack2(silu_mul2(bf16x2_to_f32x2(w[i]), bf16x2_to_f32x2(uw[i])), f[2 * i], f[2 * i + 1]);
          if (far) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float g = (i & 1) ? bf16hi_to_f32(w[i >> 1]) : bf16lo_to_f32(w[i >> 1]);
              if (g < kFarGate) f[i] = silu_mul_far(g, (i & 1) ? bf16hi_to_f32(uw[i >> 1]) : bf16lo_to_f32(uw[i >> 1]));
            }
          } else {
            gates = __vmaxu2(gates, __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3])));
          }
          m = col < K ? mx_absmax_halves(f) : 0u;           // past the gate columns lie up columns, not zeros
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) unpack2(bf16x2_to_f32x2(w[i]), f[2 * i], f[2 * i + 1]);
          m = mx_absmax_bits(mx_absmax_bits(mx_absmax_bits(w[0] & 0x7fff7fffu, w[1]), w[2]), w[3]);
        }
        const uint32_t byte = mx_block_byte(m);
        const uint32_t word = mx_gather_word(byte);
        if (p * kRowsPerPass < rows_left) dst[(int64_t)p * kRowsPerPass * (K / 8)] = mx_quantize8(f, byte);
        if (lane16 == 0) tile[mx_scale_offset(p * kRowsPerPass + row_in_pass, 0) / 4] = word;
      };
#pragma unroll
      for (int pp = 0; pp < PART_PASSES; ++pp) pass(pp, false);
      if constexpr (SWIGLU) {
        // far gates are rare: the warp's rows are then done again, so that the passes above have no branch
        // (with one in each, 109099 x 3072 took 267 us)
        if (__any_sync(0xffffffffu, col < K && max(gates & 0xffffu, gates >> 16) > kFarGateBits)) {
#pragma unroll 1
          for (int pp = 0; pp < PART_PASSES; ++pp) pass(pp, true);
        }
      }
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(empty0 + stage * 8);
      advance();
    }
    // The tile's bytes are complete; the other buffer is written next, and this one again only after
    // one more of these barriers.
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    if (threadIdx.x < kMxTileBytes / 16)
      reinterpret_cast<uint4*>(scales + (int64_t)t * kMxTileBytes)[threadIdx.x] = reinterpret_cast<const uint4*>(tile)[threadIdx.x];
    turn ^= 1;
  }
}

// The values of a quantised matrix in bf16 (exact, but where 6 * 2^e passes bf16's range): the same
// tile per CTA, four bytes of elements in and 16 bytes out per thread and row.
__global__ void __launch_bounds__(kThreads, 4)
dequantize_mxfp4_kernel(const uint32_t* __restrict__ q, const uint8_t* __restrict__ scales, uint4* __restrict__ out,
                        int M, int K, int col_tiles) {
  const int ct = blockIdx.x % col_tiles;
  const int rt = blockIdx.x / col_tiles;
  const int lane16 = threadIdx.x & 15;
  const int row_in_pass = threadIdx.x >> 4;
  const int col = ct * kMxTileCols + lane16 * 8;
  if (col >= K) return;
  const uint8_t* tile = scales + (int64_t)blockIdx.x * kMxTileBytes;
  uint32_t w[kPasses], e[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int r = p * kRowsPerPass + row_in_pass;
    const int row = rt * kMxTileRows + r;
    w[p] = row < M ? __ldg(q + (int64_t)row * (K / 8) + col / 8) : 0u;
    e[p] = __ldg(tile + mx_scale_offset(r, lane16 >> 2));
  }
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = rt * kMxTileRows + p * kRowsPerPass + row_in_pass;
    if (row >= M) break;
    const float s = mx_scale_value(e[p]);
    uint32_t h[4], o[4];
    mx_unpack8(w[p], h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      o[i] = pack_bf16x2_rn(f.x * s, f.y * s);
    }
    out[(int64_t)row * (K / 8) + col / 8] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// bf16(q * scale[row]).  One warp per row piece of 32 x 8 columns x 4; K % 8 == 0.
__global__ void __launch_bounds__(kThreads)
dequantize_int8_rows_kernel(const uint2* __restrict__ q, const float* __restrict__ scale, uint4* __restrict__ out,
                            int64_t M, int kvec) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  const int pieces = (kvec + 127) / 128;
  const int64_t total = M * pieces;
  for (int64_t t = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); t < total; t += warps) {
    const int64_t row = t / pieces;
    const int c0 = (int)(t - row * pieces) * 128 + lane;
    const float s = __ldg(scale + row);
    uint2 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c0 + 32 * i < kvec ? __ldg(q + row * kvec + c0 + 32 * i) : make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c0 + 32 * i >= kvec) break;
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = (j < 2 ? v[i].x : v[i].y) >> (16 * (j & 1));
        o[j] = pack_bf16x2_rn((float)(int8_t)(w & 0xff) * s, (float)(int8_t)((w >> 8) & 0xff) * s);
      }
      out[row * kvec + c0 + 32 * i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// Widths that are no multiple of 8: q and out start a row at the same place in their vectors, so a warp
// takes the aligned vectors that a row touches and stores those at its ends element by element.
__global__ void __launch_bounds__(kThreads)
dequantize_int8_rows_odd_kernel(const uint2* __restrict__ q, const float* __restrict__ scale, uint4* __restrict__ out,
                                int64_t M, int K) {
  const int lane = threadIdx.x & 31;
  for (int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); row < M;
       row += (int64_t)gridDim.x * (kThreads / 32)) {
    const float s = __ldg(scale + row);
    const int64_t start = row * K, v0 = start >> 3;
    const int head = (int)(start & 7), vecs = (head + K + 7) >> 3;
    for (int c = lane; c < vecs; c += 32) {
      if (c * 8 >= head && c * 8 + 8 - head <= K) {
        const uint2 v = __ldg(q + v0 + c);
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w = (j < 2 ? v.x : v.y) >> (16 * (j & 1));
          o[j] = pack_bf16x2_rn((float)(int8_t)(w & 0xff) * s, (float)(int8_t)((w >> 8) & 0xff) * s);
        }
        out[v0 + c] = make_uint4(o[0], o[1], o[2], o[3]);
      } else {
        for (int j = 0; j < 8; ++j) {
          const int col = c * 8 + j - head;
          if (col < 0 || col >= K) continue;
          reinterpret_cast<__nv_bfloat16*>(out + v0 + c)[j] =
              __float2bfloat16_rn((float)reinterpret_cast<const int8_t*>(q + v0 + c)[j] * s);
        }
      }
    }
  }
}

// Any width and alignment: one CTA per row, element by element.
__global__ void __launch_bounds__(kThreads)
dequantize_int8_rows_generic_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale,
                                    __nv_bfloat16* __restrict__ out, int64_t M, int64_t K) {
  for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
    const float s = scale[row];
    for (int64_t c = threadIdx.x; c < K; c += kThreads) out[row * K + c] = __float2bfloat16_rn((float)q[row * K + c] * s);
  }
}

int tile_grid(const char* what, int64_t M, int64_t K, int* col_tiles, unsigned* grid) {
  const int64_t rt = (M + kMxTileRows - 1) / kMxTileRows, ct = (K + kMxTileCols - 1) / kMxTileCols;
  if (rt * ct > 0x7fffffffLL || M > 0x7fffff00LL || K > 0x3fffff00LL)
    return fail(B2_TOO_LARGE, "%s: M=%lld K=%lld exceed the launch grid", what, (long long)M, (long long)K);
  *col_tiles = (int)ct;
  *grid = (unsigned)(rt * ct);
  return B2_OK;
}

}  // namespace

int launch_quantize_mxfp4(const void* x, uint8_t* q, uint8_t* scales, int64_t M, int64_t K, bool swiglu,
                          cudaStream_t stream) {
  int ct;
  unsigned tiles;
  const int st = tile_grid("quantize_mxfp4", M, K, &ct, &tiles);
  if (st != B2_OK) return st;
  static PerDeviceSetup per_device;
  const DeviceSlot* slot = nullptr;
  const int setup_status = per_device.get("quantize_mxfp4", [](int dev, DeviceSlot& s) -> int {
    const void* kernels[2] = {(const void*)quantize_mxfp4_kernel<false>, (const void*)quantize_mxfp4_kernel<true>};
    for (const void* f : kernels) {
      const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kQuantSmem);
      if (e != cudaSuccess) return fail(B2_LAUNCH_FAILED, "quantize_mxfp4: smem attribute: %s", cudaGetErrorString(e));
    }
    s.a = kNumSMsB200;
    cudaDeviceGetAttribute(&s.a, cudaDevAttrMultiProcessorCount, dev);
    return B2_OK;
  }, &slot);
  if (setup_status != B2_OK) return setup_status;
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return fail(B2_LAUNCH_FAILED, "quantize_mxfp4: cuTensorMapEncodeTiled is unavailable");
  CUtensorMap map;
  const cuuint64_t width = (cuuint64_t)K * (swiglu ? 2 : 1);
  const cuuint64_t dims[2] = {width, (cuuint64_t)M}, strides[1] = {width * 2};
  const cuuint32_t box[2] = {kMxTileCols, 64}, estr[2] = {1, 1};
  const CUresult r = enc(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(x), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B2_LAUNCH_FAILED, "quantize_mxfp4: tensor map encode failed (%d)", (int)r);
  const unsigned cap = (unsigned)slot->a * 3;
  const unsigned grid = tiles < cap ? tiles : cap;
  if (swiglu)
    quantize_mxfp4_kernel<true><<<grid, kThreads + 32, kQuantSmem, stream>>>(map, (uint32_t*)q, scales, (int)M, (int)K, ct, (int)tiles);
  else
    quantize_mxfp4_kernel<false><<<grid, kThreads + 32, kQuantSmem, stream>>>(map, (uint32_t*)q, scales, (int)M, (int)K, ct, (int)tiles);
  return check_launch("quantize_mxfp4");
}

int launch_dequantize_mxfp4(const uint8_t* q, const uint8_t* scales, void* out, int64_t M, int64_t K,
                            cudaStream_t stream) {
  int ct;
  unsigned grid;
  const int st = tile_grid("dequantize_mxfp4", M, K, &ct, &grid);
  if (st != B2_OK) return st;
  dequantize_mxfp4_kernel<<<grid, kThreads, 0, stream>>>((const uint32_t*)q, scales, (uint4*)out, (int)M, (int)K, ct);
  return check_launch("dequantize_mxfp4");
}

int launch_dequantize_int8_rows(const int8_t* q, const float* scale, void* out, int64_t M, int64_t K,
                                cudaStream_t stream) {
  if (K % 8 == 0 && K <= 0x7fffffffLL && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && aligned16(out)) {
    const int kvec = (int)(K / 8);
    const int64_t need = (M * ((kvec + 127) / 128) + kThreads / 32 - 1) / (kThreads / 32);
    const int64_t cap = (int64_t)kNumSMsB200 * 32;
    dequantize_int8_rows_kernel<<<(unsigned)(need < cap ? need : cap), kThreads, 0, stream>>>(
        (const uint2*)q, scale, (uint4*)out, M, kvec);
  } else if (K <= 0x7ffffff0LL && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && aligned16(out)) {
    const int64_t need = (M + kThreads / 32 - 1) / (kThreads / 32), cap = (int64_t)kNumSMsB200 * 32;
    dequantize_int8_rows_odd_kernel<<<(unsigned)(need < cap ? need : cap), kThreads, 0, stream>>>(
        (const uint2*)q, scale, (uint4*)out, M, (int)K);
  } else {
    const int64_t cap = (int64_t)kNumSMsB200 * 16;
    dequantize_int8_rows_generic_kernel<<<(unsigned)(M < cap ? M : cap), kThreads, 0, stream>>>(
        q, scale, (__nv_bfloat16*)out, M, K);
  }
  return check_launch("dequantize_int8_rows");
}

}  // namespace b2
