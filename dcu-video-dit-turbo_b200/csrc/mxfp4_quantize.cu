// bf16 -> MXFP4 quantiser (plain, or of the SwiGLU product) and the way back, for sm_100a; and
// the values of rowwise int8.
//
// All are bound by memory: quantising K columns of a row moves 2K (4K with SwiGLU) bytes in and
// K/2 + K/32 out.  One CTA takes one scale tile, 128 rows x 128 columns: 16 lanes hold a row's 128
// columns, one 16-byte load each (four lanes per block of 32, so the block's maximum is two
// shuffles), and a thread's eight rows are loaded before the first is used.  The tile's 512 scale
// bytes meet in shared memory and leave as full lines; written row by row they would be 4-byte
// pieces of eight lines each.
#include "b2_common.cuh"
#include "b2_launch.h"
#include "mxfp4.cuh"

namespace b2 {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerPass = kThreads / 16;                 // 16
constexpr int kPasses = kMxTileRows / kRowsPerPass;         // 8

// silu(g) * u in fp32: g / (1 + exp(-g)); the exponential and the reciprocal are the fast ones (a
// few units in the last place of fp32), five decimal digits below the step of the 4-bit elements.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float e = __expf(-g);
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * r * u;
}

// 8 fp32 of each of 4 neighbouring lanes make a block: its packed elements (returned) and byte.
__device__ __forceinline__ uint32_t quantize8(const float (&f)[8], uint32_t absmax_bits, uint32_t& byte) {
  byte = mx_scale_byte(absmax_bits >> 23);
  const float inv = mx_inverse_scale(byte);
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = f[i] * inv;
  return byte == 255u ? 0u : mx_pack8(s);
}

template <bool SWIGLU>
__global__ void __launch_bounds__(kThreads)
quantize_mxfp4_kernel(const uint4* __restrict__ x, uint32_t* __restrict__ q, uint8_t* __restrict__ scales,
                      int M, int K, int col_tiles) {
  __shared__ uint32_t tile[kMxTileBytes / 4];
  const int ct = blockIdx.x % col_tiles;
  const int rt = blockIdx.x / col_tiles;
  const int lane16 = threadIdx.x & 15;
  const int row_in_pass = threadIdx.x >> 4;
  const int col = ct * kMxTileCols + lane16 * 8;
  const bool col_ok = col < K;                              // K % 32 == 0: a block is in or out whole
  const int64_t row_vec = (SWIGLU ? 2 : 1) * (int64_t)(K / 8);
  uint4 v[kPasses], u[SWIGLU ? kPasses : 1];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = rt * kMxTileRows + p * kRowsPerPass + row_in_pass;
    const bool live = col_ok && row < M;
    const uint4* src = x + (int64_t)row * row_vec + col / 8;
    v[p] = live ? ldg_stream(src) : make_uint4(0, 0, 0, 0);
    if constexpr (SWIGLU) u[p] = live ? ldg_stream(src + K / 8) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int r = p * kRowsPerPass + row_in_pass;
    const int row = rt * kMxTileRows + r;
    const uint32_t w[4] = {v[p].x, v[p].y, v[p].z, v[p].w};
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf16lo_to_f32(w[i]);
      f[2 * i + 1] = bf16hi_to_f32(w[i]);
    }
    uint32_t m;
    if constexpr (SWIGLU) {
      const uint32_t uw[4] = {u[p].x, u[p].y, u[p].z, u[p].w};
      m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = silu_mul(f[2 * i], bf16lo_to_f32(uw[i]));
        f[2 * i + 1] = silu_mul(f[2 * i + 1], bf16hi_to_f32(uw[i]));
        m = max(m, max(__float_as_uint(f[2 * i]) & 0x7fffffffu, __float_as_uint(f[2 * i + 1]) & 0x7fffffffu));
      }
    } else {
      m = mx_absmax_bits(mx_absmax_bits(mx_absmax_bits(w[0] & 0x7fff7fffu, w[1]), w[2]), w[3]);
      m = max(m << 16, m & 0xffff0000u);                    // the larger half, as fp32 bits
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    uint32_t byte;
    const uint32_t packed = quantize8(f, m, byte);
    if (col_ok && row < M) q[(int64_t)row * (K / 8) + col / 8] = packed;
    const uint32_t word = mx_gather_word(byte, 0xffffffffu);   // rows and blocks outside hold zeros: byte 0
    if (lane16 == 0) tile[mx_scale_offset(r, 0) / 4] = word;
  }
  __syncthreads();
  if (threadIdx.x < kMxTileBytes / 16)
    reinterpret_cast<uint4*>(scales + (int64_t)blockIdx.x * kMxTileBytes)[threadIdx.x] =
        reinterpret_cast<const uint4*>(tile)[threadIdx.x];
}

// The values of a quantised matrix in bf16 (exact, but where 6 * 2^e passes bf16's range): the same
// tile per CTA, four bytes of elements in and 16 bytes out per thread and row.
__global__ void __launch_bounds__(kThreads)
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
  unsigned grid;
  const int st = tile_grid("quantize_mxfp4", M, K, &ct, &grid);
  if (st != B2_OK) return st;
  if (swiglu)
    quantize_mxfp4_kernel<true><<<grid, kThreads, 0, stream>>>((const uint4*)x, (uint32_t*)q, scales, (int)M, (int)K, ct);
  else
    quantize_mxfp4_kernel<false><<<grid, kThreads, 0, stream>>>((const uint4*)x, (uint32_t*)q, scales, (int)M, (int)K, ct);
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
  } else {
    const int64_t cap = (int64_t)kNumSMsB200 * 16;
    dequantize_int8_rows_generic_kernel<<<(unsigned)(M < cap ? M : cap), kThreads, 0, stream>>>(
        q, scale, (__nv_bfloat16*)out, M, K);
  }
  return check_launch("dequantize_int8_rows");
}

}  // namespace b2
