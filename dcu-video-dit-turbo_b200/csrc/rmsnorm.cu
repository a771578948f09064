// RMSNorm with the residual's addition and a quantised output: the producer of a quantised linear.
//
//   s = bf16(x + residual)                      (stored: the residual stream of the next layer)
//   y = s / sqrt(mean(s^2) + eps) * weight      (fp32)
//   int8    scale = max|y| / 127 per row, at least 1e-30;  q = round half even(y / scale)
//   mxfp4   per block of 32 columns (mxfp4.cuh)
//
// Bound by memory: 4 bytes in and 2 + 1 (2 + 17/32) bytes out per element.  A row is held by TPR
// threads in registers from its only read to its quantised write; y is never rounded to bf16 in
// between.  A thread keeps the same columns of every row, so the weight is read once per CTA.
// Measured: int8 109099 x 3072 376 us = 6.2 TB/s, 23638 x 3072 88 us = 5.8; MXFP4 360 and 84 us.
// Roundings: the mean, 1 / sqrt, max|y| / 127 and y / scale are each rounded once, to the nearest fp32
// (0 to 3 % more time than products with rounded reciprocals and the fast 1 / sqrt, int8 at 16384 columns 4 %).
// The elements divide by the fp32 scale that is stored, so q * scale is within half a step of y.
#include "b2_common.cuh"
#include "b2_launch.h"
#include "mxfp4.cuh"

namespace b2 {
namespace {

constexpr int kThreads = 256;   // of the generic kernel

// 1 / n as a sum of two fp32
struct Reciprocal {
  float high, low;
  __host__ __device__ constexpr explicit Reciprocal(double n) : high((float)(1.0 / n)), low((float)(1.0 / n - (double)(float)(1.0 / n))) {}
};

struct RmsArgs {
  const uint4* x;
  const uint4* residual;   // null: s = x and nothing is stored to `sum`
  const uint4* weight;
  uint4* sum;
  void* q;                 // int8 [M, C] or packed [M, C/2]
  void* scale;             // fp32 [M] or scale tiles
  int64_t M;
  int cvec;                // C / 8
  Reciprocal inv_c{1.0};   // of C
  float eps;
};

// v / n, rounded once (from within 2^-48 of itself); infinities and NaN as they are
__device__ __forceinline__ float quotient(float v, const Reciprocal& inv) {
  return fabsf(v) <= 3.4028234e38f ? fmaf(v, inv.high, v * inv.low) : v;
}
// 1 / sqrt(sum of squares / C + eps)
__device__ __forceinline__ float row_rstd(float ss, const Reciprocal& inv_c, float eps) {
  return __frsqrt_rn(__fadd_rn(quotient(ss, inv_c), eps));
}
// A row's int8 scale, from its largest magnitude, and 1 / scale as a sum of two fp32.  Rows with a NaN or an
// infinity keep that in the scale and get zero elements.
struct Int8Scale {
  float s, inv, inv_low;
  bool zero_row;
  __device__ __forceinline__ explicit Int8Scale(float absmax) {
    s = absmax != absmax ? absmax : fmaxf(quotient(absmax, Reciprocal(127.0)), 1.0e-30f);
    zero_row = !(s <= 3.4028234e38f);
    inv = __frcp_rn(s);
    inv_low = fmaf(-s, inv, 1.0f) * inv;
  }
  // Round half even of y / s for a pair, |y| <= 127 s (a unit in the last place over): the low bytes of
  // the sums.  The quotient is rounded once, to the nearest fp32: with the reciprocal's first part
  // alone it put 4 to 6 of 1000 exact ties on the wrong side.
  __device__ __forceinline__ void bits2(float y0, float y1, uint32_t& b0, uint32_t& b1) const {
    const uint64_t y = pack2(y0, y1);
    const uint64_t t = fma2(y, pack2(inv, inv), mul2(y, pack2(inv_low, inv_low)));
    float e0, e1;
    unpack2(add2(t, pack2(12582912.0f, 12582912.0f)), e0, e1);   // 1.5 * 2^23: nearest integer, ties to even
    b0 = __float_as_uint(e0) & 0xffu;
    b1 = __float_as_uint(e1) & 0xffu;
  }
};

// Asks the vectors v0 .. v0 + vecs of x and residual into L2, one request per 128-byte line.
template <int TPR, int VPT>
__device__ __forceinline__ void prefetch_row(const RmsArgs& a, int64_t v0, int vecs, int lane) {
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * TPR;
    if (c < vecs && (lane & 7) == 0) {
      asm volatile("prefetch.global.L2 [%0];" ::"l"(a.x + v0 + c));
      if (a.residual != nullptr) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.residual + v0 + c));
    }
  }
}

template <int THREADS, int TPR, int VPT, bool MX>
__global__ void __launch_bounds__(THREADS, 768 / THREADS)
rmsnorm_residual_kernel(const RmsArgs a) {
  __shared__ float red[2][THREADS / 32];
  constexpr int RPC = THREADS / TPR;
  const int slot = threadIdx.x / TPR;
  const int lane = threadIdx.x % TPR;
  uint4 wt[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * TPR;
    wt[i] = c < a.cvec ? __ldg(a.weight + c) : make_uint4(0, 0, 0, 0);
  }
  // 4-bit scales come in tiles of 128 rows: the rows that fill the last tile are walked too
  const int64_t rows = MX ? (a.M + kMxTileRows - 1) / kMxTileRows * kMxTileRows : a.M;
  const int col_tiles = (a.cvec + 15) / 16;
  int turn = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * RPC; row0 < rows; row0 += (int64_t)gridDim.x * RPC) {
    const int64_t row = row0 + slot;
    const bool live = row < a.M;
    uint4 v[VPT], r[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = lane + i * TPR;
      const bool in = live && c < a.cvec;
      v[i] = in ? ldg_stream(a.x + row * a.cvec + c) : make_uint4(0, 0, 0, 0);
      r[i] = in && a.residual != nullptr ? ldg_stream(a.residual + row * a.cvec + c) : make_uint4(0, 0, 0, 0);
    }
    // The row that this slot takes next is asked into L2 now: between the loads of two rows lie two
    // dependent reductions, and what is in flight meanwhile is all that keeps memory busy (int8,
    // 4099 x 5120: 43 -> 31 us, 8192 x 16384: 277 -> 154 us).
    const int64_t next = row + (int64_t)gridDim.x * RPC;
    if (next < a.M) prefetch_row<TPR, VPT>(a, next * a.cvec, a.cvec, lane);
    uint64_t ss2[2] = {0ull, 0ull};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = lane + i * TPR;
      uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      if (a.residual != nullptr) {
        const uint32_t rw[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = bf16x2_add_rn(w[j], rw[j]);
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
        if (live && c < a.cvec) a.sum[row * a.cvec + c] = v[i];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t e = bf16x2_to_f32x2(w[j]);
        ss2[j & 1] = fma2(e, e, ss2[j & 1]);
      }
    }
    float a0, a1, b0, b1;
    unpack2(ss2[0], a0, a1);
    unpack2(ss2[1], b0, b1);
    // consecutive reductions use the two buffers in turn
    const float ss = slot_allreduce<THREADS, TPR>((a0 + a1) + (b0 + b1), red[turn], slot, SumOp());
    turn ^= 1;
    const float rstd = row_rstd(ss, a.inv_c, a.eps);
    const uint64_t rstd2 = pack2(rstd, rstd);
    float y[VPT][8];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      const uint32_t ww[4] = {wt[i].x, wt[i].y, wt[i].z, wt[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        unpack2(mul2(mul2(bf16x2_to_f32x2(w[j]), rstd2), bf16x2_to_f32x2(ww[j])), y[i][2 * j], y[i][2 * j + 1]);
      if constexpr (MX) {
        const int c = lane + i * TPR;
        // columns outside the row (and rows outside the matrix) are zeros times rstd: not NaN unless
        // rstd is one, so they are left out
        const uint32_t byte = mx_block_byte(live && c < a.cvec ? mx_absmax_halves(y[i]) : 0u);
        const uint32_t word = mx_gather_word(byte);
        if (live && c < a.cvec) reinterpret_cast<uint32_t*>(a.q)[row * a.cvec + c] = mx_quantize8(y[i], byte);
        if ((c & 15) == 0 && c < col_tiles * 16)
          *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(a.scale) +
                                       ((row / kMxTileRows) * col_tiles + c / 16) * kMxTileBytes +
                                       mx_scale_offset((int)(row % kMxTileRows), 0)) = word;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(y[i][j]) & 0x7fffffffu);
      }
    }
    if constexpr (!MX) {
      // the weight's vector of a column outside the row is zero: such columns add nothing to the
      // maximum, but for a NaN that the row's own columns have as well
      const float absmax = slot_allreduce<THREADS, TPR>(__uint_as_float(most), red[turn], slot, NanMaxOp());
      turn ^= 1;
      const Int8Scale scale(absmax);
      if (live) {
        if (lane == 0) reinterpret_cast<float*>(a.scale)[row] = scale.s;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int c = lane + i * TPR;
          if (c < a.cvec) {
            uint2 o = make_uint2(0, 0);
            if (!scale.zero_row) {
              uint32_t b[8];
#pragma unroll
              for (int j = 0; j < 8; j += 2) scale.bits2(y[i][j], y[i][j + 1], b[j], b[j + 1]);
              o.x = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
              o.y = b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24);
            }
            reinterpret_cast<uint2*>(a.q)[row * a.cvec + c] = o;
          }
        }
      }
    }
  }
}

// int8 form for widths that are no multiple of 8.  Rows then start anywhere in a 16-byte vector, but x,
// residual, sum and q all start a row at the same place in theirs, so a row is held as the aligned
// vectors that it touches: those at its two ends are shared with its neighbours and are stored
// element by element.  The weight sits differently under every row and is read from shared memory.
// Bound by instructions (a predicate and a two-byte load per element): 2.9 TB/s at 23638 x 1001 and
// 2.5 at 8192 x 4099; one CTA per row and two bytes per load reach 1.2 and 2.0.
template <int THREADS, int TPR, int VPT>
__global__ void __launch_bounds__(THREADS, 768 / THREADS)
rmsnorm_residual_quant_odd_kernel(const RmsArgs a, const __nv_bfloat16* __restrict__ weight, int C) {
  __shared__ float red[2][THREADS / 32];
  extern __shared__ __nv_bfloat16 w_s[];
  constexpr int RPC = THREADS / TPR;
  const int slot = threadIdx.x / TPR;
  const int lane = threadIdx.x % TPR;
  for (int c = threadIdx.x; c < C; c += THREADS) w_s[c] = weight[c];
  __syncthreads();
  for (int64_t row0 = (int64_t)blockIdx.x * RPC; row0 < a.M; row0 += (int64_t)gridDim.x * RPC) {
    const int64_t row = row0 + slot;
    const bool live = row < a.M;
    const int64_t start = row * C;
    const int64_t v0 = start >> 3;
    const int head = (int)(start & 7);                      // elements of the first vector that are not this row's
    const int vecs = live ? (head + C + 7) >> 3 : 0;
    // element i of vector v is column v * 8 + i - head
    uint4 v[VPT], r[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = lane + i * TPR;
      // the tensor's last vector may be a part of one: it is read element by element
      const bool whole = c < vecs && (v0 + c) * 8 + 8 <= a.M * C;
      v[i] = whole ? ldg_stream(a.x + v0 + c) : make_uint4(0, 0, 0, 0);
      r[i] = whole && a.residual != nullptr ? ldg_stream(a.residual + v0 + c) : make_uint4(0, 0, 0, 0);
      if (c < vecs && !whole) {
        uint16_t xe[8] = {}, re[8] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c * 8 + j - head < C) {
            xe[j] = reinterpret_cast<const uint16_t*>(a.x + v0 + c)[j];
            if (a.residual != nullptr) re[j] = reinterpret_cast<const uint16_t*>(a.residual + v0 + c)[j];
          }
        v[i] = make_uint4(xe[0] | xe[1] << 16, xe[2] | xe[3] << 16, xe[4] | xe[5] << 16, xe[6] | xe[7] << 16);
        r[i] = make_uint4(re[0] | re[1] << 16, re[2] | re[3] << 16, re[4] | re[5] << 16, re[6] | re[7] << 16);
      }
    }
    const int64_t next = row + (int64_t)gridDim.x * RPC;
    if (next < a.M) prefetch_row<TPR, VPT>(a, (next * C) >> 3, C >> 3, lane);
    float y[VPT][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = lane + i * TPR;
      const bool inner = c * 8 >= head && c * 8 + 8 - head <= C;   // all eight elements are this row's
      uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      if (a.residual != nullptr) {
        const uint32_t rw[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = bf16x2_add_rn(w[j], rw[j]);
        if (c < vecs) {
          if (inner) {
            a.sum[v0 + c] = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int col = c * 8 + j - head;
              if (col >= 0 && col < C) reinterpret_cast<uint16_t*>(a.sum + v0 + c)[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int col = c * 8 + j - head;
        const float e = (j & 1) ? bf16hi_to_f32(w[j >> 1]) : bf16lo_to_f32(w[j >> 1]);
        y[i][j] = c < vecs && col >= 0 && col < C ? e : 0.f;
        ss = fmaf(y[i][j], y[i][j], ss);
      }
    }
    ss = slot_allreduce<THREADS, TPR>(ss, red[0], slot, SumOp());
    const float rstd = row_rstd(ss, a.inv_c, a.eps);
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int col = (lane + i * TPR) * 8 + j - head;
        const float w = col >= 0 && col < C ? __bfloat162float(w_s[col]) : 0.f;
        y[i][j] = y[i][j] * rstd * w;
        most = max(most, __float_as_uint(y[i][j]) & 0x7fffffffu);
      }
    const float absmax = slot_allreduce<THREADS, TPR>(__uint_as_float(most), red[1], slot, NanMaxOp());
    const Int8Scale by(absmax);
    if (!live) continue;
    if (lane == 0) reinterpret_cast<float*>(a.scale)[row] = by.s;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = lane + i * TPR;
      if (c >= vecs) break;
      uint32_t b[8] = {};
      if (!by.zero_row) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) by.bits2(y[i][j], y[i][j + 1], b[j], b[j + 1]);
      }
      uint2* dst = reinterpret_cast<uint2*>(a.q) + v0 + c;
      if (c * 8 >= head && c * 8 + 8 - head <= C) {
        *dst = make_uint2(b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24), b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = c * 8 + j - head;
          if (col >= 0 && col < C) reinterpret_cast<uint8_t*>(dst)[j] = (uint8_t)b[j];
        }
      }
    }
  }
}

// int8 form for any width and alignment: one CTA per row, which is read three times (the second and
// third time from L2).
__global__ void __launch_bounds__(kThreads)
rmsnorm_residual_quant_generic_kernel(const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ residual,
                                      const __nv_bfloat16* __restrict__ weight, __nv_bfloat16* __restrict__ sum,
                                      int8_t* __restrict__ q, float* __restrict__ scale, int64_t M, int64_t C,
                                      Reciprocal inv_c, float eps) {
  __shared__ float red[2][kThreads / 32];
  for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
    const int64_t at = row * C;
    auto value = [&](int64_t c) {
      const __nv_bfloat16 v = x[at + c];
      return residual != nullptr ? __bfloat162float(__hadd_rn(v, residual[at + c])) : __bfloat162float(v);
    };
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < C; c += kThreads) {
      const float v = value(c);
      if (residual != nullptr) sum[at + c] = __float2bfloat16_rn(v);
      ss = fmaf(v, v, ss);
    }
    ss = slot_allreduce<kThreads, kThreads>(ss, red[0], 0, SumOp());
    const float rstd = row_rstd(ss, inv_c, eps);
    uint32_t most = 0;
    for (int64_t c = threadIdx.x; c < C; c += kThreads)
      most = max(most, __float_as_uint(value(c) * rstd * __bfloat162float(weight[c])) & 0x7fffffffu);
    const float absmax = slot_allreduce<kThreads, kThreads>(__uint_as_float(most), red[1], 0, NanMaxOp());
    const Int8Scale by(absmax);
    if (threadIdx.x == 0) scale[row] = by.s;
    for (int64_t c = threadIdx.x; c < C; c += kThreads) {
      uint32_t bits = 0, other;
      if (!by.zero_row) by.bits2(value(c) * rstd * __bfloat162float(weight[c]), 0.f, bits, other);
      q[at + c] = (int8_t)bits;
    }
  }
}

}  // namespace

int launch_rmsnorm_residual(const void* x, const void* residual, const void* weight, void* sum, void* q, void* scale,
                            int64_t M, int64_t C, float eps, bool mx, cudaStream_t stream) {
  const bool aligned = aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(sum) &&
                       (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
  const bool vector = C % 8 == 0 && C <= 16384 && aligned;
  if (!vector && !(aligned && !mx && C <= 16376)) {
    if (mx) return fail(B2_NOT_WHITELISTED, "rmsnorm_residual_mxfp4: C=%lld exceeds 16384", (long long)C);
    const int64_t cap = (int64_t)kNumSMsB200 * 8;
    rmsnorm_residual_quant_generic_kernel<<<(unsigned)(M < cap ? M : cap), kThreads, 0, stream>>>(
        (const __nv_bfloat16*)x, (const __nv_bfloat16*)residual, (const __nv_bfloat16*)weight, (__nv_bfloat16*)sum,
        (int8_t*)q, (float*)scale, M, C, Reciprocal((double)C), eps);
    return check_launch("rmsnorm_residual_quant");
  }
  RmsArgs a;
  a.x = (const uint4*)x;
  a.residual = (const uint4*)residual;
  a.weight = (const uint4*)weight;
  a.sum = (uint4*)sum;
  a.q = q;
  a.scale = scale;
  a.M = M;
  a.cvec = (int)(C / 8);
  a.inv_c = Reciprocal((double)C);
  a.eps = eps;
  if (!vector) {
#define B2_RMS_ODD(THREADS, TPR, VPT)                                                                            \
  do {                                                                                                           \
    const int64_t need = (M + THREADS / TPR - 1) / (THREADS / TPR);                                              \
    const int64_t cap = (int64_t)kNumSMsB200 * 1024 / THREADS;                                                   \
    rmsnorm_residual_quant_odd_kernel<THREADS, TPR, VPT>                                                         \
        <<<(unsigned)(need < cap ? need : cap), THREADS, (size_t)C * 2, stream>>>(a, (const __nv_bfloat16*)weight, (int)C); \
  } while (0)
    // a row may touch one vector more than its width fills, besides the one that it fills in part
    const int64_t vecs = (C + 14) / 8;
    if (vecs <= 32) B2_RMS_ODD(256, 32, 1);
    else if (vecs <= 64) B2_RMS_ODD(256, 32, 2);
    else if (vecs <= 128) B2_RMS_ODD(256, 64, 2);
    else if (vecs <= 256) B2_RMS_ODD(256, 128, 2);
    else if (vecs <= 512) B2_RMS_ODD(256, 256, 2);
    else if (vecs <= 1024) B2_RMS_ODD(256, 256, 4);
    else B2_RMS_ODD(512, 512, 4);
#undef B2_RMS_ODD
    return check_launch("rmsnorm_residual_quant");
  }
  const int64_t rows = mx ? (M + kMxTileRows - 1) / kMxTileRows * kMxTileRows : M;
#define B2_RMS(THREADS, TPR, VPT)                                                            \
  do {                                                                                       \
    const int64_t need = (rows + THREADS / TPR - 1) / (THREADS / TPR);                       \
    const int64_t cap = (int64_t)kNumSMsB200 * 2048 / THREADS;                               \
    const unsigned g = (unsigned)(need < cap ? need : cap);                                  \
    if (mx)                                                                                  \
      rmsnorm_residual_kernel<THREADS, TPR, VPT, true><<<g, THREADS, 0, stream>>>(a);        \
    else                                                                                     \
      rmsnorm_residual_kernel<THREADS, TPR, VPT, false><<<g, THREADS, 0, stream>>>(a);       \
  } while (0)
  // Two vectors per thread up to 4096 columns (against four: int8 at 23638 x 1024 36 -> 35 us, MXFP4
  // at 50000 x 2048 131 -> 115 us), where they do not fill a row's threads badly; above, as few
  // threads as keep a row in registers (8192 columns: 256 threads x 4 82 us, 512 x 2 107 us).
  if (C <= 256) B2_RMS(256, 32, 1);
  else if (C <= 512) B2_RMS(256, 32, 2);
  else if (C <= 1024) B2_RMS(256, 64, 2);
  else if (C <= 2048) B2_RMS(256, 128, 2);
  else if (C <= 3072) B2_RMS(256, 128, 3);
  else if (C <= 4096) B2_RMS(256, 256, 2);
  else if (C <= 6144) B2_RMS(256, 256, 3);
  else if (C <= 8192) B2_RMS(256, 256, 4);
  else B2_RMS(512, 512, 4);
#undef B2_RMS
  return check_launch("rmsnorm_residual");
}

}  // namespace b2
