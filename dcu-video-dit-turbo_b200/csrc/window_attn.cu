// bf16 attention with a sliding window and a few first keys that stay visible, for sm_100a: shared
// key heads, queries that sit at the end of a longer key sequence (a cache), per-sequence lengths.
//
// Query i of a sequence with n keys sits at p = i + n - Sq and sees the keys j < n with
//   j <= p + right   and   (j >= p - left  or  j < sinks)
// (left, right < 0: no limit on that side).  A query that sees nothing gives zeros.
//
// The mathematics is flash_fwd.cu's (exp2-domain running softmax in fp32, a fixed share of the
// exponentials on the FMA pipe, rescaling only when the running maximum grows by more than 2^8);
// flash_common.cuh holds the shared pieces.  What differs:
//
//   rows      Query heads that share a key head are packed with the positions, row r = i * pack + head,
//             so a CTA's rows read one set of keys and span few positions.
//   keys      A CTA walks only the 128-key tiles that some row of it sees: the tiles of the first
//             keys, then those of its window.  Scores are masked in the tiles that some row does
//             not see whole ("mixed"); the others take flash_fwd.cu's path.
//   P         Weights are rounded to bf16 for P . V (the tensor core wants both operands of V's type): a relative
//             error of at most 2^-8 each, independent from key to key, so a row is off by about as much as
//             by the rounding of its output (0.0023 relative with both, 0.0017 with the output's alone).
//             Sums, maxima and O stay in fp32.
//   values    0 * NaN is NaN, so a value that a row must not see may not meet its zero weight in a
//             product: the two otherwise idle warps look through every mixed tile, clear the rows
//             at or past n (a cache's unwritten part) and set non-finite values to zero.  Those of
//             visible keys are added back to the rows that see them at the end (a path that only
//             runs if there were any).
//   tiles     window_tile_kernel: two tiles of up to 128 rows per work item.  A CTA that has finished
//             its item takes over one that has not started (cluster launch control), so loads, first
//             scores and set-up of the next item run under the output of the last: windows are a
//             dozen steps long, and starting a CTA costs three.
//   few rows  window_few_kernel, at most 128 rows per key head (single tokens): the two tiles become
//             two streams over the same rows, stream 0 takes the even tiles of keys and stream 1 the
//             odd ones.
//   splits    Where that leaves SMs empty the keys are split over CTAs.  Parts (maximum, sum, unnormalised
//             output of each row) are joined in the shared memory of a cluster, or, when there are
//             many, through memory by a second kernel.
//
// Bound by the tensor cores (4 * 128 FLOP per visible pair and head) when many rows share the keys,
// by reading K and V once for single tokens.  Measured: 24 heads x 23638, window 3344 each way, 836 first
// keys 1.82 to 1.93 ms over five GPUs, 1.10 PFLOP/s over the visible pairs at 1.83; a step of 256 rows x
// 128 keys takes 1.77 us, of which the tensor cores work 1.1: a tile's chain scores -> maximum ->
// exponentials -> P -> product -> next scores is what it waits for.  24 heads x 8192, window 511: 92 to 116
// us over these, a fifth of it the items' output.
// 8 x 6 key heads, single tokens, 4224 keys each: 104 MB in 25 us, of which 8 are set-up, first loads and
// the join.
#include "flash_common.cuh"
#include "sm100_pair.cuh"

namespace b2 {

unsigned int read_clear_status_window() { return read_and_clear_device_status(); }

namespace {

using namespace flash;

// Registers per thread of the softmax and the service warps (setmaxnreg; see flash_common.cuh for what
// bounds them).  The work loop of window_tile_kernel's service warps spills below 56 (216 / 72 takes 3 %
// less time than 232 / 40 over a clip of 23638 tokens).
constexpr int TILE_REGS_SOFTMAX = 216, TILE_REGS_SERVICE = 72;
constexpr int FEW_REGS_SOFTMAX = 232, FEW_REGS_SERVICE = 40;
static_assert(2 * TILE_REGS_SOFTMAX + TILE_REGS_SERVICE <= 3 * kLaunchRegs && 2 * FEW_REGS_SOFTMAX + FEW_REGS_SERVICE <= 3 * kLaunchRegs,
              "register split exceeds the CTA's launch allocation");
// Shared memory: Q, the K ring, the V ring, rows on their way out, barriers.  The few-row form has one tile
// of Q and a third stage in its place, and none of the rows.
template <bool FEW>
struct WinSmem {
  static constexpr int STAGES = FEW ? 3 : 2;
  static constexpr int Q = 0;
  static constexpr int K = Q + (FEW ? 1 : 2) * TILE_BYTES;
  static constexpr int V = K + STAGES * TILE_BYTES;
  static constexpr int OUT = V + STAGES * TILE_BYTES;            // rows on their way out, 4 KB per softmax warp
  static constexpr int NEXT = OUT + (FEW ? 0 : kSoftmaxWarps * 4096);   // answers of the work scheduler (2 x 16)
  static constexpr int BARS = NEXT + 32;
  // barriers; [stage] or [tile], P by part and tile
  static constexpr int QF = 0, SF = 2, OF = 4;                   // Q, S, O are there
  static constexpr int OE = 6, QE = 8;                           // O has been read / Q has been used
  static constexpr int NF = 9, NE = 11;                          // the next item is known / has been read
  static constexpr int PF = 13;
  static constexpr int KF = PF + 2 * P_PARTS, KE = KF + STAGES;  // K is there / has been used
  static constexpr int VF = KE + STAGES, VE = VF + STAGES;
  static constexpr int VC = VE + STAGES;                         // a mixed tile's values are cleared
  static constexpr int NUM = VC + STAGES;
  static constexpr int TOTAL = 1024 + BARS + NUM * 8 + 16;
  static_assert(TOTAL <= 227 * 1024, "shared memory budget");
  static_assert(OE == OF + 2 && QE == OE + 2 && NF == QE + 1 && NE == NF + 2 && PF == NE + 2, "barriers follow one another");
  // joining the parts of a cluster: each CTA's rows in the place of Q, K and V
  static constexpr int PITCH = HEAD_DIM + 4;                     // floats: rows start 4 banks apart
  static constexpr int ML = 2 * BLOCK_M * PITCH * 4;
  static_assert(ML + 2 * BLOCK_M * 8 <= NEXT, "the rows to join take the place of the operands");
};
constexpr int kFixWarp = 10, kFixThreads = 64;
constexpr int kMaxCluster = 8;                // CTAs that join their parts through shared memory

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// n / d for 0 <= n < 2^31 by a multiplication.  With shift = 31 + s, d <= 2^s, and mul = ceil(2^shift / d):
// mul * d = 2^shift + e, 0 <= e < d, and n * e < 2^31 * 2^s = 2^shift, so the quotient is exact.  Every role of
// every CTA decodes its work items: against divisions 1 to 3 % less time with short windows.
struct Divisor {
  uint32_t mul, shift;
};
__device__ __forceinline__ int quotient(int n, const Divisor& d) { return (int)(((uint64_t)(uint32_t)n * d.mul) >> d.shift); }
Divisor make_divisor(int64_t d) {
  uint32_t s = 0;
  while ((int64_t(1) << s) < d) ++s;
  return {(uint32_t)(((uint64_t(1) << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d), 31 + s};
}

struct WinArgs {
  __nv_bfloat16* out;           // [B, Sq, H, 128]
  int join;                     // the cluster's CTAs join their parts
  float* part_o;                // [parts][B * Sq * H][128]: parts for window_join_kernel, or null
  float2* part_ml;              // [parts][B * Sq * H]: (maximum in the exp2 domain, sum)
  const __nv_bfloat16* q;
  const __nv_bfloat16* v;       // for the non-finite path
  const int* lengths;           // keys per sequence, null: Sk
  int64_t q_b, q_h, q_s, v_b, v_h, v_s;   // strides in elements
  int H, share, groups, Sq, Sk;           // share = H / Hkv, groups = H / pack
  int together, last, chunks;             // row groups whose items are in order; in the last chunk; chunks
  int ascending;                          // the first positions see the most keys
  Divisor by_splits, by_chunk, by_together, by_last, by_groups, by_share;
  int pack, tile_pos, blocks;             // heads per row group; positions per tile; work items along positions
  int left, right, sinks, splits;
  int64_t total_rows;                     // B * Sq * H
  int k_swap, v_swap;
  float scale_log2;
};

// Items come in order of position, those that see the most keys first (the last of a causal call), over
// `together` row groups (heads and sequences) at a time, at least four rounds of the SMs: these run out of
// work on short items.  Row group after row group leaves SMs idle at the end; all row groups together
// read so many keys at a time that long calls lose in the steady state.  One after the other / all / so:
// 24 heads x 8192 causal 460 / 407 / 397 us; 2 x 24 heads on 8 key heads x 4099, window 1023, 144 / 132 / 126;
// 24 x 23638, window 3344 each way, 1940 / 2005 / 1932; causal 3161 / 3194 / 3117.  Without a limit on either
// side all positions see the same keys, and row groups follow one another: 24 x 8192 797 us, all 835.
// One work item: positions [pos0, pos0 + CTA positions) of `pack` heads from h0, a share of their keys.
struct Item {
  int split, block, h0, hkv, b;
};
__device__ __forceinline__ Item decode_item(const WinArgs& a, int index) {
  Item it;
  const int rest = quotient(index, a.by_splits);
  it.split = index - rest * a.splits;
  const int chunk = quotient(rest, a.by_chunk), in = rest - chunk * a.together * a.blocks;
  const bool last = chunk == a.chunks - 1;
  const int row = quotient(in, last ? a.by_last : a.by_together);
  const int heads = chunk * a.together + in - row * (last ? a.last : a.together);
  it.block = a.ascending ? row : a.blocks - 1 - row;
  it.b = quotient(heads, a.by_groups);
  it.h0 = (heads - it.b * a.groups) * a.pack;
  it.hkv = quotient(it.h0, a.by_share);
  return it;
}

// What a CTA reads: the same numbers in every role.
struct Span {
  int n;                     // keys of this sequence
  int lo_full, hi_full;      // every row sees every key of [lo_full, hi_full] (and those before `sinks`)
  int steps;                 // this CTA's share of the key tiles
  int first, sink_steps, win;   // step j starts at key first + 128 j while j < sink_steps, at win + 128 j from there
};

__device__ __forceinline__ int sequence_keys(const int* lengths, int b, int Sk) {
  return lengths == nullptr ? Sk : min(max(lengths[b], 0), Sk);
}
// j <= p + right with no limit for right < 0; positions and limits stay below 2^31 (checked by the
// entry point), the sum may not
__device__ __forceinline__ int last_key(int p, int right, int n) {
  return right < 0 ? n - 1 : (int)min((int64_t)p + right, (int64_t)n - 1);
}
__device__ __forceinline__ int first_key(int p, int left) {
  return left < 0 ? 0 : max((int)max((int64_t)p - left, (int64_t)-1), 0);
}

// positions: of the item's rows, the first at pos0
__device__ __forceinline__ Span make_span(const WinArgs& a, int pos0, int positions, int b, int split) {
  Span s;
  s.n = sequence_keys(a.lengths, b, a.Sk);
  const int p_min = pos0 + s.n - a.Sq;
  const int p_max = min(pos0 + positions, a.Sq) - 1 + s.n - a.Sq;
  s.lo_full = first_key(p_max, a.left);
  s.hi_full = last_key(p_min, a.right, s.n);
  const int end = last_key(p_max, a.right, s.n) + 1;             // <= 0: nothing is visible
  int total = 0, sink_tiles = 0, win0 = 0;
  if (end > 0) {
    // Tiles of the window start at its first key, not at a multiple of 128 (which would take two
    // thirds of a tile more on average), behind the tiles of the first keys where those reach into it.
    const int begin = first_key(p_min, a.left);
    sink_tiles = (min(min(a.sinks, begin), end) + BLOCK_N - 1) / BLOCK_N;
    win0 = max(begin, sink_tiles * BLOCK_N);
    total = sink_tiles + max(end - win0 + BLOCK_N - 1, 0) / BLOCK_N;
  }
  const int step0 = quotient(total * split, a.by_splits);   // tiles of 128 keys times at most 64 splits: below 2^31
  s.steps = quotient(total * (split + 1), a.by_splits) - step0;
  s.first = step0 * BLOCK_N;
  s.sink_steps = sink_tiles - step0;
  s.win = win0 + (step0 - sink_tiles) * BLOCK_N;
  return s;
}
// first key of the CTA's step j
__device__ __forceinline__ int step_key(const Span& s, int j) {
  return (j < s.sink_steps ? s.first : s.win) + j * BLOCK_N;
}
// some row of the CTA does not see the whole tile
__device__ __forceinline__ bool is_mixed(const WinArgs& a, const Span& s, int key0) {
  return key0 + BLOCK_N - 1 > s.hi_full || (key0 < s.lo_full && key0 + BLOCK_N > a.sinks);
}
__device__ __forceinline__ bool sees_any(const WinArgs& a, int p, int n) {
  const int last = last_key(p, a.right, n);
  return last >= 0 && (last >= first_key(p, a.left) || a.sinks > 0);
}

constexpr uint32_t kIdescQK = make_idesc(/*f32*/ 1, /*bf16*/ 1, /*bf16*/ 1, 0, 0, BLOCK_M, BLOCK_N);
constexpr uint32_t kIdescPV = make_idesc(1, 1, 1, 0, /*B MN-major*/ 1, BLOCK_M, HEAD_DIM);

__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row0, int h,
                                          int b, int swap) {
  mbar_expect_tx(bar, TILE_BYTES);
  if (swap) {
    tma_load_4d(dst, map, bar, 0, h, row0, b);
    tma_load_4d(dst + HALF_BYTES, map, bar, 64, h, row0, b);
  } else {
    tma_load_4d(dst, map, bar, 0, row0, h, b);
    tma_load_4d(dst + HALF_BYTES, map, bar, 64, row0, h, b);
  }
}

// one tile of Q: positions pos0.. of `pack` heads (positions past the sequence arrive as zeros)
__device__ __forceinline__ void load_q(uint32_t dst, const CUtensorMap* map, uint32_t bar, const WinArgs& a, int pos0,
                                       int h0, int b) {
  mbar_expect_tx(bar, (uint32_t)(a.pack * a.tile_pos) * HEAD_DIM * 2);
  tma_load_4d(dst, map, bar, 0, h0, pos0, b);
  tma_load_4d(dst + HALF_BYTES, map, bar, 64, h0, pos0, b);
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t max_bits4(uint32_t m, const uint4& v) {
  m = __vmaxu2(m, v.x & 0x7fff7fffu);
  m = __vmaxu2(m, v.y & 0x7fff7fffu);
  m = __vmaxu2(m, v.z & 0x7fff7fffu);
  return __vmaxu2(m, v.w & 0x7fff7fffu);
}
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
  const uint32_t lo = (w & 0x7f80u) == 0x7f80u ? 0u : 0xffffu, hi = (w & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u;
  return w & (lo | hi);
}

// A mixed tile of values: rows at or past `valid` become zeros, non-finite values become zeros;
// returns whether a row before `valid` held one.  64 threads, one 128-byte line half at a time.
__device__ __forceinline__ bool clean_values(uint32_t tile, int valid, int ft) {
  bool found = false;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    // thread ft owns lines ft and ft + 64 of the half tile; the order of the 16-byte chunks differs
    // from thread to thread so that the eight lanes of a phase touch different banks
#pragma unroll 1
    for (int l = 0; l < 2; ++l) {
      const int row = ft + 64 * l;
      const uint32_t line = tile + half * HALF_BYTES + row * 128;
      if (row >= valid) {
#pragma unroll
        for (int c = 0; c < 8; ++c) sts128(line + ((c ^ (row & 7)) << 4), make_uint4(0, 0, 0, 0));
        continue;
      }
      uint32_t m = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) m = max_bits4(m, lds128(line + ((c ^ (row & 7)) << 4)));
      if ((m & 0xffffu) >= 0x7f80u || (m >> 16) >= 0x7f80u) {
        found = true;
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          uint4 v = lds128(line + (c << 4));
          v.x = finite_or_zero(v.x);
          v.y = finite_or_zero(v.y);
          v.z = finite_or_zero(v.z);
          v.w = finite_or_zero(v.w);
          sts128(line + (c << 4), v);
        }
      }
    }
  }
  return found;
}

// Bits 0 .. n-1 of a word (all for n >= 32, none for n <= 0).
__device__ __forceinline__ uint32_t columns_below(int n) {
  return n <= 0 ? 0u : 0xffffffffu >> (32 - min(n, 32));
}

// What the sum of a row's parts says about the row: its multiplier, 0 for a row that sees nothing, NaN
// where the formula has 0 / 0 (keys in sight whose scores are all -inf) or a NaN.
__device__ __forceinline__ float row_inverse(const WinArgs& a, float l, int p, int n) {
  if (l == 0.f) return sees_any(a, p, n) ? __uint_as_float(0x7fc00000u) : 0.0f;
  return 1.0f / l;
}
// Joins parts one by one: weights 2^(m - max m).  The first pass finds the maximum.
struct PartSum {
  float top = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(const float2& ml, const float4& x) {
    if (ml.x == -INFINITY && ml.y == 0.f) return;   // this part saw nothing
    const float w = exp2f(ml.x - top);
    l = fmaf(w, ml.y, l);
    o.x = fmaf(w, x.x, o.x);
    o.y = fmaf(w, x.y, o.y);
    o.z = fmaf(w, x.z, o.z);
    o.w = fmaf(w, x.w, o.w);
  }
  __device__ __forceinline__ uint2 row(float inv) const {
    return make_uint2(pack_bf16x2_rn(o.x * inv, o.y * inv), pack_bf16x2_rn(o.z * inv, o.w * inv));
  }
};

// What one softmax thread knows of its row.
struct Row {
  int key_first, key_last;             // visible: these, those between and the first keys
  bool live;                           // a row of the tensor: others hold anything and must not cause a rescaling
  float top = -INFINITY, sum = 0.f;    // running maximum of the raw scores, sum of the exponentials
  __device__ __forceinline__ Row(const WinArgs& a, int position, int n, bool exists)
      : key_first(first_key(position, a.left)), key_last(last_key(position, a.right, n)), live(exists) {}
};

// One of eight score pairs takes its exponential on the FMA pipe (two in flash_fwd.cu): with masks and
// work items around the steps the softmax warps are short of issue slots before the exp2 unit is full.
// One against two: 0.7 to 2.8 % less time over windows from 511 to whole sequences; none loses 2 % on
// the long ones, three 6 %.
constexpr int WIN_EMU_MASK = 0x02;

// One step of one tile: scores from tensor memory -> masked -> P in their place, O rescaled if the
// maximum grew (`rescale` is false on the row's first step, when O holds nothing).  `publish(part)`
// hands a half of P to the MMA issuer.
template <class Publish>
__device__ __forceinline__ void softmax_step(Row& row, uint32_t s_tmem, uint32_t o_tmem, float sl2, int sinks, int key0,
                                             bool rescale, int lane, Publish publish) {
  {
    // visible columns: [first, last] and those before `sink`
    const int last = row.key_last - key0, first = row.key_first - key0, sink = sinks - key0;
    if (__builtin_expect(__any_sync(0xffffffffu, last < BLOCK_N - 1 || (first > 0 && sink < BLOCK_N)), 0)) {
      // A bit per visible column, 32 at a time: testing constant bits of a word costs a third of three
      // comparisons per score.  The masked scores go back to tensor memory: a short loop apart from the
      // path that every step takes, against 128 more selects in it, takes 1 to 3 % less time (more with
      // short windows), whole sequences included: the warps of both tiles run out of the instruction caches.
      // A tile that no row of the warp sees (a step is the CTA's, its last rows see other keys than its
      // first) has P = 0 and leaves the exp2 unit to the other warps: 2 to 6 % with windows up to 511.
      if (__all_sync(0xffffffffu, last < 0 || (first >= BLOCK_N && sink <= 0))) {
        const uint32_t zero[16] = {};
#pragma unroll
        for (int c = 0; c < 64; c += 16) tmem_st_32x32b_x16(s_tmem + c, zero);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          publish(0);
          publish(1);
        }
        return;
      }
      // from the first column that some row of the warp does not see to the last
      const int lo = __reduce_min_sync(0xffffffffu, min(first > 0 ? max(sink, 0) : 128, last + 1));
      const int hi = __any_sync(0xffffffffu, last < BLOCK_N - 1) ? 128 : __reduce_max_sync(0xffffffffu, first);
#pragma unroll 1
      for (int c = max(lo, 0) & ~31; c < min(hi, 128); c += 32) {
        const uint32_t seen = columns_below(last + 1 - c) & (~columns_below(first - c) | columns_below(sink - c));
        uint32_t x[32];
        tmem_ld_32x32b_x32(s_tmem + c, x);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!(seen & (1u << i))) x[i] = 0xff800000u;   // -inf
        tmem_st_32x32b_x16(s_tmem + c, *reinterpret_cast<uint32_t(*)[16]>(&x[0]));
        tmem_st_32x32b_x16(s_tmem + c + 16, *reinterpret_cast<uint32_t(*)[16]>(&x[16]));
      }
      tmem_wait_st();
    }
  }
  uint32_t s[128];
#pragma unroll
  for (int c = 0; c < 128; c += 32) tmem_ld_32x32b_x32(s_tmem + c, *reinterpret_cast<uint32_t(*)[32]>(&s[c]));
  tmem_wait_ld();
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 128; c += 2)
    mx[(c >> 1) & 3] = fmax3(mx[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
  const float m_row = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  const bool raise = row.live && (m_row - row.top) * sl2 > 8.0f;   // false while both are -inf (NaN)
  // a row that had seen nothing has added zeros to O so far (its values were cleared): nothing to rescale
  const bool correct = raise && rescale && row.top != -INFINITY;
  float alpha = 1.0f;
  if (raise) {
    alpha = ex2_approx((row.top - m_row) * sl2);
    row.top = m_row;
    row.sum *= alpha;
  }
  __syncwarp();
  if (__any_sync(0xffffffffu, correct)) {
#pragma unroll 1
    for (int c = 0; c < 128; c += 16) {
      uint32_t o[16];
      tmem_ld_32x32b_x16(o_tmem + c, o);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
      tmem_st_32x32b_x16(o_tmem + c, o);
    }
  }
  // a row that has seen nothing yet has only -inf scores: exp2(-inf - 0) = 0
  const float neg_ms = row.top == -INFINITY ? 0.0f : -row.top * sl2;
  const uint64_t sl2x2 = pack2(sl2, sl2), nmsx2 = pack2(neg_ms, neg_ms);
  uint64_t sm2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    uint32_t p[8];
    exp_chunk<WIN_EMU_MASK>(&s[16 * q], p, sl2x2, nmsx2, sm2);
    tmem_st_32x32b_x8(s_tmem + 8 * q, p);   // P takes the first half of S
    if ((q + 1) % 4 == 0) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) publish(q / 4);
    }
  }
  float a0, a1, b0, b1, c0, c1, d0, d1;
  unpack2(sm2[0], a0, a1);
  unpack2(sm2[1], b0, b1);
  unpack2(sm2[2], c0, c1);
  unpack2(sm2[3], d0, d1);
  row.sum += ((a0 + a1) + (b0 + b1)) + ((c0 + c1) + (d0 + d1));
}
static_assert(P_PARTS == 2, "P is published in halves");

// Adds the non-finite values that the fix warps took out of the mixed tiles to a stored row (in fp32, or in
// bf16 where it is final: an infinity or a NaN is the same there) that sees them: the steps first,
// first + stride, ... of the item.
__device__ __forceinline__ void add_nonfinite(const WinArgs& a, const Span& span, const Row& row, int first, int stride,
                                              int steps, int hkv, int b, float* part, __nv_bfloat16* out) {
#pragma unroll 1
  for (int u = first; u < steps; u += stride) {
    const int key0 = step_key(span, u);
    if (!is_mixed(a, span, key0)) continue;
#pragma unroll 1
    for (int j = key0; j < key0 + BLOCK_N && j <= row.key_last; ++j) {
      if (j < row.key_first && j >= a.sinks) continue;
      const __nv_bfloat16* src = a.v + b * a.v_b + hkv * a.v_h + (int64_t)j * a.v_s;
#pragma unroll 1
      for (int c = 0; c < HEAD_DIM; ++c) {
        const float x = __bfloat162float(src[c]);
        if (fabsf(x) <= 3.4e38f) continue;
        if (part != nullptr)
          part[c] += x;
        else
          out[c] = __float2bfloat16_rn(__bfloat162float(out[c]) + x);
      }
    }
  }
}
__device__ __forceinline__ void store_f32(float* dst, const uint32_t (&o)[32]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    reinterpret_cast<uint4*>(dst)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
}
__device__ __forceinline__ void store_bf16(__nv_bfloat16* dst, const uint32_t (&o)[32], float inv) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 w;
    w.x = pack_bf16x2_rn(__uint_as_float(o[8 * i + 0]) * inv, __uint_as_float(o[8 * i + 1]) * inv);
    w.y = pack_bf16x2_rn(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv);
    w.z = pack_bf16x2_rn(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv);
    w.w = pack_bf16x2_rn(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv);
    reinterpret_cast<uint4*>(dst)[i] = w;
  }
}

// The join of a cluster's parts: every CTA holds (slot) rows in shared memory; a warp takes a row, a
// lane four columns, and the rows go round the CTAs.  PARTS slots of a CTA belong to one row.
// row_of(r) gives the position and head of row r.
template <class L, int PARTS, class RowOf>
__device__ __forceinline__ void join_cluster(const WinArgs& a, uint32_t sbase, int warp, int lane, int split, int b, int n,
                                             int nrows, RowOf row_of) {
  for (int r = warp * a.splits + split; r < nrows; r += kSoftmaxWarps * a.splits) {
    int pos, head;
    if (!row_of(r, pos, head)) continue;
    PartSum sum;
    // lane p has part p's maximum and sum (at most 16 parts)
    const int parts = PARTS * a.splits;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < parts) ml = ld_cluster_f2(map_to_cta(sbase + L::ML + (lane % PARTS * BLOCK_M + r) * 8, lane / PARTS));
    sum.top = ml.x;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sum.top = fmaxf(sum.top, __shfl_xor_sync(0xffffffffu, sum.top, off));
    sum.top = __shfl_sync(0xffffffffu, sum.top, 0);
    const bool any_nan = __any_sync(0xffffffffu, ml.y != ml.y);
#pragma unroll 1
    for (int p0 = 0; p0 < parts; p0 += 4) {
      float4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (p0 + i < parts)
          x[i] = ld_cluster_f4(map_to_cta(sbase + (((p0 + i) % PARTS * BLOCK_M + r) * L::PITCH + lane * 4) * 4, (p0 + i) / PARTS));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (p0 + i < parts)
          sum.add(make_float2(__shfl_sync(0xffffffffu, ml.x, p0 + i), __shfl_sync(0xffffffffu, ml.y, p0 + i)), x[i]);
    }
    const float inv = any_nan ? __uint_as_float(0x7fc00000u) : row_inverse(a, sum.l, pos + n - a.Sq, n);
    reinterpret_cast<uint2*>(a.out + (((int64_t)b * a.Sq + pos) * a.H + head) * HEAD_DIM)[lane] = sum.row(inv);
  }
}

// The work scheduler: a running CTA takes the place of one that has not been launched yet.
__device__ __forceinline__ void ask_next(uint32_t answer, uint32_t bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer),
               "r"(bar)
               : "memory");
}
// index of the block taken over, -1 when there was none left
__device__ __forceinline__ int read_next(uint32_t answer) {
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(answer)
      : "memory");
  return got ? (int)x : -1;
}

__global__ void __launch_bounds__(NUM_THREADS, 1)
window_tile_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ WinArgs args) {
  using L = WinSmem<false>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::NUM);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // Set when a mixed tile held a non-finite value and never cleared: the path that it opens looks for
  // itself and adds nothing where there is nothing.
  volatile int* nonfinite = abort_flag + 1;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int idx) -> uint32_t { return bar0 + idx * 8; };
  auto wait = [&](int idx, uint32_t parity) -> bool { return mbar_wait(bar0 + idx * 8, parity & 1, abort_flag, kStatusFlashTimeout); };
  auto wait_warp = [&](int idx, uint32_t parity) -> bool { return mbar_wait_warp(bar0 + idx * 8, parity & 1, abort_flag, kStatusFlashTimeout); };
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const bool more = args.join == 0;   // a cluster's CTAs do one item

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::NUM; ++i) {
      int count = 1;
      if (i == L::OE || i == L::OE + 1 || (i >= L::PF && i < L::KF)) count = 4;   // the tile's four warps
      if (i == L::NE || i == L::NE + 1) count = kSoftmaxWarps + 4;                // every warp that asks
      if (i >= L::VE && i < L::VC) count = 1 + kFixThreads / 32;                  // MMAs done, looked through
      if (i >= L::VC) count = kFixThreads;
      mbar_init(bar(i), count);
    }
    *abort_flag = 0;
    *nonfinite = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  const int tile_rows = args.tile_pos * args.pack;
  if (tile_rows < BLOCK_M) {   // rows that no load of Q reaches: zeros, like those past the sequence
    for (int i = threadIdx.x; i < 4 * (BLOCK_M - tile_rows) * 8; i += NUM_THREADS)
      sts128(sbase + L::Q + (i & 3) * HALF_BYTES + (tile_rows + (i >> 5)) * 128 + ((i >> 2) & 7) * 16, make_uint4(0, 0, 0, 0));
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int item_pos = 2 * args.tile_pos;

  // The item after `fetch` others, or -1: for one lane of the warps that load and issue, for whole warps.
  auto next_item = [&](int fetch, auto wait_for) -> int {
    if (!more) return -1;
    const int slot = fetch & 1;
    if (!wait_for(L::NF + slot, fetch >> 1)) return -1;
    const int next = read_next(sbase + L::NEXT + slot * 16);
    fence_proxy_async_smem();   // read before the scheduler writes there again
    return next;
  };

  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TILE_REGS_SERVICE));
    if (warp == kLoadWarp) {
      if (lane == 0) {
        int index = blockIdx.x, g = 0, full_items = 0;
        bool ok = true;
        for (int fetch = 0; ok && index >= 0; ++fetch) {
          const Item it = decode_item(args, index);
          const int pos0 = it.block * item_pos;
          const Span span = make_span(args, pos0, item_pos, it.b, it.split);
          // The next item is asked for with two steps to go: early enough to load it without a pause,
          // late enough that no CTA holds an item back while another has nothing to do.
          auto ask = [&]() -> bool {
            const int slot = fetch & 1;
            if (!wait(L::NE + slot, (fetch >> 1) ^ 1)) return false;   // its last answer has been read by every warp
            ask_next(sbase + L::NEXT + slot * 16, bar(L::NF + slot));
            return true;
          };
          if (more && span.steps == 0) ok = ask();
          for (int j = 0; ok && j < span.steps; ++j) {
            const int st = (g + j) & 1;
            const uint32_t use = (uint32_t)(g + j) >> 1;
            const int key0 = step_key(span, j);
            if (!(ok = wait(L::KE + st, use ^ 1))) break;
            if (more && j == max(0, span.steps - 2) && !(ok = ask())) break;
            load_tile(sbase + L::K + st * TILE_BYTES, &tmap_k, bar(L::KF + st), key0, it.hkv, it.b, args.k_swap);
            if (j == 0) {
              // Q once the last item's scores are all computed
              if (!(ok = wait(L::QE, full_items ^ 1))) break;
              for (int t = 0; t < 2; ++t) load_q(sbase + L::Q + t * TILE_BYTES, &tmap_q, bar(L::QF + t), args, pos0 + t * args.tile_pos, it.h0, it.b);
            }
            if (!(ok = wait(L::VE + st, use ^ 1))) break;
            load_tile(sbase + L::V + st * TILE_BYTES, &tmap_v, bar(L::VF + st), key0, it.hkv, it.b, args.v_swap);
          }
          g += span.steps;
          full_items += span.steps > 0;
          if (!ok) break;
          index = next_item(fetch, wait);
          if (more) mbar_arrive(bar(L::NE + (fetch & 1)));
        }
      }
    } else if (warp >= kFixWarp) {
      const int ft = threadIdx.x - kFixWarp * 32;
      int index = blockIdx.x, g = 0;
      bool ok = true;
      for (int fetch = 0; ok && index >= 0; ++fetch) {
        const Item it = decode_item(args, index);
        const Span span = make_span(args, it.block * item_pos, item_pos, it.b, it.split);
        // every step is waited for and released, mixed or not: these warps can neither run ahead of
        // the ring by a whole phase nor fall behind it by one
        for (int j = 0; ok && j < span.steps; ++j) {
          const int key0 = step_key(span, j);
          const int st = (g + j) & 1;
          if (!(ok = wait_warp(L::VF + st, (uint32_t)(g + j) >> 1))) break;
          if (is_mixed(args, span, key0)) {
            if (clean_values(sbase + L::V + st * TILE_BYTES, span.n - key0, ft)) *nonfinite = 1;
            fence_proxy_async_smem();
            mbar_arrive(bar(L::VC + st));
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(L::VE + st));
        }
        g += span.steps;
        if (!ok) break;
        index = next_item(fetch, wait_warp);
        __syncwarp();
        if (more && lane == 0) mbar_arrive(bar(L::NE + (fetch & 1)));
      }
    } else if (elect_one() != 0) {
      // One lane does it all: a lane that only waits could fall behind by a phase of a barrier.
      const uint32_t s0 = tmem_base + COL_S0, o0 = tmem_base + COL_O0;   // tile 1: 128 columns on
      const uint32_t q0 = desc_lo(sbase + L::Q, 16);
      const uint32_t k0 = desc_lo(sbase + L::K, 16);
      const uint32_t v0 = desc_lo(sbase + L::V, HALF_BYTES);
      constexpr uint32_t TILE_UNITS = TILE_BYTES >> 4;
      uint32_t clean_phase = 0;   // bit per stage
      int index = blockIdx.x, g = 0, full_items = 0;
      bool ok = true;
      // S of tile t = Q . K^T of the stage's keys
      auto issue_qk = [&](int t, int st) {
        mma_f16_ss_kmajor_x8(s0 + t * 128, q0 + t * TILE_UNITS, k0 + st * TILE_UNITS, kIdescQK);
        tc_commit(bar(L::SF + t));
      };
      // O of tile t += P . V, each half of P as soon as it is published; `step` counts over all items
      auto issue_pv = [&](int t, int step, bool first) -> bool {
        const int st = step & 1;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (!wait(L::PF + 2 * part + t, step)) return false;
          tc_fence_after();
          if (part == 0)
            mma_f16_ts_seq<0, 4>(o0 + t * 128, s0 + t * 128, v0 + st * TILE_UNITS, kIdescPV, first ? 0u : 1u);
          else
            mma_f16_ts_seq<4, 4>(o0 + t * 128, s0 + t * 128, v0 + st * TILE_UNITS, kIdescPV, 1u);
        }
        return true;
      };
      for (int fetch = 0; ok && index >= 0; ++fetch) {
        const Item it = decode_item(args, index);
        const Span span = make_span(args, it.block * item_pos, item_pos, it.b, it.split);
        const int steps = span.steps;
        // the step's values are there, and cleared if the tile is mixed
        auto wait_v = [&](int j) -> bool {
          const int st = (g + j) & 1;
          if (!wait(L::VF + st, (uint32_t)(g + j) >> 1)) return false;
          if (is_mixed(args, span, step_key(span, j))) {
            if (!wait(L::VC + st, clean_phase >> st)) return false;
            clean_phase ^= 1u << st;
          }
          return true;
        };
        auto wait_k = [&](int j) -> bool {
          if (!wait(L::KF + ((g + j) & 1), (uint32_t)(g + j) >> 1)) return false;
          tc_fence_after();
          return true;
        };
        if (steps > 0) {
          if (!(ok = wait_k(0) && wait(L::QF, full_items))) break;
          tc_fence_after();
          issue_qk(0, g & 1);
          if (!(ok = wait(L::QF + 1, full_items))) break;
          tc_fence_after();
          issue_qk(1, g & 1);
          tc_commit(bar(L::KE + (g & 1)));
          if (steps == 1) tc_commit(bar(L::QE));
          // the softmax warps have read the last item's O
          if (full_items > 0 && !(ok = wait(L::OE, full_items - 1) && wait(L::OE + 1, full_items - 1))) break;
          if (!(ok = wait_v(0))) break;
          for (int j = 0; j < steps; ++j) {
            const int st = (g + j) & 1;
            const bool last = j + 1 == steps;
            if (!(ok = issue_pv(0, g + j, j == 0))) break;
            if (last) {
              tc_commit(bar(L::OF));
            } else {
              if (!(ok = wait_k(j + 1))) break;
              issue_qk(0, st ^ 1);
            }
            if (!(ok = issue_pv(1, g + j, j == 0))) break;
            tc_commit(bar(L::VE + st));
            if (last) {
              tc_commit(bar(L::OF + 1));
            } else {
              // the next step's values, waited for while this step's MMAs are still queued
              if (!(ok = wait_v(j + 1))) break;
              issue_qk(1, st ^ 1);
              tc_commit(bar(L::KE + (st ^ 1)));
              if (j + 2 == steps) tc_commit(bar(L::QE));
            }
          }
          if (!ok) break;
          g += steps;
          ++full_items;
        }
        index = next_item(fetch, wait);
        if (more) mbar_arrive(bar(L::NE + (fetch & 1)));
      }
    }
    if (args.join) {   // the softmax warps' two meetings
      __syncwarp();
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TILE_REGS_SOFTMAX));
    const int t = warp >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int row_pos = min(r, tile_rows - 1) / args.pack;          // position within the tile, and head
    const int row_head = min(r, tile_rows - 1) - row_pos * args.pack;
    const uint32_t lane_sel = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tmem = tmem_base + COL_S0 + t * 128 + lane_sel;
    const uint32_t o_tmem = tmem_base + COL_O0 + t * 128 + lane_sel;
    const uint32_t out_stage = sbase + L::OUT + warp * 4096;
    int index = blockIdx.x, g = 0, full_items = 0;
    bool ok = true;
    for (int fetch = 0; index >= 0; ++fetch) {
      const Item it = decode_item(args, index);
      const int pos0 = it.block * item_pos;
      const Span span = make_span(args, pos0, item_pos, it.b, it.split);
      const int steps = span.steps;
      const int pos = pos0 + t * args.tile_pos + row_pos;
      const bool row_ok = r < tile_rows && pos < args.Sq;
      const bool warp_ok = __any_sync(0xffffffffu, row_ok);
      Row row(args, min(pos, args.Sq - 1) + span.n - args.Sq, span.n, row_ok);
      for (int u = 0; u < steps; ++u) {
        if (ok) ok = wait(L::SF + t, g + u);
        tc_fence_after();
        if (!warp_ok) {   // none of the warp's rows exist: whatever P holds there goes nowhere
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bar(L::PF + t));
            mbar_arrive(bar(L::PF + 2 + t));
          }
          continue;
        }
        softmax_step(row, s_tmem, o_tmem, args.scale_log2, args.sinks, step_key(span, u), u != 0, lane,
                     [&](int part) { mbar_arrive(bar(L::PF + 2 * part + t)); });
      }
      g += steps;
      if (ok && steps > 0) ok = wait(L::OF + t, full_items);
      // the rows to join take the operands' place: no MMA of the other tile may still read them
      if (ok && args.join && steps > 0) ok = wait(L::OF + (t ^ 1), full_items);
      ok = __all_sync(0xffffffffu, ok);   // the warp goes on as one
      tc_fence_after();
      const bool parts = args.part_o != nullptr;
      const int64_t out_row = ((int64_t)it.b * args.Sq + min(pos, args.Sq - 1)) * args.H + it.h0 + row_head;
      if (ok && warp_ok) {
        const float inv = row.sum != row.sum ? 1.0f : row_inverse(args, row.sum, min(pos, args.Sq - 1) + span.n - args.Sq, span.n);
        const int slot = t * BLOCK_M + r;
        // where the row's part goes, null: the row is final
        float* part = args.join ? reinterpret_cast<float*>(smem) + slot * L::PITCH
                      : parts ? args.part_o + (it.split * args.total_rows + out_row) * HEAD_DIM
                              : nullptr;
        if (row_ok) {
          const float2 ml = make_float2(row.top * args.scale_log2, row.sum);
          if (args.join)
            reinterpret_cast<float2*>(smem + L::ML)[slot] = ml;
          else if (parts)
            args.part_ml[it.split * args.total_rows + out_row] = ml;
        }
        __syncwarp();
        const int64_t row0 = ((int64_t)it.b * args.Sq + pos0 + t * args.tile_pos) * args.H + it.h0;
        // Rows leave through 4 KB of shared memory per warp, 128 bytes of each at a time: a thread holds
        // a row, a store takes four (written from the registers, each 16 bytes of a warp are 32 lines of
        // L1, one per clock).  Short loops: straight code of this length spends its time on fetching
        // instructions, with the other tile's softmax in the same caches.
        const int rel = row_ok ? row_pos * args.H + row_head : -1;
        char* dst = (parts ? reinterpret_cast<char*>(args.part_o + (it.split * args.total_rows + row0) * HEAD_DIM)
                           : reinterpret_cast<char*>(args.out + row0 * HEAD_DIM)) + (lane & 7) * 16;
        const int pitch = parts ? HEAD_DIM * 4 : HEAD_DIM * 2;
        const uint32_t line = out_stage + lane * 128;
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t o[32];
          if (steps > 0) {
            tmem_ld_32x32b_x32(o_tmem + c, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
          if (c == 96 && steps > 0) {   // O is in registers: the next item's may be written
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(L::OE + t));
          }
          bool full = !args.join;
          if (part != nullptr) {
            const uint32_t to = full ? line : sbase + (t * BLOCK_M + r) * L::PITCH * 4 + c * 4;
            const uint32_t swz = full ? lane & 7 : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sts128(to + ((i ^ swz) << 4), make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sts128(line + ((((c >> 3) & 7) + i) ^ (lane & 7)) * 16,
                     make_uint4(pack_bf16x2_rn(__uint_as_float(o[8 * i + 0]) * inv, __uint_as_float(o[8 * i + 1]) * inv),
                                pack_bf16x2_rn(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv),
                                pack_bf16x2_rn(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv),
                                pack_bf16x2_rn(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv)));
            full = (c & 32) != 0;
          }
          __syncwarp();
          if (full) {
#pragma unroll 1
            for (int i = 0; i < 8; i += 2) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int src = 4 * (i + k) + (lane >> 3);
                const uint4 v = lds128(out_stage + src * 128 + (((lane & 7) ^ (src & 7)) << 4));
                const int to = __shfl_sync(0xffffffffu, rel, src);
                if (to >= 0) *reinterpret_cast<uint4*>(dst + (int64_t)to * pitch) = v;
              }
            }
            dst += 128;
            __syncwarp();   // the next columns take their place
          }
        }
        if (*nonfinite != 0 && row_ok)
          add_nonfinite(args, span, row, 0, 1, steps, it.hkv, it.b, part, args.out + out_row * HEAD_DIM);
        __syncwarp();
      } else if (steps > 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::OE + t));
      }
      full_items += steps > 0;
      if (args.join) {
        __syncwarp();
        cluster_sync_all();   // every CTA's rows are in its shared memory
        join_cluster<L, 1>(args, sbase, warp, lane, it.split, it.b, span.n, 2 * BLOCK_M, [&](int rr, int& p, int& h) {
          const int tt = rr / BLOCK_M, in = rr % BLOCK_M;
          const int rp = in / args.pack;
          p = pos0 + tt * args.tile_pos + rp;
          h = it.h0 + in - rp * args.pack;
          return in < tile_rows && p < args.Sq;
        });
        __syncwarp();
        cluster_sync_all();   // no CTA retires while another reads its rows
      }
      index = ok ? next_item(fetch, wait_warp) : -1;
      __syncwarp();
      if (more && lane == 0) mbar_arrive(bar(L::NE + (fetch & 1)));
    }
  }

  __syncwarp();
  if (*abort_flag != 0) {
    const long long t0 = clock64();
    while (clock64() - t0 < 200000) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// At most 128 rows per key head: the two tiles are two streams over the same rows.
__global__ void __launch_bounds__(NUM_THREADS, 1)
window_few_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                  const __grid_constant__ WinArgs args) {
  using L = WinSmem<true>;
  constexpr int STAGES = L::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::NUM);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* nonfinite = abort_flag + 1;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int idx) -> uint32_t { return bar0 + idx * 8; };
  auto wait = [&](int idx, uint32_t parity) -> bool { return mbar_wait(bar0 + idx * 8, parity & 1, abort_flag, kStatusFlashTimeout); };
  auto wait_warp = [&](int idx, uint32_t parity) -> bool { return mbar_wait_warp(bar0 + idx * 8, parity & 1, abort_flag, kStatusFlashTimeout); };
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  const Item it = decode_item(args, blockIdx.x);
  const Span span = make_span(args, 0, args.Sq, it.b, it.split);
  const int steps = span.steps;
  const int rows = args.Sq * args.pack;

  // Loads first: the ring's first stages as soon as the barriers exist, Q into registers, so that
  // memory works while tensor memory is allocated and the warps meet.
  auto start_k = [&](int j) {
    const int st = j % STAGES;
    load_tile(sbase + L::K + st * TILE_BYTES, &tmap_k, bar(L::KF + st), step_key(span, j), it.hkv, it.b, args.k_swap);
  };
  auto start_v = [&](int j) {
    const int st = j % STAGES;
    load_tile(sbase + L::V + st * TILE_BYTES, &tmap_v, bar(L::VF + st), step_key(span, j), it.hkv, it.b, args.v_swap);
  };
  if (threadIdx.x == kLoadWarp * 32) {
    for (int i = 0; i < L::NUM; ++i) {
      int count = 1;
      if (i == L::QF || (i >= L::PF && i < L::KF)) count = 4;            // the tile's four warps
      if (i >= L::VE && i < L::VC) count = 1 + kFixThreads / 32;         // MMAs done, looked through
      if (i >= L::VC) count = kFixThreads;
      mbar_init(bar(i), count);
    }
    *abort_flag = 0;
    *nonfinite = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int j = 0; j < min(steps, STAGES); ++j) {
      start_k(j);
      start_v(j);
    }
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  // the rows of Q: 16 lanes per row, 8 rows per pass
  const int tid = threadIdx.x & 127, c16 = tid & 15;
  uint4 qv[16];
  if (warp < 4 && steps > 0) {
#pragma unroll
    for (int p = 0; p < 16; ++p) {
      if (p * 8 < rows) {
        const int r = min(p * 8 + (tid >> 4), rows - 1);
        const int i = r / args.pack, h = it.h0 + r - i * args.pack;
        qv[p] = ldg_stream(reinterpret_cast<const uint4*>(args.q + it.b * args.q_b + h * args.q_h + i * args.q_s) + c16);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Rows past the last hold a copy of it up to the pass's end, and anything behind: they go nowhere.
  if (warp < 4 && steps > 0) {
#pragma unroll
    for (int p = 0; p < 16; ++p) {
      if (p * 8 < rows) {
        const int r = p * 8 + (tid >> 4);
        sts128(sbase + L::Q + (c16 >> 3) * HALF_BYTES + r * 128 + (((c16 & 7) ^ (r & 7)) << 4), qv[p]);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(L::QF));
  }

  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW_REGS_SERVICE));
    if (warp == kLoadWarp) {
      if (lane == 0) {
        // The first stages are on their way.  A step's K is free long before its V (the streams' MMAs
        // alternate), so K runs a step ahead: behind V it would wait for the other stream's product too.
        auto load_k = [&](int j) -> bool {
          if (!wait(L::KE + j % STAGES, (j / STAGES) ^ 1)) return false;
          start_k(j);
          return true;
        };
        bool ok = steps <= STAGES || load_k(STAGES);
        for (int j = STAGES; ok && j < steps; ++j) {
          ok = (j + 1 >= steps || load_k(j + 1)) && wait(L::VE + j % STAGES, (j / STAGES) ^ 1);
          if (ok) start_v(j);
        }
      }
    } else if (warp >= kFixWarp) {
      const int ft = threadIdx.x - kFixWarp * 32;
      for (int j = 0; j < steps; ++j) {   // every step, as in window_tile_kernel
        const int key0 = step_key(span, j);
        const int st = j % STAGES;
        if (!wait_warp(L::VF + st, j / STAGES)) break;
        if (is_mixed(args, span, key0)) {
          if (clean_values(sbase + L::V + st * TILE_BYTES, span.n - key0, ft)) *nonfinite = 1;
          fence_proxy_async_smem();
          mbar_arrive(bar(L::VC + st));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::VE + st));
      }
    } else if (steps > 0 && elect_one() != 0) {   // one lane, as in window_tile_kernel
      const uint32_t s0 = tmem_base + COL_S0, o0 = tmem_base + COL_O0;   // stream 1: 128 columns on
      const uint32_t q0 = desc_lo(sbase + L::Q, 16);
      const uint32_t k0 = desc_lo(sbase + L::K, 16);
      const uint32_t v0 = desc_lo(sbase + L::V, HALF_BYTES);
      constexpr uint32_t TILE_UNITS = TILE_BYTES >> 4;
      uint32_t clean_phase = 0;   // bit per stage
      // S of step j in stream j & 1
      auto issue_qk = [&](int j) -> bool {
        const int st = j % STAGES, t = j & 1;
        if (!wait(L::KF + st, j / STAGES)) return false;
        tc_fence_after();
        mma_f16_ss_kmajor_x8(s0 + t * 128, q0, k0 + st * TILE_UNITS, kIdescQK);
        tc_commit(bar(L::SF + t));
        tc_commit(bar(L::KE + st));
        return true;
      };
      bool ok = wait(L::QF, 0) && issue_qk(0) && (steps == 1 || issue_qk(1));
      for (int j = 0; ok && j < steps; ++j) {
        const int st = j % STAGES, t = j & 1;
        if (!(ok = wait(L::VF + st, j / STAGES))) break;
        if (is_mixed(args, span, step_key(span, j))) {
          if (!(ok = wait(L::VC + st, clean_phase >> st))) break;
          clean_phase ^= 1u << st;
        }
        if (!(ok = wait(L::PF + t, j >> 1))) break;
        tc_fence_after();
        mma_f16_ts_seq<0, 4>(o0 + t * 128, s0 + t * 128, v0 + st * TILE_UNITS, kIdescPV, j > 1 ? 1u : 0u);
        if (!(ok = wait(L::PF + 2 + t, j >> 1))) break;
        tc_fence_after();
        mma_f16_ts_seq<4, 4>(o0 + t * 128, s0 + t * 128, v0 + st * TILE_UNITS, kIdescPV, 1u);
        tc_commit(bar(L::VE + st));
        if (j + 2 < steps)
          ok = issue_qk(j + 2);
        else
          tc_commit(bar(L::OF + t));
      }
    }
    if (args.join) {   // the softmax warps' two meetings
      __syncwarp();
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FEW_REGS_SOFTMAX));
    const int t = warp >> 2;
    const int quarter = warp & 3;
    const int uses = (steps + 1 - t) >> 1;   // steps of this stream
    const int r = quarter * 32 + lane;
    const bool row_ok = r < rows;
    const bool warp_ok = quarter * 32 < rows;
    const int pos = min(r, rows - 1) / args.pack;
    const int head = it.h0 + min(r, rows - 1) - pos * args.pack;
    Row row(args, pos + span.n - args.Sq, span.n, row_ok);
    const uint32_t lane_sel = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tmem = tmem_base + COL_S0 + t * 128 + lane_sel;
    const uint32_t o_tmem = tmem_base + COL_O0 + t * 128 + lane_sel;
    bool ok = true;
    for (int u = 0; u < uses; ++u) {
      if (ok) ok = wait(L::SF + t, u);
      tc_fence_after();
      if (!warp_ok) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(L::PF + t));
          mbar_arrive(bar(L::PF + 2 + t));
        }
        continue;
      }
      softmax_step(row, s_tmem, o_tmem, args.scale_log2, args.sinks, step_key(span, 2 * u + t), u != 0, lane,
                   [&](int part) { mbar_arrive(bar(L::PF + 2 * part + t)); });
    }
    if (ok && uses > 0) ok = wait(L::OF + t, 0);
    // the rows to join take the operands' place: no MMA of the other stream may still read them
    if (ok && args.join && ((steps + t) >> 1) > 0) ok = wait(L::OF + (t ^ 1), 0);
    ok = __all_sync(0xffffffffu, ok);   // the warp goes on as one
    tc_fence_after();
    const bool parts = args.part_o != nullptr;
    // with nothing to join there is a single step, which is stream 0's
    if (ok && warp_ok && (t == 0 || parts || args.join)) {
      const int64_t out_row = ((int64_t)it.b * args.Sq + pos) * args.H + head;
      const int64_t part_row = (2 * it.split + t) * args.total_rows + out_row;
      const float inv = row.sum != row.sum ? 1.0f : row_inverse(args, row.sum, pos + span.n - args.Sq, span.n);
      const int slot = t * BLOCK_M + r;
      float* part = args.join ? reinterpret_cast<float*>(smem) + slot * L::PITCH
                    : parts ? args.part_o + part_row * HEAD_DIM
                            : nullptr;
      if (row_ok) {
        const float2 ml = make_float2(row.top * args.scale_log2, row.sum);
        if (args.join)
          reinterpret_cast<float2*>(smem + L::ML)[slot] = ml;
        else if (parts)
          args.part_ml[part_row] = ml;
      }
      __syncwarp();
#pragma unroll 1
      for (int c = 0; c < 128; c += 32) {
        uint32_t o[32];
        if (uses > 0) {
          tmem_ld_32x32b_x32(o_tmem + c, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (row_ok) {
          if (part != nullptr)
            store_f32(part + c, o);
          else
            store_bf16(args.out + out_row * HEAD_DIM + c, o, inv);
        }
        __syncwarp();   // the next columns are loaded by the whole warp
      }
      if (*nonfinite != 0 && row_ok)
        add_nonfinite(args, span, row, t, 2, steps, it.hkv, it.b, part, args.out + out_row * HEAD_DIM);
      __syncwarp();
    }
    if (args.join) {
      __syncwarp();
      cluster_sync_all();   // every CTA's rows are in its shared memory
      join_cluster<L, 2>(args, sbase, warp, lane, it.split, it.b, span.n, rows, [&](int rr, int& p, int& h) {
        p = rr / args.pack;
        h = it.h0 + rr - p * args.pack;
        return true;
      });
      __syncwarp();
      cluster_sync_all();   // no CTA retires while another reads its rows
    }
  }

  __syncwarp();
  if (*abort_flag != 0) {
    const long long t0 = clock64();
    while (clock64() - t0 < 200000) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Joins the parts that lie in memory: WARPS warps per row, four columns per lane.  Four parts at a time:
// their loads are under way together, the first four's under the search for the maximum (one at a
// time and one warp per row, 128 parts of a single row took 39 us more).
template <int WARPS>
__global__ void __launch_bounds__(256)
window_join_kernel(const WinArgs args, int parts) {
  __shared__ float4 sums[WARPS][32];
  __shared__ float ls[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = WARPS > 1 ? warp * 4 : 0;   // this warp's parts: first .. first + 3, and so on
  const int64_t row = WARPS > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
  if (row >= args.total_rows) return;
  const float2* ml = args.part_ml + row;
  const float4* o = reinterpret_cast<const float4*>(args.part_o) + row * (HEAD_DIM / 4) + lane;
  float2 w[4];
  float4 x[4];
  auto load = [&](int p0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = min(p0 + i, parts - 1);
      w[i] = ml[p * args.total_rows];
      x[i] = o[p * args.total_rows * (HEAD_DIM / 4)];
    }
  };
  load(first);
  PartSum sum;
  bool any_nan = false;
  for (int p = lane; p < parts; p += 32) {
    const float2 v = ml[p * args.total_rows];
    sum.top = fmaxf(sum.top, v.x);
    any_nan |= v.y != v.y;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum.top = fmaxf(sum.top, __shfl_xor_sync(0xffffffffu, sum.top, off));
  any_nan = __any_sync(0xffffffffu, any_nan);
#pragma unroll 1
  for (int p0 = first; p0 < parts;) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p0 + i < parts) sum.add(w[i], x[i]);
    p0 += 4 * WARPS;
    if (p0 < parts) load(p0);
  }
  if (WARPS > 1) {
    sums[warp][lane] = sum.o;
    if (lane == 0) ls[warp] = sum.l;
    __syncthreads();
    if (warp > 0) return;
    for (int i = 1; i < WARPS; ++i) {
      const float4 v = sums[i][lane];
      sum.l += ls[i];
      sum.o.x += v.x;
      sum.o.y += v.y;
      sum.o.z += v.z;
      sum.o.w += v.w;
    }
  }
  const int64_t bi = row / args.H;
  const int b = (int)(bi / args.Sq), i = (int)(bi - (int64_t)b * args.Sq);
  const int n = sequence_keys(args.lengths, b, args.Sk);
  const float inv = any_nan ? __uint_as_float(0x7fc00000u) : row_inverse(args, sum.l, i + n - args.Sq, n);
  reinterpret_cast<uint2*>(args.out + row * HEAD_DIM)[lane] = sum.row(inv);
}

// How a call is laid over the GPU: few-row form or not, splits of the key sequence, parts to join.
struct WinPlan {
  bool few, join;
  int pack, tile_pos;          // heads per row group, positions per tile
  int blocks, splits, parts;   // parts: to be joined by window_join_kernel (1: none)
};
WinPlan make_plan(int B, int H, int Hkv, int Sq, int Sk, int left, int right, int sinks) {
  WinPlan p;
  const int share = H / Hkv;
  const int64_t rows = (int64_t)Sq * share;
  p.few = rows <= BLOCK_M;
  // Heads per row group: as many of those that share a key head as fill seven eighths of a tile's 128
  // rows (fewer positions per item see fewer keys in vain: 2 x 24 heads x 4099, three to a key
  // head, window 1023: 126 rows in threes 158 us, 128 rows of one head 180 us).
  p.pack = share;
  if (!p.few) {
    p.pack = 1;
    for (int d = 2; d <= share && d <= BLOCK_M; ++d)
      if (share % d == 0 && BLOCK_M / d * d >= 112) p.pack = d;
  }
  p.tile_pos = p.few ? Sq : BLOCK_M / p.pack;
  p.blocks = p.few ? 1 : (Sq + 2 * p.tile_pos - 1) / (2 * p.tile_pos);
  // the most 128-key steps that a CTA can have: its positions, the window around them, the first
  // keys; one more for a window that starts inside a tile
  const int64_t positions = min((int64_t)Sq, (int64_t)(p.few ? 1 : 2) * p.tile_pos);
  int64_t keys = Sk;
  if (left >= 0 && right >= 0) keys = min(keys, (int64_t)left + right + positions);
  int64_t steps = (keys + BLOCK_N - 1) / BLOCK_N + (keys < Sk ? 1 : 0);
  if (left >= 0) steps += (min(sinks, Sk) + BLOCK_N - 1) / BLOCK_N;
  steps = max((int64_t)1, min(steps, ((int64_t)Sk + BLOCK_N - 1) / BLOCK_N));
  // One CTA runs per SM, so a grid takes rounds of (its steps + a fixed part: set-up, first loads,
  // output).  The figures are microseconds measured on a B200 with 24, 48 and 96 CTAs before
  // splitting: a few-row step takes 0.83 alone and what 64 KB per CTA take from memory when many run; a
  // full step 1.85.  A cluster joins its parts for one (few rows) or nine (256 rows), but leaves
  // SMs without a place; parts in memory take a second kernel and 1040 bytes per row and part, there
  // and back.  24 heads' single tokens over 8192 keys: 65.5 us unsplit, 32.7 in clusters of four, 33.9 in
  // four parts through memory; 24 x 300 rows over 8192 keys: 121 unsplit, 84 in clusters of two, 78.8 in
  // two parts through memory, 62.5 in three; 2 heads x 700 over 16384: 49 in clusters of eight, 36 in 24 parts.
  constexpr int kSlots[kMaxCluster + 1] = {0, 148, 148, 135, 132, 130, 132, 105, 120};
  const int64_t ctas = (int64_t)p.blocks * (H / p.pack) * B;
  double best = 1e30;
  p.splits = 1;
  p.join = false;
  auto consider = [&](int s, bool cluster) {
    const int64_t n = ctas * s, slots = cluster ? kSlots[s] : kNumSMsB200;
    const double rounds = (double)((n + slots - 1) / slots);
    const double running = (double)(n < slots ? n : slots);
    const double step = p.few ? (running * 0.0109 > 0.83 ? running * 0.0109 : 0.83) : 1.85;
    double cost = rounds * ((double)steps / s * step + (p.few ? 8.0 : 5.0));
    if (cluster && (s > 1 || p.few)) cost += p.few ? 1.0 : 9.0 * rounds;
    if (!cluster) cost += 6.0 + 2.1e-4 * (double)((int64_t)Sq * H * B) * s * (p.few ? 2 : 1);
    if (cost < best) {
      best = cost;
      p.splits = s;
      p.join = cluster;
    }
  };
  for (int s = 1; s <= 64 && s <= steps; ++s) {
    if (s <= kMaxCluster) consider(s, true);
    if (s > 1) consider(s, false);
  }
  p.parts = p.join ? 1 : p.splits * (p.few ? 2 : 1);
  // nothing to join: whole rows of one CTA, or a few-row call of one step (its second stream has none)
  if (p.join && p.splits == 1 && (!p.few || steps == 1)) p.join = false;
  return p;
}

// Q as (channel, head, position, batch): a box is `pack` heads of `positions` positions, which lands
// as rows position * pack + head.
int encode_q_map(CUtensorMap* map, const void* base, int B, int H, int S, const int64_t* st, int pack, int positions) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return fail(B2_LAUNCH_FAILED, "window_fwd: cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[4] = {HEAD_DIM, (cuuint64_t)H, (cuuint64_t)S, (cuuint64_t)B};
  const cuuint64_t strides[3] = {(cuuint64_t)st[1] * 2, (cuuint64_t)st[2] * 2, (cuuint64_t)st[0] * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)pack, (cuuint32_t)positions, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B2_LAUNCH_FAILED, "window_fwd: tensor map encode failed (%d)", (int)r);
  return B2_OK;
}

}  // namespace

int64_t window_fwd_workspace_bytes(int B, int H, int Hkv, int Sq, int Sk, int left, int right, int sinks) {
  const WinPlan p = make_plan(B, H, Hkv, Sq, Sk, left, right, sinks);
  return p.parts == 1 ? 0 : (int64_t)p.parts * B * H * Sq * (HEAD_DIM * 4 + 8);
}

int launch_window_fwd(const void* q, const void* k, const void* v, void* out, void* workspace, const int* lengths,
                      int B, int H, int Hkv, int Sq, int Sk, const int64_t* qs, const int64_t* ks, const int64_t* vs,
                      float scale, int left, int right, int sinks, cudaStream_t stream) {
  static PerDeviceSetup per_device;
  const DeviceSlot* slot = nullptr;
  const int setup_status = per_device.get("window_fwd", [](int, DeviceSlot&) -> int {
    const void* kernels[2] = {(const void*)window_tile_kernel, (const void*)window_few_kernel};
    const int split[2] = {2 * TILE_REGS_SOFTMAX + TILE_REGS_SERVICE, 2 * FEW_REGS_SOFTMAX + FEW_REGS_SERVICE};
    const int bytes[2] = {WinSmem<false>::TOTAL, WinSmem<true>::TOTAL};
    for (int i = 0; i < 2; ++i) {
      const void* f = kernels[i];
      cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes[i]);
      if (e != cudaSuccess) return fail(B2_LAUNCH_FAILED, "window_fwd: smem attribute: %s", cudaGetErrorString(e));
      cudaFuncAttributes fa;
      e = cudaFuncGetAttributes(&fa, f);
      if (e != cudaSuccess) return fail(B2_LAUNCH_FAILED, "window_fwd: attributes: %s", cudaGetErrorString(e));
      if (split[i] > 3 * ((fa.numRegs + 7) / 8 * 8))
        return fail(B2_LAUNCH_FAILED, "window_fwd: a register split of %d does not fit %d launch registers", split[i], fa.numRegs);
    }
    return B2_OK;
  }, &slot);
  if (setup_status != B2_OK) return setup_status;
  const WinPlan plan = make_plan(B, H, Hkv, Sq, Sk, left, right, sinks);
  const int64_t items = (int64_t)plan.blocks * plan.splits * (H / plan.pack) * B;
  if (items > 0x7fffffffLL) return fail(B2_TOO_LARGE, "window_fwd: too many work items");
  CUtensorMap tq, tk, tv;
  WinArgs a;
  int st = encode_qkv_map(&tk, k, B, Hkv, Sk, ks, &a.k_swap);
  if (st != B2_OK) return st;
  st = encode_qkv_map(&tv, v, B, Hkv, Sk, vs, &a.v_swap);
  if (st != B2_OK) return st;
  if (!plan.few) {
    st = encode_q_map(&tq, q, B, H, Sq, qs, plan.pack, plan.tile_pos);
    if (st != B2_OK) return st;
  }
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.total_rows = (int64_t)B * Sq * H;
  a.join = plan.join ? 1 : 0;
  a.part_o = plan.parts == 1 ? nullptr : reinterpret_cast<float*>(workspace);
  a.part_ml = plan.parts == 1 ? nullptr : reinterpret_cast<float2*>(a.part_o + plan.parts * a.total_rows * HEAD_DIM);
  a.q = reinterpret_cast<const __nv_bfloat16*>(q);
  a.v = reinterpret_cast<const __nv_bfloat16*>(v);
  a.lengths = lengths;
  a.q_b = qs[0];
  a.q_h = qs[1];
  a.q_s = qs[2];
  a.v_b = vs[0];
  a.v_h = vs[1];
  a.v_s = vs[2];
  const int64_t all = (int64_t)(H / plan.pack) * B;
  const int64_t least = left < 0 && right < 0 ? 1 : (4 * kNumSMsB200 + plan.blocks - 1) / plan.blocks;
  const int64_t chunks = all > least ? all / least : 1, together = (all + chunks - 1) / chunks;
  a.together = (int)together;
  a.ascending = left >= 0 && right < 0 ? 1 : 0;
  a.chunks = (int)((all + together - 1) / together);
  a.last = (int)(all - (a.chunks - 1) * together);
  a.groups = H / plan.pack;
  a.by_splits = make_divisor(plan.splits);
  a.by_chunk = make_divisor(together * plan.blocks);
  a.by_together = make_divisor(together);
  a.by_last = make_divisor(a.last);
  a.by_groups = make_divisor(a.groups);
  a.by_share = make_divisor(H / Hkv);
  a.H = H;
  a.share = H / Hkv;
  a.Sq = Sq;
  a.Sk = Sk;
  a.pack = plan.pack;
  a.tile_pos = plan.tile_pos;
  a.blocks = plan.blocks;
  a.left = left;
  a.right = right;
  a.sinks = left < 0 ? 0 : sinks;
  a.splits = plan.splits;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)items);
  cfg.blockDim = dim3(NUM_THREADS);
  cfg.dynamicSmemBytes = plan.few ? WinSmem<true>::TOTAL : WinSmem<false>::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = plan.join ? (unsigned)plan.splits : 1u;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = plan.few ? cudaLaunchKernelEx(&cfg, window_few_kernel, tk, tv, a)
                                 : cudaLaunchKernelEx(&cfg, window_tile_kernel, tq, tk, tv, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(B2_LAUNCH_FAILED, "window_fwd: launch failed: %s", cudaGetErrorString(e));
  }
  if (plan.parts == 1) return B2_OK;
  // a block per row where a warp would read many parts in turn
  if (plan.parts >= 16 && a.total_rows <= 8192)
    window_join_kernel<8><<<(unsigned)a.total_rows, 256, 0, stream>>>(a, plan.parts);
  else
    window_join_kernel<1><<<(unsigned)((a.total_rows + 7) / 8), 256, 0, stream>>>(a, plan.parts);
  return check_launch("window_fwd (join)");
}

}  // namespace b2
