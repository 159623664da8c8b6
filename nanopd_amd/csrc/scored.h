// Attention with changed scores over the paged pool: what its kernels share.
//
// Of query row at position p, head h, and key j of the same sequence:
//   t = scale * q.k_j;  with a cap c:  t = c * tanh(t / c);
//   with slopes:        t -= slope[h] * |p - j|
//   seen(j) = first <= j and (lo <= j <= p, or j < prefix),
//   lo = first, or with a window w the later of first and p - w + 1
//   out = sum over seen j of softmax(t)_j v_j; zeros where no key is seen.
// Scores and the running maximum are kept in log2 units (t * log2 e), sums and
// outputs in fp32; P is rounded to the 2-byte type for the P.V product, and the
// row sum adds the rounded values, so that the weights used add up to one.
//
// Partial results of a key range are (m, l, O[d]): m the exponents' reference,
// l = sum 2^(t - m), O = sum 2^(t - m) v. A range without a seen key has
// m = -inf, l = 0, O = 0. Ranges merge as M = max m, w = 2^(m - M),
// out = sum w O / sum w l.
#pragma once

#include <type_traits>

#include "common.h"

namespace npd {
namespace scored {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoRef = 3.402823466e38f;   // exponent offset of a row without a reference
constexpr int kTileRows = 128;              // rows of a workgroup of the rows kernel
// ... and how many of them run at once on a compute unit at (padded) head dim d
// (FP8 bytes pass through registers: at three, steps of 128 dims spill; 96 tokens in
// three groups take 130 us, 112 at two)
__host__ __device__ constexpr int rows_per_cu(int64_t d, bool fp8) {
  return d > 128 ? 1 : d > 64 ? (fp8 ? 2 : 3) : 4;
}
// Waves of the stream kernel on a SIMD at (padded) head dim d, by its registers.
__host__ __device__ constexpr int stream_per_simd(int64_t d, bool fp8) {
  return d > 128 ? 2 : d > 64 ? (fp8 ? 2 : 3) : (fp8 ? 4 : 3);
}
constexpr int kStepKeys = 32;               // keys per step of the rows kernel
// Shares of the rows kernel's workgroups, in steps: what a piece of a tile costs
// besides its steps, the smallest share (but for its tilt), and how near a tile's edge no cut is made.
constexpr int kTileCost = 6;
constexpr int kMinShare = 16;
constexpr int kNearEdge = 4;
constexpr int kListTiles = 512;             // most tiles per kv head that are cut into parts
constexpr int kUnitHeads = 16;              // most heads of a stream unit (MFMA columns)

// One call. Rows are (token, head) pairs of a kv head's G query heads.
struct Args {
  uint16_t* out;
  const uint16_t* q;
  const char* k_cache;
  const char* v_cache;
  const int32_t* block_tables;
  const int32_t* seq_lens;        // context lengths
  const int32_t* cu_seqlens_q;    // chunks (null: one token per sequence)
  const int32_t* first_keys;      // null: 0
  const int32_t* prefix_lens;     // null: 0
  const float* slopes;            // null: no distance term
  const float* k_scale;           // FP8 pools: per-kv-head scales
  const float* v_scale;
  const int32_t* cu_groups;       // shared prefixes: sequences of group g are
  const int32_t* shared_lens;     // cu_groups[g] .. cu_groups[g + 1] - 1
  float* tile_o;                  // partials of the rows kernel [slot][kv head][row][D]
  float* tile_ml;                 // their (m, l)
  int32_t* tile_items;            // [tile][kv head][4]: first slot, first and last workgroup
  float* unit_o;                  // partials of the stream kernel [seq][head][part][D]
  float* unit_ml;
  int num_seqs, num_groups, total_q, max_shared;
  int num_heads, num_kv_heads, group, head_dim;
  int block_size, bs_shift, num_blocks, max_bps;   // bs_shift < 0: no power of two
  int tiles;                      // rows kernel: tiles of all groups, or tiles_max of each sequence
  int tiles_max;                  // ... chunks: most tiles of one sequence
  int room;                       // ... workgroups per kv head (chunks without a list: whole tiles)
  int room1;                      // ... of them in one round over the compute units
  bool list;                      // ... that share the steps of all tiles evenly
  int cost_shift;                 // ... whose cost is counted in 2^shift steps
  int unit_splits;                // stream kernel: most parts of a unit
  int part_keys;                  // ... fewest keys of one
  float stream_waves;             // ... waves that run at once
  int subs, sub_heads;            // stream kernel: units per kv head, heads of a unit
  int window;                     // 0: none
  float scale_log2;               // scale * log2(e)
  float cap_in, cap_log2;         // cap: 2 log2(e) scale / cap, and cap * log2(e) (0: no cap)
  bool cap_wide;                  // cap past kCapPlain
  int64_t q_stride_token, q_stride_head, out_stride_token, out_stride_head;
};

// Capped score in log2 units: A tanh(y) with e^(2y) = 2^(x * cin) and A = cap *
// log2(e), as A - 2A / (1 + e^(2y)). Past the range of the exponential the
// quotient is 0 or 2A: the cap itself. The difference leaves an absolute error
// of about A * 2^-23, that of the exponential of a score at the cap; so a cap up
// to 256 needs no more. A larger one also stands for scores far below it, whose
// error should go by their own size: |y| < 1/4 takes the odd series (its first
// dropped term is below 2^-23 of y there).
constexpr float kCapPlain = 256.f;
__device__ __forceinline__ float cap_plain(float x, float cin, float A) {
  const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * cin) + 1.f);
  return fmaf(-2.f * A, r, A);
}
__device__ __forceinline__ float cap_exact(float x, float cin, float A) {
  const float y = x * cin * 0.34657359027997264f;   // ln 2 / 2
  const float z = y * y;
  float p = fmaf(z, 0.021869488536155203f, -0.053968253968253971f);
  p = fmaf(z, p, 0.13333333333333333f);
  p = fmaf(z, p, -0.33333333333333331f);
  p = fmaf(z * y, p, y);
  return fabsf(y) < 0.25f ? A * p : cap_plain(x, cin, A);
}

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// The keys a row sees: [lo, hi) and [first, pre), hi <= context.
struct alignas(16) Keys {
  int first, lo, hi, pre;
};
__device__ __forceinline__ Keys row_keys(int pos, int ctx, int first, int pre, int window) {
  Keys k{0, 0, 0, 0};
  if (pos < 0 || pos >= ctx) return k;
  k.first = first < 0 ? 0 : first;
  k.lo = window > 0 && pos - window + 1 > k.first ? pos - window + 1 : k.first;
  k.hi = pos + 1;
  if (k.lo > k.hi) k.lo = k.hi;
  k.pre = clampi(pre, 0, ctx);
  if (k.pre <= k.first) k.pre = k.first = 0;
  return k;
}

// The group of sequence s: its first sequence, shared keys and first tile of the
// rows kernel (tiles of kTileRows flattened (sequence, head) rows per group).
// Groups are taken 64 at a time, one per lane.
struct Group {
  int seq0, seqs, shared, tile0;
};
__device__ __forceinline__ Group group_at(const Args& a, int g) {
  Group r;
  r.seq0 = clampi(a.cu_groups[g], 0, a.num_seqs);
  r.seqs = clampi(a.cu_groups[g + 1], r.seq0, a.num_seqs) - r.seq0;
  r.shared = clampi(a.shared_lens[g], 0, a.max_shared);
  r.tile0 = 0;
  return r;
}
// The group that holds sequence x (its first tile of the rows kernel too). false:
// none.
__device__ __forceinline__ bool find_group(const Args& a, int x, int lane, Group& out) {
  int base = 0;
  for (int g0 = 0; g0 < a.num_groups; g0 += 64) {
    Group r{0, 0, 0, 0};
    int n = 0;
    if (g0 + lane < a.num_groups) {
      r = group_at(a, g0 + lane);
      n = (int)(((int64_t)r.seqs * a.group + kTileRows - 1) / kTileRows);
    }
    const int incl = wave_scan_i(n);
    const int t0 = base + incl - n;
    const uint64_t m = __ballot(x >= r.seq0 && x < r.seq0 + r.seqs);
    if (m != 0) {
      const int sel = __builtin_ctzll(m);
      out.seq0 = __builtin_amdgcn_readlane(r.seq0, sel);
      out.seqs = __builtin_amdgcn_readlane(r.seqs, sel);
      out.shared = __builtin_amdgcn_readlane(r.shared, sel);
      out.tile0 = __builtin_amdgcn_readlane(t0, sel);
      return true;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// v_mfma operand layouts (16x16: 4 groups g4 of 16 lanes; 32x32: 2 halves):
//   16x16x32  A[m = lane%16][k = 8*(lane/16) + e], B[k][n = lane%16],
//             D[m = 4*(lane/16) + i][n = lane%16]
//   16x16x16  A[m = lane%16][k = 4*(lane/16) + e], B and D likewise
//   32x32x16  A[m = lane%32][k = 8*(lane/32) + e], B[k][n = lane%32],
//             D[m = 8*(i/4) + 4*(lane/32) + i%4][n = lane%32]
template <class TT>
struct Mma;
template <>
struct Mma<BF16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 k32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b),
                                                   c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 k16(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a),
                                                     __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 m32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b),
                                                   c, 0, 0, 0);
  }
};
template <>
struct Mma<F16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 k32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b),
                                                  c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 k16(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                                 __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 m32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b),
                                                  c, 0, 0, 0);
  }
};

// ds_read_b64_tr_b16: in a group of 16 lanes, lane j receives element j%4 of the
// 8-byte chunks addressed by lanes 4e + j/4, e = 0..3
__device__ __forceinline__ u32x2 lds_read_tr(const void* p) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
}

// Eight e4m3 bytes -> four pairs of TT, exact.
template <class TT>
__device__ __forceinline__ u32x4 e4m3x8_to(uint32_t lo, uint32_t hi) {
  return u32x4{e4m3x2_to<TT, false>(lo), e4m3x2_to<TT, true>(lo), e4m3x2_to<TT, false>(hi),
               e4m3x2_to<TT, true>(hi)};
}

// Launcher by padded head dim (scored_rows_d*.hip): chunks, or groups (the shared
// keys and the sequences' own ones in one launch).
template <int D>
void launch_rows(const Args& a, int32_t dtype, hipStream_t st);

}  // namespace scored
}  // namespace npd
