// Decode attention with changed scores (scored.h): the unit that streams the keys
// of one token.
//
// Work unit: one wave per (sequence, kv head, up to 16 of its query heads, part
// of the keys that the token sees). All heads of a unit see the same keys, so
// masks are no part of the loop: the keys seen are two ranges (prefix and own
// range), taken as one list of pool rows in LDS, which also makes any block size,
// window start and head dim one path. Per step of 16 keys:
//   S^T = K . Q^T on v_mfma_f32_16x16x32, K read from the pool in its operand
//     layout (16 bytes per lane, the heads padded to 16 columns);
//   the head's reference moves only when a step's maximum passes it by 2^8;
//   O^T += V^T . P^T on v_mfma_f32_16x16x16, V through LDS for the transposing
//     reads of its operand.
// Loads run kRing steps ahead in registers (8 to 16 KB of a wave in flight).
// Bound: HBM, the units' K/V bytes (64 sequences of 128 to 4096 keys, 32 / 8 heads of
// 128, bf16: 117 us, 4.83 TB/s of the 4.92 that a large copy reaches). Short ones
// are bound by the chain length -> table -> K -> step, 9 us a call with its launch.
// Parts: a unit's keys are cut into near-equal parts, from the lengths on the device
// (part_len); the parts meet in a merge kernel. At 1000 and 4000 keys of one
// sequence, parts of 64 keys take 11 and 13 us where parts of 256 take 22 and 27;
// four deep rings of 128 dims (64 KB in flight) took 5% longer over full batches,
// and at 256 dims spill.
#pragma once

#include "scored.h"

namespace npd {
namespace scored {

// Waves of a stream launch, about: for ragged lengths several rounds of them, for
// lengths within a quarter of their mean the one round that runs at once (40 tokens
// with 4160 keys each in a window, FP8: 75 us against 92; 64 of 4000: 101 against
// 115; ragged to 4000 or 16000 one round takes 85 against 77 and 183 against 156).
// Parts shorter than kLongPart keys spend more on their start and merge than they
// spare once there are kFewItems of them.
constexpr int kTargetItems = 4096;
constexpr int kFewItems = 1024;
constexpr int kLongPart = 256;
constexpr int kListKeys = 1024;      // rows listed in LDS at a time (a multiple of every ring)
constexpr float kTau = 8.f;          // a reference moves by more than this (log2 units)

// Nontemporal: a pool row is read once per call (by one unit per kv head).
__device__ __forceinline__ u32x4 ld_stream(const char* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

// Between a wave's own LDS writes and reads (which it issues in order).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Keys of sequence s that its stream units take (past the shared ones).
__device__ __forceinline__ void unit_keys(const Args& a, int s, int lane, int& pos, int& a0, int& na,
                                          int& b0, int& nb) {
  const int ctx = clampi(a.seq_lens[s], 0, a.max_bps * a.block_size);
  pos = ctx - 1;
  const Keys k = row_keys(pos, ctx, a.first_keys ? a.first_keys[s] : 0,
                          a.prefix_lens ? a.prefix_lens[s] : 0, a.window);
  int from = 0;
  if (a.cu_groups) {
    Group g;
    if (find_group(a, s, lane, g)) from = g.shared;
  }
  b0 = k.lo < from ? from : k.lo;
  nb = k.hi > b0 ? k.hi - b0 : 0;
  a0 = k.first < from ? from : k.first;
  const int ae = k.pre < b0 ? k.pre : b0;
  na = ae > a0 ? ae - a0 : 0;
  // prefix keys past the token: none (pre <= context = position + 1)
}
// Keys of a part, of one length for all units: beside the rows kernel and for units
// that are not cut the host's, else by all keys (of each stride-th sequence, where
// there are many) over the waves wanted.
// (The merge comes to the same length: no operation may be contracted in one of them.)
__device__ __forceinline__ int part_len(const Args& a, int lane) {
#pragma clang fp contract(off)
  if (a.cu_groups || a.unit_splits == 1) return a.part_keys;
  const int stride = (a.num_seqs + 511) / 512;
  float sum = 0.f, most = 0.f, count = 0.f;
  for (int s = lane * stride; s < a.num_seqs; s += 64 * stride) {
    const int ctx = clampi(a.seq_lens[s], 0, a.max_bps * a.block_size);
    const Keys k = row_keys(ctx - 1, ctx, a.first_keys ? a.first_keys[s] : 0,
                            a.prefix_lens ? a.prefix_lens[s] : 0, a.window);
    const float keys = (float)(k.hi - k.lo) + (float)max(0, min(k.pre, k.lo) - k.first);
    sum += keys;
    most = fmaxf(most, keys);
    count += 1.f;
  }
  sum = wave_sum_f(sum);
  count = wave_sum_f(count);
  const float units = (float)(a.num_kv_heads * a.subs), total = sum * units * (float)stride;
  // one round of even lengths: each unit's last part is half a part long on average
  const bool even = wave_max_f(most) * count <= 1.25f * sum;
  const float items = even ? fmaxf(a.stream_waves - 0.5f * units * (float)a.num_seqs, 0.5f * a.stream_waves)
                           : (float)kTargetItems;
  const int few = (int)fminf(total * (1.f / kFewItems), 1e9f);
  const int n = (int)fminf(total / items, 1e9f);
  return max(a.part_keys, (max(n, min(few, kLongPart)) + 15) / 16 * 16);
}
__device__ __forceinline__ int unit_parts(const Args& a, int keys, int lane) {
  const int len = part_len(a, lane);
  const int p = keys / len + (keys % len != 0);
  return p < a.unit_splits ? p : a.unit_splits;
}

// DP: the head dim padded to 64, 128 or 256. Chunks past the row's end load its
// last chunk against zero queries; their output dims are not stored.
// One wave; the LDS is its own.
template <int DP>
struct StreamLds {
  uint16_t v[16 * (DP + 16)];      // rows of DP + 16 elements: an 8-bank shift per row
  int row[kListKeys];
};
template <class TT, int DP, bool kF8, int kRing>
__device__ __forceinline__ void stream_unit(const Args& a, int item, int lane, StreamLds<DP>& lds) {
  constexpr int EB = kF8 ? 1 : 2;                  // bytes per element
  constexpr int CPR = DP * EB / 16;                // 16-byte chunks per (padded) row
  constexpr int NKL = CPR / 4;                     // K loads per lane and step
  constexpr int TPL = 64 / CPR;                    // rows per V load
  constexpr int NVL = 16 / TPL;                    // V loads per lane and step
  constexpr int NKC = DP / 32;                     // S MFMAs per step
  constexpr int NOB = DP / 16;                     // 16-dim blocks of O^T
  constexpr int VROW = DP + 16;
  static_assert(NKL >= 1 && NVL >= 1, "row shape");
  uint16_t* s_v = lds.v;
  int* s_row = lds.row;
  const int g4 = lane >> 4, n16 = lane & 15;
  const int units = a.num_seqs * a.num_kv_heads * a.subs;
  const int part = item / units, unit = item - part * units;
  if (part >= a.unit_splits) return;
  const int sub = unit % a.subs, kh = unit / a.subs % a.num_kv_heads;
  const int s = unit / a.subs / a.num_kv_heads;
  const int h0 = kh * a.group + sub * a.sub_heads;
  const int heads = min(a.sub_heads, a.group - sub * a.sub_heads);
  const int d = a.head_dim;

  int pos, a0, na, b0, nb;
  unit_keys(a, s, lane, pos, a0, na, b0, nb);
  const int keys = na + nb;
  const int parts = unit_parts(a, keys, lane);
  const bool direct = !a.cu_groups && parts <= 1;
  uint16_t* orow = a.out + s * a.out_stride_token + (h0 + n16) * a.out_stride_head;
  if (part >= parts) {
    if (part == 0 && direct && n16 < heads)   // no key at all: zero rows
      for (int e = g4 * 4; e < d; e += 16) *reinterpret_cast<u32x2*>(orow + e) = u32x2{0, 0};
    return;
  }
  const int span = ((keys + parts - 1) / parts + 15) / 16 * 16;
  const int k0 = part * span < keys ? part * span : keys;
  const int k1 = k0 + span < keys ? k0 + span : keys;

  // Q^T as the B operand: lane (g4, n16) = head n16, the dims of the K operand
  // (2-byte pools: chunk c = dims 32c + 8 g4 ..; FP8: load c covers dims 64c +
  // 16 g4 .., converted in two halves)
  u32x4 qb[NKC];
  {
    const uint16_t* qrow = a.q + s * a.q_stride_token + (h0 + n16) * a.q_stride_head;
#pragma unroll
    for (int c = 0; c < NKC; ++c) {
      const int at = kF8 ? 64 * (c / 2) + 16 * g4 + 8 * (c % 2) : 32 * c + 8 * g4;
      qb[c] = n16 < heads && at < d ? *reinterpret_cast<const u32x4*>(qrow + at) : u32x4{0, 0, 0, 0};
    }
  }
  const float kscale = kF8 ? a.k_scale[kh] : 1.f;
  const float oscale = kF8 ? a.v_scale[kh] : 1.f;
  const bool cap = a.cap_log2 > 0.f;
  const float c2 = a.scale_log2 * kscale, cin = a.cap_in * kscale;
  const float slope = a.slopes && n16 < heads ? a.slopes[h0 + n16] * kLog2e : 0.f;
  const int64_t rowb = (int64_t)d * EB;
  const int last = (int)(rowb / 16) - 1;            // the row's last chunk
  const int j = lane % CPR, r = lane / CPR;         // V: chunk and row of this lane's loads
  const int vcol = (j < last ? j : last) * 16;
  int kcol[NKL];
#pragma unroll
  for (int c = 0; c < NKL; ++c) kcol[c] = (4 * c + g4 < last ? 4 * c + g4 : last) * 16;

  f32x4 oacc[NOB];
#pragma unroll
  for (int b = 0; b < NOB; ++b) oacc[b] = f32x4{0, 0, 0, 0};
  float mref = -INFINITY, lp = 0.f;   // head n16's reference; this lane's sum of its P
  const uint16_t* vl = s_v + (g4 * 4 + (n16 >> 2)) * VROW + 4 * (n16 & 3);

  for (int t0 = k0; t0 < k1; t0 += kListKeys) {
    const int ntok = k1 - t0 < kListKeys ? k1 - t0 : kListKeys;
    const int nsteps = ((ntok + 15) / 16 + kRing - 1) / kRing * kRing;
    // pool rows of the keys; entries past them repeat the last one
    wave_sync();
    for (int e = lane; e < nsteps * 16; e += 64) {
      const int x = t0 + (e < ntok ? e : ntok - 1);
      const int key = x < na ? a0 + x : b0 + (x - na);
      const int lb = a.bs_shift >= 0 ? key >> a.bs_shift : key / a.block_size;
      const int bid = clampi(a.block_tables[(int64_t)s * a.max_bps + lb], 0, a.num_blocks - 1);
      s_row[e] = (bid * a.num_kv_heads + kh) * a.block_size + (key - lb * a.block_size);
    }
    wave_sync();
    auto load_k = [&](u32x4* buf, int st) {
      const char* p = a.k_cache + (int64_t)s_row[st * 16 + n16] * rowb;
#pragma unroll
      for (int c = 0; c < NKL; ++c) buf[c] = ld_stream(p + kcol[c]);
    };
    auto load_v = [&](u32x4* buf, int st) {
#pragma unroll
      for (int i = 0; i < NVL; ++i)
        buf[i] = ld_stream(a.v_cache + (int64_t)s_row[st * 16 + i * TPL + r] * rowb + vcol);
    };
    auto step = [&](const u32x4* kraw, const u32x4* vraw, int st) {
      // V rows into LDS; past the last key zeros, so that an infinity there
      // meets no zero probability
      const bool tail = st * 16 + 16 > ntok;
#pragma unroll
      for (int i = 0; i < NVL; ++i) {
        const int row = i * TPL + r;
        u32x4 v = vraw[i];
        if (tail && st * 16 + row >= ntok) v = u32x4{0, 0, 0, 0};
        if constexpr (kF8) {
          *reinterpret_cast<u32x4*>(&s_v[row * VROW + j * 16]) = e4m3x8_to<TT>(v.x, v.y);
          *reinterpret_cast<u32x4*>(&s_v[row * VROW + j * 16 + 8]) = e4m3x8_to<TT>(v.z, v.w);
        } else {
          *reinterpret_cast<u32x4*>(&s_v[row * VROW + j * 8]) = v;
        }
      }
      f32x4 sacc = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < NKL; ++c) {
        if constexpr (kF8) {
          sacc = Mma<TT>::k32(e4m3x8_to<TT>(kraw[c].x, kraw[c].y), qb[2 * c], sacc);
          sacc = Mma<TT>::k32(e4m3x8_to<TT>(kraw[c].z, kraw[c].w), qb[2 * c + 1], sacc);
        } else {
          sacc = Mma<TT>::k32(kraw[c], qb[c], sacc);
        }
      }
      float sv[4];
      const int e0 = st * 16 + 4 * g4;
#pragma unroll
      for (int i = 0; i < 4; ++i) sv[i] = cap ? cap_exact(sacc[i], cin, a.cap_log2) : sacc[i] * c2;
      if (a.slopes) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = t0 + e0 + i;
          const int key = x < na ? a0 + x : b0 + (x - na);
          sv[i] = fmaf(-slope, (float)(pos - key), sv[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sv[i] = e0 + i < ntok ? sv[i] : -INFINITY;
      const float x = row_max4(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])));
      float f = 1.f;
      if (x > mref + kTau) {
        f = mref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref - x);
        mref = x;
      }
      if (__ballot(f != 1.f) != 0) {   // the first step, then rarely
        lp *= f;
#pragma unroll
        for (int b = 0; b < NOB; ++b) oacc[b] *= f;
      }
      const float ref = mref == -INFINITY ? 0.f : mref;
      const uint32_t p01 = TT::pack2(__builtin_amdgcn_exp2f(sv[0] - ref), __builtin_amdgcn_exp2f(sv[1] - ref));
      const uint32_t p23 = TT::pack2(__builtin_amdgcn_exp2f(sv[2] - ref), __builtin_amdgcn_exp2f(sv[3] - ref));
      lp += (TT::lo(p01) + TT::hi(p01)) + (TT::lo(p23) + TT::hi(p23));
      const u32x2 pb = u32x2{p01, p23};
#pragma unroll
      for (int b = 0; b < NOB; ++b) oacc[b] = Mma<TT>::k16(lds_read_tr(vl + b * 16), pb, oacc[b]);
    };
    u32x4 kb[kRing][NKL], vb[kRing][NVL];
#pragma unroll
    for (int b = 0; b < kRing; ++b) {
      load_k(kb[b], b);
      load_v(vb[b], b);
    }
    int st0 = 0;
    for (; st0 + kRing < nsteps; st0 += kRing) {
#pragma unroll
      for (int b = 0; b < kRing; ++b) {
        step(kb[b], vb[b], st0 + b);
        load_k(kb[b], st0 + kRing + b);
        load_v(vb[b], st0 + kRing + b);
      }
    }
#pragma unroll
    for (int b = 0; b < kRing; ++b) step(kb[b], vb[b], st0 + b);
  }
  const float lsum = row_sum4(lp);
  if (n16 >= heads) return;
  if (direct) {
    const float inv = lsum > 0.f || lsum != lsum ? oscale / lsum : 0.f;
#pragma unroll
    for (int b = 0; b < NOB; ++b)
      if (b * 16 + 4 * g4 < d)
        *reinterpret_cast<u32x2*>(orow + b * 16 + 4 * g4) =
            u32x2{TT::pack2(oacc[b].x * inv, oacc[b].y * inv), TT::pack2(oacc[b].z * inv, oacc[b].w * inv)};
    return;
  }
  const int64_t slot = ((int64_t)s * a.num_heads + h0 + n16) * a.unit_splits + part;
#pragma unroll
  for (int b = 0; b < NOB; ++b)
    if (b * 16 + 4 * g4 < d) *reinterpret_cast<f32x4*>(a.unit_o + slot * d + b * 16 + 4 * g4) = oacc[b];
  if (g4 == 0) {
    a.unit_ml[slot * 2] = mref;
    a.unit_ml[slot * 2 + 1] = lsum;
  }
}

}  // namespace scored
}  // namespace npd
