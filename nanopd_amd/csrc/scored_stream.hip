// Decode attention with changed scores (scored.h): the kernel that streams the
// keys of one token per sequence, the merge of partial results, and the C
// entries of the scored attention ops.
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
// Loads run kRing steps ahead in registers (about 16 KB of a wave in flight at
// any head dim). Bound: HBM, the unit's K/V bytes.
// Parts: a unit's keys are cut into near-equal parts of at least kMinPart keys,
// as many as the launch has waves for it (unit_splits), from the lengths on the
// device; the parts meet in the merge kernel.
#include "scored.h"

namespace npd {
namespace scored {
namespace {

constexpr int kListKeys = 1024;      // rows listed in LDS at a time (a multiple of every ring)
constexpr int kMinPart = 256;        // shortest part of a unit (keys)
constexpr float kTau = 8.f;          // a reference moves by more than this (log2 units)
constexpr int kTargetItems = 4096;   // waves of a launch, about

// Nontemporal: a pool row is read once per call (by one unit per kv head).
__device__ __forceinline__ u32x4 ld_stream(const char* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
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
    if (find_group<true>(a, s, lane, g)) from = g.shared;
  }
  b0 = k.lo < from ? from : k.lo;
  nb = k.hi > b0 ? k.hi - b0 : 0;
  a0 = k.first < from ? from : k.first;
  const int ae = k.pre < b0 ? k.pre : b0;
  na = ae > a0 ? ae - a0 : 0;
  // prefix keys past the token: none (pre <= context = position + 1)
}
__device__ __forceinline__ int unit_parts(const Args& a, int keys) {
  const int p = (keys + kMinPart - 1) / kMinPart;
  return p < a.unit_splits ? p : a.unit_splits;
}

// DP: the head dim padded to 64, 128 or 256. Chunks past the row's end load its
// last chunk against zero queries; their output dims are not stored.
template <class TT, int DP, bool kF8>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2)))
void stream_kernel(Args a) {
  constexpr int kRing = DP == 64 || (kF8 && DP == 128) ? 4 : (DP == 128 || kF8 ? 2 : 1);
  constexpr int EB = kF8 ? 1 : 2;                  // bytes per element
  constexpr int CPR = DP * EB / 16;                // 16-byte chunks per (padded) row
  constexpr int NKL = CPR / 4;                     // K loads per lane and step
  constexpr int TPL = 64 / CPR;                    // rows per V load
  constexpr int NVL = 16 / TPL;                    // V loads per lane and step
  constexpr int NKC = DP / 32;                     // S MFMAs per step
  constexpr int NOB = DP / 16;                     // 16-dim blocks of O^T
  constexpr int VROW = DP + 16;                    // V row in LDS: an 8-bank shift per row
  static_assert(NKL >= 1 && NVL >= 1, "row shape");
  __shared__ __attribute__((aligned(16))) uint16_t s_v[16 * VROW];
  __shared__ int s_row[kListKeys];
  const int lane = threadIdx.x, g4 = lane >> 4, n16 = lane & 15;
  const int units = a.num_seqs * a.num_kv_heads * a.subs;
  const int part = (int)blockIdx.x / units, unit = (int)blockIdx.x - part * units;
  const int sub = unit % a.subs, kh = unit / a.subs % a.num_kv_heads;
  const int s = unit / a.subs / a.num_kv_heads;
  const int h0 = kh * a.group + sub * a.sub_heads;
  const int heads = min(a.sub_heads, a.group - sub * a.sub_heads);
  const int d = a.head_dim;

  int pos, a0, na, b0, nb;
  unit_keys(a, s, lane, pos, a0, na, b0, nb);
  const int keys = na + nb;
  const int parts = unit_parts(a, keys);
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
    __syncthreads();
    for (int e = lane; e < nsteps * 16; e += 64) {
      const int x = t0 + (e < ntok ? e : ntok - 1);
      const int key = x < na ? a0 + x : b0 + (x - na);
      const int lb = a.bs_shift >= 0 ? key >> a.bs_shift : key / a.block_size;
      const int bid = clampi(a.block_tables[(int64_t)s * a.max_bps + lb], 0, a.num_blocks - 1);
      s_row[e] = (bid * a.num_kv_heads + kh) * a.block_size + (key - lb * a.block_size);
    }
    __syncthreads();
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

// Merge: one wave per (token, head) row. The row's partials are the parts of its
// stream units and, with groups, of its group's tiles (chunks: of its tile).
// LPR lanes hold four dims each; the 64 / LPR lane groups take slots in turn.
template <class TT, int LPR>
__global__ __launch_bounds__(256) void merge_kernel(Args a) {
  constexpr int SG = 64 / LPR;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int h = (int)(row % a.num_heads);
  const int tok = (int)(row / a.num_heads);
  if (tok >= a.total_q) return;
  const int kh = h / a.group, hh = h - kh * a.group, d = a.head_dim;
  int nt = 0, nu = 0;        // partials of tiles and of stream units
  int64_t tslot = 0, uslot = 0;
  const int64_t tstep = (int64_t)a.num_kv_heads * kTileRows;   // slots between a tile's parts
  if (a.cu_seqlens_q) {
    // the sequence of the token: the last that starts at or before it (binary search)
    int lo = 0, hi = a.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu_seqlens_q[mid] <= tok) lo = mid; else hi = mid - 1;
    }
    const int q0 = clampi(a.cu_seqlens_q[lo], 0, a.total_q);
    const int q1 = clampi(a.cu_seqlens_q[lo + 1], q0, a.total_q);
    if (tok < q0 || tok >= q1) return;
    const int f = (tok - q0) * a.group + hh;
    if (f / kTileRows >= a.tiles_max) return;
    const int64_t tile = (int64_t)q0 * a.group / kTileRows + lo + f / kTileRows;
    const int32_t* ti = a.tile_items + 2 * (tile * a.num_kv_heads + kh);
    nt = ti[1];
    if (nt <= 1) return;     // written by the rows kernel itself
    tslot = ((int64_t)ti[0] * a.num_kv_heads + kh) * kTileRows + f % kTileRows;
  } else {
    int pos, a0, na, b0, nb;
    unit_keys(a, tok, lane, pos, a0, na, b0, nb);
    nu = unit_parts(a, na + nb);
    if (!a.cu_groups && nu <= 1) return;   // written by the stream kernel itself
    uslot = ((int64_t)tok * a.num_heads + h) * a.unit_splits;
    Group g;
    if (a.cu_groups && find_group<true>(a, tok, lane, g) && g.shared > 0) {
      const int64_t f = (int64_t)(tok - g.seq0) * a.group + hh;
      const int64_t tile = g.tile0 + f / kTileRows;
      if (tile < a.tiles) {
        const int32_t* ti = a.tile_items + 2 * (tile * a.num_kv_heads + kh);
        nt = ti[1];
        tslot = ((int64_t)ti[0] * a.num_kv_heads + kh) * kTileRows + f % kTileRows;
      }
    }
  }
  // (lists that do not ascend may leave an entry unwritten: stay in the buffer)
  const int64_t room = (int64_t)a.items * a.num_kv_heads * kTileRows;
  if (tslot < 0 || nt < 0 || tslot + nt * tstep > room + tstep - kTileRows) nt = 0;
  const int n = nt + nu;
  auto ml = [&](int i) {
    return i < nt ? a.tile_ml + (tslot + i * tstep) * 2 : a.unit_ml + (uslot + i - nt) * 2;
  };
  auto ov = [&](int i) {
    return i < nt ? a.tile_o + (tslot + i * tstep) * d : a.unit_o + (uslot + i - nt) * d;
  };
  float M = -INFINITY;
  for (int i = lane; i < n; i += 64) M = fmaxf(M, ml(i)[0]);
  M = wave_max_f(M);
  const int c = (lane % LPR) * 4;
  f32x4 o = f32x4{0, 0, 0, 0};
  float L = 0.f;
  if (M > -INFINITY) {
    for (int i = lane / LPR; i < n; i += SG) {
      const float* p = ml(i);
      if (p[0] == -INFINITY) continue;   // a part without a key
      const float w = __builtin_amdgcn_exp2f(p[0] - M);
      L = fmaf(p[1], w, L);
      if (c < d) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(ov(i) + c);
        o.x = fmaf(x.x, w, o.x);
        o.y = fmaf(x.y, w, o.y);
        o.z = fmaf(x.z, w, o.z);
        o.w = fmaf(x.w, w, o.w);
      }
    }
  }
#pragma unroll
  for (int k = LPR; k < 64; k <<= 1) {
    L += __shfl_xor(L, k, 64);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = o[e];
      o[e] = v + __shfl_xor(v, k, 64);
    }
  }
  if (lane < LPR && c < d) {
    const float inv = L > 0.f || L != L ? (a.v_scale ? a.v_scale[kh] : 1.f) / L : 0.f;
    uint16_t* dst = a.out + tok * a.out_stride_token + h * a.out_stride_head + c;
    *reinterpret_cast<u32x2*>(dst) =
        u32x2{TT::pack2(o.x * inv, o.y * inv), TT::pack2(o.z * inv, o.w * inv)};
  }
}

template <class TT, int DP>
void launch_stream_d(const Args& a, int64_t items, hipStream_t st) {
  const dim3 g((unsigned)items), b(64);
  if (a.k_scale)
    hipLaunchKernelGGL((stream_kernel<TT, DP, true>), g, b, 0, st, a);
  else
    hipLaunchKernelGGL((stream_kernel<TT, DP, false>), g, b, 0, st, a);
}
template <class TT>
void launch_stream(const Args& a, hipStream_t st) {
  const int64_t items = (int64_t)a.num_seqs * a.num_kv_heads * a.subs * a.unit_splits;
  if (a.head_dim <= 64) launch_stream_d<TT, 64>(a, items, st);
  else if (a.head_dim <= 128) launch_stream_d<TT, 128>(a, items, st);
  else launch_stream_d<TT, 256>(a, items, st);
}
template <class TT>
void launch_merge(const Args& a, hipStream_t st) {
  const dim3 g((unsigned)(((int64_t)a.total_q * a.num_heads + 3) / 4)), b(256);
  if (a.head_dim <= 64) hipLaunchKernelGGL((merge_kernel<TT, 16>), g, b, 0, st, a);
  else if (a.head_dim <= 128) hipLaunchKernelGGL((merge_kernel<TT, 32>), g, b, 0, st, a);
  else hipLaunchKernelGGL((merge_kernel<TT, 64>), g, b, 0, st, a);
}
void launch_rows_any(const Args& a, int32_t dtype, hipStream_t st) {
  if (a.head_dim <= 64) launch_rows<64>(a, dtype, st);
  else if (a.head_dim <= 128) launch_rows<128>(a, dtype, st);
  else launch_rows<256>(a, dtype, st);
}

// Units of at most kUnitHeads heads: the fewest near-equal ones.
int64_t subs_of(int64_t group) { return (group + kUnitHeads - 1) / kUnitHeads; }

// Most parts of a unit: as many as bring the launch to kTargetItems waves, no
// more than the table's tokens (or the window's) have parts of kMinPart keys.
int64_t unit_splits_of(int64_t units, int64_t max_keys) {
  int64_t w = (kTargetItems + units - 1) / units;
  const int64_t most = (max_keys + kMinPart - 1) / kMinPart;
  w = w < most ? w : most;
  return w < 1 ? 1 : w;
}

// Workgroups of the rows kernel that run at once per kv head.
int64_t rows_room(int64_t head_dim, int64_t num_kv_heads) {
  const int64_t n = rows_per_cu(head_dim) * (int64_t)device_cus() / num_kv_heads;
  return n < 1 ? 1 : n;
}

int64_t pad256(int64_t x) { return (x + 255) / 256 * 256; }

// Sizes of a call's partials; the workspace is the counter region (which these
// ops leave alone, so that one buffer serves every attention op), then the
// tiles' partials and part counts, then the units'.
struct Plan {
  int64_t tiles = 0, tiles_max = 0, items = 0, room = 1, unit_splits = 1;
  bool list = false;
  int64_t tile_slots = 0, unit_slots = 0, head_dim = 0, kv_heads = 0;
  int64_t tile_items_at() const { return kCounterBytes; }
  int64_t tile_o_at() const { return tile_items_at() + (tile_slots ? pad256(tiles * kv_heads * 8) : 0); }
  int64_t tile_ml_at() const { return tile_o_at() + pad256(tile_slots * head_dim * 4); }
  int64_t unit_o_at() const { return tile_ml_at() + pad256(tile_slots * 8); }
  int64_t unit_ml_at() const { return unit_o_at() + pad256(unit_slots * head_dim * 4); }
  int64_t bytes() const {
    return tile_slots || unit_slots ? unit_ml_at() + pad256(unit_slots * 8) : 0;
  }
};

int64_t window_keys(int64_t max_keys, int64_t window, bool prefix) {
  return window > 0 && !prefix && window < max_keys ? window : max_keys;
}
Plan decode_plan(int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                 int64_t max_keys) {
  Plan p;
  p.head_dim = head_dim;
  p.kv_heads = num_kv_heads;
  p.unit_splits = unit_splits_of(num_seqs * num_kv_heads * subs_of(num_heads / num_kv_heads), max_keys);
  p.unit_slots = p.unit_splits > 1 ? num_seqs * num_heads * p.unit_splits : 0;
  return p;
}
Plan shared_plan(int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                 int64_t max_keys, int64_t num_groups, int64_t max_shared) {
  Plan p = decode_plan(num_seqs, num_heads, num_kv_heads, head_dim, max_keys);
  p.unit_slots = num_seqs * num_heads * p.unit_splits;   // always merged
  p.tiles = num_seqs * (num_heads / num_kv_heads) / kTileRows + num_groups;
  p.list = true;
  p.room = rows_room(head_dim, num_kv_heads);
  // parts of target steps: at most room + one round-up per tile, nor more than
  // the shared keys' steps
  const int64_t most = p.tiles * (max_shared / kStepKeys + 1);
  p.items = p.room + p.tiles < most ? p.room + p.tiles : most;
  p.tile_slots = p.items * num_kv_heads * kTileRows;
  return p;
}
Plan chunk_plan(int64_t num_seqs, int64_t total_q, int64_t num_heads, int64_t num_kv_heads,
                int64_t head_dim, int64_t max_q_len, int64_t max_keys) {
  Plan p;
  const int64_t g = num_heads / num_kv_heads;
  p.head_dim = head_dim;
  p.kv_heads = num_kv_heads;
  p.tiles = total_q * g / kTileRows + num_seqs;
  p.tiles_max = (max_q_len * g + kTileRows - 1) / kTileRows;
  p.room = rows_room(head_dim, num_kv_heads);
  p.items = num_seqs * p.tiles_max;
  const int64_t most = p.tiles < p.items ? p.tiles : p.items;
  // cut into parts unless whole tiles fill the chip three times over, or hold so
  // few keys that none would be cut
  p.list = p.items <= kListTiles && most < 3 * p.room && max_keys > 8 * kStepKeys;
  if (p.list) {
    p.items = p.room + most;
    p.tile_slots = p.items * num_kv_heads * kTileRows;
  }
  return p;
}

struct Call {
  const char* name;
  void* out;
  const void* query;
  const void* key_cache;
  const void* value_cache;
  const int32_t* block_tables;
  const int32_t* lens;
  int64_t num_seqs, total_q, num_heads, num_kv_heads, head_dim, num_blocks, block_size, max_bps;
  float scale, softcap;
  const float* slopes;
  int64_t window;
  const float* k_scale;
  const float* v_scale;
  int64_t q_stride_token, q_stride_head, out_stride_token, out_stride_head;
  int32_t dtype;
};

int check_call(const Call& c) {
  if (c.dtype != NPD_DTYPE_F16 && c.dtype != NPD_DTYPE_BF16)
    return fail(NPD_E_DTYPE, "%s: unsupported dtype code %d (fp16/bf16 only)", c.name, c.dtype);
  if (c.num_seqs < 0 || c.total_q < 0 || c.num_heads <= 0 || c.num_kv_heads <= 0 ||
      c.num_blocks <= 0 || c.block_size <= 0 || c.max_bps <= 0)
    return fail(NPD_E_INVALID,
                "%s: bad sizes (seqs %lld, heads %lld, kv heads %lld, blocks %lld, block %lld, "
                "max blocks/seq %lld)", c.name, (long long)c.num_seqs, (long long)c.num_heads,
                (long long)c.num_kv_heads, (long long)c.num_blocks, (long long)c.block_size,
                (long long)c.max_bps);
  if (c.num_heads % c.num_kv_heads != 0)
    return fail(NPD_E_INVALID, "%s: num_heads %lld is not a multiple of num_kv_heads %lld", c.name,
                (long long)c.num_heads, (long long)c.num_kv_heads);
  const bool fp8 = c.k_scale != nullptr || c.v_scale != nullptr;
  const int64_t step = fp8 ? 16 : 8;
  if (c.head_dim < 32 || c.head_dim > 256 || c.head_dim % step != 0)
    return fail(NPD_E_INVALID, "%s: head_dim %lld is not a multiple of %lld in [32, 256]", c.name,
                (long long)c.head_dim, (long long)step);
  if (c.num_blocks > INT32_MAX / c.block_size / c.num_kv_heads ||
      c.max_bps > INT32_MAX / c.block_size)
    return fail(NPD_E_INVALID, "%s: pool exceeds int32 row indexing", c.name);
  if (c.num_seqs > INT32_MAX || c.total_q > INT32_MAX / c.num_heads ||
      c.num_seqs > INT32_MAX / c.num_heads)
    return fail(NPD_E_INVALID, "%s: too many (token, head) rows", c.name);
  if (!(c.scale > 0.f) || c.scale > 3e38f)
    return fail(NPD_E_INVALID, "%s: scale must be positive and finite", c.name);
  if (!(c.softcap >= 0.f) || c.softcap > 1e30f || (c.softcap > 0.f && c.softcap < 1e-30f))
    return fail(NPD_E_INVALID, "%s: softcap must be 0 (none) or from 1e-30 to 1e30", c.name);
  if (c.window < 0 || c.window > INT32_MAX)
    return fail(NPD_E_INVALID, "%s: window must be 0 (none) or a positive int32", c.name);
  if (c.q_stride_token % 8 || c.q_stride_head % 8 || c.out_stride_token % 8 || c.out_stride_head % 8 ||
      c.q_stride_token < 0 || c.q_stride_head < 0 || c.out_stride_token < 0 || c.out_stride_head < 0)
    return fail(NPD_E_ALIGN, "%s: query/out strides must be non-negative multiples of 8 elements",
                c.name);
  if (c.num_seqs == 0 || c.total_q == 0) return NPD_OK;
  if (!c.out || !c.query || !c.key_cache || !c.value_cache || !c.block_tables || !c.lens)
    return fail(NPD_E_INVALID, "%s: null pointer", c.name);
  if (fp8 && (!c.k_scale || !c.v_scale))
    return fail(NPD_E_INVALID, "%s: pass both k_scale and v_scale (FP8 pool) or neither", c.name);
  if (!aligned16(c.out) || !aligned16(c.query) || !aligned16(c.key_cache) || !aligned16(c.value_cache))
    return fail(NPD_E_ALIGN, "%s: out, query and caches must be 16-byte aligned", c.name);
  return NPD_OK;
}

int check_workspace(const Call& c, const Plan& p, const void* workspace, int64_t bytes) {
  const int64_t need = p.bytes();
  if (need == 0) return NPD_OK;
  if (!workspace || bytes < need)
    return fail(NPD_E_WORKSPACE, "%s: workspace of %lld bytes needed, %lld given", c.name,
                (long long)need, (long long)bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return fail(NPD_E_ALIGN, "%s: workspace must be 256-byte aligned", c.name);
  return NPD_OK;
}

Args make_args(const Call& c, const Plan& p, void* workspace) {
  Args a{};
  a.out = static_cast<uint16_t*>(c.out);
  a.q = static_cast<const uint16_t*>(c.query);
  a.k_cache = static_cast<const char*>(c.key_cache);
  a.v_cache = static_cast<const char*>(c.value_cache);
  a.block_tables = c.block_tables;
  a.seq_lens = c.lens;
  a.slopes = c.slopes;
  a.k_scale = c.k_scale;
  a.v_scale = c.v_scale;
  char* ws = static_cast<char*>(workspace);
  if (p.tile_slots) {
    a.tile_items = reinterpret_cast<int32_t*>(ws + p.tile_items_at());
    a.tile_o = reinterpret_cast<float*>(ws + p.tile_o_at());
    a.tile_ml = reinterpret_cast<float*>(ws + p.tile_ml_at());
  }
  if (p.unit_slots) {
    a.unit_o = reinterpret_cast<float*>(ws + p.unit_o_at());
    a.unit_ml = reinterpret_cast<float*>(ws + p.unit_ml_at());
  }
  a.num_seqs = (int)c.num_seqs;
  a.total_q = (int)c.total_q;
  a.num_heads = (int)c.num_heads;
  a.num_kv_heads = (int)c.num_kv_heads;
  a.group = (int)(c.num_heads / c.num_kv_heads);
  a.head_dim = (int)c.head_dim;
  a.block_size = (int)c.block_size;
  a.bs_shift = (c.block_size & (c.block_size - 1)) == 0 ? __builtin_ctzll((uint64_t)c.block_size) : -1;
  a.num_blocks = (int)c.num_blocks;
  a.max_bps = (int)c.max_bps;
  a.tiles = (int)p.tiles;
  a.tiles_max = (int)p.tiles_max;
  a.items = (int)p.items;
  a.room = (int)p.room;
  a.list = p.list;
  a.unit_splits = (int)p.unit_splits;
  a.subs = (int)subs_of(a.group);
  a.sub_heads = (a.group + a.subs - 1) / a.subs;
  a.window = (int)c.window;
  a.scale_log2 = c.scale * kLog2e;
  if (c.softcap > 0.f) {
    a.cap_in = 2.f * (a.scale_log2 / c.softcap);
    a.cap_log2 = c.softcap * kLog2e;
    a.cap_wide = c.softcap > kCapPlain;
  }
  a.q_stride_token = c.q_stride_token;
  a.q_stride_head = c.q_stride_head;
  a.out_stride_token = c.out_stride_token;
  a.out_stride_head = c.out_stride_head;
  return a;
}

bool grid_ok(int64_t n) { return n <= INT32_MAX; }

}  // namespace
}  // namespace scored
}  // namespace npd

using namespace npd;
using namespace npd::scored;

extern "C" int64_t npd_paged_attention_scored_workspace_size(int64_t num_seqs, int64_t num_heads,
                                                             int64_t num_kv_heads, int64_t head_dim,
                                                             int64_t block_size,
                                                             int64_t max_blocks_per_seq,
                                                             int64_t window, int32_t has_prefix) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      max_blocks_per_seq <= 0 || max_blocks_per_seq > INT32_MAX / block_size ||
      num_seqs > INT32_MAX / num_heads)
    return 0;
  return decode_plan(num_seqs, num_heads, num_kv_heads, head_dim,
                     window_keys(block_size * max_blocks_per_seq, window, has_prefix != 0)).bytes();
}

extern "C" int npd_paged_attention_scored(
    void* out, const void* query, const void* key_cache, const void* value_cache,
    const int32_t* block_tables, const int32_t* seq_lens, int64_t num_seqs, int64_t num_heads,
    int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
    int64_t max_blocks_per_seq, float scale, float softcap, const float* alibi_slopes,
    int64_t window, const int32_t* first_keys, const int32_t* prefix_lens, const float* k_scale,
    const float* v_scale, int64_t q_stride_seq, int64_t q_stride_head, int64_t out_stride_seq,
    int64_t out_stride_head, void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream) {
  const Call c{"npd_paged_attention_scored", out, query, key_cache, value_cache, block_tables,
               seq_lens, num_seqs, num_seqs, num_heads, num_kv_heads, head_dim, num_blocks,
               block_size, max_blocks_per_seq, scale, softcap, alibi_slopes, window, k_scale,
               v_scale, q_stride_seq, q_stride_head, out_stride_seq, out_stride_head, dtype};
  int rc = check_call(c);
  if (rc != NPD_OK || num_seqs == 0) return rc;
  const Plan p = decode_plan(num_seqs, num_heads, num_kv_heads, head_dim,
                             window_keys(block_size * max_blocks_per_seq, window, prefix_lens != nullptr));
  rc = check_workspace(c, p, workspace, workspace_bytes);
  if (rc != NPD_OK) return rc;
  Args a = make_args(c, p, workspace);
  a.first_keys = first_keys;
  a.prefix_lens = prefix_lens;
  if (!grid_ok(num_seqs * num_kv_heads * a.subs * p.unit_splits))
    return fail(NPD_E_INVALID, "%s: too many (seq, kv-head) units", c.name);
  hipStream_t st = as_stream(stream);
  if (dtype == NPD_DTYPE_BF16) launch_stream<BF16>(a, st);
  else launch_stream<F16>(a, st);
  if (p.unit_slots) {
    if (dtype == NPD_DTYPE_BF16) launch_merge<BF16>(a, st);
    else launch_merge<F16>(a, st);
  }
  return check_launch(c.name);
}

extern "C" int64_t npd_paged_attention_shared_workspace_size(int64_t num_seqs, int64_t num_heads,
                                                             int64_t num_kv_heads, int64_t head_dim,
                                                             int64_t block_size,
                                                             int64_t max_blocks_per_seq,
                                                             int64_t num_groups,
                                                             int64_t max_shared_len) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      max_blocks_per_seq <= 0 || max_blocks_per_seq > INT32_MAX / block_size ||
      num_seqs > INT32_MAX / num_heads || num_groups <= 0 || num_groups > INT32_MAX)
    return 0;
  return shared_plan(num_seqs, num_heads, num_kv_heads, head_dim, block_size * max_blocks_per_seq,
                     num_groups, max_shared_len < 0 ? 0 : max_shared_len).bytes();
}

extern "C" int npd_paged_attention_shared(
    void* out, const void* query, const void* key_cache, const void* value_cache,
    const int32_t* block_tables, const int32_t* seq_lens, const int32_t* cu_groups,
    const int32_t* shared_lens, int64_t num_seqs, int64_t num_groups, int64_t max_shared_len,
    int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks,
    int64_t block_size, int64_t max_blocks_per_seq, float scale, float softcap,
    const float* alibi_slopes, int64_t window, const float* k_scale, const float* v_scale,
    int64_t q_stride_seq, int64_t q_stride_head, int64_t out_stride_seq, int64_t out_stride_head,
    void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream) {
  const Call c{"npd_paged_attention_shared", out, query, key_cache, value_cache, block_tables,
               seq_lens, num_seqs, num_seqs, num_heads, num_kv_heads, head_dim, num_blocks,
               block_size, max_blocks_per_seq, scale, softcap, alibi_slopes, window, k_scale,
               v_scale, q_stride_seq, q_stride_head, out_stride_seq, out_stride_head, dtype};
  int rc = check_call(c);
  if (rc != NPD_OK) return rc;
  if (num_groups <= 0 || num_groups > INT32_MAX || max_shared_len < 0)
    return fail(NPD_E_INVALID, "%s: %lld groups, shared keys up to %lld", c.name,
                (long long)num_groups, (long long)max_shared_len);
  if (num_seqs == 0) return NPD_OK;
  if (!cu_groups || !shared_lens) return fail(NPD_E_INVALID, "%s: null pointer", c.name);
  const int64_t max_keys = block_size * max_blocks_per_seq;
  const Plan p = shared_plan(num_seqs, num_heads, num_kv_heads, head_dim, max_keys, num_groups,
                             max_shared_len);
  rc = check_workspace(c, p, workspace, workspace_bytes);
  if (rc != NPD_OK) return rc;
  Args a = make_args(c, p, workspace);
  a.cu_groups = cu_groups;
  a.shared_lens = shared_lens;
  a.num_groups = (int)num_groups;
  a.max_shared = (int)(max_shared_len < max_keys ? max_shared_len : max_keys);
  if (!grid_ok(num_seqs * num_kv_heads * a.subs * p.unit_splits) ||
      !grid_ok(p.items * num_kv_heads))
    return fail(NPD_E_INVALID, "%s: too many work items", c.name);
  hipStream_t st = as_stream(stream);
  launch_rows_any(a, dtype, st);
  if (dtype == NPD_DTYPE_BF16) {
    launch_stream<BF16>(a, st);
    launch_merge<BF16>(a, st);
  } else {
    launch_stream<F16>(a, st);
    launch_merge<F16>(a, st);
  }
  return check_launch(c.name);
}

extern "C" int64_t npd_paged_prefill_scored_workspace_size(int64_t num_seqs, int64_t total_q,
                                                           int64_t num_heads, int64_t num_kv_heads,
                                                           int64_t head_dim, int64_t max_q_len,
                                                           int64_t max_context_len) {
  if (num_seqs <= 0 || total_q <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      max_q_len <= 0 || max_context_len <= 0 || total_q > INT32_MAX / num_heads ||
      num_seqs > INT32_MAX / num_heads || max_q_len > INT32_MAX / num_heads)
    return 0;
  return chunk_plan(num_seqs, total_q, num_heads, num_kv_heads, head_dim, max_q_len,
                    max_context_len).bytes();
}

extern "C" int npd_paged_prefill_scored(
    void* out, const void* query, const void* key_cache, const void* value_cache,
    const int32_t* block_tables, const int32_t* cu_seqlens_q, const int32_t* context_lens,
    int64_t num_seqs, int64_t total_q, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
    int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_seq, int64_t max_q_len,
    int64_t max_context_len, float scale, float softcap, const float* alibi_slopes, int64_t window,
    const int32_t* first_keys, const int32_t* prefix_lens, const float* k_scale,
    const float* v_scale, int64_t q_stride_token, int64_t q_stride_head, int64_t out_stride_token,
    int64_t out_stride_head, void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream) {
  const Call c{"npd_paged_prefill_scored", out, query, key_cache, value_cache, block_tables,
               context_lens, num_seqs, total_q, num_heads, num_kv_heads, head_dim, num_blocks,
               block_size, max_blocks_per_seq, scale, softcap, alibi_slopes, window, k_scale,
               v_scale, q_stride_token, q_stride_head, out_stride_token, out_stride_head, dtype};
  int rc = check_call(c);
  if (rc != NPD_OK || num_seqs == 0 || total_q == 0) return rc;
  if (!cu_seqlens_q) return fail(NPD_E_INVALID, "%s: null pointer", c.name);
  if (max_q_len <= 0 || max_q_len > INT32_MAX / num_heads || max_context_len < 0)
    return fail(NPD_E_INVALID, "%s: max_q_len %lld, max_context_len %lld", c.name,
                (long long)max_q_len, (long long)max_context_len);
  // the workspace is sized without the window: one buffer serves every layer
  const Plan p = chunk_plan(num_seqs, total_q, num_heads, num_kv_heads, head_dim, max_q_len,
                            max_context_len);
  rc = check_workspace(c, p, workspace, workspace_bytes);
  if (rc != NPD_OK) return rc;
  Args a = make_args(c, p, workspace);
  a.cu_seqlens_q = cu_seqlens_q;
  a.first_keys = first_keys;
  a.prefix_lens = prefix_lens;
  if (!grid_ok(p.items * num_kv_heads))
    return fail(NPD_E_INVALID, "%s: too many work items", c.name);
  hipStream_t st = as_stream(stream);
  launch_rows_any(a, dtype, st);
  if (p.tile_slots) {
    if (dtype == NPD_DTYPE_BF16) launch_merge<BF16>(a, st);
    else launch_merge<F16>(a, st);
  }
  return check_launch(c.name);
}
