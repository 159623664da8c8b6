// Attention with changed scores (scored.h): the kernel for many query rows that
// read the same keys -- prompt chunks, and the tokens of a group of sequences
// over their shared prefix.
//
// Workgroup: 4 waves = 128 flattened (token, head) rows of one kv head, and a
// part of the keys they see. K/V tiles of 64 keys load straight into LDS
// (global_load_lds, 16 bytes per lane; FP8 bytes through registers, converted
// exactly), two tiles of each, the next one loading under the step. Per step a
// wave forms
//   S^T = K . Q^T     (32x32x16 MFMA, its 32 query rows in registers),
//   P   = 2^(t - m)   (scored.h; masks only in steps that some row sees in part),
//   O^T += V^T . P^T  (V through transposing LDS reads).
// A row's reference m moves only where a P grew past a bound (kPast), so no
// maximum is taken in the usual step. Steps run from the last key back: the
// newest keys come first, which with a distance term hold the largest scores.
//
// Masked keys: P is 0 by selection, but 0 times an infinity or NaN in V is NaN,
// and rows of a tile do not see the same keys. So a row whose result is not
// finite is computed again, key by key over what it sees (redo_row); a finite
// result had no such product.
//
// Bound: the MFMAs and the exponentials share the issue of a SIMD. Two
// workgroups per compute unit run unsynchronised (head dims up to 128), one's
// MFMAs under the other's exponentials.
#pragma once

#include "scored.h"

namespace npd {
namespace scored {

constexpr int kThreads = 256;
constexpr int kListBlocks = 2048;    // pool blocks listed in LDS at a time (8 KB)

// LDS position of 16-byte chunk c of tile row r is c ^ swz(r): rows are D * 2
// bytes apart without padding (direct loads write 1 KB runs), and the swizzle
// spreads both kinds of reads over the banks.
template <int D>
__device__ __forceinline__ int swz(int row) {
  if (D == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  return ((row & 3) << 2) | (((row >> 2) & 1) << 1) | ((row >> 3) & 1);
}
template <int D>
constexpr int swz8() { return D == 64 ? 32 : 16; }   // bytes that differ between rows r and r + 8

// 64 lanes x 16 bytes from p (per lane) straight into LDS at lds .. lds + 1023
__device__ __forceinline__ void load_to_lds(uint32_t lds, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds), "v"(p) : "memory", "m0");
}
// Every load and LDS access of this wave is done; then the workgroup's barrier.
__device__ __forceinline__ void wait_all_and_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// When a row's reference moves. bf16: it sits kBias above the maximum it was
// taken from, and a P of 2 or more (bit 14 of a half) asks for a new one. fp16
// keeps it at the maximum, and asks where a lane's 32 P of a step come to 2^8 or
// more: one of them then passed it by kMove.
template <class TT>
struct Bound;
template <>
struct Bound<BF16> {
  static constexpr float kBias = 7.f, kMove = 0.f, kPast = 0.f;
};
template <>
struct Bound<F16> {
  static constexpr float kBias = 0.f, kMove = 2.f, kPast = 256.f;
};

__device__ __forceinline__ int wave_min_i(int x) { return -wave_max_i(-x); }

// The item of a workgroup: rows f0 .. of a tile, and where they come from.
struct Item {
  int s;        // block table row
  int row0;     // first token row of q / out (chunks: of the chunk; groups: sequence)
  int rows;     // flattened rows of the chunk or group
  int t;        // tile of them
  int limit;    // keys at or past it belong to no row here (context, or shared keys)
  int ctx;      // chunks: context; groups: unused
  int qlen;     // chunks: tokens
};

template <class TT, int D, bool kF8, bool kCap, bool kBias>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2)))
void rows_kernel(Args a) {
  constexpr int KT = kStepKeys;
  constexpr int RB = 2 * D;                 // bytes of a tile row
  constexpr int TB = KT * RB;               // bytes of a tile
  constexpr int NI = TB / 4096;             // 1 KB loads per wave and tile
  constexpr int NC = D / 16, NS = KT / 32, KB = KT / 16, DB = D / 32;
  constexpr int EB = kF8 ? 1 : 2;
  __shared__ __attribute__((aligned(1024))) char s_k[2 * TB];
  __shared__ __attribute__((aligned(1024))) char s_v[2 * TB];
  __shared__ int s_row[kListBlocks];
  __shared__ int s_red[4][4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, c32 = lane & 31;
  const int G = a.group, d = a.head_dim, bs = a.block_size;
  const int cap_keys = a.max_bps * bs;

  // ---- the item: kv head fastest (with 8 of them each XCD's L2 serves one),
  // the last tile of a chunk first (it sees the most keys)
  int id = blockIdx.x;
  const int kh = id % a.num_kv_heads;
  id /= a.num_kv_heads;
  Item it;
  int part;
  int64_t tile;      // of all sequences or groups
  if (a.cu_seqlens_q) {
    const int per = a.tiles_max * a.num_seqs;
    part = id / per;
    id -= part * per;
    it.s = id / a.tiles_max;
    it.t = a.tiles_max - 1 - (id - it.s * a.tiles_max);
    const int q0 = clampi(a.cu_seqlens_q[it.s], 0, a.total_q);
    it.qlen = clampi(a.cu_seqlens_q[it.s + 1], q0, a.total_q) - q0;
    it.ctx = clampi(a.seq_lens[it.s], 0, cap_keys);
    it.row0 = q0;
    it.rows = it.qlen * G;
    it.limit = it.ctx;
    tile = (int64_t)q0 * G / kTileRows + it.s + it.t;
  } else {
    part = id / a.tiles;
    tile = id - part * a.tiles;
    Group g;
    if (!find_group<false>(a, (int)tile, lane, g)) return;
    it.s = it.row0 = g.seq0;
    it.qlen = g.seqs;
    it.rows = g.seqs * G;
    it.t = (int)tile - g.tile0;
    it.limit = g.shared;
    it.ctx = 0;
  }
  if (it.t * kTileRows >= it.rows) return;

  // ---- this lane's row (past the last: a copy of it, not stored)
  const int f0 = it.t * kTileRows + wave * 32;
  const bool row_ok = f0 + c32 < it.rows;
  const int f = row_ok ? f0 + c32 : it.rows - 1;
  const int tok = f / G;
  const int h = kh * G + (f - tok * G);
  const int qrow = it.row0 + tok;
  int pos, ctx = it.ctx;
  if (a.cu_seqlens_q) {
    pos = ctx - it.qlen + tok;
  } else {
    ctx = clampi(a.seq_lens[qrow], 0, cap_keys);
    pos = ctx - 1;
  }
  Keys see = row_keys(pos, ctx, a.first_keys ? a.first_keys[qrow] : 0,
                      a.prefix_lens ? a.prefix_lens[it.s] : 0, a.window);
  see.hi = see.hi < it.limit ? see.hi : it.limit;
  see.pre = see.pre < it.limit ? see.pre : it.limit;
  if (see.lo >= see.hi) see.lo = see.hi = 0;          // empty ranges are [0, 0)
  if (see.first >= see.pre) see.first = see.pre = 0;

  // ---- the wave's and the workgroup's ranges: near [lo, hi), far [first, pre)
  constexpr int kFar = 0x7fffffff;
  const int w_lo = wave_min_i(see.hi > 0 ? see.lo : kFar), w_hi = wave_max_i(see.hi);
  const int w_first = wave_min_i(see.pre > 0 ? see.first : kFar), w_pre = wave_max_i(see.pre);
  // keys that every row of the wave sees: [w_lo1, w_hi0) and [w_first1, w_pre0)
  const int w_lo1 = wave_max_i(see.lo), w_hi0 = wave_min_i(see.hi);
  const int w_first1 = wave_max_i(see.first), w_pre0 = wave_min_i(see.pre);
  if (lane == 0) {
    s_red[0][wave] = w_lo;
    s_red[1][wave] = w_hi;
    s_red[2][wave] = w_first;
    s_red[3][wave] = w_pre;
  }
  __syncthreads();
  auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int nlo = uni(min(min(s_red[0][0], s_red[0][1]), min(s_red[0][2], s_red[0][3])));
  const int nhi = uni(max(max(s_red[1][0], s_red[1][1]), max(s_red[1][2], s_red[1][3])));
  const int flo = uni(min(min(s_red[2][0], s_red[2][1]), min(s_red[2][2], s_red[2][3])));
  const int fhi = uni(max(max(s_red[3][0], s_red[3][1]), max(s_red[3][2], s_red[3][3])));
  // step ranges [fs0, fs1) and [ns0, ns1), one range where they meet; key
  // bounds of each for the loads
  int ns0 = nhi > 0 ? nlo / KT : 0, ns1 = (nhi + KT - 1) / KT;
  int fs0 = fhi > 0 ? flo / KT : 0, fs1 = (fhi + KT - 1) / KT;
  int nk0 = nlo, nk1 = nhi, fk0 = flo, fk1 = fhi;
  if (fs1 > fs0 && ns1 > ns0 && fs1 >= ns0) {
    ns0 = min(ns0, fs0);
    ns1 = max(ns1, fs1);
    nk0 = min(nk0, fk0);
    nk1 = max(nk1, fk1);
    fs0 = fs1 = 0;
  }
  const int nfar = fs1 - fs0, nsteps = nfar + ns1 - ns0;
  int nsp = 0;
  if (nsteps > 0) {
    nsp = (nsteps + 3) / 4;      // a part has four steps at least
    nsp = nsp < a.tile_splits ? nsp : a.tile_splits;
  }
  const bool merged = a.cu_groups || nsp > 1;
  if (a.tile_parts && part == 0 && tid == 0)
    a.tile_parts[tile * a.num_kv_heads + kh] = nsp;
  uint16_t* op = a.out + (int64_t)qrow * a.out_stride_token + (int64_t)h * a.out_stride_head;
  if (part >= nsp) {
    if (part == 0 && !a.cu_groups && row_ok)   // no key at all: zero rows
      for (int e = hf * 4; e < d; e += 8) *reinterpret_cast<u32x2*>(op + e) = u32x2{0, 0};
    return;
  }
  const int base = nsteps / nsp, rem = nsteps - base * nsp;
  const int st0 = part * base + min(part, rem), st1 = st0 + base + (part < rem ? 1 : 0);

  // ---- queries as B operands: qb[c] = Q[row][16c + 8 hf ..], zeros past the row
  const uint16_t* qp = a.q + (int64_t)qrow * a.q_stride_token + (int64_t)h * a.q_stride_head;
  u32x4 qb[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
    qb[c] = c * 16 + hf * 8 < d ? *reinterpret_cast<const u32x4*>(qp + c * 16 + hf * 8) : u32x4{0, 0, 0, 0};
  const float kscale = kF8 ? a.k_scale[kh] : 1.f;
  const float c2 = a.scale_log2 * kscale, cin = a.cap_in * kscale, capA = a.cap_log2;
  const float slope = kBias ? a.slopes[h] * kLog2e : 0.f;

  // ---- tile loads. Chunks past the row's end repeat its last one (zero queries
  // meet them in S, and their output dims are not stored).
  const int64_t rowb = (int64_t)d * EB;
  const int last16 = (int)(rowb / 16) - 1;
  constexpr int LROW = kF8 ? D / 16 : RB / 16;         // lanes per row
  constexpr int NR = kF8 ? KT * D / (kThreads * 16) : NI;
  static_assert(NR >= 1, "tile shape");
  int lrow[NR], lcol[NR];
#pragma unroll
  for (int e = 0; e < NR; ++e) {
    int c;
    if (kF8) {
      lrow[e] = (tid + kThreads * e) / LROW;
      c = (tid + kThreads * e) % LROW;
    } else {
      const int o = (wave * NI + e) * 1024 + lane * 16;
      lrow[e] = o / RB;
      c = (o % RB / 16) ^ swz<D>(lrow[e]);
    }
    lcol[e] = (c < last16 ? c : last16) * 16;
  }
  const uint32_t lds_k = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_k;
  const uint32_t lds_v = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_v;
  int blk0 = 0, key_lo = 0, key_hi = 0;    // of the segment: first block listed, keys loaded
  auto div_bs = [&](int x) { return a.bs_shift >= 0 ? x >> a.bs_shift : x / bs; };
  auto pool_row = [&](int step, int e) -> int64_t {
    const int key = clampi(step * KT + lrow[e], key_lo, key_hi - 1);
    const int lb = div_bs(key);
    return (int64_t)s_row[lb - blk0] + (key - lb * bs);
  };
  auto load = [&](int step, int b) {        // 2-byte pools
#pragma unroll
    for (int e = 0; e < NR; ++e) {
      const int64_t off = pool_row(step, e) * rowb + lcol[e];
      const uint32_t run = (uint32_t)(b * TB + (wave * NI + e) * 1024);
      load_to_lds(lds_k + run, a.k_cache + off);
      load_to_lds(lds_v + run, a.v_cache + off);
    }
  };
  u32x4 rk[kF8 ? NR : 1], rv[kF8 ? NR : 1];
  auto fetch = [&](int step) {              // FP8 pools: bytes into registers ...
#pragma unroll
    for (int e = 0; e < NR; ++e) {
      const int64_t off = pool_row(step, e) * rowb + lcol[e];
      rk[kF8 ? e : 0] = *reinterpret_cast<const u32x4*>(a.k_cache + off);
      rv[kF8 ? e : 0] = *reinterpret_cast<const u32x4*>(a.v_cache + off);
    }
  };
  auto stash = [&](int b) {                 // ... and converted into LDS
#pragma unroll
    for (int e = 0; e < NR; ++e) {
      const int c = (tid + kThreads * e) % LROW * 2, sw = swz<D>(lrow[e]);
      const int at = b * TB + lrow[e] * RB;
      const u32x4 k = rk[kF8 ? e : 0], v = rv[kF8 ? e : 0];
      *reinterpret_cast<u32x4*>(s_k + at + ((c ^ sw) << 4)) = e4m3x8_to<TT>(k.x, k.y);
      *reinterpret_cast<u32x4*>(s_k + at + (((c + 1) ^ sw) << 4)) = e4m3x8_to<TT>(k.z, k.w);
      *reinterpret_cast<u32x4*>(s_v + at + ((c ^ sw) << 4)) = e4m3x8_to<TT>(v.x, v.y);
      *reinterpret_cast<u32x4*>(s_v + at + (((c + 1) ^ sw) << 4)) = e4m3x8_to<TT>(v.z, v.w);
    }
  };

  f32x16 oacc[DB];     // O^T[dim 32 db + 8 (i/4) + 4 hf + i%4][row c32]
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) oacc[db][i] = 0.f;
  float mref = -INFINITY, nmref = kNoRef, lsum = 0.f;

  const int kofs = c32 * RB + ((hf ^ swz<D>(c32)) << 4);
  const int vrow = 4 * hf + ((lane & 15) >> 2);
  const int vofs = vrow * RB + (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ swz<D>(vrow)) << 4) +
                   (lane & 1) * 8;
  auto compute = [&](int step, int b) {
    const int key0 = step * KT;
    const bool some = (key0 < w_hi && key0 + KT > w_lo) || (key0 < w_pre && key0 + KT > w_first);
    if (!some) return;     // no row of this wave sees a key here
    f32x16 sacc[NS];       // S^T[key 32 n + 8 (i/4) + 4 hf + i%4][row c32]
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) sacc[n][i] = 0.f;
#pragma unroll
    for (int x = 0; x < NS * NC; ++x) {
      const u32x4 ka = *reinterpret_cast<const u32x4*>(s_k + ((b * TB + kofs) ^ (x / NS << 5)) +
                                                       x % NS * 32 * RB);
      sacc[x % NS] = Mma<TT>::m32(ka, qb[x / NS], sacc[x % NS]);
    }
    // scores in log2 units (without a cap or slopes: times c2 in the exponent)
    if constexpr (kCap) {
      if (__builtin_expect(a.cap_wide, 0)) {
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) sacc[n][i] = cap_exact(sacc[n][i], cin, capA);
      } else {
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) sacc[n][i] = cap_plain(sacc[n][i], cin, capA);
      }
    }
    if constexpr (kBias) {
      const float dist0 = (float)(pos - key0 - 4 * hf);
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float dist = fabsf(dist0 - (float)(n * 32 + 8 * (i >> 2) + (i & 3)));
          const float x = sacc[n][i];
          sacc[n][i] = fmaf(-slope, dist, kCap ? x : x * c2);
        }
    }
    const bool all = (key0 >= w_lo1 && key0 + KT <= w_hi0) || (key0 >= w_first1 && key0 + KT <= w_pre0);
    if (!all) {
      const int o = key0 + 4 * hf;
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = o + n * 32 + 8 * (i >> 2) + (i & 3);
          const bool seen = (key >= see.lo && key < see.hi) || (key >= see.first && key < see.pre);
          const float x = sacc[n][i];
          sacc[n][i] = seen ? x : -INFINITY;
        }
    }
    constexpr bool kScaled = !kCap && !kBias;
    const float cs = kScaled ? c2 : 1.f;
    u32x4 pb[KB];   // P^T as B operands: slots e < 4 -> key 4 hf + e, e >= 4 -> 8 + 4 hf + e - 4
    auto expo = [&]() {
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float x = sacc[n][i], y = sacc[n][i + 1];
          pb[n * 2 + (i >> 3)][(i & 7) >> 1] =
              TT::pack2(__builtin_amdgcn_exp2f(kScaled ? fmaf(x, cs, nmref) : x + nmref),
                        __builtin_amdgcn_exp2f(kScaled ? fmaf(y, cs, nmref) : y + nmref));
        }
    };
    auto sum_p = [&](float x) {
      float ps[4] = {x, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) ps[i] = TT::dot2(pb[kb][i], TT::kOne2, ps[i]);
      return (ps[0] + ps[1]) + (ps[2] + ps[3]);
    };
    expo();
    constexpr bool kBySum = std::is_same<TT, F16>::value;
    float st = 0.f;
    bool past;
    if constexpr (kBySum) {
      st = sum_p(0.f);
      past = !(st < Bound<TT>::kPast);
    } else {
      uint32_t o = 0;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        o = o | pb[kb][0] | pb[kb][1];
        o = o | pb[kb][2] | pb[kb][3];
      }
      past = (o & 0x40004000u) != 0;
    }
    if (__ballot(past) != 0) {
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sacc[n][i]);
      mx = half_max(mx) * cs;
      const bool nd = mx > mref + Bound<TT>::kMove;
      const float mnew = nd ? mx + Bound<TT>::kBias : mref;
      const float alpha = nd ? __builtin_amdgcn_exp2f(mref - mnew) : 1.f;   // 0 from -inf
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[db] *= alpha;
      lsum *= alpha;
      mref = mnew;
      nmref = mnew == -INFINITY ? kNoRef : -mnew;
      expo();
      if constexpr (kBySum) st = sum_p(0.f);
    }
    if constexpr (kBySum) lsum += st;
    else lsum = sum_p(lsum);
    const int vt = b * TB + vofs;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const int at = vt ^ (db << 6);
        const u32x2 lo = lds_read_tr(s_v + at + kb * 16 * RB);
        const u32x2 hi = lds_read_tr(s_v + (at ^ swz8<D>()) + (kb * 16 + 8) * RB);
        oacc[db] = Mma<TT>::m32(u32x4{lo.x, lo.y, hi.x, hi.y}, pb[kb], oacc[db]);
      }
  };

  // ---- the part's steps, from the last back: near ones, then far ones, each in
  // segments whose blocks fit the list
  const int64_t list_steps = (int64_t)(kListBlocks - 2) * bs / KT;
  const int seg = list_steps < 1 ? 1 : (list_steps > 1 << 20 ? 1 << 20 : (int)list_steps);
  for (int range = 1; range >= 0; --range) {
    // steps of this range in the part: [r0, r1)
    const int r0 = range ? ns0 + max(st0 - nfar, 0) : fs0 + min(st0, nfar);
    const int r1 = range ? ns0 + max(st1 - nfar, 0) : fs0 + min(st1, nfar);
    const int k0 = range ? nk0 : fk0, k1 = range ? nk1 : fk1;
    for (int e1 = r1; e1 > r0; e1 -= seg) {
      const int e0 = e1 - seg > r0 ? e1 - seg : r0;
      key_lo = max(k0, e0 * KT);
      key_hi = min(k1, e1 * KT);
      __syncthreads();       // the last segment's reads are done
      blk0 = div_bs(key_lo);
      const int nblk = div_bs(key_hi - 1) + 1 - blk0;
      for (int e = tid; e < nblk; e += kThreads) {
        const int bid = clampi(a.block_tables[(int64_t)it.s * a.max_bps + blk0 + e], 0, a.num_blocks - 1);
        s_row[e] = (bid * a.num_kv_heads + kh) * bs;
      }
      wait_all_and_barrier();
      if constexpr (kF8) {
        fetch(e1 - 1);
        stash(0);
      } else {
        load(e1 - 1, 0);
      }
      for (int i = e1 - 1, b = 0; i >= e0; --i, b ^= 1) {
        wait_all_and_barrier();    // tile i is there, and all waves have left the other buffer
        if (i > e0) {
          if constexpr (kF8) fetch(i - 1); else load(i - 1, b ^ 1);
        }
        compute(i, b);
        if constexpr (kF8) {
          if (i > e0) stash(b ^ 1);
        }
      }
    }
  }

  // ---- results
  const float ltot = half_sum(lsum);
  float chk = ltot;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) chk = fmaf(oacc[db][i], 0.f, chk);
  const bool bad = !(chk < INFINITY);          // an infinity or NaN among the row's sums
  const uint32_t bad32 = (uint32_t)__ballot(bad) | (uint32_t)(__ballot(bad) >> 32);
  const bool mine_bad = (bad32 >> c32) & 1;
  const float oscale = kF8 ? a.v_scale[kh] : 1.f;
  const int64_t slot0 = ((tile * a.num_kv_heads + kh) * a.tile_splits + part) * kTileRows + wave * 32;
  if (row_ok && !mine_bad) {
    if (!merged) {
      const float inv = ltot > 0.f ? oscale / ltot : 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = db * 32 + i * 8 + hf * 4;
          if (e < d)
            *reinterpret_cast<u32x2*>(op + e) =
                u32x2{TT::pack2(oacc[db][4 * i] * inv, oacc[db][4 * i + 1] * inv),
                      TT::pack2(oacc[db][4 * i + 2] * inv, oacc[db][4 * i + 3] * inv)};
        }
    } else {
      float* po = a.tile_o + (slot0 + c32) * d;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = db * 32 + i * 8 + hf * 4;
          if (e < d)
            *reinterpret_cast<f32x4*>(po + e) = f32x4{oacc[db][4 * i], oacc[db][4 * i + 1],
                                                      oacc[db][4 * i + 2], oacc[db][4 * i + 3]};
        }
      if (hf == 0) {
        a.tile_ml[(slot0 + c32) * 2] = mref;
        a.tile_ml[(slot0 + c32) * 2 + 1] = ltot;
      }
    }
  }
  if (__builtin_expect(bad32 == 0, 1)) return;

  // ---- redo of rows whose sums are not finite: one key after another, over the
  // keys that the row sees in this part; lane l holds dims 4l .. 4l + 3
  for (int r = 0; r < 32; ++r) {
    if (!((bad32 >> r) & 1) || f0 + r >= it.rows) continue;
    auto of = [&](int x) { return __builtin_amdgcn_readlane(x, r); };
    const int rlo = of(see.lo), rhi = of(see.hi), rfirst = of(see.first), rpre = of(see.pre);
    const int rpos = of(pos), rtok = of(qrow), rh = of(h);
    const float rslope = kBias ? a.slopes[rh] * kLog2e : 0.f;
    const int e0 = lane * 4;
    const bool on = e0 < d;
    float qv[4] = {0, 0, 0, 0}, o[4] = {0, 0, 0, 0};
    if (on) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(a.q + (int64_t)rtok * a.q_stride_token +
                                                      (int64_t)rh * a.q_stride_head + e0);
      qv[0] = TT::lo(w.x), qv[1] = TT::hi(w.x), qv[2] = TT::lo(w.y), qv[3] = TT::hi(w.y);
    }
    float m = -INFINITY, l = 0.f;
    for (int i = st0; i < st1; ++i) {
      const int step = i < nfar ? fs0 + i : ns0 + (i - nfar);
      for (int key = step * KT; key < step * KT + KT; ++key) {
        if (!((key >= rlo && key < rhi) || (key >= rfirst && key < rpre))) continue;
        const int lb = div_bs(key);
        const int bid = clampi(a.block_tables[(int64_t)it.s * a.max_bps + lb], 0, a.num_blocks - 1);
        const int64_t off = ((int64_t)(bid * a.num_kv_heads + kh) * bs + (key - lb * bs)) * rowb + e0 * EB;
        float kv[4] = {0, 0, 0, 0}, vv[4] = {0, 0, 0, 0};
        if (on) {
          u32x2 kw, vw;
          if constexpr (kF8) {
            const uint32_t kb = *reinterpret_cast<const uint32_t*>(a.k_cache + off);
            const uint32_t vb = *reinterpret_cast<const uint32_t*>(a.v_cache + off);
            kw = u32x2{e4m3x2_to<TT, false>(kb), e4m3x2_to<TT, true>(kb)};
            vw = u32x2{e4m3x2_to<TT, false>(vb), e4m3x2_to<TT, true>(vb)};
          } else {
            kw = *reinterpret_cast<const u32x2*>(a.k_cache + off);
            vw = *reinterpret_cast<const u32x2*>(a.v_cache + off);
          }
          kv[0] = TT::lo(kw.x), kv[1] = TT::hi(kw.x), kv[2] = TT::lo(kw.y), kv[3] = TT::hi(kw.y);
          vv[0] = TT::lo(vw.x), vv[1] = TT::hi(vw.x), vv[2] = TT::lo(vw.y), vv[3] = TT::hi(vw.y);
        }
        float t = fmaf(qv[0], kv[0], qv[1] * kv[1]) + fmaf(qv[2], kv[2], qv[3] * kv[3]);
        t = wave_sum_f(t);
        t = kCap ? cap_exact(t, cin, capA) : t * c2;
        if (kBias) t = fmaf(-rslope, fabsf((float)(rpos - key)), t);
        const float mn = fmaxf(m, t);
        const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        const float p = __builtin_amdgcn_exp2f(t - mn);   // NaN scores, and +inf ones, give NaN
        l = l * al + p;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * al + p * vv[e];
        m = mn;
      }
    }
    if (!merged) {
      const float inv = l > 0.f || l != l ? oscale / l : 0.f;
      if (on)
        *reinterpret_cast<u32x2*>(a.out + (int64_t)rtok * a.out_stride_token +
                                  (int64_t)rh * a.out_stride_head + e0) =
            u32x2{TT::pack2(o[0] * inv, o[1] * inv), TT::pack2(o[2] * inv, o[3] * inv)};
    } else {
      if (on) *reinterpret_cast<f32x4*>(a.tile_o + (slot0 + r) * d + e0) = f32x4{o[0], o[1], o[2], o[3]};
      if (lane == 0) {
        a.tile_ml[(slot0 + r) * 2] = m;
        a.tile_ml[(slot0 + r) * 2 + 1] = l;
      }
    }
  }
}

template <class TT, int D, bool kF8>
void launch_rows_f(const Args& a, hipStream_t st) {
  const int64_t tiles = a.cu_seqlens_q ? (int64_t)a.num_seqs * a.tiles_max : a.tiles;
  const dim3 g((unsigned)(tiles * a.num_kv_heads * a.tile_splits)), b(kThreads);
  const bool cap = a.cap_log2 > 0.f, bias = a.slopes != nullptr;
  if (cap && bias) hipLaunchKernelGGL((rows_kernel<TT, D, kF8, true, true>), g, b, 0, st, a);
  else if (cap) hipLaunchKernelGGL((rows_kernel<TT, D, kF8, true, false>), g, b, 0, st, a);
  else if (bias) hipLaunchKernelGGL((rows_kernel<TT, D, kF8, false, true>), g, b, 0, st, a);
  else hipLaunchKernelGGL((rows_kernel<TT, D, kF8, false, false>), g, b, 0, st, a);
}

template <int D>
void launch_rows(const Args& a, int32_t dtype, hipStream_t st) {
  if (dtype == NPD_DTYPE_BF16) {
    if (a.k_scale) launch_rows_f<BF16, D, true>(a, st);
    else launch_rows_f<BF16, D, false>(a, st);
  } else {
    if (a.k_scale) launch_rows_f<F16, D, true>(a, st);
    else launch_rows_f<F16, D, false>(a, st);
  }
}

}  // namespace scored
}  // namespace npd
