// Attention with changed scores (scored.h): the kernel for many query rows that
// read the same keys -- prompt chunks, and the tokens of a group of sequences
// over their shared prefix.
//
// Workgroup: 4 waves of 32 flattened (token, head) rows of one kv head, and a part
// of the keys they see. K/V tiles of 32 keys load straight into LDS
// (global_load_lds, 16 bytes per lane; FP8 bytes through registers, converted
// exactly), the next ones under the step. Per step a wave forms
//   S^T = K . Q^T     (32x32x16 MFMA, its 32 query rows in registers),
//   P   = 2^(t - m)   (scored.h; masks only in steps that some row sees in part),
//   O^T += V^T . P^T  (V through transposing LDS reads).
// A row's reference m moves only where a P grew past a bound (kPast), so no
// maximum is taken in the usual step. Steps run from the last key back: the
// newest keys come first, which with a distance term hold the largest scores.
//
// What bounds it: three things of like size that do not overlap fully. Of a step at
// 128 dims (128 rows by 32 keys) a compute unit's MFMAs take 0.22 us, the issue of a
// capped softmax 0.25 (per score two exponentials or reciprocals and one more, 8
// cycles an instruction, others 4; both together, measured in registers alone, 0.31)
// and the LDS reads of K and V operands, 64 KB, 0.21; in place a step takes 0.6.
// Workgroups of one compute unit run unsynchronised, one's waits under another's
// issue: three (168 registers, operands read two ahead of their MFMA) take 1359 us
// over 12000 tokens of 32 / 8 heads of 128, capped (868 TFLOP/s of the 1263 that a
// large matrix product reaches), two 1436. At 256 dims one workgroup has the unit:
// for two, 200 bytes of registers spill within the loop (packed documents: 221 us
// against 130).
//
// Masked keys: P is 0 by selection, but 0 times an infinity or NaN in V is NaN,
// and rows of a tile do not see the same keys. So a row whose result is not
// finite is computed again, key by key over what it sees (redo_row); a finite
// result had no such product.
//
// Shares: where whole tiles would leave the chip uneven, its workgroups take equal
// shares of all tiles' steps, laid end to end (rows_share), from the lengths on the
// device. A share may end one tile, hold whole ones and begin another; the pieces
// of a tile meet in the merge kernel. A piece costs 10 to 13 us besides its steps
// (finding it 4, its rows and ranges 4, its list of blocks 1.4, the first tiles 2,
// storing 2.5), a step 0.65 us of a compute unit. Chunks of 300 to 512 tokens over
// 3000, shared out: 112 us; cut into equal parts of each tile: 122.
#pragma once

#include "scored_stream.h"

namespace npd {
namespace scored {

constexpr int kThreads = 256;
constexpr int kListEntries = 512;    // pool blocks listed in LDS at a time
constexpr int kPieces = 4;           // pieces of a share listed at a time

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
// At most N direct loads of this wave are in flight, its LDS accesses are done;
// then the workgroup's barrier.
template <int N>
__device__ __forceinline__ void wait_and_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}
constexpr int kWaitVm0 = 0x0f70;            // s_waitcnt vmcnt(0), the other counters free

// When a row's reference moves. bf16: it sits kBias above the maximum it was
// taken from, and a P of 2 or more (bit 14 of a half) asks for a new one. fp16
// keeps it at the maximum, and asks where a lane's 16 P of a step come to 2^8 or
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

// A piece of a workgroup's work: cost units from / est .. to / est of a tile.
struct Piece {
  int s;          // block table row
  int row0;       // first token row of q / out
  int tokens;     // tokens of the chunk, or sequences of the group
  int t;          // tile of them
  int limit;      // keys at or past it belong to no row here (context, or shared keys)
  int tile;       // index of the tile among all
  int from, to, est;
};

// Pieces from cost `done` on of the share of workgroup id, up to kPieces, by one
// wave into out (past the share's end: est == 0). The tiles,
// each at its cost, are laid end to end (chunks: from the last of the last
// sequence; a tile's steps are those of its causal range, window and first
// document, an estimate: what its rows see decides) and cut at multiples of the
// share; a cut near a tile's edge moves there. sum: running costs (kListEntries).
__device__ __forceinline__ void rows_share(const Args& a, int id, int done, int lane, int* sum, Piece* out) {
  const int G = a.group, cap = a.max_bps * a.block_size, shift = a.cost_shift;
  const bool chunks = a.cu_seqlens_q != nullptr;
  auto cost = [&](int steps) { return max(1, (steps + kTileCost) >> shift); };
  auto chunk = [&](int sq, int& q0, int& ql, int& cx) {
    q0 = clampi(a.cu_seqlens_q[sq], 0, a.total_q);
    ql = clampi(a.cu_seqlens_q[sq + 1], q0, a.total_q) - q0;
    cx = clampi(a.seq_lens[sq], 0, cap);
  };
  auto group_tiles = [&](const Group& g) { return (int)(((int64_t)g.seqs * G + kTileRows - 1) / kTileRows); };
  auto group_cost = [&](const Group& g) { return g.shared > 0 ? cost((g.shared + kStepKeys - 1) / kStepKeys) : 0; };
  // entry e: tile all - 1 - e of num_seqs * tiles_max, or `per` groups
  const int all = a.num_seqs * a.tiles_max;
  const int per = chunks ? 1 : (a.num_groups + kListEntries - 1) / kListEntries;
  const int n = chunks ? all : (a.num_groups + per - 1) / per;
  int total = 0;
#pragma unroll 1
  for (int e0 = 0; e0 < n; e0 += 64) {
    const int e = e0 + lane;
    int c = 0;
    if (e < n) {
      if (chunks) {
        const int i = all - 1 - e, sq = i / a.tiles_max, t = i - sq * a.tiles_max;
        int q0, ql, cx;
        chunk(sq, q0, ql, cx);
        if (t * kTileRows < ql * G) {
          const int tok = t * kTileRows / G;
          const int p0 = cx - ql + tok, p1 = cx - ql + min(ql, ((t + 1) * kTileRows + G - 1) / G);
          int lo = a.first_keys ? a.first_keys[q0 + tok] : 0;
          if (a.window > 0) lo = max(lo, p0 - a.window + 1);
          c = cost(max(0, (max(p1, 0) + kStepKeys - 1) / kStepKeys - max(lo, 0) / kStepKeys));
        }
      } else {
#pragma unroll 1
        for (int g = e * per; g < min((e + 1) * per, a.num_groups); ++g) {
          const Group r = group_at(a, g);
          c += group_tiles(r) * group_cost(r);
        }
      }
    }
    c = total + wave_scan_i(c);
    sum[e] = c;
    total = __builtin_amdgcn_readlane(c, 63);
  }
  wave_sync();
  // cut k of `shares`, at k / shares of the total but for the tilt: the workgroups
  // of a compute unit do not run equally fast, its waves issue in the order of
  // their age (three of them: steps of 1.45, 1.9 and 2.45 us; shares that are all
  // alike end at 64, 81 and 93 us, tilted ones together)
  // (shares in whole rounds over the compute units, where they are more than one)
  int shares = min(a.room, total / kMinShare + 1);
  if (shares > a.room1) shares -= shares % a.room1;
  const int tilt = clampi(3 * (shares - a.room1) / a.room1, 0, 6);   // sixteenths
  Piece pc{};
  // the tile at cost x: its number in its entry, where it begins, its cost
  int at, own;
  auto find = [&](int x) {
    int e = 0;
#pragma unroll 1
    for (int e0 = 0; e0 < n; e0 += 64) {
      const uint64_t m = __ballot(e0 + lane < n && sum[e0 + lane] > x);
      if (m != 0) {
        e = e0 + __builtin_ctzll(m);
        break;
      }
    }
    at = e > 0 ? sum[e - 1] : 0;
    own = sum[e] - at;
    if (chunks) {
      const int i = all - 1 - e;
      pc.s = i / a.tiles_max;
      pc.t = i - pc.s * a.tiles_max;
    } else {
      Group r = group_at(a, e * per);
#pragma unroll 1
      for (int g = e * per + 1; g < min((e + 1) * per, a.num_groups); ++g) {
        const int c = group_tiles(r) * group_cost(r);
        if (x < at + c) break;
        at += c;
        r = group_at(a, g);
      }
      own = max(1, group_cost(r));
      pc.t = (x - at) / own;
      at += pc.t * own;
      pc.s = pc.row0 = r.seq0;
      pc.tokens = r.seqs;
      pc.limit = r.shared;
    }
  };
  // a cut between shares
  auto edge = [&](int k) {
    if (k >= shares) return total;
    const int u = (int)((int64_t)total * k / shares);
    const int x = u + (int)((int64_t)u * (shares - k) / shares * tilt / 16);
    find(x);
    return x - at < kNearEdge ? at : at + own - x < kNearEdge ? at + own : x;
  };
  int g = edge(id) + done;
  const int g1 = edge(id + 1);
#pragma unroll 1
  for (int p = 0; p < kPieces; ++p) {
    pc = Piece{};
    if (g < g1) {
      find(g);
      bool ok = true;
      if (chunks) {
        chunk(pc.s, pc.row0, pc.tokens, pc.limit);
        pc.tile = pc.s * a.tiles_max + pc.t;
      } else {
        Group r;
        ok = find_group(a, pc.s, lane, r) && r.tile0 + pc.t < a.tiles;   // (not: groups that overlap)
        pc.tile = r.tile0 + pc.t;
      }
      pc.from = g - at;
      pc.to = min(g1 - at, own);
      g += pc.to - pc.from;
      // (not: costs past 2^31, of lists that do not ascend)
      if (ok && pc.t >= 0 && pc.from >= 0 && pc.to > pc.from) pc.est = own;
      else g = g1;
    }
    if (lane == 0) out[p] = pc;
  }
}

// kCapped: no cap, a plain one, or one past kCapPlain.
enum Capped { kNoCap, kPlainCap, kWideCap };
template <int D>
struct RowsLds {
  static constexpr int kBufs = D > 128 ? 2 : 3;    // K and V tiles
  char k[kBufs * kStepKeys * D * 2];
  char v[kBufs * kStepKeys * D * 2];
  Keys see[kTileRows];        // keys of the rows (read where a step masks)
  int row[kListEntries];      // pool rows of the segment's blocks
  int red[4][4];
  Piece piece[kPieces];
};
// One piece of workgroup id of kv head kh.
template <class TT, int D, bool kF8, Capped kCapped, bool kBias>
__device__ __forceinline__ void rows_piece(const Args& a, const Piece& it, int id, int kh, bool first,
                                           int tid, RowsLds<D>& lds) {
  constexpr int KT = kStepKeys;
  constexpr int TR = kTileRows;
  constexpr int kBufs = RowsLds<D>::kBufs;
  constexpr int kAhead = D > 128 ? 4 : 2;   // LDS operand reads ahead of their MFMA
  constexpr int RB = 2 * D;                 // bytes of a tile row
  constexpr int TB = KT * RB;               // bytes of a tile
  constexpr int NI = TB / 4096;             // 1 KB loads per wave and tile
  constexpr int NC = D / 16, KB = KT / 16, DB = D / 32;
  constexpr int EB = kF8 ? 1 : 2;
  constexpr bool kCap = kCapped != kNoCap;
  static_assert(KT == 32 && NI >= 1, "one 32-key block per step");
  char* s_k = lds.k;
  char* s_v = lds.v;
  int* s_row = lds.row;
  auto& s_red = lds.red;
  Keys* s_see = lds.see;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, c32 = lane & 31;
  const int G = a.group, d = a.head_dim, bs = a.block_size;
  const int cap_keys = a.max_bps * bs;
  auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };

  const int frows = it.tokens * G;

  // ---- this lane's row (past the last: a copy of it, not stored)
  const int f0 = it.t * TR + wave * 32;
  struct Row {
    bool ok;
    int tok, h, q;     // token of the chunk or sequence of the group, head, row of q / out
    __device__ int64_t strides(int64_t token, int64_t head) const { return q * token + h * head; }
  };
  auto row_of = [&](int c) {
    Row r;
    r.ok = f0 + c < frows;
    const int f = r.ok ? f0 + c : frows - 1;
    r.tok = f / G;
    r.h = kh * G + (f - r.tok * G);
    r.q = it.row0 + r.tok;
    return r;
  };
  const Row row = row_of(c32);
  const int row_len = a.cu_seqlens_q ? 0 : a.seq_lens[row.q];
  const int row_first = a.first_keys ? a.first_keys[row.q] : 0;
  const int row_pre = a.prefix_lens ? a.prefix_lens[it.s] : 0;

  // ---- queries as B operands: qb[c] = Q[row][16c + 8 hf ..], zeros past the row
  u32x4 qb[NC];
  {
    const uint16_t* qp = a.q + row.strides(a.q_stride_token, a.q_stride_head);
#pragma unroll
    for (int c = 0; c < NC; ++c)
      qb[c] = c * 16 + hf * 8 < d ? *reinterpret_cast<const u32x4*>(qp + c * 16 + hf * 8)
                                  : u32x4{0, 0, 0, 0};
  }
  int pos, ctx;
  if (a.cu_seqlens_q) {
    ctx = it.limit;
    pos = ctx - it.tokens + row.tok;
  } else {
    ctx = clampi(row_len, 0, cap_keys);
    pos = ctx - 1;
  }
  Keys see = row_keys(pos, ctx, row_first, row_pre, a.window);
  see.hi = min(see.hi, it.limit);
  see.pre = min(see.pre, it.limit);
  if (see.lo >= see.hi) see.lo = see.hi = 0;          // empty ranges are [0, 0)
  if (see.first >= see.pre) see.first = see.pre = 0;
  if (hf == 0) s_see[wave * 32 + c32] = see;

  // ---- ranges: near [lo, hi), far [first, pre); of the wave (none where it has no
  // row to store) and of the workgroup the keys that some row sees, and of the wave
  // those that every row sees
  constexpr int kFarKey = 0x7fffffff;
  const bool idle = f0 >= frows;
  const int w_lo = idle ? kFarKey : wave_min_i(see.hi > 0 ? see.lo : kFarKey);
  const int w_hi = idle ? 0 : wave_max_i(see.hi);
  const int w_first = idle ? kFarKey : wave_min_i(see.pre > 0 ? see.first : kFarKey);
  const int w_pre = idle ? 0 : wave_max_i(see.pre);
  // (a wave without a row masks nothing: its results go nowhere)
  const int w_lo1 = idle ? 0 : wave_max_i(see.lo), w_hi0 = idle ? kFarKey : wave_min_i(see.hi);
  const int w_first1 = wave_max_i(see.first), w_pre0 = wave_min_i(see.pre);
  if (lane == 0) {
    s_red[0][wave] = w_lo;
    s_red[1][wave] = w_hi;
    s_red[2][wave] = w_first;
    s_red[3][wave] = w_pre;
  }
  __syncthreads();
  auto least = [&](const int (&x)[4]) { return uni(min(min(x[0], x[1]), min(x[2], x[3]))); };
  auto most = [&](const int (&x)[4]) { return uni(max(max(x[0], x[1]), max(x[2], x[3]))); };
  const int nlo = least(s_red[0]), nhi = most(s_red[1]), flo = least(s_red[2]), fhi = most(s_red[3]);
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
  // steps of the piece; where its results go: rows of out, or a slot of partials
  // (a share's first piece may begin within a tile, its last end within one)
  const bool whole_tile = it.from == 0 && it.to == it.est;
  const bool merged = a.cu_groups || !whole_tile;
  const int64_t slot = whole_tile ? 2 * (int64_t)a.room + it.tile : 2 * (int64_t)id + (first ? 0 : 1);
  if (tid == 0 && a.tile_items) {
    int32_t* e = a.tile_items + 4 * ((int64_t)it.tile * a.num_kv_heads + kh);
    if (it.from == 0) {
      e[0] = (int)slot;
      e[1] = id;
    }
    if (it.to == it.est) e[2] = id;
  }
  const int st0 = (int)((int64_t)it.from * nsteps / it.est);
  const int st1 = (int)((int64_t)it.to * nsteps / it.est);

  const float kscale = kF8 ? a.k_scale[kh] : 1.f;
  const float c2 = a.scale_log2 * kscale, cin = a.cap_in * kscale, capA = a.cap_log2;
  const float slope = kBias ? a.slopes[row.h] * kLog2e : 0.f;

  // ---- tile loads. Chunks past the row's end repeat its last one (zero queries
  // meet them in S, and their output dims are not stored).
  const int64_t rowb = (int64_t)d * EB;
  const int last16 = (int)(rowb / 16) - 1;
  constexpr int LROW = kF8 ? D / 16 : RB / 16;         // lanes per row
  constexpr int NR = kF8 ? (KT * LROW + kThreads - 1) / kThreads : NI;
  constexpr bool kSome = kF8 && KT * LROW < kThreads;  // some threads load
  // load e of a lane: tile row lrow0 + e * kRows, column lcol[e]
  constexpr int kRows = kF8 ? kThreads / LROW : 1024 / RB;
  const int lrow0 = kF8 ? tid / LROW : (wave * NI * 1024 + lane * 16) / RB;
  uint32_t lcol[NR];
#pragma unroll
  for (int e = 0; e < NR; ++e) {
    const int c = kF8 ? tid % LROW : (lane * 16 % RB / 16) ^ swz<D>(lrow0 + e * kRows);
    lcol[e] = (uint32_t)(c < last16 ? c : last16) * 16;
  }
  const uint32_t lds_k = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_k;
  const uint32_t lds_v = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_v;
  // s_row lists the first pool row of each block, or, where the block size is no
  // power of two, of each key. A step that lies within the keys to load takes its
  // rows by a list entry and an offset in the block that are a part of the lane's
  // and a part of the step's; the others clamp key by key.
  const int sh = a.bs_shift >= 0 ? a.bs_shift : 0, in_blk = (1 << sh) - 1;
  int ent0 = 0, key_lo = 0, key_hi = 0;    // of the segment: first entry listed, keys loaded
  // Of the tile loaded next: pool rows less the offsets off_blk + row_o (added where
  // they are used, so that the wait for the list falls there)
  int rows[NR], row_o = 0;
  auto off_blk = [&](int e) { return (lrow0 + e * kRows) & in_blk; };
  auto find_rows = [&](int step) {
    const int k0 = step * KT;
    row_o = k0 & in_blk;   // (0 for blocks up to KT)
    if (k0 >= key_lo && k0 + KT <= key_hi) {
      const int ent = (k0 >> sh) - ent0;
#pragma unroll
      for (int e = 0; e < NR; ++e) rows[e] = s_row[ent + ((lrow0 + e * kRows) >> sh)];
    } else {
#pragma unroll
      for (int e = 0; e < NR; ++e) {
        const int key = max(key_lo, min(key_hi - 1, k0 + lrow0 + e * kRows));
        rows[e] = s_row[(key >> sh) - ent0] + (key & in_blk) - off_blk(e) - row_o;
      }
    }
  };
  auto byte_at = [&](int e) {   // of this lane's load e
    return (int64_t)((uint64_t)(uint32_t)(rows[e] + off_blk(e) + row_o) * (uint32_t)rowb) + lcol[e];
  };
  auto load = [&](int buf) {   // 2-byte pools: the tile of `rows`
#pragma unroll
    for (int e = 0; e < NR; ++e) {
      const int64_t at = byte_at(e);
      const uint32_t run = (uint32_t)(buf * TB + (wave * NI + e) * 1024);
      load_to_lds(lds_k + run, a.k_cache + at);
      load_to_lds(lds_v + run, a.v_cache + at);
    }
  };
  struct Raw {
    u32x4 w[kF8 ? NR : 1];
  };
  auto fetch = [&](Raw& rk, Raw& rv) {   // FP8 pools: the bytes of `rows` into registers ...
    if (kSome && tid >= KT * LROW) return;
#pragma unroll
    for (int e = 0; e < NR; ++e) {
      const int64_t at = byte_at(e);
      rk.w[kF8 ? e : 0] = *reinterpret_cast<const u32x4*>(a.k_cache + at);
      rv.w[kF8 ? e : 0] = *reinterpret_cast<const u32x4*>(a.v_cache + at);
    }
  };
  auto stash = [&](const Raw& rk, const Raw& rv, int buf) {   // ... and converted into LDS
    if (kSome && tid >= KT * LROW) return;
#pragma unroll
    for (int e = 0; e < NR; ++e) {
      const int c = tid % LROW * 2, row = lrow0 + e * kRows, sw = swz<D>(row);
      const int at = buf * TB + row * RB;
      const u32x4 k = rk.w[kF8 ? e : 0], v = rv.w[kF8 ? e : 0];
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
  float nmref = kNoRef, lsum = 0.f;   // the reference's negative (kNoRef: none yet); P's sum

  const int kofs = c32 * RB + ((hf ^ swz<D>(c32)) << 4);
  const int vrow = 4 * hf + ((lane & 15) >> 2);
  const int vofs = vrow * RB + (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ swz<D>(vrow)) << 4) +
                   (lane & 1) * 8;
  // Exponent arguments are S * cs + off + nmref. Without a cap or slopes S is the
  // product itself; with a plain cap S = 1 / (1 + e^2y), whose last step A - 2A S
  // joins the exponent's FMA; else S is the score in log2 units.
  constexpr bool kUnit = kBias || kCapped == kWideCap, kRecip = kCapped == kPlainCap && !kBias;
  const float cs = kUnit ? 1.f : (kRecip ? -2.f * capA : c2);
  const float off = kRecip ? capA : 0.f;
  const float hidden = kRecip ? INFINITY : -INFINITY;   // S of a masked key
  constexpr bool kBySum = std::is_same<TT, F16>::value;
  constexpr int NPV = KB * DB;    // P.V operands of a step
  constexpr f32x16 kZero = {0};

  // Step i over the K and V tiles kt, vt
  auto step = [&](int i, const char* kt, const char* vt) {
    const int key0 = i * KT;
    // (products first where waves of a SIMD compete: their operands come from LDS)
    __builtin_amdgcn_s_setprio(1);
    f32x16 s;   // S^T[key 8 (i/4) + 4 hf + i%4][row c32]
    {
      u32x4 ka[NC];
      auto read = [&](int x) { ka[x] = *reinterpret_cast<const u32x4*>(kt + (kofs ^ (x << 5))); };
#pragma unroll
      for (int x = 0; x < kAhead; ++x) read(x);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        if (x + kAhead < NC) read(x + kAhead);
        s = Mma<TT>::m32(ka[x], qb[x], x == 0 ? kZero : s);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (kCapped == kPlainCap) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = s[e];
        const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * cin) + 1.f);
        s[e] = kBias ? fmaf(-2.f * capA, r, capA) : r;
      }
    } else if constexpr (kCapped == kWideCap) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = s[e];
        s[e] = cap_exact(x, cin, capA);
      }
    }
    if constexpr (kBias) {
      const float dist0 = (float)(pos - key0 - 4 * hf);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = s[e], dist = fabsf(dist0 - (float)(8 * (e >> 2) + (e & 3)));
        s[e] = fmaf(-slope, dist, kCap ? x : x * c2);
      }
    }
    const bool whole = (key0 >= w_lo1 && key0 + KT <= w_hi0) || (key0 >= w_first1 && key0 + KT <= w_pre0);
    if (!whole) {
      const Keys ks = s_see[wave * 32 + c32];
      const int o = key0 + 4 * hf;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = o + 8 * (e >> 2) + (e & 3);
        const bool seen = (key >= ks.lo && key < ks.hi) || (key >= ks.first && key < ks.pre);
        const float x = s[e];
        s[e] = seen ? x : hidden;
      }
    }
    // P^T as B operands: slots e < 4 -> key 4 hf + e, e >= 4 -> 8 + 4 hf + e - 4
    // (pairs of scalars up to the products: vectors here are put together in an
    // else branch of the rare case below, and every accumulator is copied for it)
    uint32_t pb[8];
    auto expo = [&]() {
      const float o = off + nmref;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float x = s[e], y = s[e + 1];
        pb[e >> 1] = TT::pack2(__builtin_amdgcn_exp2f(kUnit ? x + o : fmaf(x, cs, o)),
                                             __builtin_amdgcn_exp2f(kUnit ? y + o : fmaf(y, cs, o)));
      }
    };
    auto sum_p = [&](float x) {
      float y = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        x = TT::dot2(pb[e], TT::kOne2, x);
        y = TT::dot2(pb[e + 1], TT::kOne2, y);
      }
      return x + y;
    };
    expo();
    float st = 0.f;
    bool past;
    if constexpr (kBySum) {
      st = sum_p(0.f);
      past = !(st < Bound<TT>::kPast);
    } else {
      uint32_t o = pb[0] | pb[1] | pb[2];
      o = o | pb[3] | pb[4];
      o = o | pb[5] | pb[6];
      past = ((o | pb[7]) & 0x40004000u) != 0;
    }
    if (__builtin_expect(__ballot(past) != 0, 0)) {
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = s[e];
        mx = fmaxf(mx, kUnit ? x : fmaf(x, cs, off));
      }
      mx = half_max(mx);
      // (without a reference -nmref is below any score, and alpha 0)
      const bool nd = mx > Bound<TT>::kMove - nmref;
      const float mnew = mx + Bound<TT>::kBias;
      const float alpha = nd ? __builtin_amdgcn_exp2f(-nmref - mnew) : 1.f;
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[db] *= alpha;
      lsum *= alpha;
      nmref = nd ? -mnew : nmref;
      expo();
      if constexpr (kBySum) st = sum_p(0.f);
    }
    __builtin_amdgcn_s_setprio(1);
    u32x4 va[NPV];
    auto read = [&](int x) {   // 16-key block x / DB, 32-dim block x % DB
      const int at = vofs ^ (x % DB << 6);
      const u32x2 lo = lds_read_tr(vt + at + x / DB * 16 * RB);
      const u32x2 hi = lds_read_tr(vt + (at ^ swz8<D>()) + (x / DB * 16 + 8) * RB);
      va[x] = u32x4{lo.x, lo.y, hi.x, hi.y};
    };
#pragma unroll
    for (int x = 0; x < kAhead; ++x) read(x);
    if constexpr (kBySum) lsum += st;
    else lsum = sum_p(lsum);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < NPV; ++x) {
      if (x + kAhead < NPV) read(x + kAhead);
      oacc[x % DB] = Mma<TT>::m32(va[x], u32x4{pb[x / DB * 4], pb[x / DB * 4 + 1], pb[x / DB * 4 + 2],
                                               pb[x / DB * 4 + 3]}, oacc[x % DB]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };

  // ---- the part's steps, from the last back: near ones, then far ones, each in
  // segments whose blocks fit the list. Count n up from a segment's last step; tile
  // n + kBufs - 1 starts loading in step n, into the buffer that step n - 1 read.
  const int64_t list_steps = ((int64_t)(kListEntries - 2) << sh) / KT;
  const int seg = list_steps > 1 << 20 ? 1 << 20 : (int)list_steps;
  Raw rk, rv;
  for (int c = st1 - 1; c >= st0;) {
    const bool near = c >= nfar;
    const int c0 = max(max(st0, near ? nfar : 0), c - seg + 1);
    const int N = c - c0 + 1, top = near ? ns0 + (c - nfar) : fs0 + c;
    c = c0 - 1;
    key_lo = max(near ? nk0 : fk0, (top + 1 - N) * KT);
    key_hi = min(near ? nk1 : fk1, (top + 1) * KT);
    __syncthreads();       // the last segment's reads are done
    ent0 = key_lo >> sh;
    const int nent = ((key_hi - 1) >> sh) + 1 - ent0;
    for (int e = tid; e < nent; e += kThreads) {
      const int key = (ent0 + e) << sh, lb = a.bs_shift >= 0 ? ent0 + e : key / bs;
      const int bid = clampi(a.block_tables[(int64_t)it.s * a.max_bps + lb], 0, a.num_blocks - 1);
      s_row[e] = (bid * a.num_kv_heads + kh) * bs + (key - lb * bs);
    }
    // none of the compiler's own loads stays in flight: its waits inside the loop
    // would cover the tile loads too
    __builtin_amdgcn_s_waitcnt(kWaitVm0);
    __syncthreads();
    find_rows(top);
    if constexpr (kF8) {
      fetch(rk, rv);
      stash(rk, rv, 0);
      if (N > 1) find_rows(top - 1);
    } else {
      load(0);
      if (N > 1) find_rows(top - 1);
      if (kBufs > 2) {
        if (N > 1) load(1);
        if (N > 2) find_rows(top - 2);
      }
    }
    // step n over the tiles in buffer `buf` (a constant)
    auto body = [&](int n, int buf) {
      constexpr int kFar = kF8 ? 1 : kBufs - 1;   // steps that loads start ahead
      if constexpr (kF8) {
        wait_and_barrier<63>();
        if (n + kFar < N) fetch(rk, rv);
      } else {
        if (kBufs > 2 && n + 1 < N) wait_and_barrier<2 * NR>();   // tile n + 1 may be in flight
        else wait_and_barrier<0>();
        if (n + kFar < N) load((buf + kBufs - 1) % kBufs);
      }
      if (n + kFar + 1 < N) find_rows(top - n - kFar - 1);
      step(top - n, s_k + buf * TB, s_v + buf * TB);
      if constexpr (kF8) {
        if (n + 1 < N) stash(rk, rv, (buf + 1) % kBufs);
      }
    };
    for (int n = 0; n < N;) {
      body(n, 0);
      if (++n >= N) break;
      body(n, 1);
      if (++n >= N) break;
      if constexpr (kBufs > 2) {
        body(n, 2);
        ++n;
      }
    }
  }

  // ---- results
  const float ltot = half_sum(lsum);
  float chk = ltot;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = oacc[db][i];
      chk = fmaf(x, 0.f, chk);
    }
  const uint64_t bad = __ballot(!(chk < INFINITY));   // an infinity or NaN among the row's sums
  const uint32_t bad_rows = (uint32_t)bad | (uint32_t)(bad >> 32);
  const float oscale = kF8 ? a.v_scale[kh] : 1.f;
  const int64_t slot0 = (slot * a.num_kv_heads + kh) * TR + wave * 32;
  int c = c32;   // (opaque: the row is found again, not kept through the loop)
  asm volatile("" : "+v"(c));
  const Row dst = row_of(c);
  uint16_t* op = a.out + dst.strides(a.out_stride_token, a.out_stride_head);
  if (dst.ok && !((bad_rows >> c) & 1)) {
    const float inv = ltot > 0.f ? oscale / ltot : 0.f;
    if (merged) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = db * 32 + i * 8 + hf * 4;
          if (e >= d) continue;
          *reinterpret_cast<f32x4*>(a.tile_o + (slot0 + c) * d + e) =
              f32x4{oacc[db][4 * i], oacc[db][4 * i + 1], oacc[db][4 * i + 2], oacc[db][4 * i + 3]};
        }
    } else {
      // of 16 dims the lane has 4 hf .. + 3 and 8 + 4 hf ..; the other half of the wave,
      // which holds the same row, gives it those that make eight in a row
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const int e = db * 32 + i * 8 + hf * 8;
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = TT::pack2(oacc[db][4 * i + 2 * k] * inv, oacc[db][4 * i + 2 * k + 1] * inv);
          const auto p = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
          const auto q = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
          if (e < d) *reinterpret_cast<u32x4*>(op + e) = u32x4{p[0], q[0], p[1], q[1]};
        }
    }
    if (merged && hf == 0) {
      a.tile_ml[(slot0 + c) * 2] = nmref == kNoRef ? -INFINITY : -nmref;
      a.tile_ml[(slot0 + c) * 2 + 1] = ltot;
    }
  }
  if (__builtin_expect(bad_rows == 0, 1)) return;

  // ---- redo of rows whose sums are not finite: one key after another, over the
  // keys that the row sees in this part; lane l holds dims 4l .. 4l + 3
  for (int w = 0; w < 32; ++w) {
    if (!((bad_rows >> w) & 1) || f0 + w >= frows) continue;
    const Keys ks = s_see[wave * 32 + w];
    const Row rr = row_of(w);
    const int rh = rr.h, rpos = a.cu_seqlens_q ? it.limit - it.tokens + rr.tok
                                               : clampi(a.seq_lens[rr.q], 0, cap_keys) - 1;
    const float rslope = kBias ? a.slopes[rh] * kLog2e : 0.f;
    const int d0 = lane * 4;
    const bool on = d0 < d;
    auto widen = [](u32x2 x, float (&f)[4]) {
      f[0] = TT::lo(x.x), f[1] = TT::hi(x.x), f[2] = TT::lo(x.y), f[3] = TT::hi(x.y);
    };
    float qv[4] = {0, 0, 0, 0}, o[4] = {0, 0, 0, 0};
    if (on)
      widen(*reinterpret_cast<const u32x2*>(a.q + rr.strides(a.q_stride_token, a.q_stride_head) + d0), qv);
    float m = -INFINITY, l = 0.f;
    for (int i = st0; i < st1; ++i) {
      const int step = i < nfar ? fs0 + i : ns0 + (i - nfar);
      for (int key = step * KT; key < step * KT + KT; ++key) {
        if (!((key >= ks.lo && key < ks.hi) || (key >= ks.first && key < ks.pre))) continue;
        const int lb = a.bs_shift >= 0 ? key >> a.bs_shift : key / bs;
        const int bid = clampi(a.block_tables[(int64_t)it.s * a.max_bps + lb], 0, a.num_blocks - 1);
        const int64_t at = ((int64_t)(bid * a.num_kv_heads + kh) * bs + (key - lb * bs)) * rowb + d0 * EB;
        float kv[4] = {0, 0, 0, 0}, vv[4] = {0, 0, 0, 0};
        if (on) {
          if constexpr (kF8) {
            const uint32_t kw = *reinterpret_cast<const uint32_t*>(a.k_cache + at);
            const uint32_t vw = *reinterpret_cast<const uint32_t*>(a.v_cache + at);
            widen(u32x2{e4m3x2_to<TT, false>(kw), e4m3x2_to<TT, true>(kw)}, kv);
            widen(u32x2{e4m3x2_to<TT, false>(vw), e4m3x2_to<TT, true>(vw)}, vv);
          } else {
            widen(*reinterpret_cast<const u32x2*>(a.k_cache + at), kv);
            widen(*reinterpret_cast<const u32x2*>(a.v_cache + at), vv);
          }
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
        *reinterpret_cast<u32x2*>(a.out + rr.strides(a.out_stride_token, a.out_stride_head) + d0) =
            u32x2{TT::pack2(o[0] * inv, o[1] * inv), TT::pack2(o[2] * inv, o[3] * inv)};
    } else {
      if (on) *reinterpret_cast<f32x4*>(a.tile_o + (slot0 + w) * d + d0) = f32x4{o[0], o[1], o[2], o[3]};
      if (lane == 0) {
        a.tile_ml[(slot0 + w) * 2] = m;
        a.tile_ml[(slot0 + w) * 2 + 1] = l;
      }
    }
  }
}

// All pieces of workgroup `block` (kv head fastest: with 8 of them each XCD's L2
// serves one). Each piece takes the arguments and its thread number afresh, so
// that nothing derived from them stays in registers from piece to piece.
template <class TT, int D, bool kF8, Capped kCapped, bool kBias>
__device__ __forceinline__ void rows_group(int block, RowsLds<D>& lds) {
  typedef const Args __attribute__((address_space(4))) KernArgs;
  auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  for (int done = 0, n = 0;; ++n) {
    KernArgs* ka = (KernArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    int tid = threadIdx.x;
    asm volatile("" : "+s"(ka), "+v"(tid));
    const Args& a = *(const Args*)ka;
    const int id = block / a.num_kv_heads, kh = block - id * a.num_kv_heads;
    Piece it;
    if (a.list) {
      __syncthreads();   // the last piece's reads are done
      if (n % kPieces == 0) {
        if (uni(tid >> 6) == 0) rows_share(a, id, done, tid & 63, lds.row, lds.piece);
        __syncthreads();
      }
      const Piece& p = lds.piece[n % kPieces];
      it = Piece{uni(p.s), uni(p.row0), uni(p.tokens), uni(p.t), uni(p.limit), uni(p.tile),
                 uni(p.from), uni(p.to), uni(p.est)};
      if (it.est == 0) return;
    } else {
      // whole tiles of chunks, the last of a sequence first (it sees the most keys)
      it.s = id / a.tiles_max;
      it.t = a.tiles_max - 1 - (id - it.s * a.tiles_max);
      it.row0 = clampi(a.cu_seqlens_q[it.s], 0, a.total_q);
      it.tokens = clampi(a.cu_seqlens_q[it.s + 1], it.row0, a.total_q) - it.row0;
      it.limit = clampi(a.seq_lens[it.s], 0, a.max_bps * a.block_size);
      it.tile = it.from = 0;
      it.to = it.est = 1;
      if ((int64_t)it.t * kTileRows >= (int64_t)it.tokens * a.group) return;
    }
    rows_piece<TT, D, kF8, kCapped, kBias>(a, it, id, kh, n == 0, tid, lds);
    if (!a.list) return;
    done += it.to - it.from;
  }
}

template <class TT, int D, bool kF8, Capped kCapped, bool kBias>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(rows_per_cu(D, kF8), rows_per_cu(D, kF8))))
void chunks_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) RowsLds<D> lds;
  rows_group<TT, D, kF8, kCapped, kBias>(blockIdx.x, lds);
}

// Groups: workgroups for the shared keys, then four stream units each for the
// sequences' own keys: the one kind waits on the matrix cores, the other on HBM.
template <class TT, int D, bool kF8, Capped kCapped, bool kBias>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(rows_per_cu(D, kF8), rows_per_cu(D, kF8))))
void shared_kernel(Args a) {
  union Lds {
    RowsLds<D> rows;
    StreamLds<D> stream[kThreads / 64];
  };
  __shared__ __attribute__((aligned(1024))) Lds lds;
  const int n = a.room * a.num_kv_heads;
  if ((int)blockIdx.x < n) {
    rows_group<TT, D, kF8, kCapped, kBias>(blockIdx.x, lds.rows);
  } else {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int kRing = D == 64 || (kF8 && D == 128) ? 4 : (D == 128 || kF8 ? 2 : 1);
    stream_unit<TT, D, kF8, kRing>(a, ((int)blockIdx.x - n) * (kThreads / 64) + wave, threadIdx.x & 63,
                            lds.stream[wave]);
  }
}

template <class TT, int D, bool kF8, Capped kCapped, bool kBias>
void launch_rows_k(const Args& a, hipStream_t st) {
  int64_t n = (int64_t)a.room * a.num_kv_heads;
  if (a.cu_seqlens_q) {
    hipLaunchKernelGGL((chunks_kernel<TT, D, kF8, kCapped, kBias>), dim3((unsigned)n), dim3(kThreads), 0, st, a);
  } else {
    const int64_t units = (int64_t)a.num_seqs * a.num_kv_heads * a.subs * a.unit_splits;
    n += (units + kThreads / 64 - 1) / (kThreads / 64);
    hipLaunchKernelGGL((shared_kernel<TT, D, kF8, kCapped, kBias>), dim3((unsigned)n), dim3(kThreads), 0, st, a);
  }
}
template <class TT, int D, bool kF8>
void launch_rows_f(const Args& a, hipStream_t st) {
  const bool bias = a.slopes != nullptr;
  if (a.cap_log2 <= 0.f) {
    if (bias) launch_rows_k<TT, D, kF8, kNoCap, true>(a, st);
    else launch_rows_k<TT, D, kF8, kNoCap, false>(a, st);
  } else if (a.cap_wide) {
    if (bias) launch_rows_k<TT, D, kF8, kWideCap, true>(a, st);
    else launch_rows_k<TT, D, kF8, kWideCap, false>(a, st);
  } else {
    if (bias) launch_rows_k<TT, D, kF8, kPlainCap, true>(a, st);
    else launch_rows_k<TT, D, kF8, kPlainCap, false>(a, st);
  }
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
