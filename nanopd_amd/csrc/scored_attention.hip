// Attention with changed scores over the paged pool: the C entries, the decode
// kernel (units of scored_stream.h) and the merges of partial results.
#include "scored_stream.h"

namespace npd {
namespace scored {
namespace {

constexpr int kOnePart = 256;        // keys up to which a unit is not cut (no merge: 9 us, not 11)
constexpr int kDecodePart = 64;      // shortest part of a unit that is (keys)
// Rows of which each has a workgroup to merge it: many parts are then read side by
// side (64 tokens over 8192 shared keys: 48 us against 51.5; one token of 4000 keys:
// 13 against 16). More rows fill the chip with a few lanes each.
constexpr int kWideRows = 2048;
constexpr int kSharedPart = 256;     // ... beside the rows kernel

template <class TT, int DP, bool kF8>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(stream_per_simd(DP, kF8))))
void stream_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) StreamLds<DP> lds;
  constexpr int kRing = DP == 64 || (kF8 && DP == 128) ? 4 : (DP == 128 || kF8 ? 2 : 1);
  stream_unit<TT, DP, kF8, kRing>(a, blockIdx.x, threadIdx.x, lds);
}

// Partials of a row: `nt` of its tile (slot t0 and then every second from t1 on,
// tstep apart) and `nu` of its stream units (consecutive from u0).
struct Parts {
  int nt, nu;
  int64_t t0, t1, tstep, u0;
  __device__ __forceinline__ bool tile(int i) const { return i < nt; }
  __device__ __forceinline__ int64_t slot(int i) const {
    return i >= nt ? u0 + (i - nt) : i == 0 ? t0 : t1 + i * tstep;
  }
};
// The merge of a row by LPR lanes (four dims each), every part's sum weighted by
// 2^(m - M); kFlight parts' loads at a time.
template <class TT, int LPR>
__device__ __forceinline__ void merge_row(const Args& a, const Parts& p, int lane, uint16_t* dst,
                                          float oscale) {
  constexpr int kFlight = 4;
  const int n = p.nt + p.nu, d = a.head_dim, j = lane % LPR, c = j * 4;
  auto ml = [&](int i) { return (p.tile(i) ? a.tile_ml : a.unit_ml) + p.slot(i) * 2; };
  float M = -INFINITY;
  for (int i = j; i < n; i += LPR) M = fmaxf(M, ml(i)[0]);
#pragma unroll
  for (int k = 1; k < LPR; k <<= 1) M = fmaxf(M, __shfl_xor(M, k, 64));
  f32x4 o = f32x4{0, 0, 0, 0};
  float L = 0.f;
  if (M > -INFINITY) {
    for (int i0 = 0; i0 < n; i0 += kFlight) {
      float w[kFlight], l[kFlight];
      f32x4 x[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int i = i0 + k < n ? i0 + k : n - 1;
        const float* q = ml(i);
        w[k] = i0 + k < n ? q[0] : -INFINITY;
        l[k] = q[1];
        x[k] = f32x4{0, 0, 0, 0};
        // (a part without a key has no sums)
        if (w[k] != -INFINITY && c < d)
          x[k] = *reinterpret_cast<const f32x4*>((p.tile(i) ? a.tile_o : a.unit_o) + p.slot(i) * d + c);
      }
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const float f = __builtin_amdgcn_exp2f(w[k] - M);
        if (w[k] != -INFINITY) L = fmaf(l[k], f, L);
        o.x = fmaf(x[k].x, f, o.x);
        o.y = fmaf(x[k].y, f, o.y);
        o.z = fmaf(x[k].z, f, o.z);
        o.w = fmaf(x[k].w, f, o.w);
      }
    }
  }
  if (c < d) {
    const float inv = L > 0.f || L != L ? oscale / L : 0.f;
    *reinterpret_cast<u32x2*>(dst + c) =
        u32x2{TT::pack2(o.x * inv, o.y * inv), TT::pack2(o.z * inv, o.w * inv)};
  }
}

// A tile's entry as the parts of its row r (none where lists that do not ascend
// left no such entry: stay in the buffer).
__device__ __forceinline__ void tile_parts(const Args& a, int64_t tile, int kh, int r, Parts& p) {
  const int32_t* e = a.tile_items + 4 * (tile * a.num_kv_heads + kh);
  const int slot0 = e[0], wg = e[1], parts = e[2] - wg + 1;
  p.nt = 0;
  if (parts < 1 || parts > a.room || wg < 0 || wg + parts > a.room || slot0 < 0 ||
      slot0 >= 2 * a.room + a.tiles)
    return;
  p.nt = parts;
  p.t0 = ((int64_t)slot0 * a.num_kv_heads + kh) * kTileRows + r;
  p.t1 = ((int64_t)2 * wg * a.num_kv_heads + kh) * kTileRows + r;
  p.tstep = (int64_t)2 * a.num_kv_heads * kTileRows;
}

// The parts of one token's row (by a whole wave).
__device__ __forceinline__ void token_parts(const Args& a, int s, int h, int lane, Parts& p) {
  int pos, a0, na, b0, nb;
  unit_keys(a, s, lane, pos, a0, na, b0, nb);
  p.nu = unit_parts(a, na + nb, lane);
  p.u0 = ((int64_t)s * a.num_heads + h) * a.unit_splits;
  Group g;
  if (a.cu_groups && find_group(a, s, lane, g) && g.shared > 0) {
    const int kh = h / a.group;
    const int64_t f = (int64_t)(s - g.seq0) * a.group + (h - kh * a.group);
    const int64_t tile = g.tile0 + f / kTileRows;
    if (tile < a.tiles) tile_parts(a, tile, kh, (int)(f % kTileRows), p);
  }
}
// One token per sequence: a wave takes 64 / LPR heads of a token.
template <class TT, int LPR>
__global__ __launch_bounds__(256) void merge_tokens_kernel(Args a) {
  constexpr int R = 64 / LPR;
  const int lane = threadIdx.x & 63;
  const int per = (a.num_heads + R - 1) / R;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int s = (int)(w / per), h = (int)(w - (int64_t)s * per) * R + lane / LPR;
  if (s >= a.num_seqs) return;   // whole waves
  Parts p{};
  token_parts(a, s, h < a.num_heads ? h : a.num_heads - 1, lane, p);
  if (h >= a.num_heads || (!a.cu_groups && p.nu <= 1)) return;   // (one part: written by its unit)
  merge_row<TT, LPR>(a, p, lane, a.out + s * a.out_stride_token + h * a.out_stride_head,
                     a.v_scale ? a.v_scale[h / a.group] : 1.f);
}

// Few rows, or many parts of each: a workgroup per row, its lane groups at a part each.
template <class TT, int LPR>
__global__ __launch_bounds__(256) void merge_wide_kernel(Args a) {
  constexpr int kGroups = 256 / LPR;
  __shared__ f32x4 s_o[4][LPR];
  __shared__ float s_l[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = a.head_dim, c = lane % LPR * 4;
  const int s = blockIdx.x / a.num_heads, h = blockIdx.x - s * a.num_heads;
  Parts p{};
  token_parts(a, s, h, lane, p);
  const int n = p.nt + p.nu;
  if (!a.cu_groups && n <= 1) return;   // written by its unit
  auto ml = [&](int i) { return (p.tile(i) ? a.tile_ml : a.unit_ml) + p.slot(i) * 2; };
  float M = -INFINITY;
  for (int i = lane; i < n; i += 64) M = fmaxf(M, ml(i)[0]);
  M = wave_max_f(M);
  f32x4 o = f32x4{0, 0, 0, 0};
  float L = 0.f;
  if (M > -INFINITY) {
    constexpr int kFlight = 4;
    for (int i0 = threadIdx.x / LPR; i0 < n; i0 += kFlight * kGroups) {
      float m[kFlight], l[kFlight];
      f32x4 x[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int i = i0 + k * kGroups < n ? i0 + k * kGroups : i0;
        const float* q = ml(i);
        m[k] = i0 + k * kGroups < n ? q[0] : -INFINITY;
        l[k] = q[1];
        x[k] = f32x4{0, 0, 0, 0};
        if (c < d) x[k] = *reinterpret_cast<const f32x4*>((p.tile(i) ? a.tile_o : a.unit_o) + p.slot(i) * d + c);
      }
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        // (a part without a key has no sums)
        const bool has = m[k] != -INFINITY;
        const float f = __builtin_amdgcn_exp2f(m[k] - M);
        L = has ? fmaf(l[k], f, L) : L;
        o.x = has ? fmaf(x[k].x, f, o.x) : o.x;
        o.y = has ? fmaf(x[k].y, f, o.y) : o.y;
        o.z = has ? fmaf(x[k].z, f, o.z) : o.z;
        o.w = has ? fmaf(x[k].w, f, o.w) : o.w;
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
  if (lane < LPR) s_o[wave][lane] = o;
  if (lane == 0) s_l[wave] = L;
  __syncthreads();
  if (threadIdx.x >= LPR || c >= d) return;
  L = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
  o = (s_o[0][lane] + s_o[1][lane]) + (s_o[2][lane] + s_o[3][lane]);
  const float inv = L > 0.f || L != L ? (a.v_scale ? a.v_scale[h / a.group] : 1.f) / L : 0.f;
  *reinterpret_cast<u32x2*>(a.out + s * a.out_stride_token + h * a.out_stride_head + c) =
      u32x2{TT::pack2(o.x * inv, o.y * inv), TT::pack2(o.z * inv, o.w * inv)};
}

// Chunks: a workgroup takes a tile's rows of one kv head, kSlice of them.
constexpr int kSlice = 16;
template <class TT, int LPR>
__global__ __launch_bounds__(256) void merge_tiles_kernel(Args a) {
  const int lane = threadIdx.x & 63;
  int id = blockIdx.x;
  const int slice = id % (kTileRows / kSlice);
  id /= kTileRows / kSlice;
  const int kh = id % a.num_kv_heads;
  const int tile = id / a.num_kv_heads, sq = tile / a.tiles_max, t = tile - sq * a.tiles_max;
  const int q0 = clampi(a.cu_seqlens_q[sq], 0, a.total_q);
  const int q1 = clampi(a.cu_seqlens_q[sq + 1], q0, a.total_q);
  const int rows = (q1 - q0) * a.group;
  if (t * kTileRows >= rows) return;
  const float oscale = a.v_scale ? a.v_scale[kh] : 1.f;
  for (int r = slice * kSlice + threadIdx.x / LPR; r < (slice + 1) * kSlice; r += 256 / LPR) {
    const int f = t * kTileRows + r;
    if (f >= rows) break;
    Parts p{};
    tile_parts(a, tile, kh, r, p);
    if (p.nt <= 1) return;     // written by the rows kernel itself
    const int tok = f / a.group, h = kh * a.group + (f - tok * a.group);
    merge_row<TT, LPR>(a, p, lane, a.out + (int64_t)(q0 + tok) * a.out_stride_token + h * a.out_stride_head,
                       oscale);
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
template <class TT, int LPR>
void launch_merge_d(const Args& a, hipStream_t st) {
  if (a.cu_seqlens_q) {
    const int64_t n = (int64_t)a.tiles * a.num_kv_heads * (kTileRows / kSlice);
    hipLaunchKernelGGL((merge_tiles_kernel<TT, LPR>), dim3((unsigned)n), dim3(256), 0, st, a);
  } else if ((int64_t)a.num_seqs * a.num_heads <= kWideRows) {
    hipLaunchKernelGGL((merge_wide_kernel<TT, LPR>), dim3((unsigned)(a.num_seqs * a.num_heads)), dim3(256), 0, st, a);
  } else {
    constexpr int R = 64 / LPR;
    const int64_t waves = (int64_t)a.num_seqs * ((a.num_heads + R - 1) / R);
    hipLaunchKernelGGL((merge_tokens_kernel<TT, LPR>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a);
  }
}
template <class TT>
void launch_merge_t(const Args& a, hipStream_t st) {
  if (a.head_dim <= 64) launch_merge_d<TT, 16>(a, st);
  else if (a.head_dim <= 128) launch_merge_d<TT, 32>(a, st);
  else launch_merge_d<TT, 64>(a, st);
}
void launch_merge(const Args& a, int32_t dtype, hipStream_t st) {
  if (dtype == NPD_DTYPE_BF16) launch_merge_t<BF16>(a, st);
  else launch_merge_t<F16>(a, st);
}

// Units of at most kUnitHeads heads: the fewest near-equal ones.
int64_t subs_of(int64_t group) { return (group + kUnitHeads - 1) / kUnitHeads; }

// Workgroups of the rows kernel that run at once per kv head.
int64_t rows_room(int64_t head_dim, int64_t num_kv_heads, bool fp8) {
  const int64_t n = rows_per_cu(head_dim, fp8) * (int64_t)device_cus() / num_kv_heads;
  return n < 1 ? 1 : n;
}

int64_t pad256(int64_t x) { return (x + 255) / 256 * 256; }

// Sizes of a call's partials; the workspace is the counter region (which these
// ops leave alone, so that one buffer serves every attention op), then the
// tiles' partials and part counts, then the units'.
struct Plan {
  int64_t part_keys = 0;
  int64_t tiles = 0, tiles_max = 0, room = 1, unit_splits = 1;
  bool list = false, groups = false;
  int64_t tile_slots = 0, unit_slots = 0, head_dim = 0, kv_heads = 0;
  int64_t tile_items_at() const { return kCounterBytes; }
  int64_t tile_o_at() const { return tile_items_at() + (tile_slots ? pad256(tiles * kv_heads * 16) : 0); }
  int64_t tile_ml_at() const { return tile_o_at() + pad256(tile_slots * head_dim * 4); }
  int64_t unit_o_at() const { return tile_ml_at() + pad256(tile_slots * 8); }
  int64_t unit_ml_at() const { return unit_o_at() + pad256(unit_slots * head_dim * 4); }
  int64_t bytes() const {
    return tile_slots || unit_slots ? unit_ml_at() + pad256(unit_slots * 8) : 0;
  }
};

// Most parts of a unit: twice what makes kTargetItems waves of units that are all
// alike, for the longest of a ragged batch; no more than the table's tokens (or the
// window's) have parts of `least` keys.
void cut_units(Plan& p, int64_t units, int64_t max_keys, int64_t least) {
  const int64_t w = max_keys <= kOnePart ? 1 : 2 * ((kTargetItems + units - 1) / units);
  const int64_t most = (max_keys + least - 1) / least;
  p.part_keys = least;
  p.unit_splits = units >= kTargetItems ? 1 : w < most ? w : most;
  if (p.unit_splits < 1) p.unit_splits = 1;
}

int64_t window_keys(int64_t max_keys, int64_t window, bool prefix) {
  return window > 0 && !prefix && window < max_keys ? window : max_keys;
}
Plan decode_plan(int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                 int64_t max_keys, int64_t least = kDecodePart) {
  Plan p;
  p.head_dim = head_dim;
  p.kv_heads = num_kv_heads;
  cut_units(p, num_seqs * num_kv_heads * subs_of(num_heads / num_kv_heads), max_keys, least);
  p.unit_slots = p.unit_splits > 1 ? num_seqs * num_heads * p.unit_splits : 0;
  return p;
}
// Slots of the rows kernel's partials: two per workgroup (its first tile may have
// begun before it and its last may go on after it); groups also one per tile (the
// parts of whole tiles meet those of the stream units).
// Elements of K up to which shared keys are read once per sequence after all: a
// launch without the rows kernel spares its fixed work, about the time of reading
// 128 MB. Measured with 4 to 64 sequences, 2 and 8 kv heads, head dims of 64 to 256,
// once per sequence against shared: at 17 M elements 18 to 24 us against 25 to 35,
// at 34 M 28 to 34 against 26 to 39, at 67 M 36 to 55 against 28 to 42.
constexpr int64_t kReadAgain = int64_t(1) << 25;
// Shares over at most `tiles` tiles of a kv head with at most `steps` steps each.
void plan_list(Plan& p, int64_t tiles, int64_t steps) {
  const int64_t total = tiles * (steps + kTileCost), most = (total + kMinShare - 1) / kMinShare;
  p.list = true;
  p.room = p.room < most ? p.room : most < 1 ? 1 : most;
}
Plan shared_plan(int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                 int64_t max_keys, int64_t num_groups, int64_t max_shared) {
  max_shared = max_shared < max_keys ? max_shared : max_keys;
  if (num_seqs * num_kv_heads * max_shared <= kReadAgain / head_dim)
    return decode_plan(num_seqs, num_heads, num_kv_heads, head_dim, max_keys);
  Plan p = decode_plan(num_seqs, num_heads, num_kv_heads, head_dim, max_keys, kSharedPart);
  p.groups = true;
  p.unit_slots = num_seqs * num_heads * p.unit_splits;   // always merged
  p.tiles = num_seqs * (num_heads / num_kv_heads) / kTileRows + num_groups;
  p.room = rows_room(head_dim, num_kv_heads, false);
  plan_list(p, p.tiles, max_shared / kStepKeys + 1);
  p.tile_slots = (2 * p.room + p.tiles) * num_kv_heads * kTileRows;
  return p;
}
Plan chunk_plan(int64_t num_seqs, int64_t total_q, int64_t num_heads, int64_t num_kv_heads,
                int64_t head_dim, int64_t max_q_len, int64_t max_keys) {
  Plan p;
  const int64_t g = num_heads / num_kv_heads;
  p.head_dim = head_dim;
  p.kv_heads = num_kv_heads;
  p.tiles_max = (max_q_len * g + kTileRows - 1) / kTileRows;
  p.room = rows_room(head_dim, num_kv_heads, false);
  const int64_t all = num_seqs * p.tiles_max, rows = total_q * g / kTileRows + num_seqs;
  const int64_t most = rows < all ? rows : all;
  // shared out evenly unless whole tiles fill the chip twice over
  if (all <= kListTiles && most < 2 * p.room) {
    p.tiles = all;
    plan_list(p, all, max_keys / kStepKeys + 2);
    p.tile_slots = p.room > 1 ? 2 * p.room * num_kv_heads * kTileRows : 0;
  } else {
    p.room = all;
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
  a.room = (int)p.room;
  if (p.list) {   // (the workspace is sized for either kind of pool)
    const int64_t room = rows_room(c.head_dim, c.num_kv_heads, c.k_scale != nullptr);
    a.room = (int)(room < p.room ? room : p.room);
  }
  a.room1 = (int)((device_cus() + c.num_kv_heads - 1) / c.num_kv_heads);
  a.list = p.list;
  // (units in which all tiles' costs stay below 2^30, whatever the lengths)
  if (p.list)
    while (a.cost_shift < 30 &&
           ((c.block_size * c.max_bps / kStepKeys + kTileCost) >> a.cost_shift) + 1 > (INT32_MAX / 2) / p.tiles)
      ++a.cost_shift;
  a.unit_splits = (int)p.unit_splits;
  a.part_keys = (int)p.part_keys;
  a.stream_waves = (float)(stream_per_simd(c.head_dim, c.k_scale != nullptr) * 4 * device_cus());
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

int run_decode(const Call& c, const Plan& p, const Args& a, hipStream_t st) {
  if (!grid_ok(c.num_seqs * c.num_kv_heads * a.subs * p.unit_splits))
    return fail(NPD_E_INVALID, "%s: too many (seq, kv-head) units", c.name);
  if (c.dtype == NPD_DTYPE_BF16) launch_stream<BF16>(a, st);
  else launch_stream<F16>(a, st);
  if (p.unit_slots) launch_merge(a, c.dtype, st);
  return check_launch(c.name);
}

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
  return run_decode(c, p, a, as_stream(stream));
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
  if (!p.groups) return run_decode(c, p, a, as_stream(stream));
  a.cu_groups = cu_groups;
  a.shared_lens = shared_lens;
  a.num_groups = (int)num_groups;
  a.max_shared = (int)(max_shared_len < max_keys ? max_shared_len : max_keys);
  if (!grid_ok(num_seqs * num_kv_heads * a.subs * p.unit_splits + p.room * num_kv_heads))
    return fail(NPD_E_INVALID, "%s: too many work items", c.name);
  hipStream_t st = as_stream(stream);
  if (head_dim <= 64) launch_rows<64>(a, dtype, st);
  else if (head_dim <= 128) launch_rows<128>(a, dtype, st);
  else launch_rows<256>(a, dtype, st);
  launch_merge(a, dtype, st);
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
  if (!grid_ok(p.room * num_kv_heads))
    return fail(NPD_E_INVALID, "%s: too many work items", c.name);
  hipStream_t st = as_stream(stream);
  if (head_dim <= 64) launch_rows<64>(a, dtype, st);
  else if (head_dim <= 128) launch_rows<128>(a, dtype, st);
  else launch_rows<256>(a, dtype, st);
  if (p.tile_slots) launch_merge(a, dtype, st);
  return check_launch(c.name);
}
