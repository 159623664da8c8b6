// The norms around a block of a layer that norms what the block returns too: the
// norm after the block, its gate, the residual add and the norm before the next
// block, one launch.
//   d     = delta * rsqrt(mean(delta^2) + eps) * post   (post null: delta)
//   x_out = residual_scale * x + gate * d               (gate null: d), rounded
//   h     = x_out * rsqrt(mean(x_out^2) + eps) * weight (weight null: no h)
// Sums, statistics and d are fp32; x_out is rounded once, and the second norm
// reads the rounded value, as the next layer does; h is rounded once.
//
// Bound by HBM bytes at many rows (x and delta read, x_out and h written, each
// once: the row stays in registers between the two statistics), by the latency
// of load, two reductions and store at few. 16384 rows of 5120, gated per row:
// 128 us, 5.2 TB/s; 527 of 4096: 5.5 us, 3.2 TB/s; one row of 4096: 3.3 us.
#include "common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kThreads = 256;
constexpr int kWaveWidth = 2048;   // widest row that one wave takes

struct NormArgs {
  u32x4* x_out;
  u32x4* h;
  const u32x4* x;
  const u32x4* delta;
  const u32x4* post;
  const u32x4* weight;
  const uint16_t* gate;
  int64_t gate_row, rows;   // gate elements between rows
  bool gate_scalar;         // one gate per row (else eight per chunk, 16-byte aligned)
  int chunks;               // 8-element chunks per row
  float inv_e, scale, eps;
};

template <class TT>
__device__ __forceinline__ void widen(u32x4 w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = TT::lo(w[i]);
    f[2 * i + 1] = TT::hi(w[i]);
  }
}

// Sum over the threads of a row: a wave (TPR 64) or the workgroup (TPR 256).
template <int TPR>
__device__ __forceinline__ float row_total(float x, float* s_sum) {
  x = npd::wave_sum_f(x);
  if constexpr (TPR == 64) return x;
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = x;
  __syncthreads();
  return (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

// A row's threads hold its chunks tid + TPR e, e < NCH, in registers.
template <class TT, int TPR, int NCH>
__global__ __launch_bounds__(kThreads) void block_norms_kernel(NormArgs a) {
  __shared__ float s_sum[2][kThreads / 64];
  const int tid = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
  if (row >= a.rows) return;   // whole waves
  const int64_t base = row * a.chunks;
  u32x4 xv[NCH], dv[NCH], pv[NCH], gv[NCH], wv[NCH];
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < NCH; ++e) {
    const int c = tid + TPR * e;
    xv[e] = dv[e] = pv[e] = gv[e] = wv[e] = u32x4{0, 0, 0, 0};
    if (c < a.chunks) {
      dv[e] = a.delta[base + c];
      xv[e] = a.x[base + c];
      if (a.post) pv[e] = a.post[c];
      if (a.gate && !a.gate_scalar)
        gv[e] = *reinterpret_cast<const u32x4*>(a.gate + row * a.gate_row + (int64_t)c * 8);
      if (a.weight) wv[e] = a.weight[c];
    }
  }
  float g = 1.f;
  if (a.gate && a.gate_scalar) g = TT::lo(a.gate[row * a.gate_row]);
  float r = 1.f;
  if (a.post) {
#pragma unroll
    for (int e = 0; e < NCH; ++e) {
      float f[8];
      widen<TT>(dv[e], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
    }
    r = rsqrtf(row_total<TPR>(ss, s_sum[0]) * a.inv_e + a.eps);
  }
  ss = 0.f;
#pragma unroll
  for (int e = 0; e < NCH; ++e) {
    float x[8], d[8], p[8], gg[8];
    widen<TT>(xv[e], x);
    widen<TT>(dv[e], d);
    widen<TT>(pv[e], p);
    widen<TT>(gv[e], gg);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float y = a.post ? d[i] * r * p[i] : d[i];
      if (a.gate) y *= a.gate_scalar ? g : gg[i];
      x[i] = fmaf(a.scale, x[i], y);
    }
    const int c = tid + TPR * e;
#pragma unroll
    for (int i = 0; i < 4; ++i) xv[e][i] = TT::pack2(x[2 * i], x[2 * i + 1]);
    if (c < a.chunks) a.x_out[base + c] = xv[e];
    widen<TT>(xv[e], x);
    if (c < a.chunks) {
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
    }
  }
  if (!a.weight) return;
  r = rsqrtf(row_total<TPR>(ss, s_sum[1]) * a.inv_e + a.eps);
#pragma unroll
  for (int e = 0; e < NCH; ++e) {
    const int c = tid + TPR * e;
    float x[8], w[8];
    widen<TT>(xv[e], x);
    widen<TT>(wv[e], w);
    u32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      y[i] = TT::pack2(x[2 * i] * r * w[2 * i], x[2 * i + 1] * r * w[2 * i + 1]);
    if (c < a.chunks) a.h[base + c] = y;
  }
}

template <class TT>
void launch(const NormArgs& a, hipStream_t st) {
  const int tpr = a.chunks * 8 <= kWaveWidth ? 64 : kThreads;
  const int per = kThreads / tpr;
  const dim3 g((unsigned)((a.rows + per - 1) / per)), b(kThreads);
  const int nch = (a.chunks + tpr - 1) / tpr;
  if (tpr == 64) {
    if (nch == 1) hipLaunchKernelGGL((block_norms_kernel<TT, 64, 1>), g, b, 0, st, a);
    else if (nch == 2) hipLaunchKernelGGL((block_norms_kernel<TT, 64, 2>), g, b, 0, st, a);
    else hipLaunchKernelGGL((block_norms_kernel<TT, 64, 4>), g, b, 0, st, a);
  } else {
    if (nch == 2) hipLaunchKernelGGL((block_norms_kernel<TT, 256, 2>), g, b, 0, st, a);
    else if (nch == 3) hipLaunchKernelGGL((block_norms_kernel<TT, 256, 3>), g, b, 0, st, a);
    else hipLaunchKernelGGL((block_norms_kernel<TT, 256, 4>), g, b, 0, st, a);
  }
}

}  // namespace

extern "C" int npd_block_norms(void* x_out, void* h, const void* x, const void* delta,
                               const void* post_weight, const void* weight, const void* gate,
                               int64_t gate_stride_row, int64_t gate_stride_col, int64_t rows,
                               int64_t width, float residual_scale, float eps, int32_t dtype,
                               void* stream) {
  using namespace npd;
  const char* name = "npd_block_norms";
  if (dtype != NPD_DTYPE_F16 && dtype != NPD_DTYPE_BF16)
    return fail(NPD_E_DTYPE, "%s: unsupported dtype code %d (fp16/bf16 only)", name, dtype);
  if (rows < 0 || rows > INT32_MAX || width <= 0 || width % 8 != 0 || width > 8192)
    return fail(NPD_E_INVALID, "%s: %lld rows of %lld (a multiple of 8 up to 8192 wanted)", name,
                (long long)rows, (long long)width);
  if (!(eps >= 0.f)) return fail(NPD_E_INVALID, "%s: eps must be non-negative", name);
  if ((h == nullptr) != (weight == nullptr))
    return fail(NPD_E_INVALID, "%s: pass both h and weight or neither", name);
  if (rows == 0) return NPD_OK;
  if (!x_out || !x || !delta) return fail(NPD_E_INVALID, "%s: null pointer", name);
  if (!aligned16(x_out) || !aligned16(h) || !aligned16(x) || !aligned16(delta) ||
      !aligned16(post_weight) || !aligned16(weight))
    return fail(NPD_E_ALIGN, "%s: pointers must be 16-byte aligned", name);
  if (gate) {
    if (gate_stride_row < 0 || (gate_stride_col != 0 && gate_stride_col != 1))
      return fail(NPD_E_INVALID, "%s: gate strides %lld, %lld", name, (long long)gate_stride_row,
                  (long long)gate_stride_col);
    if (gate_stride_col == 1 && (!aligned16(gate) || gate_stride_row % 8 != 0))
      return fail(NPD_E_ALIGN, "%s: gate rows must be 16-byte aligned", name);
  }
  NormArgs a;
  a.x_out = static_cast<u32x4*>(x_out);
  a.h = static_cast<u32x4*>(h);
  a.x = static_cast<const u32x4*>(x);
  a.delta = static_cast<const u32x4*>(delta);
  a.post = static_cast<const u32x4*>(post_weight);
  a.weight = static_cast<const u32x4*>(weight);
  a.gate = static_cast<const uint16_t*>(gate);
  a.gate_row = gate_stride_row;
  a.gate_scalar = gate_stride_col == 0;
  a.rows = rows;
  a.chunks = (int)(width / 8);
  a.inv_e = 1.f / (float)width;
  a.scale = residual_scale;
  a.eps = eps;
  hipStream_t st = as_stream(stream);
  if (dtype == NPD_DTYPE_BF16) launch<BF16>(a, st);
  else launch<F16>(a, st);
  return check_launch(name);
}
