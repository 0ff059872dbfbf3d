// RMS norm with the residual's addition and an 8-bit output, and its gradient
// (HBM-bound streaming kernels, sm_100a).
//
//   forward   h = bf16(x + residual)                  (h = x without a residual)
//             rstd = 1 / sqrt(mean(h^2) + eps)         fp32, kept for the backward pass
//             y = h * rstd * w                         fp32, unrounded
//             (q, sfa) = 1x128 quant of y (kQuantFinite), or out = bf16(y)
//   backward  g = dy * w,  xhat = h * rstd
//             dx = rstd * (g - xhat * mean(g * xhat)) + dh       (x and the residual share it)
//             dw = sum over tokens of dy * xhat
//
// A row is held in registers between the reduction and the output: kWarps warps share
// it, each thread owning kChunks runs of 16 consecutive values (two 16-byte loads), so
// 8 lanes hold one 1x128 group and its abs-max is three shuffles.
#pragma once

#include "quant.cuh"

namespace ltxfp8 {

constexpr int kRunLen = 16;  // consecutive values of one thread

// 16 consecutive bf16 <-> fp32 pairs.
struct Run16 {
  uint4 a, b;
};
__device__ __forceinline__ Run16 ld_run(const __nv_bfloat16* p) {
  const uint4* v = reinterpret_cast<const uint4*>(p);
  return Run16{v[0], v[1]};
}
__device__ __forceinline__ void st_run(__nv_bfloat16* p, const Run16& r) {
  uint4* v = reinterpret_cast<uint4*>(p);
  v[0] = r.a;
  v[1] = r.b;
}
__device__ __forceinline__ void run_to_f2(const Run16& r, float2 (&f)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
__device__ __forceinline__ Run16 f2_to_run(const float2 (&f)[8]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(f[i].x, f[i].y);
  return Run16{make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
}
__device__ __forceinline__ Run16 zero_run() { return Run16{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)}; }

// 16 gain values, bf16 or fp32 (w == nullptr: ones).
__device__ __forceinline__ void ld_gain(const void* w, bool w_f32, int col, float2 (&f)[8]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = make_float2(1.0f, 1.0f);
  } else if (w_f32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + col);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = __ldg(p + i);
      f[2 * i] = make_float2(v.x, v.y);
      f[2 * i + 1] = make_float2(v.z, v.w);
    }
  } else {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w) + col);
    run_to_f2(Run16{__ldg(p), __ldg(p + 1)}, f);
  }
}

// 1x128 quantisation (kQuantFinite) of the 16 values this lane holds of a group; the
// other 112 are in the 7 lanes that share its aligned eighth-of-a-warp.  All 32 lanes call.
__device__ __forceinline__ uint4 quant_run16(const float2 (&f)[8], float& inv) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmax_nan(amax, fmax_nan(fabsf(f[i].x), fabsf(f[i].y)));
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) amax = fmax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  float s;
  group_scale<kQuantFinite>(amax, s, inv);
  const float2 s2 = make_float2(s, s);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 lo = __fmul2_rn(f[2 * i], s2), hi = __fmul2_rn(f[2 * i + 1], s2);
    w[i] = static_cast<uint32_t>(f32x2_to_e4m3x2_inrange(lo.x, lo.y)) |
           (static_cast<uint32_t>(f32x2_to_e4m3x2_inrange(hi.x, hi.y)) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sum over the kWarps warps of this thread's row (every thread gets it).  `red` holds
// one float per warp of the block; with more than one warp a row this is a block-wide
// barrier, which callers alternate over two buffers so one barrier a row is enough.
template <int kWarps>
__device__ __forceinline__ float row_sum(float v, float* red, int warp) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if constexpr (kWarps == 1) {
    return v;
  } else {
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    const int w0 = warp / kWarps * kWarps;
    float s = red[w0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) s += red[w0 + i];
    return s;
  }
}

struct NormFwdParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* res;  // null: no residual
  int64_t x_ld, res_ld, M;
  int H;
  const void* w;  // null: no gain
  bool w_f32;
  float eps;
  __nv_bfloat16* h;  // [M, H], with a residual
  uint8_t* q;        // [M, H] or null
  float* sfa;
  int64_t sfa_ld;
  __nv_bfloat16* out;  // [M, H] when q is null
  float* rstd;         // [M] or null
};

template <int kWarps>
constexpr int norm_threads = kWarps > 8 ? kWarps * 32 : 256;

template <int kWarps, int kChunks, bool kRes, bool kQuant>
__global__ void __launch_bounds__(norm_threads<kWarps>) rms_norm_fwd_kernel(const NormFwdParams p) {
  constexpr int kRows = norm_threads<kWarps> / (32 * kWarps);  // rows of a block
  __shared__ float red[norm_threads<kWarps> / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + warp / kWarps;
  const bool row_ok = row < p.M;
  const int t = (warp % kWarps) * 32 + lane;

  Run16 v[kChunks];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int col = (i * kWarps * 32 + t) * kRunLen;
    v[i] = (row_ok && col < p.H) ? ld_run(p.x + row * p.x_ld + col) : zero_run();
  }
  if constexpr (kRes) {
    Run16 r[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (i * kWarps * 32 + t) * kRunLen;
      r[i] = (row_ok && col < p.H) ? ld_run(p.res + row * p.res_ld + col) : zero_run();
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (i * kWarps * 32 + t) * kRunLen;
      float2 a[8], b[8];
      run_to_f2(v[i], a);
      run_to_f2(r[i], b);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = __fadd2_rn(a[j], b[j]);
      v[i] = f2_to_run(a);  // the stored residual stream is what is normalised
      if (row_ok && col < p.H) st_run(p.h + row * p.H + col, v[i]);
    }
  }
  float acc = 0.0f;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    float2 a[8], s = make_float2(0.0f, 0.0f);
    run_to_f2(v[i], a);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __ffma2_rn(a[j], a[j], s);
    acc += s.x + s.y;
  }
  const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(row_sum<kWarps>(acc, red, warp) / static_cast<float>(p.H) + p.eps));
  if (p.rstd != nullptr && row_ok && t == 0) p.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int col = (i * kWarps * 32 + t) * kRunLen;
    const bool ok = row_ok && col < p.H;
    float2 a[8], w[8];
    run_to_f2(v[i], a);
    ld_gain(p.w, p.w_f32, col < p.H ? col : 0, w);
    const float2 r2 = make_float2(rstd, rstd);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = __fmul2_rn(__fmul2_rn(a[j], r2), w[j]);
    if constexpr (kQuant) {
      float inv;
      const uint4 codes = quant_run16(a, inv);
      if (ok) {
        *reinterpret_cast<uint4*>(p.q + row * p.H + col) = codes;
        if ((lane & 7) == 0) p.sfa[static_cast<int64_t>(col / 128) * p.sfa_ld + row] = inv;
      }
    } else {
      if (ok) st_run(p.out + row * p.H + col, f2_to_run(a));
    }
  }
}

struct NormBwdParams {
  const __nv_bfloat16* dy;
  const __nv_bfloat16* h;
  const __nv_bfloat16* dh;  // null: no gradient of the residual stream to add
  int64_t dy_ld, h_ld, dh_ld, M;
  int H;
  const float* rstd;
  const void* w;  // null: no gain
  bool w_f32;
  __nv_bfloat16* dx;  // [M, H]
  float* dw_part;     // [gridDim.x, H] partial sums over the block's rows, or null
};

// A persistent grid: block b takes the row groups b, b + gridDim.x, ... and keeps the
// gain gradient of its rows in registers; the blocks' partial sums are added by
// col_sum_kernel in block order, so the result does not depend on scheduling.
template <int kWarps, int kChunks>
__global__ void __launch_bounds__(norm_threads<kWarps>) rms_norm_bwd_kernel(const NormBwdParams p) {
  constexpr int kRows = norm_threads<kWarps> / (32 * kWarps);
  __shared__ float red[2][norm_threads<kWarps> / 32];
  __shared__ float dw_rows[kRows > 1 ? kRows * kWarps * 32 * kChunks * kRunLen : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = (warp % kWarps) * 32 + lane;
  const float inv_h = 1.0f / static_cast<float>(p.H);

  float2 dw[kChunks][8];
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = make_float2(0.0f, 0.0f);

  int phase = 0;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows; r0 < p.M;
       r0 += static_cast<int64_t>(gridDim.x) * kRows, phase ^= 1) {
    const int64_t row = r0 + warp / kWarps;
    const bool row_ok = row < p.M;
    const float rstd = row_ok ? __ldg(p.rstd + row) : 0.0f;
    Run16 vy[kChunks], vh[kChunks], vd[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (i * kWarps * 32 + t) * kRunLen;
      const bool ok = row_ok && col < p.H;
      vy[i] = ok ? ld_run(p.dy + row * p.dy_ld + col) : zero_run();
      vh[i] = ok ? ld_run(p.h + row * p.h_ld + col) : zero_run();
      vd[i] = (ok && p.dh != nullptr) ? ld_run(p.dh + row * p.dh_ld + col) : zero_run();
    }
    float acc = 0.0f;
    const float2 r2 = make_float2(rstd, rstd);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (i * kWarps * 32 + t) * kRunLen;
      float2 y[8], x[8], w[8], s = make_float2(0.0f, 0.0f);
      run_to_f2(vy[i], y);
      run_to_f2(vh[i], x);
      ld_gain(p.w, p.w_f32, col < p.H ? col : 0, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 yx = __fmul2_rn(y[j], __fmul2_rn(x[j], r2));  // dy * xhat
        dw[i][j] = __fadd2_rn(dw[i][j], yx);
        s = __ffma2_rn(yx, w[j], s);
      }
      acc += s.x + s.y;
    }
    const float c = row_sum<kWarps>(acc, red[phase], warp) * inv_h;
    const float2 c2 = make_float2(-c, -c);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (i * kWarps * 32 + t) * kRunLen;
      float2 y[8], x[8], w[8], d[8];
      run_to_f2(vy[i], y);
      run_to_f2(vh[i], x);
      run_to_f2(vd[i], d);
      ld_gain(p.w, p.w_f32, col < p.H ? col : 0, w);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        d[j] = __ffma2_rn(r2, __ffma2_rn(__fmul2_rn(x[j], r2), c2, __fmul2_rn(y[j], w[j])), d[j]);
      if (row_ok && col < p.H) st_run(p.dx + row * p.H + col, f2_to_run(d));
    }
  }
  if (p.dw_part == nullptr) return;
  float* part = p.dw_part + static_cast<int64_t>(blockIdx.x) * p.H;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (i * kWarps * 32 + t) * kRunLen;
      if (col < p.H) {
        float4* dst = reinterpret_cast<float4*>(part + col);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          dst[j] = make_float4(dw[i][2 * j].x, dw[i][2 * j].y, dw[i][2 * j + 1].x, dw[i][2 * j + 1].y);
      }
    }
  } else {
    // The block's row groups are added in row order.
    constexpr int kRowLen = kWarps * 32 * kChunks * kRunLen;
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<float2*>(dw_rows + (warp / kWarps) * kRowLen + (i * kWarps * 32 + t) * kRunLen + 2 * j) =
            dw[i][j];
    __syncthreads();
    for (int col = threadIdx.x; col < p.H; col += norm_threads<kWarps>) {
      float s = dw_rows[col];
#pragma unroll
      for (int r = 1; r < kRows; ++r) s += dw_rows[r * kRowLen + col];
      part[col] = s;
    }
  }
}

// out[n] = sum over p of part[p, n], in the type of `out` (fp32 or bf16): a block sums 32
// columns, its 8 warps every eighth partial row each, in a fixed order.
__global__ void __launch_bounds__(256) col_sum_kernel(const float* __restrict__ part, int parts, int N, void* out,
                                                      bool out_f32) {
  __shared__ float red[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (n < N) {
#pragma unroll 8
    for (int i = warp; i < parts; i += 8) s += part[static_cast<int64_t>(i) * N + n];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && n < N) {
#pragma unroll
    for (int w = 1; w < 8; ++w) s += red[w][lane];
    if (out_f32)
      static_cast<float*>(out)[n] = s;
    else
      static_cast<__nv_bfloat16*>(out)[n] = __float2bfloat16_rn(s);
  }
}

}  // namespace ltxfp8
