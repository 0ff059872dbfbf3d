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
// 8 lanes hold one 1x128 group and its abs-max is three shuffles.  Every value is read once
// and written once: the floor is memory traffic (7.03 bytes a value forward with a residual and
// codes, 8 backward with dh).  Measured, tokens x width, in a chain of launches over 600 MB of inputs in
// rotation: forward 24576 x 4096 107 us (6.6 TB/s in a burst at 1965 MHz, a plain copy 6.5; 117 us in
// calls that last, under the power cap), 1003 x 2048 without a residual 3.3 us, 8 x 4096 2.0 us (a
// launch); backward with the gain's gradient 24576 x 4096 124 us (6.5 TB/s; 130 in calls that last),
// 1003 x 2048 8.5 us, of which the sum of the blocks' partial gains, a second launch, is 3.
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
  int stages;         // of the shared-memory ring, at most kNormMaxStages
};

// A persistent grid: block b takes the row groups b, b + gridDim.x, ... and keeps the
// gain gradient of its rows in registers; the blocks' partial sums are added by
// col_sum_kernel in block order, so the result does not depend on scheduling.
//
// HBM-bound, but a row is a reduction, a barrier and a second pass: with register loads too
// few bytes are in flight behind them (24576 x 4096: 167 us, 143 with the ring).  So bulk copies
// bring the rows through a ring of `stages` shared-memory stages; a stage is free again at
// the row's own barrier, when every thread has its values in registers.  Narrow rows are bound by
// a pass's instructions instead (300 a warp, 1.1 us for the 16 warps of an SM; below 512 columns
// part of the lanes idle): 6474 x 640 12 us against 4 of traffic.
enum NormStatus : unsigned int { kStNormLoad = 0x4E010001u, kStNormDrain = 0x4E010002u };
constexpr int kNormMaxStages = 8;

template <int kWarps, int kChunks>
__global__ void __launch_bounds__(norm_threads<kWarps>) rms_norm_bwd_kernel(const NormBwdParams p) {
  constexpr int kRows = norm_threads<kWarps> / (32 * kWarps);
  __shared__ float red[2][norm_threads<kWarps> / 32];
  __shared__ uint64_t full[kNormMaxStages];
  extern __shared__ __align__(128) uint8_t ring[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = (warp % kWarps) * 32 + lane;
  const float inv_h = 1.0f / static_cast<float>(p.H);
  const int inputs = p.dh != nullptr ? 3 : 2;
  const uint32_t row_bytes = static_cast<uint32_t>(p.H) * 2u;
  const uint32_t stage_bytes = row_bytes * kRows * inputs;
  const int64_t row_groups = (p.M + kRows - 1) / kRows;
  const int passes = static_cast<int>((row_groups - blockIdx.x + gridDim.x - 1) / gridDim.x);

  // Warp 0: fetch the rows of pass j (input i's row r at (i * kRows + r)), a copy per input where
  // its rows are contiguous, else one per row: many small copies cost more than their bytes
  // (20000 x 128: 15.0 us, 19.1 one by one).
  auto load_pass = [&](int j) {
    const int64_t r0 = (blockIdx.x + static_cast<int64_t>(j) * gridDim.x) * kRows;
    const int rows = static_cast<int>(p.M - r0 < kRows ? p.M - r0 : kRows);
    uint64_t* bar = &full[j % p.stages];
    if (lane == 0) mbar_arrive_expect_tx(bar, row_bytes * rows * inputs);
    __syncwarp();
    const int i = lane / kRows, r = lane - i * kRows;
    if (i < inputs && r < rows) {
      const __nv_bfloat16* base = i == 0 ? p.dy : i == 1 ? p.h : p.dh;
      const int64_t ld = i == 0 ? p.dy_ld : i == 1 ? p.h_ld : p.dh_ld;
      const bool whole = ld == p.H;
      if (!whole || r == 0)
        bulk_load(bar, ring + (j % p.stages) * stage_bytes + lane * row_bytes, base + (r0 + r) * ld,
                  whole ? row_bytes * rows : row_bytes);
    }
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    fence_mbarrier_init();
  }
  __syncthreads();
  grid_launch_dependents();  // the grid is one wave: the column sums' blocks can only queue behind it
  if (warp == 0)
    for (int j = 0; j < p.stages && j < passes; ++j) load_pass(j);

  // The gain stays in registers (16 a thread): its first load overlaps the first rows', and the
  // passes need none.  With two runs a thread there is no room, and it is read per row.
  constexpr bool kHoldGain = kChunks == 1;
  float2 gain[kHoldGain ? 1 : kChunks][8];
  if constexpr (kHoldGain) ld_gain(p.w, p.w_f32, t * kRunLen < p.H ? t * kRunLen : 0, gain[0]);

  float2 dw[kChunks][8];
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = make_float2(0.0f, 0.0f);

  const int64_t row_step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + warp / kWarps;
  float rstd_next = row < p.M ? __ldg(p.rstd + row) : 0.0f;
  bool ok = true;
  int j = 0;
  for (; j < passes; ++j, row += row_step) {
    const bool row_ok = row < p.M;
    const float rstd = rstd_next;
    rstd_next = row + row_step < p.M ? __ldg(p.rstd + row + row_step) : 0.0f;
    ok = mbar_wait(&full[j % p.stages], (j / p.stages) & 1u, kStNormLoad);
    const uint8_t* src = ring + (j % p.stages) * stage_bytes + (warp / kWarps) * row_bytes;
    Run16 vy[kChunks], vh[kChunks], vd[kChunks];
    float acc = 0.0f;
    const float2 r2 = make_float2(rstd, rstd);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (i * kWarps * 32 + t) * kRunLen;
      const bool in = row_ok && col < p.H;
      const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(src) + col;
      vy[i] = in ? ld_run(v) : zero_run();
      vh[i] = in ? ld_run(v + kRows * p.H) : zero_run();
      vd[i] = (in && inputs == 3) ? ld_run(v + 2 * kRows * p.H) : zero_run();
      float2 y[8], x[8], s = make_float2(0.0f, 0.0f);
      run_to_f2(vy[i], y);
      run_to_f2(vh[i], x);
      if constexpr (!kHoldGain) ld_gain(p.w, p.w_f32, col < p.H ? col : 0, gain[i]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 yx = __fmul2_rn(y[k], __fmul2_rn(x[k], r2));  // dy * xhat
        dw[i][k] = __fadd2_rn(dw[i][k], yx);
        s = __ffma2_rn(yx, gain[kHoldGain ? 0 : i][k], s);
      }
      acc += s.x + s.y;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    if (lane == 0) red[j & 1][warp] = acc;
    if (!__syncthreads_and(ok)) break;
    if (warp == 0 && j + p.stages < passes) load_pass(j + p.stages);
    float c = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) c += red[j & 1][warp / kWarps * kWarps + i];
    c *= -inv_h;
    const float2 c2 = make_float2(c, c);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (i * kWarps * 32 + t) * kRunLen;
      float2 y[8], x[8], d[8];
      run_to_f2(vy[i], y);
      run_to_f2(vh[i], x);
      run_to_f2(vd[i], d);
      if constexpr (!kHoldGain) ld_gain(p.w, p.w_f32, col < p.H ? col : 0, gain[i]);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        d[k] = __ffma2_rn(r2, __ffma2_rn(__fmul2_rn(x[k], r2), c2, __fmul2_rn(y[k], gain[kHoldGain ? 0 : i][k])), d[k]);
      if (row_ok && col < p.H) st_run(p.dx + row * p.H + col, f2_to_run(d));
    }
  }
  if (j < passes) {
    // A wait gave up: let the copies already issued land before the block exits.
    const int issued = j + p.stages < passes ? j + p.stages : passes;
    for (int i = j; i < issued; ++i) mbar_wait(&full[i % p.stages], (i / p.stages) & 1u, kStNormDrain);
    return;
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
        for (int k = 0; k < 4; ++k)
          dst[k] = make_float4(dw[i][2 * k].x, dw[i][2 * k].y, dw[i][2 * k + 1].x, dw[i][2 * k + 1].y);
      }
    }
  } else {
    // The block's row groups are added in row order, through the ring (all passes are consumed).
    constexpr int kRowLen = kWarps * 32 * kChunks * kRunLen;
    float* dw_rows = reinterpret_cast<float*>(ring);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        *reinterpret_cast<float2*>(dw_rows + (warp / kWarps) * kRowLen + (i * kWarps * 32 + t) * kRunLen + 2 * k) =
            dw[i][k];
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
// columns, its kColSumWarps warps every kColSumWarps-th partial row each, in a fixed order.
// Latency-bound (296 rows at most of a norm: ten dependent loads a thread would be, in one batch
// of loads here): 2.5 to 3 us with the launch, whose start overlaps the first kernel's end.  `part` is
// not __restrict__: it is being written when this kernel starts.
constexpr int kColSumWarps = 32;
__global__ void __launch_bounds__(kColSumWarps * 32)
    col_sum_kernel(const float* part, int parts, int N, void* out, bool out_f32) {
  __shared__ float red[kColSumWarps][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = blockIdx.x * 32 + lane;
  float s = 0.0f;
  grid_wait_dependencies();
  if (n < N) {
#pragma unroll 8
    for (int i = warp; i < parts; i += kColSumWarps) s += part[static_cast<int64_t>(i) * N + n];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && n < N) {
#pragma unroll
    for (int w = 1; w < kColSumWarps; ++w) s += red[w][lane];
    if (out_f32)
      static_cast<float*>(out)[n] = s;
    else
      static_cast<__nv_bfloat16*>(out)[n] = __float2bfloat16_rn(s);
  }
}

}  // namespace ltxfp8
