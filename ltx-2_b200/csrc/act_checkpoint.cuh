// An activation function with the 8-bit checkpoint of its input, and its use in the
// backward pass (streaming kernels, sm_100a).
//
//   forward   (yq, ys) = 1x128 quant of act(z)   the next GEMM's operand
//             (zq, zs) = 1x128 quant of z        all that the backward pass keeps of z
//   backward  z~ = zq * zs,  dz = dy * act'(z~), as bf16 (weight gradients), as 1x128 codes
//             (the input-gradient GEMM's operand) and summed over tokens (bias gradient)
//
// The activations and their derivatives are in activation.cuh; everything is fp32 and unrounded
// up to the outputs' own rounding.
#pragma once

#include "activation.cuh"
#include "residual_norm.cuh"

namespace ltxfp8 {

// 16 e4m3 codes -> fp32 (exact).
__device__ __forceinline__ void codes16_to_f2(const uint4& v, float2 (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __half22float2(__half2(
        __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] & 0xFFFFu), __NV_E4M3)));
    f[2 * i + 1] =
        __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] >> 16), __NV_E4M3)));
  }
}

struct ActSaveParams {
  const __nv_bfloat16* z;
  int64_t z_ld, M, N;
  uint32_t groups;  // N / 128
  uint32_t magic;   // ceil(2^32 / groups): k / groups = umulhi(k, magic) for the k used here
  uint8_t* yq;
  float* ys;
  int64_t ys_ld;
  uint8_t* zq;  // kSave: the checkpoint
  float* zs;
  int64_t zs_ld;
};

constexpr int kActSaveUnroll = 2;
constexpr int kActSaveGroups = 32 * kActSaveUnroll;  // 1x128 groups of a 256-thread block

// One pass, 8 lanes a group (its abs-max is three shuffles), two groups a thread in flight.  Without
// a checkpoint it is an instantiation of its own: as a branch it cost 180 bytes of spills (113
// against 71 us at 6144 x 16384).
// Measured, GELU with the checkpoint at 6144 x 16384: 72 us, 5.7 TB/s; the floor is 63 us of
// traffic (4.06 bytes a value).  What it spends besides are instructions: 17 a value, two of them on
// the exponential unit (exp2 and the reciprocal, 43 us of that unit alone); at a clock of 1.4 GHz
// under the power cap the same launch takes 93 us.
template <int kAct, bool kSave>
__global__ void __launch_bounds__(256, 6) act_quantize_save_kernel(const ActSaveParams p) {
  const int64_t g0 = static_cast<int64_t>(blockIdx.x) * kActSaveGroups;
  const int64_t row0 = g0 / p.groups;
  const uint32_t kb0 = static_cast<uint32_t>(g0 - row0 * p.groups);
  const int l8 = threadIdx.x & 7;
  Run16 v[kActSaveUnroll];
  int64_t row[kActSaveUnroll];
  uint32_t kb[kActSaveUnroll];
#pragma unroll
  for (int u = 0; u < kActSaveUnroll; ++u) {
    const uint32_t k = kb0 + (threadIdx.x >> 3) + 32u * u;
    const uint32_t dr = p.groups == 1 ? k : __umulhi(k, p.magic);
    row[u] = row0 + dr;
    kb[u] = k - dr * p.groups;
    v[u] = row[u] < p.M ? ld_run(p.z + row[u] * p.z_ld + kb[u] * 128 + l8 * kRunLen) : zero_run();
  }
#pragma unroll
  for (int u = 0; u < kActSaveUnroll; ++u) {
    float2 z[8], y[8];
    run_to_f2(v[u], z);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = act_apply<kAct>(z[j]);
    float zi = 0.0f, yi;
    uint4 zc;
    if constexpr (kSave) zc = quant_run16(z, zi);
    const uint4 yc = quant_run16(y, yi);
    if (row[u] < p.M) {
      const int64_t off = row[u] * p.N + kb[u] * 128 + l8 * kRunLen;
      *reinterpret_cast<uint4*>(p.yq + off) = yc;
      if constexpr (kSave) *reinterpret_cast<uint4*>(p.zq + off) = zc;
      if (l8 == 0) {
        p.ys[static_cast<int64_t>(kb[u]) * p.ys_ld + row[u]] = yi;
        if constexpr (kSave) p.zs[static_cast<int64_t>(kb[u]) * p.zs_ld + row[u]] = zi;
      }
    }
  }
}

struct ActBwdParams {
  const __nv_bfloat16* dy;
  int64_t dy_ld, M, N;
  const uint8_t* zq;
  const float* zs;
  int64_t zs_ld;
  int groups;                    // N / 128
  int col_groups, rows, passes;  // 1x128 groups of a column block, rows of a pass, passes over M
  __nv_bfloat16* dz;             // [M, N] or null
  uint8_t* dzq;                  // [M, N] or null
  float* dzs;
  int64_t dzs_ld;
  float* db_part;  // [gridDim.y, N] partial column sums, or null
};

// Block (x, y) owns column block x and walks the passes y, y + gridDim.y, ... of `rows` rows
// each, so the bias gradient of its columns stays in registers; the partial sums of the
// gridDim.y row shares are added by col_sum_kernel in a fixed order.  8 lanes hold a group.
//
// HBM-bound (6 bytes a value); the loop's arithmetic (two exponential-unit instructions and
// about 20 others a value) hides the loads only if many are in flight, so bulk copies bring
// dy and the codes through a ring of shared-memory stages.  A stage is released by one
// arrival per warp as soon as its values are in registers.
// Measured with dz in both forms and dbias at 6143 x 16384: 107 to 109 us, 5.6 TB/s (floor 94 us of
// traffic); three stages (108 KB in flight on an SM) are best: two 109, four 109, six 111; loads to
// registers alone took 134 us where the first ring took 122.
// kDirect: a few rows (one share, so no partial sums and no second launch): the loads go straight
// to registers.
enum ActStatus : unsigned int { kStActLoad = 0x41010001u, kStActFree = 0x41010002u, kStActDrain = 0x41010003u };
constexpr int kActBwdMaxGroups = 32;  // 4096 columns = 256 threads x 16
constexpr int kActBwdStages = 3;
constexpr uint32_t kActBwdDyBytes = kActBwdMaxGroups * 256;                    // 8 KB a pass
constexpr uint32_t kActBwdStageBytes = kActBwdDyBytes + kActBwdMaxGroups * 128;  // + 4 KB of codes
constexpr uint32_t kActBwdSmemBytes = kActBwdStages * kActBwdStageBytes;       // 36 KB

template <int kAct, bool kDirect>
__global__ void __launch_bounds__(256, 3) act_backward_kernel(const ActBwdParams p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kActBwdStages], freed[kActBwdStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kb0 = blockIdx.x * p.col_groups;
  const int ngroups = min(p.col_groups, p.groups - kb0);  // of this block
  const int runs = p.col_groups * 8;
  const int r = threadIdx.x / runs, t = threadIdx.x - r * runs;
  const int kb = kb0 + t / 8;
  const bool mine = r < p.rows && t < ngroups * 8;
  const int64_t col0 = static_cast<int64_t>(kb0) * 128, col = col0 + t * kRunLen;
  const int npass = (p.passes - static_cast<int>(blockIdx.y) + static_cast<int>(gridDim.y) - 1) /
                    static_cast<int>(gridDim.y);

  // Warp 0: fetch pass j of this block, its dy and its codes: one copy each where the block's rows
  // are contiguous, else one per row and lane (many small copies cost more than their bytes).
  const bool whole_q = p.col_groups == p.groups, whole_y = whole_q && p.dy_ld == p.N;
  auto load_pass = [&](int j) {
    const int s = j % kActBwdStages;
    const int64_t m0 = (blockIdx.y + static_cast<int64_t>(j) * gridDim.y) * p.rows;
    const int rows = static_cast<int>(p.M - m0 < p.rows ? p.M - m0 : p.rows);
    if (lane == 0) mbar_arrive_expect_tx(&full[s], static_cast<uint32_t>(rows * ngroups) * 384u);
    __syncwarp();
    if (lane < rows) {
      uint8_t* st = ring + s * kActBwdStageBytes;
      const int64_t m = m0 + lane;
      if (!whole_y || lane == 0)
        bulk_load(&full[s], st + lane * p.col_groups * 256, p.dy + m * p.dy_ld + col0,
                  ngroups * 256u * (whole_y ? rows : 1));
      if (!whole_q || lane == 0)
        bulk_load(&full[s], st + kActBwdDyBytes + lane * p.col_groups * 128, p.zq + m * p.N + col0,
                  ngroups * 128u * (whole_q ? rows : 1));
    }
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < kActBwdStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&freed[s], 8);
    }
    fence_mbarrier_init();
  }
  __syncthreads();
  if constexpr (!kDirect) {
    grid_launch_dependents();
    if (warp == 0)
      for (int j = 0; j < kActBwdStages && j < npass; ++j) load_pass(j);
  }

  float2 db[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) db[k] = make_float2(0.0f, 0.0f);
  const int64_t step = static_cast<int64_t>(gridDim.y) * p.rows;
  int64_t m = static_cast<int64_t>(blockIdx.y) * p.rows + r;
  const float* zs = p.zs + static_cast<int64_t>(mine ? kb : 0) * p.zs_ld;
  float sc_next = (mine && m < p.M) ? __ldg(zs + m) : 0.0f;
  int j = 0;
  for (; j < npass; ++j, m += step) {
    const int s = j % kActBwdStages;
    const uint32_t ph = (j / kActBwdStages) & 1u;
    const bool in = mine && m < p.M;
    const float sc = act_grad_scale(sc_next);
    sc_next = (mine && m + step < p.M) ? __ldg(zs + m + step) : 0.0f;
    Run16 vy = zero_run();
    uint4 vz = make_uint4(0, 0, 0, 0);
    if constexpr (kDirect) {
      if (in) {
        vy = ld_run(p.dy + m * p.dy_ld + col);
        vz = *reinterpret_cast<const uint4*>(p.zq + m * p.N + col);
      }
    } else {
      if (!warp_wait(&full[s], ph, kStActLoad)) break;
      const uint8_t* st = ring + s * kActBwdStageBytes;
      if (in) {
        vy = ld_run(reinterpret_cast<const __nv_bfloat16*>(st) + threadIdx.x * kRunLen);
        vz = *reinterpret_cast<const uint4*>(st + kActBwdDyBytes + threadIdx.x * kRunLen);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&freed[s]);
    }
    float2 d[8], z[8];
    run_to_f2(vy, d);
    codes16_to_f2(vz, z);
    const float2 s2 = make_float2(sc, sc);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      d[k] = __fmul2_rn(d[k], act_grad<kAct>(__fmul2_rn(z[k], s2)));
      db[k] = __fadd2_rn(db[k], d[k]);
    }
    if (p.dz != nullptr && in) st_run(p.dz + m * p.N + col, f2_to_run(d));
    if (p.dzq != nullptr) {
      float inv;
      const uint4 c = quant_run16(d, inv);
      if (in) {
        *reinterpret_cast<uint4*>(p.dzq + m * p.N + col) = c;
        if ((t & 7) == 0) p.dzs[static_cast<int64_t>(kb) * p.dzs_ld + m] = inv;
      }
    }
    if (!kDirect && warp == 0 && j + kActBwdStages < npass) {
      if (!warp_wait(&freed[s], ph, kStActFree)) break;
      load_pass(j + kActBwdStages);
    }
  }
  if (!kDirect && j < npass && warp == 0) {
    // A wait gave up: let the copies already issued land before the block exits.
    const int issued = j + kActBwdStages < npass ? j + kActBwdStages : npass;
    for (int i = j; i < issued; ++i) warp_wait(&full[i % kActBwdStages], (i / kActBwdStages) & 1u, kStActDrain);
  }
  __syncthreads();
  if (p.db_part == nullptr) return;
  // The block's rows are added in row order, through the ring (every pass is consumed).
  float* db_rows = reinterpret_cast<float*>(ring);
  if (mine) {
#pragma unroll
    for (int k = 0; k < 8; ++k) *reinterpret_cast<float2*>(db_rows + threadIdx.x * kRunLen + 2 * k) = db[k];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < ngroups * 128; c += 256) {
    float s = db_rows[c];
    for (int i = 1; i < p.rows; ++i) s += db_rows[i * p.col_groups * 128 + c];
    p.db_part[static_cast<int64_t>(blockIdx.y) * p.N + col0 + c] = s;
  }
}

// Transpose of a blockwise-FP8 weight: codes [N, K] -> [K, N], scales [N/128, K/128] ->
// [K/128, N/128], one 128 x 128 block per thread block: the operand of the input-gradient
// GEMM dX = dY W.  Codes pass through a padded shared tile in 4 x 4 byte squares.
__global__ void __launch_bounds__(256) transpose_weight_kernel(const uint8_t* __restrict__ q,
                                                               const float* __restrict__ s, int64_t N, int64_t K,
                                                               uint8_t* __restrict__ qt, float* __restrict__ st) {
  __shared__ uint32_t tile[128][33];  // row n, four codes a word
  const int64_t kb = blockIdx.x, nb = blockIdx.y;
  const uint8_t* src = q + nb * 128 * K + kb * 128;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 32 + (threadIdx.x >> 3), c = threadIdx.x & 7;
    const uint4 v = *reinterpret_cast<const uint4*>(src + row * K + c * 16);
    tile[row][c * 4] = v.x;
    tile[row][c * 4 + 1] = v.y;
    tile[row][c * 4 + 2] = v.z;
    tile[row][c * 4 + 3] = v.w;
  }
  __syncthreads();
  uint8_t* dst = qt + kb * 128 * N + nb * 128;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // square (n4, k4): rows n4*4 .. +3 of word k4 -> rows k4*4 .. +3, word n4
    const int n4 = threadIdx.x & 31, k4 = i * 8 + (threadIdx.x >> 5);
    const uint32_t a = tile[n4 * 4][k4], b = tile[n4 * 4 + 1][k4], c = tile[n4 * 4 + 2][k4], d = tile[n4 * 4 + 3][k4];
    const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
    const uint32_t cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
    uint32_t* o = reinterpret_cast<uint32_t*>(dst + static_cast<int64_t>(k4) * 4 * N) + n4;
    const int64_t ld = N / 4;
    o[0] = __byte_perm(ab0, cd0, 0x5410);
    o[ld] = __byte_perm(ab0, cd0, 0x7632);
    o[2 * ld] = __byte_perm(ab1, cd1, 0x5410);
    o[3 * ld] = __byte_perm(ab1, cd1, 0x7632);
  }
  if (threadIdx.x == 0) st[kb * (N / 128) + nb] = s[nb * (K / 128) + kb];
}

}  // namespace ltxfp8
