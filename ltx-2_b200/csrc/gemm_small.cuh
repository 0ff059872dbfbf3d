// Blockwise FP8 GEMM with the residual epilogue for a few tokens (M <= 16, sm_100a):
//
//   D[m, n] = bf16( act( sum_kb sfa[m,kb] sfb[n/128,kb] (A[m,kb] . W[n,kb]) + bias[n] ) + residual[m, n] )
//
// Bound by reading the weight once: 7 x 4096 x 4096 takes 6.6 us in a chain of launches over 1 GB of
// weights (2.5 TB/s: 256 blocks ask for their 64 KB each at once and wait for it once), 5.1 us with
// the weight in L2 and 9 to 10 us as a launch alone behind an L2 flush, its start included.  The tensor-core kernel's 128-row tiles leave it 144 busy
// CTAs, a workspace of partial sums and a second launch; here a block owns 16 weight rows, each
// of its 8 warps an eighth of their K blocks (consecutive, so that a row is read in long
// stretches), and mma.sync m16n8k32 multiplies 16 weight rows by 8 tokens straight from registers:
// nothing passes through shared memory but the eight warps' sums at the end.  Within a K block the
// products may be summed in any order, so a lane takes the 32 bytes of a row that two 16-byte
// loads give it (bytes 16 t and 64 + 16 t, t = lane % 4) as its fragments, the same bytes of the
// weight and of the tokens.
#pragma once

#include "gemm.cuh"

namespace ltxfp8 {

constexpr int kSmallWarps = 8;
constexpr int kSmallRows = 16;  // weight rows of a block

struct GemmSmallParams {
  const uint8_t* a;
  const float* sfa;
  int64_t sfa_ld;
  const uint8_t* w;
  const float* sfb;
  const float* bias;         // null: none
  const __nv_bfloat16* res;  // null: none
  int64_t res_ld;
  __nv_bfloat16* d;
  int M, N, K, kb;  // kb = K / 128
};

__device__ __forceinline__ void mma_e4m3_16n8k32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// kT: groups of 8 tokens; kU: K blocks in flight per warp.  One 16-row tile a block, three blocks
// an SM: a block that walked several tiles with the next one's loads in flight needed twice the
// registers and took 12 % longer at 16384 x 4096, 40 % at 4096 x 4096.
template <int kAct, int kT, int kU>
__global__ void __launch_bounds__(kSmallWarps * 32) gemm_small_kernel(const GemmSmallParams p) {
  __shared__ float red[kSmallWarps][kT][8][kSmallRows];  // [warp][token group][token][row]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kSmallRows;
  const uint8_t* w0 = p.w + static_cast<int64_t>(n0 + g) * p.K + t * 16;
  const uint8_t* w1 = w0 + static_cast<int64_t>(8) * p.K;
  const float* sb_row = p.sfb + static_cast<int64_t>(n0 / 128) * p.kb;
  float acc[kT][4];
#pragma unroll
  for (int i = 0; i < kT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  const uint4 zero = make_uint4(0, 0, 0, 0);

  const int share = (p.kb + kSmallWarps - 1) / kSmallWarps;
  const int kb_end = min(p.kb, (warp + 1) * share);
  for (int kb0 = warp * share; kb0 < kb_end; kb0 += kU) {
    uint4 wa[kU][4], xb[kU][kT][2];
    float sb[kU], sa[kU][kT][2];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int kb = kb0 + u;
      const bool in = kb < kb_end;
      const int off = kb * 128;
      wa[u][0] = in ? __ldg(reinterpret_cast<const uint4*>(w0 + off)) : zero;
      wa[u][1] = in ? __ldg(reinterpret_cast<const uint4*>(w0 + off + 64)) : zero;
      wa[u][2] = in ? __ldg(reinterpret_cast<const uint4*>(w1 + off)) : zero;
      wa[u][3] = in ? __ldg(reinterpret_cast<const uint4*>(w1 + off + 64)) : zero;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int kb = kb0 + u;
      const bool in = kb < kb_end;
      sb[u] = in ? __ldg(sb_row + kb) : 0.0f;
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        const int m = i * 8 + g;
        const uint8_t* x = p.a + static_cast<int64_t>(m) * p.K + kb * 128 + t * 16;
        xb[u][i][0] = in && m < p.M ? __ldg(reinterpret_cast<const uint4*>(x)) : zero;
        xb[u][i][1] = in && m < p.M ? __ldg(reinterpret_cast<const uint4*>(x + 64)) : zero;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int mc = i * 8 + 2 * t + c;  // the accumulator's token columns
          sa[u][i][c] = in && mc < p.M ? __ldg(p.sfa + static_cast<int64_t>(kb) * p.sfa_ld + mc) : 0.0f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma_e4m3_16n8k32(c, wa[u][0].x, wa[u][2].x, wa[u][0].y, wa[u][2].y, xb[u][i][0].x, xb[u][i][0].y);
        mma_e4m3_16n8k32(c, wa[u][0].z, wa[u][2].z, wa[u][0].w, wa[u][2].w, xb[u][i][0].z, xb[u][i][0].w);
        mma_e4m3_16n8k32(c, wa[u][1].x, wa[u][3].x, wa[u][1].y, wa[u][3].y, xb[u][i][1].x, xb[u][i][1].y);
        mma_e4m3_16n8k32(c, wa[u][1].z, wa[u][3].z, wa[u][1].w, wa[u][3].w, xb[u][i][1].z, xb[u][i][1].w);
        const float s0 = sa[u][i][0] * sb[u], s1 = sa[u][i][1] * sb[u];
        acc[i][0] = fmaf(s0, c[0], acc[i][0]);
        acc[i][1] = fmaf(s1, c[1], acc[i][1]);
        acc[i][2] = fmaf(s0, c[2], acc[i][2]);
        acc[i][3] = fmaf(s1, c[3], acc[i][3]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kT; ++i) {
    red[warp][i][2 * t][g] = acc[i][0];
    red[warp][i][2 * t + 1][g] = acc[i][1];
    red[warp][i][2 * t][g + 8] = acc[i][2];
    red[warp][i][2 * t + 1][g + 8] = acc[i][3];
  }
  __syncthreads();
  for (int o = threadIdx.x; o < kT * 8 * kSmallRows; o += kSmallWarps * 32) {
    const int r = o % kSmallRows, m = o / kSmallRows;
    if (m >= p.M) break;  // later outputs of this thread are later tokens
    const float* src = &red[0][0][0][0] + o;
    float z = src[0];
#pragma unroll
    for (int w = 1; w < kSmallWarps; ++w) z += src[w * kT * 8 * kSmallRows];
    const int n = n0 + r;
    if (p.bias != nullptr) z += __ldg(p.bias + n);
    float y = act_apply<kAct>(make_float2(z, z)).x;
    if (p.res != nullptr) y += __bfloat162float(p.res[static_cast<int64_t>(m) * p.res_ld + n]);
    p.d[static_cast<int64_t>(m) * p.N + n] = __float2bfloat16_rn(y);
  }
}

}  // namespace ltxfp8
