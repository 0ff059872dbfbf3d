// Weight gradient from an 8-bit activation checkpoint (tcgen05 + TMEM + TMA, sm_100a):
//
//   out[n, k] = bf16( alpha * sum_m g[m, n] * x~[m, k] ),   x~ = bf16(code[m, k] * scale[m, k/128])
//
// g bf16 [M, N] is the gradient of the layer's output, x the layer's input as the forward
// pass quantised it (e4m3 codes and 1x128 scales) or as bf16.  The scales vary along the
// summed axis, so they cannot be applied to partial sums as the forward GEMM does; the
// codes are expanded to bf16 on the way into the tensor core's operand tile instead (one
// rounding per value, 2^-9 relative at most, which a sum over tokens averages out).  No
// bf16 copy of x exists in memory.
//
// Both operands have the summed axis as their row axis, so they are MN-major operands of
// tcgen05.mma.kind::f16.  A CTA computes a 256 (k) x nt (n <= 256) tile as two M = 128
// accumulators that share the g tile; 64 tokens a stage.
//   warp 0      TMA producer: codes [64, 256] (16 KB) into the raw ring, g [64, nt] into its
//               own ring (bf16 x: straight into the operand ring)
//   warp 1      MMA issuer: 2 x 4 MMAs (M128 N=nt K16) a stage
//   warps 4-19  two groups of 8 that expand alternate stages of raw codes into the swizzled
//               MN-major operand tile; after the unit's last stage, all drain the accumulators
// The summed axis is divided among `splits` units where the tiles alone would not fill the
// GPU; those write fp32 partials that wgrad_reduce_kernel adds in split order.
#pragma once

#include "act_checkpoint.cuh"

namespace ltxfp8 {

constexpr int kWgTileK = 256;
constexpr int kWgStageM = 64;
constexpr int kWgGroups = 2;        // expanding warp groups; stage i belongs to group i % 2
constexpr int kWgThreads = 128 + kWgGroups * 256;
constexpr int kWgRawStages = 4;   // 16 KB each
constexpr int kWgGStages = 3;     // 32 KB each
constexpr int kWgOpStages = 2;    // 32 KB each (3 when x is bf16: no raw ring)
constexpr uint32_t kWgRawBytes = kWgStageM * kWgTileK;
constexpr uint32_t kWgOpBytes = kWgStageM * kWgTileK * 2;
constexpr uint32_t kWgGBytes = kWgStageM * 256 * 2;
constexpr uint32_t kWgAtomBytes = kWgStageM * 128;  // 64 M/N values x 64 tokens
constexpr uint32_t kWgSmemBytes = kWgRawStages * kWgRawBytes + kWgOpStages * kWgOpBytes + kWgGStages * kWgGBytes +
                                  1024 /*align*/ + 256 /*barriers*/;
static_assert(kWgRawStages * kWgRawBytes >= kWgOpBytes, "the bf16 form's third operand stage takes the raw ring's place");

enum WgradStatus : unsigned int {
  kStWgProducer = 0x57010001u,
  kStWgMma = 0x57010002u,
  kStWgConvert = 0x57010003u,
  kStWgAccFull = 0x57010004u,
  kStWgAccEmpty = 0x57010005u,
  kStWgDrain = 0x57010006u,
};

struct WgradParams {
  int M, N, K;
  int stages, stages_per_split, splits;  // token stages of 64
  int k_tiles, n_tiles, nt;              // nt: multiple of 16, <= 256
  int groups;                            // K / 128
  const float* xs;                       // element (m, kb) at xs[kb * xs_ld + m]
  int64_t xs_ld;
  float alpha;
  __nv_bfloat16* out;  // element (n, k) at out[n * ld_n + k * ld_k]; one of the strides is 1
  int64_t ld_n, ld_k;
  float* ws;  // splits > 1: partial of unit u at ws[u * nt * 256], row n, column k
};

struct WgradUnit {
  int k0, n0, first, count;  // first token stage and their number
};

__device__ __forceinline__ WgradUnit wgrad_unit(int u, const WgradParams& p) {
  const int tile = u / p.splits, split = u - tile * p.splits;
  const int nt = tile / p.k_tiles, kt = tile - nt * p.k_tiles;
  WgradUnit w;
  w.k0 = kt * kWgTileK;
  w.n0 = nt * p.nt;
  w.first = split * p.stages_per_split;
  w.count = min(p.stages_per_split, p.stages - w.first);
  return w;
}

// Expand 16 codes to bf16 (code * scale, rounded once) as two 16-byte operand chunks.
__device__ __forceinline__ void expand16(const uint4& v, float s, uint4& lo, uint4& hi) {
  float2 f[8];
  codes16_to_f2(v, f);
  const float2 s2 = make_float2(s, s);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = __fmul2_rn(f[j], s2);
  const Run16 r = f2_to_run(f);
  lo = r.a;
  hi = r.b;
}

template <bool kXFp8>
__global__ void __launch_bounds__(kWgThreads, 1)
    wgrad_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmG,
                 const WgradParams p) {
  constexpr int kOpStages = kXFp8 ? kWgOpStages : kWgOpStages + 1;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* s_op = smem;                                    // operand ring (x, bf16)
  uint8_t* s_raw = s_op + kWgOpStages * kWgOpBytes;        // raw ring; the bf16 form's third operand stage
  uint8_t* s_g = s_raw + kWgRawStages * kWgRawBytes;       // g ring
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(s_g + kWgGStages * kWgGBytes);
  uint64_t* raw_empty = raw_full + kWgRawStages;
  uint64_t* g_full = raw_empty + kWgRawStages;
  uint64_t* g_empty = g_full + kWgGStages;
  uint64_t* op_full = g_empty + kWgGStages;
  uint64_t* op_empty = op_full + kWgOpStages + 1;
  uint64_t* acc_full = op_empty + kWgOpStages + 1;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* drain = acc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0);
  const int lane = static_cast<int>(lane_id());

  if (threadIdx.x == 0) {
    for (int s = 0; s < kWgRawStages; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 8);
    }
    for (int s = 0; s < kWgGStages; ++s) {
      mbar_init(&g_full[s], 1);
      mbar_init(&g_empty[s], 1);
    }
    for (int s = 0; s < kOpStages; ++s) {
      mbar_init(&op_full[s], kXFp8 ? 8 : 1);
      mbar_init(&op_empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, kWgGroups * 8);
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmG);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int units = p.k_tiles * p.n_tiles * p.splits;

  if (warp == 0 && lane == 0) {
    // -------------------------------------------------------------- TMA producer
    const int boxes = (p.nt + 63) / 64;
    uint32_t it = 0;
    bool ok = true, x_sent = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const WgradUnit w = wgrad_unit(u, p);
      const int halves = w.k0 + 128 < p.K ? 2 : 1;
      for (int i = 0; i < w.count; ++i, ++it) {
        const int m0 = (w.first + i) * kWgStageM;
        x_sent = false;
        if constexpr (kXFp8) {
          const uint32_t s = it % kWgRawStages, ph = (it / kWgRawStages) & 1u;
          if (!mbar_wait(&raw_empty[s], ph ^ 1u, kStWgProducer)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&raw_full[s], halves * (kWgRawBytes / 2));
          for (int h = 0; h < halves; ++h)
            tma_load_2d(&tmX, &raw_full[s], s_raw + s * kWgRawBytes + h * (kWgRawBytes / 2), w.k0 + h * 128, m0);
        } else {
          const uint32_t s = it % kOpStages, ph = (it / kOpStages) & 1u;
          if (!mbar_wait(&op_empty[s], ph ^ 1u, kStWgProducer)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&op_full[s], halves * (kWgOpBytes / 2));
          for (int h = 0; h < 2 * halves; ++h)
            tma_load_2d(&tmX, &op_full[s], s_op + s * kWgOpBytes + h * kWgAtomBytes, w.k0 + h * 64, m0);
        }
        x_sent = true;
        const uint32_t s = it % kWgGStages, ph = (it / kWgGStages) & 1u;
        if (!mbar_wait(&g_empty[s], ph ^ 1u, kStWgProducer)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&g_full[s], boxes * kWgAtomBytes);
        for (int b = 0; b < boxes; ++b)
          tma_load_2d(&tmG, &g_full[s], s_g + s * kWgGBytes + b * kWgAtomBytes, w.n0 + b * 64, m0);
      }
    }
    if (!ok) {
      // Let the loads already in flight land before the CTA exits.
      const uint32_t x_it = it + (x_sent ? 1u : 0u);
      const uint32_t xs = kXFp8 ? kWgRawStages : kOpStages;
      uint64_t* xf = kXFp8 ? raw_full : op_full;
      for (uint32_t i = x_it > xs ? x_it - xs : 0u; i < x_it; ++i) mbar_wait(&xf[i % xs], (i / xs) & 1u, kStWgDrain);
      for (uint32_t i = it > kWgGStages ? it - kWgGStages : 0u; i < it; ++i)
        mbar_wait(&g_full[i % kWgGStages], (i / kWgGStages) & 1u, kStWgDrain);
    }
  } else if (warp == 1 && lane == 0) {
    // -------------------------------------------------------------- MMA issuer
    const uint32_t idesc =
        make_idesc(1u, 128u, static_cast<uint32_t>(p.nt)) | kIdescAMnMajor | kIdescBMnMajor;
    uint32_t it = 0, tcount = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x, ++tcount) {
      const WgradUnit w = wgrad_unit(u, p);
      const int halves = w.k0 + 128 < p.K ? 2 : 1;
      if (!mbar_wait(acc_empty, (tcount & 1u) ^ 1u, kStWgAccEmpty)) break;
      tc_fence_after_sync();
      for (int i = 0; i < w.count; ++i, ++it) {
        const uint32_t so = it % kOpStages, po = (it / kOpStages) & 1u;
        const uint32_t sg = it % kWgGStages, pg = (it / kWgGStages) & 1u;
        if (!mbar_wait(&g_full[sg], pg, kStWgMma) || !mbar_wait(&op_full[so], po, kStWgMma)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint64_t bdesc = sw128_mnmajor_desc(smem_u32(s_g + sg * kWgGBytes), kWgAtomBytes);
        for (int h = 0; h < halves; ++h) {
          const uint64_t adesc =
              sw128_mnmajor_desc(smem_u32(s_op + so * kWgOpBytes + h * (kWgOpBytes / 2)), kWgAtomBytes);
#pragma unroll
          for (int j = 0; j < 4; ++j)  // 16 tokens = 2048 B of every atom
            mma_f16(tmem_base + h * 256, adesc + 128u * j, bdesc + 128u * j, idesc, (i > 0 || j > 0) ? 1u : 0u);
        }
        tc_commit(&op_empty[so]);
        tc_commit(&g_empty[sg]);
      }
      if (ok) tc_commit(acc_full);
    }
    // Every MMA this thread issued has completed once `drain` flips.
    tc_commit(drain);
    mbar_wait(drain, 0u, kStWgDrain);
  } else if (warp >= 4) {
    // -------------------------------------------------------------- expansion, epilogue
    const int t = (static_cast<int>(threadIdx.x) - 128) & 255, grp = (warp - 4) >> 3;
    const int c = t & 7, rsub = t >> 3;  // 16-code chunk of a 128-code row, row modulo 32
    const int sp = warp & 3, half = ((warp - 4) >> 2) & 1;
    uint32_t it = 0, tcount = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x, ++tcount) {
      const WgradUnit w = wgrad_unit(u, p);
      if constexpr (kXFp8) {
        // Item j of a thread: half j >> 1, token row (j & 1) * 32 + rsub.
        const int g0 = w.k0 / 128;
        auto load_scales = [&](int i, float(&s)[4]) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int m = (w.first + i) * kWgStageM + (j & 1) * 32 + rsub, g = g0 + (j >> 1);
            s[j] = (i < w.count && m < p.M && g < p.groups) ? __ldg(p.xs + static_cast<int64_t>(g) * p.xs_ld + m) : 0.0f;
          }
        };
        float sc[4], nx[4];
        int i = static_cast<int>(it + grp) & (kWgGroups - 1);  // this group's first stage of the unit
        load_scales(i, sc);
        const uint32_t it0 = it;
        for (; i < w.count; i += kWgGroups) {
          it = it0 + i;
          load_scales(i + kWgGroups, nx);
          const uint32_t sr = it % kWgRawStages, pr = (it / kWgRawStages) & 1u;
          const uint32_t so = it % kOpStages, po = (it / kOpStages) & 1u;
          if (!__all_sync(0xffffffffu, mbar_wait(&raw_full[sr], pr, kStWgConvert)) ||
              !__all_sync(0xffffffffu, mbar_wait(&op_empty[so], po ^ 1u, kStWgConvert))) {
            ok = false;
            break;
          }
          const uint8_t* src = s_raw + sr * kWgRawBytes;
          uint8_t* dst = s_op + so * kWgOpBytes;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int h = j >> 1, row = (j & 1) * 32 + rsub;
            if (g0 + h >= p.groups) break;  // block-uniform: the tile's second group is outside K
            const uint4 v = *reinterpret_cast<const uint4*>(src + h * (kWgRawBytes / 2) + row * 128 + ((c ^ (row & 7)) * 16));
            uint4 lo, hi;
            expand16(v, sc[j], lo, hi);
            // Chunk c covers k = 16 c .. 16 c + 15 of the group: atom c >> 2, 16-byte positions
            // 2 (c & 3) and + 1, swizzled by the row.  Lanes of the second atom write their odd
            // position first, so the eight lanes of a row touch all 32 banks at once.
            uint8_t* atom = dst + h * (kWgOpBytes / 2) + (c >> 2) * kWgAtomBytes + row * 128;
            const int q0 = 2 * (c & 3) + (c >> 2), q1 = 2 * (c & 3) + 1 - (c >> 2);
            *reinterpret_cast<uint4*>(atom + ((q0 ^ (row & 7)) * 16)) = (c >> 2) ? hi : lo;
            *reinterpret_cast<uint4*>(atom + ((q1 ^ (row & 7)) * 16)) = (c >> 2) ? lo : hi;
          }
          fence_proxy_async_smem();  // the tensor core reads these bytes through the async proxy
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&raw_empty[sr]);
            mbar_arrive(&op_full[so]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[j] = nx[j];
        }
        if (!ok) break;
        it = it0 + w.count;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full, tcount & 1u, kStWgAccFull))) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      const int k = w.k0 + half * 128 + sp * 32 + lane;
      const bool k_ok = w.k0 + half * 128 < p.K;  // warp-uniform: K % 128 == 0
      if (k_ok) {
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(sp * 32) << 16) + half * 256;
        for (int c0 = grp * 32; c0 < p.nt; c0 += 32 * kWgGroups) {  // columns past nt are stale and not stored
          uint32_t r[32];
          tmem_ld_32x32b_x32(taddr + c0, r);
          tmem_wait_ld();
          if (p.splits > 1) {
            float* wsu = p.ws + (static_cast<int64_t>(u) * p.nt + c0) * kWgTileK + half * 128 + sp * 32 + lane;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c0 + j < p.nt) wsu[static_cast<int64_t>(j) * kWgTileK] = __uint_as_float(r[j]);
          } else if (p.ld_k == 1) {
            // Neighbouring lanes hold neighbouring k of the same columns: they trade so that the
            // even lane stores the pair of column j and the odd lane that of column j + 1.
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float a = __uint_as_float(r[j]) * p.alpha, b = __uint_as_float(r[j + 1]) * p.alpha;
              const float o = __shfl_xor_sync(0xffffffffu, (lane & 1) ? a : b, 1);
              const uint32_t v = (lane & 1) ? pack_bf16x2(o, b) : pack_bf16x2(a, o);
              const int n = w.n0 + c0 + j + (lane & 1);
              if (c0 + j < p.nt && n < p.N)
                *reinterpret_cast<uint32_t*>(p.out + static_cast<int64_t>(n) * p.ld_n + (k & ~1)) = v;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {  // N % 16 == 0: a run of 8 columns is all in or all out
              uint32_t v[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                v[i] = pack_bf16x2(__uint_as_float(r[j + 2 * i]) * p.alpha, __uint_as_float(r[j + 2 * i + 1]) * p.alpha);
              if (c0 + j < p.nt && w.n0 + c0 + j < p.N)
                *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(k) * p.ld_k + w.n0 + c0 + j) =
                    make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty);
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

// out = bf16(alpha * sum over splits of the partials), in split order: one thread per four
// neighbouring k of one n.
__global__ void __launch_bounds__(256) wgrad_reduce_kernel(const WgradParams p) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int kq = static_cast<int>(id & 63);
  const int64_t rowid = id >> 6;
  const int tile = static_cast<int>(rowid / p.nt), nr = static_cast<int>(rowid - static_cast<int64_t>(tile) * p.nt);
  if (tile >= p.k_tiles * p.n_tiles) return;
  const int ntile = tile / p.k_tiles, kt = tile - ntile * p.k_tiles;
  const int n = ntile * p.nt + nr, k = kt * kWgTileK + kq * 4;
  if (n >= p.N || k >= p.K) return;
  const int64_t stride = static_cast<int64_t>(p.nt) * kWgTileK;
  const float* src = p.ws + static_cast<int64_t>(tile) * p.splits * stride + static_cast<int64_t>(nr) * kWgTileK + kq * 4;
  float4 s = *reinterpret_cast<const float4*>(src);
#pragma unroll 4
  for (int i = 1; i < p.splits; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(src + i * stride);
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  if (p.ld_k == 1) {
    *reinterpret_cast<uint2*>(p.out + static_cast<int64_t>(n) * p.ld_n + k) =
        make_uint2(pack_bf16x2(s.x * p.alpha, s.y * p.alpha), pack_bf16x2(s.z * p.alpha, s.w * p.alpha));
  } else {
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p.out[static_cast<int64_t>(k + i) * p.ld_k + n * p.ld_n] = __float2bfloat16_rn(v[i] * p.alpha);
  }
}

}  // namespace ltxfp8
