// Weight gradient from an 8-bit activation checkpoint (tcgen05 + TMEM + TMA, sm_100a):
//
//   out[n, k] = bf16( alpha * sum_m g[m, n] * x~[m, k] ),   x~ = bf16(code[m, k] * scale[m, k/128])
//
// g bf16 [M, N] is the gradient of the layer's output, x the layer's input as the forward
// pass quantised it (e4m3 codes and 1x128 scales) or as bf16.  The scales vary along the
// summed axis, so they cannot be applied to partial sums as the forward GEMM does; the
// codes are expanded to bf16 on the way into the tensor core's operand tile instead: one
// rounding per value, 2^-8 of it at most and of either sign: about as much again as the result's
// own rounding (0.0022 against 0.0017 in the root mean square, measured), and a 16th of the
// codes' (e4m3, 2^-4).  Rounding the scales into g would round as often.  No bf16 copy of x
// exists in memory.
//
// Both operands have the summed axis as their row axis, so they are MN-major operands of
// tcgen05.mma.kind::f16, 64 tokens a stage.  A CTA computes a 256 (k) x nt (n <= 256) tile as
// two M = 128 accumulators that share the g tile.
//   warp 0      TMA producer of x: codes [64, 256] (16 KB) into the raw ring (bf16 x: straight
//               into the operand ring)
//   warp 2      TMA producer of g [64, nt] into its own ring: a stage of codes is free as soon as
//               its values are in registers, one of g only after its MMAs
//   warp 1      MMA issuer: 2 x 4 MMAs (K16) a stage
//   warps 4-19  two groups of 8 that expand alternate stages of codes into the swizzled MN-major
//               operand ring; after the unit's last stage, all drain the accumulators
// The producers' and the issuer's instructions share the schedulers with 16 busy warps (about
// 100 cycles each at one thread a warp): their loops run warp-uniform, with as few copies and
// waits as the layouts allow.
// kPair: two CTAs of a cluster work on one 512 (k) x nt tile with cta_group::2 MMAs (M = 256):
// each expands its own 256 k and loads half of the g tile, the leader issues the MMAs.  What
// bounds the kernel for wide g is shared-memory bandwidth (128 B a cycle): per stage of 1024
// MMA cycles at nt = 256 one CTA alone moves 48 KB of TMA writes, 48 KB of expansion and 96 KB
// of operand reads (1500 cycles); in a pair the g tile is stored once per pair and each SM's
// tensor core reads half of it: 144 KB (1150 cycles), and the traffic from L2 falls from 48 KB
// to 32 KB a stage and SM.
// Measured, 2 M N K / time: 6144 x 4096 x 4096 151 us (1366 TFLOP/s, tensor pipe 86 % active; the
// library's product of bf16 operands, without the expansion, takes 138), 24576 x 4096 x 4096 565 us
// (1460 TFLOP/s).  For few columns of g (LoRA factors) the expansion bounds it, 16 codes a cycle
// and SM, for many tokens: 24576 x 128 x 4096 takes 38 us against 17 of traffic, about 22 of them
// expansion.  At 6143 x 32 x 4096 (15 us against 4) it is 11 stages of some 924 cycles a unit, 5 us; the
// rest is fixed: launch, set-up and drain, the fp32 partials' way through memory, the second launch.
// The summed axis is divided among `splits` units where the tiles alone would not fill the
// GPU; those write fp32 partials that wgrad_reduce_kernel adds in split order.
#pragma once

#include "act_checkpoint.cuh"

namespace ltxfp8 {

constexpr int kWgTileK = 256;  // of one CTA
constexpr int kWgStageM = 64;
constexpr int kWgExpandWarps = 16;
constexpr int kWgGroups = 2;  // of expanding warps
// A multiple of the groups, so that a raw slot always serves the same group: with an odd count a
// group could run ahead, meet a slot whose earlier load (the other group's, completing late) is
// still pending, and take the phase before that for its own.
constexpr int kWgRawStages[2] = {4, 2};
static_assert(kWgRawStages[0] % kWgGroups == 0 && kWgRawStages[1] % kWgGroups == 0, "a raw slot belongs to one group");
constexpr int kWgGroupWarps = kWgExpandWarps / kWgGroups;
constexpr int kWgThreads = 128 + kWgExpandWarps * 32;
constexpr int kWgMaxStages = 8;   // of any ring
constexpr uint32_t kWgRawBytes = kWgStageM * kWgTileK;
constexpr uint32_t kWgOpBytes = kWgStageM * kWgTileK * 2;
constexpr uint32_t kWgAtomBytes = kWgStageM * 128;  // 64 M/N values x 64 tokens
constexpr uint32_t kWgRingBytes = 224 * 1024;       // all rings
constexpr uint32_t kWgSmemBytes = kWgRingBytes + 1024 /*align*/ + 512 /*barriers*/;

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
  float* ws;  // splits > 1: partial of unit u (and CTA r of a pair) at ws[(u * pair + r) * nt * 256], [n][k]
  int op_stages, raw_stages, g_stages;  // of the rings (bf16 x: no raw ring)
};

// Position in a ring of n stages.
struct RingPos {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next(int n) {
    if (++s == n) {
      s = 0;
      ph ^= 1u;
    }
  }
};

struct WgradUnit {
  int k0, n0, first, count;  // first token stage and their number
};

// `ctas`: CTAs that share a unit; k0 is the first one's.
__device__ __forceinline__ WgradUnit wgrad_unit(int u, const WgradParams& p, int ctas) {
  const int tile = u / p.splits, split = u - tile * p.splits;
  const int nt = tile / p.k_tiles, kt = tile - nt * p.k_tiles;
  WgradUnit w;
  w.k0 = kt * kWgTileK * ctas;
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

template <bool kXFp8, bool kPair>
__global__ void __launch_bounds__(kWgThreads, 1)
    wgrad_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmG,
                 const WgradParams p) {
  constexpr int kCtas = kPair ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  const int g_cols = p.nt / kCtas;  // columns of g that this CTA loads
  const int boxes = (g_cols + 63) / 64;
  const uint32_t g_bytes = boxes * kWgAtomBytes;
  uint8_t* s_op = smem;                                 // operand ring (x, bf16)
  uint8_t* s_raw = s_op + p.op_stages * kWgOpBytes;     // raw ring (codes)
  uint8_t* s_g = s_raw + p.raw_stages * kWgRawBytes;    // g ring
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(smem + kWgRingBytes);
  uint64_t* raw_empty = raw_full + kWgMaxStages;
  uint64_t* g_full = raw_empty + kWgMaxStages;   // in a pair: the leader's are used
  uint64_t* g_empty = g_full + kWgMaxStages;
  uint64_t* op_full = g_empty + kWgMaxStages;    // in a pair: the leader's are used
  uint64_t* op_empty = op_full + kWgMaxStages;
  uint64_t* acc_full = op_empty + kWgMaxStages;
  uint64_t* acc_empty = acc_full + 1;            // in a pair: the leader's is used
  uint64_t* drain = acc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0);
  const int lane = static_cast<int>(lane_id());
  const int rank = kPair ? static_cast<int>(cluster_ctarank()) : 0;
  const bool leader = rank == 0;
  const int team = static_cast<int>(blockIdx.x) / kCtas, teams = static_cast<int>(gridDim.x) / kCtas;

  if (threadIdx.x < kWgMaxStages) {
    const int s = static_cast<int>(threadIdx.x);
    mbar_init(&raw_full[s], 1);
    mbar_init(&raw_empty[s], kWgGroupWarps);
    mbar_init(&g_full[s], 1);
    mbar_init(&g_empty[s], 1);
    mbar_init(&op_full[s], kXFp8 ? kWgGroupWarps * kCtas : 1);
    mbar_init(&op_empty[s], 1);
    if (s == 0) {
      mbar_init(acc_full, 1);
      mbar_init(acc_empty, kWgExpandWarps * kCtas);
      mbar_init(drain, 1);
    }
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmG);
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  if constexpr (kPair) cluster_sync();
  else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int units = p.k_tiles * p.n_tiles * p.splits;
  grid_launch_dependents();

  if (warp == 0 || warp == 2) {
    // -------------------------------------------------------------- TMA producers: x, g
    // Columns beyond K or N and rows beyond M arrive as zeros.  In a pair the copies that the
    // leader's MMAs wait for directly (g, bf16 x) complete on the leader's barriers.
    const bool is_x = warp == 0;
    const bool shared_bar = kPair && !(kXFp8 && is_x);
    uint64_t* full = !is_x ? g_full : kXFp8 ? raw_full : op_full;
    uint64_t* empty = !is_x ? g_empty : kXFp8 ? raw_empty : op_empty;
    const int stages = !is_x ? p.g_stages : kXFp8 ? p.raw_stages : p.op_stages;
    const uint32_t bytes = !is_x ? g_bytes : kXFp8 ? kWgRawBytes : kWgOpBytes;
    uint8_t* ring = !is_x ? s_g : kXFp8 ? s_raw : s_op;
    const uint32_t full_l = shared_bar ? mapa_shared(smem_u32(full), 0) : 0u;
    RingPos pos;
    uint32_t sent = 0;
    bool ok = true;
    for (int u = team; u < units && ok; u += teams) {
      const WgradUnit w = wgrad_unit(u, p, kCtas);
      const int col = is_x ? w.k0 + rank * kWgTileK : w.n0 + rank * g_cols;
      const int copies = !is_x ? boxes : kXFp8 ? 1 : kWgTileK / 64;
      for (int i = 0; i < w.count; ++i) {
        const int m0 = (w.first + i) * kWgStageM;
        if (!warp_wait(&empty[pos.s], pos.ph ^ 1u, kStWgProducer)) {
          ok = false;
          break;
        }
        uint8_t* dst = ring + pos.s * bytes;
        uint64_t* bar = &full[pos.s];
        if (elect_one()) {
          if (!shared_bar) mbar_arrive_expect_tx(bar, bytes);
          else if (leader) mbar_arrive_expect_tx(bar, 2u * bytes);
          const CUtensorMap* map = is_x ? &tmX : &tmG;
          for (int b = 0; b < copies; ++b) {
            if (kPair && shared_bar)
              tma_load_2d_pair(map, full_l + pos.s * 8u, dst + b * kWgAtomBytes, col + b * 64, m0);
            else
              tma_load_2d(map, bar, dst + b * kWgAtomBytes, col + b * 64, m0);
          }
        }
        __syncwarp();
        pos.next(stages);
        ++sent;
      }
    }
    if (!ok && (!shared_bar || leader)) {
      // Let the loads already in flight land before the CTA exits.
      for (uint32_t i = sent > static_cast<uint32_t>(stages) ? sent - stages : 0u; i < sent; ++i)
        warp_wait(&full[i % stages], (i / stages) & 1u, kStWgDrain);
    }
  } else if (warp == 1 && leader) {
    // -------------------------------------------------------------- MMA issuer
    const uint32_t idesc =
        make_idesc(1u, 128u * kCtas, static_cast<uint32_t>(p.nt)) | kIdescAMnMajor | kIdescBMnMajor;
    auto commit = [](uint64_t* bar) {
      if constexpr (kPair) tc_commit_pair_mc(bar, 0x3);
      else tc_commit(bar);
    };
    RingPos op, gp;
    uint32_t tcount = 0;
    bool ok = true;
    for (int u = team; u < units && ok; u += teams, ++tcount) {
      const WgradUnit w = wgrad_unit(u, p, kCtas);
      const int halves = w.k0 + 128 < p.K ? 2 : 1;
      if (!warp_wait(acc_empty, (tcount & 1u) ^ 1u, kStWgAccEmpty)) break;
      tc_fence_after_sync();
      for (int i = 0; i < w.count; ++i) {
        if (!warp_wait(&g_full[gp.s], gp.ph, kStWgMma) || !warp_wait(&op_full[op.s], op.ph, kStWgMma)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint64_t adesc = sw128_mnmajor_desc(smem_u32(s_op + op.s * kWgOpBytes), kWgAtomBytes);
        const uint64_t bdesc = sw128_mnmajor_desc(smem_u32(s_g + gp.s * g_bytes), kWgAtomBytes);
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h < halves) {
#pragma unroll
              for (int j = 0; j < kWgStageM / 16; ++j) {  // 16 tokens = 2048 B of every atom
                const uint64_t ad = adesc + (kWgOpBytes / 2 / 16) * h + 128u * j, bd = bdesc + 128u * j;
                const uint32_t acc = (i > 0 || j > 0) ? 1u : 0u;
                if constexpr (kPair) mma_f16_pair(tmem_base + h * 256, ad, bd, idesc, acc);
                else mma_f16(tmem_base + h * 256, ad, bd, idesc, acc);
              }
            }
          }
          commit(&op_empty[op.s]);
          commit(&g_empty[gp.s]);
          if (i == w.count - 1) commit(acc_full);
        }
        __syncwarp();
        op.next(p.op_stages);
        gp.next(p.g_stages);
      }
    }
    // Every MMA issued above has completed once `drain` flips (in both CTAs of a pair).
    if (elect_one()) commit(drain);
    __syncwarp();
    warp_wait(drain, 0u, kStWgDrain);
  } else if (warp >= 4) {
    // -------------------------------------------------------------- expansion, epilogue
    const uint32_t op_full_l = kPair ? mapa_shared(smem_u32(op_full), 0) : 0u;
    constexpr int kRowStep = kWgGroupWarps * 4;           // token rows a group covers at once
    constexpr int kItems = 2 * kWgStageM / kRowStep;       // 16-code chunks of a thread and stage
    const int grp = (warp - 4) / kWgGroupWarps;
    const int t = (static_cast<int>(threadIdx.x) - 128) % (kWgGroupWarps * 32);
    const int c = t & 7, row0 = t >> 3;  // chunk of each 128-code group, first token row of the stage
    const int sp = warp & 3, half = ((warp - 4) >> 2) & 1, colhalf = (warp - 4) >> 3;
    RingPos raw, op;
    for (int j = 0; kXFp8 && j < grp; ++j) {  // group j starts j stages behind
      raw.next(p.raw_stages);
      op.next(p.op_stages);
    }
    uint32_t it = 0, tcount = 0;  // stages and units so far
    bool ok = true;
    for (int u = team; u < units && ok; u += teams, ++tcount) {
      const WgradUnit w = wgrad_unit(u, p, kCtas);
      const int k0 = w.k0 + rank * kWgTileK;
      if constexpr (kXFp8) {
        const int g0 = k0 / 128;
        // Item j of a thread: 128-code group j & 1, token row (j >> 1) * kRowStep + row0.
        auto load_scales = [&](int i, float(&s)[kItems]) {
#pragma unroll
          for (int j = 0; j < kItems; ++j) {
            const int m = (w.first + i) * kWgStageM + (j >> 1) * kRowStep + row0, g = g0 + (j & 1);
            s[j] = (i < w.count && m < p.M && g < p.groups) ? __ldg(p.xs + static_cast<int64_t>(g) * p.xs_ld + m) : 0.0f;
          }
        };
        float sc[kItems], nx[kItems];
        int i = static_cast<int>((grp + kWgGroups - it % kWgGroups) % kWgGroups);  // its first stage of the unit
        load_scales(i, sc);
        for (; i < w.count; i += kWgGroups) {
          load_scales(i + kWgGroups, nx);
          if (!warp_wait(&raw_full[raw.s], raw.ph, kStWgConvert)) {
            ok = false;
            break;
          }
          const uint8_t* src = s_raw + raw.s * kWgRawBytes + row0 * kWgTileK + c * 16;
          uint8_t* dst = s_op + op.s * kWgOpBytes + (c >> 2) * kWgAtomBytes + row0 * 128;
          uint4 v[kItems];
#pragma unroll
          for (int j = 0; j < kItems; ++j)  // all loads before the first store, which they could alias
            v[j] = *reinterpret_cast<const uint4*>(src + (j >> 1) * (kRowStep * kWgTileK) + (j & 1) * 128);
          if (!warp_wait(&op_empty[op.s], op.ph ^ 1u, kStWgConvert)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive(&raw_empty[raw.s]);  // the warp's codes are in registers (the vote above)
#pragma unroll
          for (int j = 0; j < kItems; ++j) {
            // (A group outside K expands to zeros: its codes arrived as zeros, its scale is 0.)
            uint4 lo, hi;
            expand16(v[j], sc[j], lo, hi);
            // Chunk c covers k = 16 c .. 16 c + 15 of the group: atom c >> 2, 16-byte positions
            // 2 (c & 3) and + 1, swizzled by the row.  Lanes of the second atom write their odd
            // position first, so the eight lanes of a row touch all 32 banks at once.
            uint8_t* atom = dst + (j & 1) * (kWgOpBytes / 2) + (j >> 1) * (kRowStep * 128);
            const int q0 = 2 * (c & 3) + (c >> 2), q1 = 2 * (c & 3) + 1 - (c >> 2), sw = row0 & 7;  // kRowStep % 8 == 0
            *reinterpret_cast<uint4*>(atom + ((q0 ^ sw) * 16)) = (c >> 2) ? hi : lo;
            *reinterpret_cast<uint4*>(atom + ((q1 ^ sw) * 16)) = (c >> 2) ? lo : hi;
          }
          fence_proxy_async_smem();  // the tensor core reads these bytes through the async proxy
          __syncwarp();
          // The operand bytes are read by this SM's tensor core, through the async proxy that the
          // fence above orders them for; to the leader of a pair the arrival is only a signal.
          if (lane == 0) {
            if constexpr (kPair) mbar_arrive_cluster(op_full_l + op.s * 8u);
            else mbar_arrive(&op_full[op.s]);
          }
#pragma unroll
          for (int j = 0; j < kItems; ++j) sc[j] = nx[j];
#pragma unroll
          for (int j = 0; j < kWgGroups; ++j) {
            raw.next(p.raw_stages);
            op.next(p.op_stages);
          }
        }
        if (!ok) break;
        it += static_cast<uint32_t>(w.count);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full, tcount & 1u, kStWgAccFull))) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      const int k = k0 + half * 128 + sp * 32 + lane;
      const bool k_ok = k0 + half * 128 < p.K;  // warp-uniform: K % 128 == 0
      if (k_ok) {
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(sp * 32) << 16) + half * 256;
        for (int c0 = colhalf * 32; c0 < p.nt; c0 += 64) {  // columns past nt are stale and not stored
          uint32_t r[32];
          tmem_ld_32x32b_x32(taddr + c0, r);
          tmem_wait_ld();
          if (p.splits > 1) {
            float* wsu = p.ws + (static_cast<int64_t>(u * kCtas + rank) * p.nt + c0) * kWgTileK + half * 128 + sp * 32 + lane;
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
      if (lane == 0) {
        if constexpr (kPair) mbar_arrive_cluster_release(mapa_shared(smem_u32(acc_empty), 0));
        else mbar_arrive(acc_empty);
      }
    }
  }
  if constexpr (kPair) {
    if (!leader && warp == 1) warp_wait(drain, 0u, kStWgDrain);  // the pair's MMAs read this CTA too
  }

  __syncwarp();
  tc_fence_before_sync();
  if constexpr (kPair) cluster_sync();  // no CTA leaves while its peer may still reach its memory
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    if constexpr (kPair) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

// out = bf16(alpha * sum over splits of the partials), in split order: one thread per four
// neighbouring k of one n of one CTA tile.
__global__ void __launch_bounds__(256) wgrad_reduce_kernel(const WgradParams p, int ctas) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int kq = static_cast<int>(id & 63);
  const int64_t rowid = id >> 6;
  const int part = static_cast<int>(rowid / p.nt), nr = static_cast<int>(rowid - static_cast<int64_t>(part) * p.nt);
  const int tile = part / ctas, rank = part - tile * ctas;
  if (tile >= p.k_tiles * p.n_tiles) return;
  const int ntile = tile / p.k_tiles, kt = tile - ntile * p.k_tiles;
  const int n = ntile * p.nt + nr, k = (kt * ctas + rank) * kWgTileK + kq * 4;
  if (n >= p.N || k >= p.K) return;
  const int64_t block = static_cast<int64_t>(p.nt) * kWgTileK;
  const float* src = p.ws + (static_cast<int64_t>(tile) * p.splits * ctas + rank) * block +
                     static_cast<int64_t>(nr) * kWgTileK + kq * 4;
  grid_wait_dependencies();
  float4 s = *reinterpret_cast<const float4*>(src);
#pragma unroll 4
  for (int i = 1; i < p.splits; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(src + i * ctas * block);
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
