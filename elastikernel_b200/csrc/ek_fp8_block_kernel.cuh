// Dense e4m3 product with block scales for more than 128 tokens:
//   C[m, n] = sum over K blocks b of  sa[m, b] sw[n / 128, b] (sum over k in b of a[m, k] w[n, k])
// and the gate/up pair of the feed-forward block, whose epilogue applies the gate
// function and quantises the activations per 1 x 128 group.
//
// A cluster of two CTAs computes 256 x 256 tiles with the 2-SM MMA (kind::f8f6f4),
// each CTA loading its 128 token rows and half of the tile's weight rows. The
// scales are fp32, so the tensor cores cannot apply them: each 128-wide K block is
// multiplied into one of two TMEM buffers, and while the next block's MMA runs, the
// epilogue warps read the product, multiply it by its one scale per row and half
// tile (a 128-column half lies in one weight block) and add it to fp32
// accumulators in registers. 256 threads hold 128 accumulators each; setmaxnreg
// gives them the registers that the loading and issuing warps do not need.
//
//   warp 0  TMA producer; warp 1  TMEM and MMA; warps 2, 3  idle
//   warps 4..11  epilogue, two per TMEM lane quarter: plain tiles half of the
//   columns each, gate tiles 64 gate columns and the same features' 64 up columns
#pragma once
#include "ek_stream_kernel.cuh"

namespace ek {

template <bool kGate_>
struct Fp8BlockCfg {
  static constexpr bool kGate = kGate_;
  static constexpr int STAGES = 6, HALF_BYTES = 128 * 128, STAGE_BYTES = 2 * HALF_BYTES;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 128 + 32 * EPI_WARPS;
  // 384 threads are launched with 168 registers each: 4 x 32 x 56 + 8 x 32 x 224 = 64512 = 384 x 168
  static constexpr int REGS_LOAD = 56, REGS_EPI = 224;
  static constexpr uint32_t IDESC = umma_idesc(0u, false, 256, 256);
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*amax*/ + 256 + 1024;
};

struct Fp8BlockParams {
  int M, N;              // tokens, columns (gate: features)
  int tiles_m, tiles_n, k_blocks, splits, num_units;
  const float* a_scale;   // [M][k_blocks]
  const float* w_scale;   // [w_blocks][k_blocks]; gate: W1's
  const float* w_scale2;  // gate: W3's
  int w_blocks;
  void* C;               // plain result
  int out_type;          // OutType
  int wide;              // rows of C are a multiple of 16 bytes
  float* ws;             // splits > 1: fp32 sums [splits][M][N]
  int gate;
  uint8_t* codes;        // gate: a [M][N] and its scales [M][ceil(N / 128)]
  float* scales;
};

// 32 consecutive columns of a row, from column col
__device__ __forceinline__ void fp8_block_store32(const Fp8BlockParams& p, void* base, int type, size_t row_at, int col,
                                                  const float2* v2) {
  const float* v = reinterpret_cast<const float*>(v2);
  if (p.wide || type == kOutFP32) {
    if (type == kOutFP32) {
      float* out = reinterpret_cast<float*>(base) + row_at + col;
      if (p.wide) {
#pragma unroll
        for (int g = 0; g < 8; ++g)
          if (col + g * 4 < p.N) *reinterpret_cast<float4*>(out + g * 4) = make_float4(v[4 * g], v[4 * g + 1],
                                                                                   v[4 * g + 2], v[4 * g + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col + j < p.N) out[j] = v[j];
      }
    } else if (type == kOutBF16) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (col + g * 8 < p.N) store8<kBF16>(base, row_at + col + g * 8, v + g * 8);
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (col + g * 8 < p.N) store8<kFP16>(base, row_at + col + g * 8, v + g * 8);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (col + j < p.N) store_out(base, type, row_at + col + j, v[j]);
  }
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
    fp8_block_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmB2, const Fp8BlockParams p) {
  constexpr int STAGES = Cfg::STAGES, HB = Cfg::HALF_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_amax = reinterpret_cast<float*>(smem + STAGES * Cfg::STAGE_BYTES);  // [2][128]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(s_amax + 256);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* kfull_bar = empty_bar + STAGES;
  uint64_t* kempty_bar = kfull_bar + 2;
  uint64_t* drain_bar = kempty_bar + 2;
  uint32_t* s_tmem_base = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem_base + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  const bool leader = rank == 0;
  const int unit0 = (int)cluster_id_x(), unit_step = (int)nclusters_x();
  const int KB = p.k_blocks;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&kfull_bar[b], 1);
      mbar_init(&kempty_bar[b], Cfg::EPI_WARPS * 2);
    }
    mbar_init(drain_bar, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<2>(s_tmem_base, 512);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers exist before anyone signals them
  tc_fence_after();
  const uint32_t tmem_base = *s_tmem_base;

  struct U {
    int tm, tn, split, kb0, kb1;
  };
  auto unit = [&](int u) {
    U w;
    const int tile = u / p.splits;
    w.split = u - tile * p.splits;
    raster(tile, p.tiles_m, p.tiles_n, 8, w.tm, w.tn);
    w.kb0 = (int)((long long)w.split * KB / p.splits);
    w.kb1 = (int)((long long)(w.split + 1) * KB / p.splits);
    return w;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_LOAD));
    if (warp == 0 && lane == 0) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      if (Cfg::kGate) tma_prefetch_desc(&tmB2);
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t full0 = mapa_shared(smem_u32(&full_bar[0]), 0);  // both CTAs' loads complete on the leader's
      const CUtensorMap* tb = (Cfg::kGate && !leader) ? &tmB2 : &tmB;
      for (int u = unit0; u < p.num_units && ok; u += unit_step) {
        const U w = unit(u);
        const int a_row = w.tm * 256 + rank * 128;
        const int b_row = Cfg::kGate ? w.tn * 128 : w.tn * 256 + rank * 128;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, s_abort)) { ok = false; break; }
          uint8_t* dst = smem + stage * Cfg::STAGE_BYTES;
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * Cfg::STAGE_BYTES);
          tma_load_2d_pair(dst, &tmA, full0 + stage * 8, kb * 128, a_row);
          tma_load_2d_pair(dst + HB, tb, full0 + stage * 8, kb * 128, b_row);
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok && leader) wait_copies<STAGES>(full_bar, issued);
    } else if (warp == 1 && lane == 0 && leader) {
      int stage = 0, gkb = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = unit0; u < p.num_units && ok; u += unit_step) {
        const U w = unit(u);
        for (int kb = w.kb0; kb < w.kb1; ++kb, ++gkb) {
          const int buf = gkb & 1;
          if (!mbar_wait(&kempty_bar[buf], ((gkb >> 1) & 1) ^ 1, s_abort) ||
              !mbar_wait(&full_bar[stage], phase, s_abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + stage * Cfg::STAGE_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_pair<true>(tmem_base + buf * 256, umma_desc_sw128(a0 + k * 32, 16, 1024),
                            umma_desc_sw128(a0 + HB + k * 32, 16, 1024), Cfg::IDESC, k > 0 ? 1u : 0u);
          umma_commit_pair(&empty_bar[stage], 0x3);
          umma_commit_pair(&kfull_bar[buf], 0x3);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      umma_commit_pair(drain_bar, 0x3);  // every MMA has completed (in both CTAs) before TMEM is freed
      volatile int never = 0;
      mbar_wait(drain_bar, 0, &never);
    } else if (warp == 1 && lane == 0) {
      volatile int never = 0;
      mbar_wait(drain_bar, 0, &never);
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_EPI));
    const int q = warp & 3, wg = (warp - 4) >> 2;
    const int lrow = q * 32 + lane;
    const uint32_t kempty0 = mapa_shared(smem_u32(&kempty_bar[0]), 0);
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    int gkb = 0;
    for (int u = unit0; u < p.num_units; u += unit_step) {
      const U w = unit(u);
      const int row = w.tm * 256 + rank * 128 + lrow;
      const bool row_ok = row < p.M;
      const float* sa = p.a_scale + (size_t)(row_ok ? row : 0) * KB;
      const int blk = Cfg::kGate ? w.tn : w.tn * 2 + wg;
      const bool blk_ok = blk < p.w_blocks;
      const float* sw = p.w_scale + (size_t)(blk_ok ? blk : 0) * KB;
      const float* sw2 = Cfg::kGate ? p.w_scale2 + (size_t)blk * KB : sw;
      float2 acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = make_float2(0.f, 0.f);
      // scales of this K block and the two after it
      float s0 = 0.f, s1 = 0.f, g0 = 0.f, g1 = 0.f, h0 = 0.f, h1 = 0.f;
      s0 = __ldg(sa + w.kb0);
      g0 = __ldg(sw + w.kb0);
      h0 = Cfg::kGate ? __ldg(sw2 + w.kb0) : g0;
      if (w.kb0 + 1 < w.kb1) {
        s1 = __ldg(sa + w.kb0 + 1);
        g1 = __ldg(sw + w.kb0 + 1);
        h1 = Cfg::kGate ? __ldg(sw2 + w.kb0 + 1) : g1;
      }
      bool good = true;
      for (int kb = w.kb0; kb < w.kb1; ++kb, ++gkb) {
        float s2 = 0.f, g2 = 0.f, h2 = 0.f;
        if (kb + 2 < w.kb1) {
          s2 = __ldg(sa + kb + 2);
          g2 = __ldg(sw + kb + 2);
          h2 = Cfg::kGate ? __ldg(sw2 + kb + 2) : g2;
        }
        const int buf = gkb & 1;
        const bool got = mbar_wait(&kfull_bar[buf], (gkb >> 1) & 1, s_abort);
        good = __all_sync(0xffffffffu, got);  // the TMEM loads are warp-collective
        if (!good) break;
        tc_fence_after();
        const uint32_t t0 = t_row + buf * 256 + (Cfg::kGate ? wg * 64 : wg * 128);
        // columns 0..63 and 64..127 of this warp: gate tiles have the up columns 128 further on
        const uint32_t t1 = Cfg::kGate ? t0 + 128 : t0 + 64;
        const float2 sg = make_float2(s0 * g0, s0 * g0), sh = make_float2(s0 * h0, s0 * h0);
        uint32_t ra[32], rb[32];
        auto add = [&](uint32_t(&r)[32], int base, float2 s) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[base + j] = fma2(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), s, acc[base + j]);
        };
        tmem_ld32(t0, ra);
        tmem_ld_wait(ra);
        tmem_ld32(t0 + 32, rb);
        add(ra, 0, sg);
        tmem_ld_wait(rb);
        tmem_ld32(t1, ra);
        add(rb, 16, sg);
        tmem_ld_wait(ra);
        tmem_ld32(t1 + 32, rb);
        add(ra, 32, sh);
        tmem_ld_wait(rb);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(kempty0 + buf * 8);
        add(rb, 48, sh);
        s0 = s1; g0 = g1; h0 = h1;
        s1 = s2; g1 = g2; h1 = h2;
      }
      if constexpr (Cfg::kGate) {
        // one decision for the eight warps: they meet for the groups' largest values
        if (named_bar_red_or(1, 32 * Cfg::EPI_WARPS, good ? 0 : 1)) break;
        float* a = reinterpret_cast<float*>(acc);  // [0, 64) gate, [64, 128) up
        float m = 0.f;
        with_gate(p.gate, [&](auto fn) {
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            a[j] = gate_f<decltype(fn)::value>(a[j]) * a[64 + j];
            m = fmaxf(m, fabsf(a[j]));  // features past N are zero
          }
        });
        s_amax[wg * 128 + lrow] = m;
        named_bar_sync(1, 32 * Cfg::EPI_WARPS);
        m = fmaxf(m, s_amax[(wg ^ 1) * 128 + lrow]);
        named_bar_sync(1, 32 * Cfg::EPI_WARPS);
        const float s = m > 0.f ? m / 448.0f : 1.0f;
        if (row_ok) {
          const int col = w.tn * 128 + wg * 64;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (col + g * 16 < p.N) {
              uint32_t pk[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float* v = a + g * 16 + i * 4;
                pk[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[0] / s, v[1] / s), __NV_SATFINITE, __NV_E4M3) |
                        ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[2] / s, v[3] / s), __NV_SATFINITE, __NV_E4M3)
                         << 16);
              }
              *reinterpret_cast<uint4*>(p.codes + (size_t)row * p.N + col + g * 16) =
                  make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
          }
          if (wg == 0) p.scales[(size_t)row * p.tiles_n + w.tn] = s;
        }
      } else {
        if (!good) break;
        if (row_ok) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int col = w.tn * 256 + wg * 128 + c * 32;
            if (p.splits > 1)
              fp8_block_store32(p, p.ws + (size_t)w.split * p.M * p.N, kOutFP32, (size_t)row * p.N, col, acc + c * 16);
            else
              fp8_block_store32(p, p.C, p.out_type, (size_t)row * p.N, col, acc + c * 16);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem_base, 512);
  }
}

// out[i] = sum over the slices, in slice order, of ws[s][i]
__global__ void __launch_bounds__(256) fp8_block_reduce_kernel(const float* __restrict__ ws, int splits, long long n,
                                                               void* __restrict__ out, int type) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += __ldcg(ws + s * n + i);
    store_out(out, type, (size_t)i, v);
  }
}

}  // namespace ek
