// Dense e4m3 product with block scales for more tokens than stream_kernel takes (past 128
// always, from 65 on where it is the faster: fp8_streams):
//   C[m, n] = sum over K blocks b of  sa[m, b] sw[n / 128, b] (sum over k in b of a[m, k] w[n, k])
// and the gate/up pair of the feed-forward block, whose epilogue applies the gate
// function and quantises the activations per 1 x 128 group.
//
// A cluster of two CTAs computes 256 x 256 tiles with the 2-SM MMA (kind::f8f6f4),
// each CTA loading its 128 token rows and half of the tile's weight rows. The
// scales are fp32, so the tensor cores cannot apply them: each 128-wide K block is
// multiplied into one of two TMEM buffers, and while the next block's MMA runs, the
// epilogue warps read the product, multiply it by its one scale per row and weight
// block and add it to fp32 accumulators in registers. Scales whose product is no normal
// number are applied one after the other (scale_pair): four blocks' scales are tested at
// once, which is 0.3 to 1.4 % of the time (4096 x 14336 x 4096: 220.8 and 221.4 us).
//
// 4096 x 14336 x 4096 takes 220 us (2190 TFLOP/s; the product with a scale per row, whose
// MMA never waits for an epilogue, 176).
//
//   warp 0  TMA producer; warp 1  TMEM and MMA; warps 2, 3  idle
//   warps 4..11  epilogue, two per TMEM lane quarter, 128 accumulators a thread: group
//   g has of a plain tile the columns [128 g, +128), of a gate tile 64 gate columns
//   and the same features' 64 up columns. setmaxnreg gives them the registers that
//   the other warps do not need. The loads from TMEM are of 64 columns, so that a K
//   block costs two waits: the epilogue's chain of waits, not its sums, is what bounds
//   the kernel (4096 x 18944 x 4096: 279 us, 302 with 32 columns a load and the next
//   load in flight; 16 epilogue warps of half the accumulators 373; 232 with the loads and
//   sums taken out).
#pragma once
#include "ek_stream_kernel.cuh"

namespace ek {

template <bool kGate_>
struct Fp8BlockCfg {
  static constexpr bool kGate = kGate_;
  static constexpr int HALF_BYTES = 128 * 128, STAGE_BYTES = 2 * HALF_BYTES;
  static constexpr int STAGES = 5;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 128 + 32 * EPI_WARPS;
  // 384 threads are launched with 168 registers each: 128 x 56 + 256 x 224 = 64512 = 384 x 168
  static constexpr int REGS_LOAD = 56, REGS_EPI = 224;
  static constexpr uint32_t IDESC = umma_idesc(0u, false, 256, 256);
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_WARPS * 8192 + 1024 /*largest values*/ + 256 + 1024;
};

struct Fp8BlockParams {
  int M, N;              // tokens, columns (gate: features)
  int tiles_m, tiles_n, k_blocks, splits, num_units;
  const float* a_scale;   // [M][k_blocks]
  const float* w_scale;   // [w_blocks][k_blocks]; gate: W1's
  const float* w_scale2;  // gate: W3's
  int w_blocks;
  int scale4;            // rows of scales are a multiple of 16 bytes
  void* C;               // plain result
  int out_type;          // OutType
  int wide;              // rows of C are a multiple of 16 bytes
  float* ws;             // splits > 1: fp32 sums [splits][M][N] (gate: [splits][M][2 N])
  int gate;
  uint8_t* codes;        // gate: a [M][N] and its scales [M][ceil(N / 128)]
  float* scales;
};

// 64 fp32 sums of the lane's row to out[row0 + lane][col0 ..], n columns in rows of ld
// elements, n a multiple of 4; by way of 8 KB of shared memory as below
__device__ __forceinline__ void store_sums64(uint8_t* tile, int lane, float* out, long long ld, int row0, int rows, int col0,
                                             int n, const float* v) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 16; ++j)
    *reinterpret_cast<uint4*>(tile + lane * 256 + ((j ^ (lane & 7)) << 4)) = *reinterpret_cast<const uint4*>(v + j * 4);
  __syncwarp();
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int r = 2 * i + (lane >> 4), row = row0 + r, col = col0 + (lane & 15) * 4;
    if (row < rows && col < n)
      *reinterpret_cast<uint4*>(out + row * ld + col) =
          *reinterpret_cast<const uint4*>(tile + r * 256 + (((lane & 15) ^ (r & 7)) << 4));
  }
}

// The warp's 32 rows x 128 columns from (row0, col0), lane's row in v, to the result or to
// a slice's sums. They cross 8 KB of shared memory, 32 rows of 16 pieces of 16 bytes (a
// piece's place permuted by the row, so that no bank is met twice), so that a warp stores
// 256 contiguous bytes of two rows at a time: 0.3 us a tile where pieces of 16 bytes of 32
// rows took 3.5.
__device__ __forceinline__ void fp8_block_store(const Fp8BlockParams& p, uint8_t* tile, int lane, int split, int row0,
                                                int col0, const float* v) {
  auto piece = [&](int r, int j) -> uint4& { return *reinterpret_cast<uint4*>(tile + r * 256 + ((j ^ (r & 7)) << 4)); };
  const bool sums = p.splits > 1;
  if (p.wide && !sums && p.out_type != kOutFP32) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) piece(lane, j) = p.out_type == kOutBF16 ? pack8<kBF16>(v + j * 8) : pack8<kFP16>(v + j * 8);
    __syncwarp();
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const int r = 2 * i + (lane >> 4), row = row0 + r, col = col0 + (lane & 15) * 8;
      if (row < p.M && col < p.N)
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.C) + (size_t)row * p.N + col) = piece(r, lane & 15);
    }
    return;
  }
  float* out = sums ? p.ws + (size_t)split * p.M * p.N : reinterpret_cast<float*>(p.C);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) piece(lane, j) = *reinterpret_cast<const uint4*>(v + half * 64 + j * 4);
    __syncwarp();
    const int c0 = col0 + half * 64;
    if (p.wide) {
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const int r = 2 * i + (lane >> 4), row = row0 + r, col = c0 + (lane & 15) * 4;
        if (row < p.M && col < p.N) *reinterpret_cast<uint4*>(out + (size_t)row * p.N + col) = piece(r, lane & 15);
      }
    } else {
      // Rows that no 16-byte piece fits: consecutive lanes, consecutive elements, four rows
      // read before any is stored (1111 x 2113 x 7184, fp32: 33 us; row by row 37)
      const int type = sums ? kOutFP32 : p.out_type;
      void* to = sums ? p.ws + (size_t)split * p.M * p.N : p.C;
#pragma unroll 1
      for (int r0 = 0; r0 < 32 && row0 + r0 < p.M; r0 += 4) {
        float x[4][2];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = (i & 1) * 32 + lane;
          x[i >> 1][i & 1] = reinterpret_cast<const float*>(&piece(r0 + (i >> 1), c >> 2))[c & 3];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = row0 + r0 + (i >> 1), c = c0 + (i & 1) * 32 + lane;
          if (row < p.M && c < p.N) store_out(to, type, (size_t)row * p.N + c, x[i >> 1][i & 1]);
        }
      }
    }
  }
}

// 32 lanes x 64 consecutive 32-bit columns: one wait where two loads of 32 take two.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
      :
        "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr));
}
// Wait for it, tying the registers to the wait.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[64]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      :
        "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
        "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
        "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]),
        "+r"(r[32]), "+r"(r[33]), "+r"(r[34]), "+r"(r[35]), "+r"(r[36]), "+r"(r[37]), "+r"(r[38]), "+r"(r[39]),
        "+r"(r[40]), "+r"(r[41]), "+r"(r[42]), "+r"(r[43]), "+r"(r[44]), "+r"(r[45]), "+r"(r[46]), "+r"(r[47]),
        "+r"(r[48]), "+r"(r[49]), "+r"(r[50]), "+r"(r[51]), "+r"(r[52]), "+r"(r[53]), "+r"(r[54]), "+r"(r[55]),
        "+r"(r[56]), "+r"(r[57]), "+r"(r[58]), "+r"(r[59]), "+r"(r[60]), "+r"(r[61]), "+r"(r[62]), "+r"(r[63])
      :
      : "memory");
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
    fp8_block_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmB2, const Fp8BlockParams p) {
  constexpr int STAGES = Cfg::STAGES, HB = Cfg::HALF_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_tile = smem + STAGES * Cfg::STAGE_BYTES;                           // [EPI_WARPS] of 8 KB
  float* s_amax = reinterpret_cast<float*>(s_tile + Cfg::EPI_WARPS * 8192);     // [2][128]
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
  pdl_wait();
  pdl_launch();

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
    if (warp == 0) {
      if (elect_one()) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        if (Cfg::kGate) tma_prefetch_desc(&tmB2);
      }
      __syncwarp();
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
          ok = mbar_wait(&empty_bar[stage], phase ^ 1, s_abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (elect_one()) {
            uint8_t* dst = smem + stage * Cfg::STAGE_BYTES;
            if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * Cfg::STAGE_BYTES);
            tma_load_2d_pair(dst, &tmA, full0 + stage * 8, kb * 128, a_row);
            tma_load_2d_pair(dst + HB, tb, full0 + stage * 8, kb * 128, b_row);
          }
          __syncwarp();
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok && leader) wait_copies<STAGES>(full_bar, issued);
    } else if (warp == 1 && leader) {
      // the whole warp walks the loop and one elected lane issues, so that what it
      // issues is uniform (elect_one)
      int stage = 0, gkb = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t a_desc = umma_desc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t b_desc = umma_desc_sw128(smem_u32(smem) + HB, 16, 1024);
      for (int u = unit0; u < p.num_units && ok; u += unit_step) {
        const U w = unit(u);
        for (int kb = w.kb0; kb < w.kb1; ++kb, ++gkb) {
          const int buf = gkb & 1;
          ok = mbar_wait(&full_bar[stage], phase, s_abort) && mbar_wait(&kempty_bar[buf], ((gkb >> 1) & 1) ^ 1, s_abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint32_t off = stage * (Cfg::STAGE_BYTES >> 4);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_pair<true>(tmem_base + buf * 256, a_desc + off + 2 * k, b_desc + off + 2 * k, Cfg::IDESC, k > 0);
            umma_commit_pair(&kfull_bar[buf], 0x3);
            umma_commit_pair(&empty_bar[stage], 0x3);
          }
          __syncwarp();
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (elect_one()) umma_commit_pair(drain_bar, 0x3);  // every MMA has completed (in both CTAs) before TMEM is freed
      __syncwarp();
      volatile int never = 0;
      mbar_wait(drain_bar, 0, &never);
    } else if (warp == 1) {
      volatile int never = 0;
      mbar_wait(drain_bar, 0, &never);
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_EPI));
    const int q = warp & 3, wg = (warp - 4) >> 2;
    const int lrow = q * 32 + lane;
    uint8_t* tile = s_tile + (warp - 4) * 8192;
    const uint32_t kempty0 = mapa_shared(smem_u32(&kempty_bar[0]), 0);
    // group g reads half g: 64 columns of the first weight block (gate), 64 of the second (up)
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const uint32_t run0 = Cfg::kGate ? wg * 64 : wg * 128, run1 = Cfg::kGate ? 128 + wg * 64 : wg * 128 + 64;
    int gkb = 0;
    for (int u = unit0; u < p.num_units; u += unit_step) {
      const U w = unit(u);
      const int row0 = w.tm * 256 + rank * 128 + q * 32;
      float2 acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = make_float2(0.f, 0.f);
      uint32_t r[64];
      auto add = [&](int base, float x) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          acc[base + j] = fma2(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), make_float2(x, x),
                               acc[base + j]);
      };
      // The scales of four K blocks at a time, fetched four blocks ahead
      const int row = row0 + lane;
      const float* sa = p.a_scale + (size_t)(row < p.M ? row : 0) * KB;
      const int blk0 = Cfg::kGate ? w.tn : 2 * w.tn + wg, blk = blk0 < p.w_blocks ? blk0 : 0;
      const float* sw0 = p.w_scale + (size_t)blk * KB;
      const float* sw1 = Cfg::kGate ? p.w_scale2 + (size_t)blk * KB
                                    : sw0;
      const bool quads = p.scale4 && w.kb0 % 4 == 0;  // a slice of K may begin anywhere
      float xa[4], xw[4], xv[4];                       // of the next four blocks
      auto fetch = [&](int kb) {
        if (quads && kb + 4 <= KB) {
          const float4 a = __ldg(reinterpret_cast<const float4*>(sa + kb));
          const float4 b = __ldg(reinterpret_cast<const float4*>(sw0 + kb));
          const float4 c = __ldg(reinterpret_cast<const float4*>(sw1 + kb));
          xa[0] = a.x; xa[1] = a.y; xa[2] = a.z; xa[3] = a.w;
          xw[0] = b.x; xw[1] = b.y; xw[2] = b.z; xw[3] = b.w;
          xv[0] = c.x; xv[1] = c.y; xv[2] = c.z; xv[3] = c.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = min(kb + j, KB - 1);
            xa[j] = __ldg(sa + k);
            xw[j] = __ldg(sw0 + k);
            xv[j] = __ldg(sw1 + k);
          }
        }
      };
      fetch(w.kb0);
      // A failed wait has raised the abort flag: the loop then runs out without waiting and
      // the tile is not stored.
      auto block = [&](auto pairs, float f0, float x0, float f1, float x1) {
        auto scale = [&](float f) {
          if constexpr (decltype(pairs)::value) {
#pragma unroll
            for (int j = 0; j < 64; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * f);
          }
        };
        const int buf = gkb & 1;
        mbar_wait_soon(&kfull_bar[buf], (gkb >> 1) & 1, s_abort);
        __syncwarp();
        tc_fence_after();
        tmem_ld64(t_row + buf * 256 + run0, r);
        tmem_ld_wait(r);
        scale(f0);
        add(0, x0);
        tmem_ld64(t_row + buf * 256 + run1, r);
        tmem_ld_wait(r);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(kempty0 + buf * 8);
        scale(f1);
        add(32, x1);
        ++gkb;
      };
#pragma unroll 1
      for (int kb = w.kb0; kb < w.kb1; kb += 4) {
        float s0[4], s1[4], lo = 1.f, hi = 1.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s0[j] = xa[j] * xw[j];
          s1[j] = Cfg::kGate ? xa[j] * xv[j] : s0[j];
          lo = fminf(lo, fminf(fabsf(s0[j]), fabsf(s1[j])));
          hi = fmaxf(hi, fmaxf(fabsf(s0[j]), fabsf(s1[j])));
        }
        // a product of scales below or past fp32's normal numbers (scale_pair)
        const bool far = lo < 0x1p-126f || hi > 0x1.fffffep127f;
        if (kb + 4 < w.kb1) fetch(kb + 4);
        if (__any_sync(0xffffffffu, far)) {
#pragma unroll 1
          for (int k = kb; k < min(kb + 4, w.kb1); ++k) {
            float f0 = __ldg(sw0 + k), x0 = __ldg(sa + k), f1 = __ldg(sw1 + k), x1 = x0;
            scale_pair(x0, f0);
            scale_pair(x1, f1);
            block(std::true_type{}, f0, x0, f1, x1);
          }
          continue;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (kb + j < w.kb1) block(std::false_type{}, 1.f, s0[j], 1.f, s1[j]);
      }
      const bool good = !__any_sync(0xffffffffu, *s_abort);
      if (Cfg::kGate && p.splits > 1) {
        if (!good) break;
        const float* a = reinterpret_cast<const float*>(acc);  // [0, 64) gate, [64, 128) up
        float* out = p.ws + (size_t)w.split * p.M * (2ll * p.N);
        store_sums64(tile, lane, out, 2ll * p.N, row0, p.M, w.tn * 128 + wg * 64, p.N, a);
        store_sums64(tile, lane, out + p.N, 2ll * p.N, row0, p.M, w.tn * 128 + wg * 64, p.N, a + 64);
      } else if constexpr (Cfg::kGate) {
        // one decision for the epilogue warps: they meet for the groups' largest values
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
        // The codes are those of the quotients a / s, correctly rounded, as everywhere else. By
        // Markstein's theorem (IBM J. Res. Dev. 34, 1990): with rs = 1 / s correctly rounded and q
        // within an ulp of the quotient, q + (a - q s) rs is the quotient, the residue being
        // exact; a product with rs is within 1.5 ulp, the first step makes it less than one. Where
        // s is so small or large that a residue might leave fp32's range: divisions, which
        // for all would add 5 % to the 8-bit block of 2048 x 4096 x 14336 and 55 % to that of
        // 1000 x 512 x 8192, whose tiles are nearly all epilogue (this: nothing and 5 %).
        const float s = act_scale(m), rs = 1.0f / s;
        uint32_t c[16];
        if (s >= 0x1p-90f && s <= 0x1p110f) {
          auto quotient = [&](float x, float y) {
            const float2 v2 = make_float2(x, y), r2 = make_float2(rs, rs), n2 = make_float2(-s, -s);
            float2 q = mul2(v2, r2);
            q = fma2(fma2(n2, q, v2), r2, q);
            return fma2(fma2(n2, q, v2), r2, q);
          };
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float* v = a + i * 4;
            const float2 lo = quotient(v[0], v[1]), hi = quotient(v[2], v[3]);
            c[i] = e4m3x4(lo.x, lo.y, hi.x, hi.y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float* v = a + i * 4;
            c[i] = e4m3x4(v[0] / s, v[1] / s, v[2] / s, v[3] / s);
          }
        }
        uint4 pk[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) pk[g] = make_uint4(c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]);
        store_warp<16>(WarpTile{tile, lane}, pk, p.codes, row0, p.M, w.tn * 128 + wg * 64, p.N);
        if (wg == 0 && row < p.M) p.scales[(size_t)row * p.tiles_n + w.tn] = s;
      } else {
        if (!good) break;
        fp8_block_store(p, tile, lane, w.split, row0, w.tn * 256 + wg * 128, reinterpret_cast<const float*>(acc));
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

// What a gate tile's epilogue does, from the slices' sums: a warp per token and 128 features
__global__ void __launch_bounds__(256)
    fp8_gate_reduce_kernel(const float* __restrict__ ws, int splits, const StreamOut o) {
  pdl_wait();
  pdl_launch();
  const int t = blockIdx.y * 8 + (threadIdx.x >> 5), f = blockIdx.x * 128 + (threadIdx.x & 31) * 4;
  if (t >= o.T) return;
  float4 h1 = make_float4(0.f, 0.f, 0.f, 0.f), h3 = h1;
  if (f < o.N)
    for (int s = 0; s < splits; ++s) {
      const float* src = ws + ((size_t)s * o.T + t) * (2ll * o.N) + f;
      add4(h1, __ldcg(reinterpret_cast<const float4*>(src)));
      add4(h3, __ldcg(reinterpret_cast<const float4*>(src + o.N)));
    }
  finish_gate(o, t, blockIdx.x, h1, h3);
}

// out[i] = sum over the slices, in slice order, of ws[s][i]
__global__ void __launch_bounds__(256) fp8_block_reduce_kernel(const float* __restrict__ ws, int splits, long long n,
                                                               void* __restrict__ out, int type) {
  pdl_wait();
  pdl_launch();
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += __ldcg(ws + s * n + i);
    store_out(out, type, (size_t)i, v);
  }
}

}  // namespace ek
