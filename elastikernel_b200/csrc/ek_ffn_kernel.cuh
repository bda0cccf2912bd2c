// Products of the gated feed-forward block on tcgen05 CTA pairs, bf16 and fp16.
//
//   gate/up   h1 = x W1^T, h3 = x W3^T, a = f(h1) h3          (ffn_gemm_kernel, kFfnGate)
//   down      y = a W2^T                                      (kFfnStore)
//   backward  da = dy W2; dh1 = da h3 f'(h1); dh3 = da f(h1)  (kFfnGateGrad)
//             dx = dh1 W1 + dh3 W3, dW1 = dh1^T x, dW3 = dh3^T x, dW2 = dy^T a
//                                                             (ffn_grad_kernel)
//
// A persistent cluster of two CTAs computes a 256 x 256 (few tiles: 256 x 128) tile
// with the 2-SM MMA: each CTA loads its own 128 rows of A and half of the tile's B
// (32 KB per 64 of K, no multicast) and its TMEM receives its 128 rows. Operands are
// used where they lie: one whose reduction axis is not the contiguous one (the
// weights in a backward pass, everything under a weight's gradient) is read MN-major
// by the MMA, so nothing is transposed. The two weights of the gate, and the two
// planes of the pre-activations, are separate tensor maps, so no tail of one is ever
// read as the other's (gate/up: the first half of a tile's columns is W1's, the second
// W3's, chosen by the CTA's rank).
//
// Bound by the tensor cores: 4096 x 4096 x 14336 in bf16 takes 925 us forward with the
// pre-activations kept (1560 TFLOP/s, 0.95 of the measured burst) and 1791 us backward (1612,
// 0.98), on a device whose power cap does not bind; the gate's gradient alone is bound by L2
// (its five planes of activations beside the operands: 400 us, 335 without them).
//
//   warp 0      TMA producer; warp 1  TMEM and MMA issue
//   warps 2..9  epilogue, two per TMEM lane quarter, half of the columns each
//
// A TMEM lane is a row, so a thread holds 32 consecutive columns of one row. What it
// reads and writes goes through 2 KB of shared memory per warp: a global access
// then covers 64 contiguous bytes of each of 8 rows, not 16 of each of 32. The
// gradient's pre-activations are fetched a chunk ahead.
//
// Few tiles: K is split over `splits` units per tile whose fp32 sums go to a
// workspace, and the ffn_*_reduce kernels add them in slice order and do what the
// epilogue would have done. No atomics.
#pragma once
#include <type_traits>

#include "ek_act.cuh"
#include "ek_gemm_kernel.cuh"

namespace ek {

// Programmatic dependent launch. A call's first launch waits for whatever precedes it on
// the stream before it reads, writes or lets its successor start, so that from then on
// nothing the caller launched is still running: later launches of the call may fetch
// the weights (which no launch of the call writes) before their own wait.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// One lane of a converged warp, always the same. A loop that a whole warp walks with an
// elected lane issuing keeps the operands of tcgen05.mma uniform; issued from inside a
// one-lane branch they are moved to the uniform registers one by one, at about 100
// clocks an instruction (a 128-byte K block of a 256 x 256 tile: 730 clocks of issue
// for 512 of multiplying).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// mbar_wait for a phase that is expected within a microsecond or so: the clock is read
// only when it has not come by then.
__device__ __forceinline__ bool mbar_wait_soon(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const uint32_t a = smem_u32(bar);
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(a, parity)) return true;
  return mbar_wait(bar, parity, abort_flag);
}

enum FfnEpi : int { kFfnStore = 0, kFfnGate = 1, kFfnGateGrad = 2 };

template <int kElem_, bool kBMN_, int kEpi_, int BN_>
struct FfnCfg {
  static constexpr int kElem = kElem_;
  static constexpr bool kBMN = kBMN_;  // B stored with its reduction axis outermost
  static constexpr int kEpi = kEpi_;
  static constexpr int BN = BN_, BK = 64;       // tile columns (gate/up: half gate, half up); K per stage
  static constexpr int A_BYTES = 128 * 128;     // a CTA's 128 rows (MN-major: two chunks of 64 columns) of A
  static constexpr int B_BYTES = BN / 2 * 128;  // and its half of B
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES, STAGES = BN == 256 ? 6 : 8;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_WARPS * 2048 + 1024 + 256;
  static constexpr uint32_t IDESC =
      umma_idesc(kElem == kBF16 ? 1u : 0u, kBMN, 256, BN);
};

struct FfnParams {
  int M, N;              // rows and columns of the result
  int tiles_m, tiles_n, k_blocks, splits, num_units;
  int b_full;            // MN-major B: columns in whole 64-column chunks (see load_half)
  int gate;              // GateFn
  void* C;               // result; gate: a; gate gradient: dh
  long long c_plane;     // gate gradient: elements between dh1 and dh3
  void* H;               // gate: the pre-activations to write (or null); gate gradient: those to read
  long long h_plane;
  void* Act;             // gate gradient: a
  float* ws;             // splits > 1: fp32 sums [splits][M][N] (gate/up: [splits][M][2 N])
};

template <int kElem>
struct Elem16;
template <>
struct Elem16<kBF16> {
  __device__ static uint32_t pack(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ static float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
};
template <>
struct Elem16<kFP16> {
  __device__ static uint32_t pack(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ static float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
};

// 8 consecutive elements to or from global memory, 16-byte aligned.
template <int kElem>
__device__ __forceinline__ void store8(void* base, size_t at, const float* v) {
  uint4 pk;
  pk.x = Elem16<kElem>::pack(v[0], v[1]);
  pk.y = Elem16<kElem>::pack(v[2], v[3]);
  pk.z = Elem16<kElem>::pack(v[4], v[5]);
  pk.w = Elem16<kElem>::pack(v[6], v[7]);
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + at) = pk;
}
template <int kElem>
__device__ __forceinline__ void unpack8(const uint4& pk, float* v) {
  const uint32_t w[4] = {pk.x, pk.y, pk.z, pk.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem16<kElem>::unpack(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// A producer that gave up waits (with a limit) for the copies it has in flight:
// `issued` stages were filled in ring order. In a pair the leader's barriers count
// both CTAs' copies, and neither CTA leaves before the closing cluster barrier.
template <int kStages>
__device__ __forceinline__ void wait_copies(uint64_t* full_bar, int issued) {
  volatile int never = 0;
  for (int i = max(0, issued - kStages); i < issued; ++i)
    if (!mbar_wait(&full_bar[i % kStages], (i / kStages) & 1, &never)) return;
}

// A 32-row x 64-byte tile of a warp in shared memory: written or read as one row per
// lane, or as 64 bytes of 8 rows at a time (4 lanes a row). The 16-byte pieces of a
// row are permuted by its number, so neither way meets a bank twice.
struct WarpTile {
  uint8_t* base;
  int lane;
  __device__ uint4& own(int j) const {
    return *reinterpret_cast<uint4*>(base + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4));
  }
  __device__ uint4& across(int i) const {
    const int r = i * 8 + (lane >> 2);
    return *reinterpret_cast<uint4*>(base + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
  }
};

// Where lane's piece i of a warp's rows [row0, row0 + 32) x 16-byte groups from
// element col0 lies in a [rows, n] matrix (kPer elements per piece); < 0: outside.
template <int kPer>
__device__ __forceinline__ long long warp_at(int i, int lane, int row0, int rows, int col0, int n, long long ld) {
  const int r = row0 + i * 8 + (lane >> 2), c = col0 + (lane & 3) * kPer;
  return r < rows && c < n ? (long long)r * ld + c : -1;
}

// 64 bytes of each of the warp's rows, the lane's own in v, to out[row0 + lane][col0 ..]
// of a [rows, n] matrix with kPer elements per 16 bytes and rows of ld (0: n) elements
template <int kPer>
__device__ __forceinline__ void store_warp(const WarpTile& w, const uint4 (&v)[4], void* out, int row0, int rows, int col0,
                                           int n, long long ld = 0) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) w.own(j) = v[j];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long at = warp_at<kPer>(i, w.lane, row0, rows, col0, n, ld ? ld : n);
    if (at >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out) + at * (16 / kPer)) = w.across(i);
  }
}
// 32 columns of fp32, 16 at a time
__device__ __forceinline__ void store_warp32(const WarpTile& w, const uint32_t (&r)[32], float* out, int row0, int rows,
                                             int col0, int n, long long ld) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t* q = r + half * 16 + j * 4;
      v[j] = make_uint4(q[0], q[1], q[2], q[3]);
    }
    store_warp<4>(w, v, out, row0, rows, col0 + half * 16, n, ld);
  }
}

template <int kElem>
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(Elem16<kElem>::pack(v[0], v[1]), Elem16<kElem>::pack(v[2], v[3]), Elem16<kElem>::pack(v[4], v[5]),
                    Elem16<kElem>::pack(v[6], v[7]));
}
template <int kElem>
__device__ __forceinline__ void pack32(const uint32_t (&r)[32], uint4 (&v)[4]) {
#pragma unroll
  for (int g = 0; g < 4; ++g) v[g] = pack8<kElem>(reinterpret_cast<const float*>(r) + g * 8);
}

// A CTA's kRows of an operand's mn axis x 64 of K, from (mn, k0): K-major one box. MN-major
// 128 columns are two chunks of 64, the swizzle's width: one 3-D box of map m where both are
// whole (the columns up to `full`, whatever follows them), else a 2-D box each of map m2,
// whose bounds fill the rest with zeros. (8192 x 2048 x 14000, no multiple of 64: the
// gradients take 2166 us so and 2253 with 2-D boxes throughout.)
template <bool kMN, int kRows>
__device__ __forceinline__ void load_half(uint8_t* dst, const CUtensorMap* m, const CUtensorMap* m2, uint32_t bar, int full,
                                          int mn, int k0) {
  if constexpr (!kMN) {
    tma_load_2d_pair(dst, m, bar, k0, mn);
  } else if (kRows == 128 && mn + 128 <= full) {
    tma_load_3d_pair(dst, m, bar, 0, k0, mn / 64);
  } else {
    tma_load_2d_pair(dst, m2, bar, mn, k0);
    if constexpr (kRows == 128) tma_load_2d_pair(dst + 64 * 128, m2, bar, mn + 64, k0);
  }
}

struct FfnUnit {
  int tm, tn, split, kb0, kb1;
};

template <class Cfg>
__device__ __forceinline__ FfnUnit ffn_unit(const FfnParams& p, int u) {
  FfnUnit w;
  const int tile = u / p.splits;
  w.split = u - tile * p.splits;
  raster(tile, p.tiles_m, p.tiles_n, 8, w.tm, w.tn);
  w.kb0 = (int)((long long)w.split * p.k_blocks / p.splits);
  w.kb1 = (int)((long long)(w.split + 1) * p.k_blocks / p.splits);
  return w;
}

// dh1, dh3 and a of 8 elements from da and the pre-activations
template <int kFn>
__device__ __forceinline__ void gate_grad8(const float* da, const float* h1, const float* h3, float* d1, float* d3,
                                           float* a) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float f, df;
    gate_f_df<kFn>(h1[j], f, df);
    d1[j] = da[j] * h3[j] * df;
    d3[j] = da[j] * f;
    a[j] = f * h3[j];
  }
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
    ffn_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmB2, const FfnParams p) {
  constexpr int STAGES = Cfg::STAGES, BN = Cfg::BN, BK = Cfg::BK, AB = Cfg::A_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES + Cfg::EPI_WARPS * 2048);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* drain_bar = tempty_bar + 2;
  uint32_t* s_tmem_base = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem_base + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  const bool leader = rank == 0;
  const int unit0 = (int)cluster_id_x(), unit_step = (int)nclusters_x();

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], Cfg::EPI_WARPS * 2);
    }
    mbar_init(drain_bar, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<2>(s_tmem_base, 2 * BN);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers exist before anyone signals them
  tc_fence_after();
  const uint32_t tmem_base = *s_tmem_base;
  pdl_wait();
  pdl_launch();

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      tma_prefetch_desc(&tmB2);
    }
    __syncwarp();
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full0 = mapa_shared(smem_u32(&full_bar[0]), 0);  // both CTAs' loads complete on the leader's
    for (int u = unit0; u < p.num_units && ok; u += unit_step) {
      const FfnUnit w = ffn_unit<Cfg>(p, u);
      const int a_mn = w.tm * 256 + rank * 128;
      const int b_mn = Cfg::kEpi == kFfnGate ? w.tn * (BN / 2) : w.tn * BN + rank * (BN / 2);
      // tmB2: gate/up W3's map, MN-major B its 2-D map
      const CUtensorMap* tb = Cfg::kEpi == kFfnGate && rank ? &tmB2 : &tmB;
      for (int kb = w.kb0; kb < w.kb1; ++kb) {
        ok = mbar_wait(&empty_bar[stage], phase ^ 1, s_abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* a_dst = smem + stage * Cfg::STAGE_BYTES;
          const uint32_t fb = full0 + stage * 8;
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * Cfg::STAGE_BYTES);
          tma_load_2d_pair(a_dst, &tmA, fb, kb * BK, a_mn);
          load_half<Cfg::kBMN, BN / 2>(a_dst + AB, tb, &tmB2, fb, p.b_full, b_mn, kb * BK);
        }
        __syncwarp();
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok && leader) wait_copies<STAGES>(full_bar, issued);
    __syncwarp();
  } else if (warp == 1) {
    if (leader) {
      int stage = 0, acc_i = 0;
      uint32_t phase = 0;
      bool ok = true;
      // MN-major: 16 rows of K are 2 KB on, the 64-column chunks BK * 128 bytes apart
      constexpr uint32_t b_step = Cfg::kBMN ? 2048 >> 4 : 32 >> 4;
      const uint64_t a_desc = umma_desc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t b_desc = umma_desc_sw128(smem_u32(smem) + AB, Cfg::kBMN ? BK * 128 : 16, 1024);
      for (int u = unit0; u < p.num_units && ok; u += unit_step, ++acc_i) {
        const FfnUnit w = ffn_unit<Cfg>(p, u);
        const int buf = acc_i & 1;
        ok = mbar_wait(&tempty_bar[buf], ((acc_i >> 1) & 1) ^ 1, s_abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * BN;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          ok = mbar_wait(&full_bar[stage], phase, s_abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint32_t off = stage * (Cfg::STAGE_BYTES >> 4);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              umma_pair<false>(d_tmem, a_desc + off + 2 * k, b_desc + off + k * b_step, Cfg::IDESC,
                               (kb > w.kb0 || k > 0) ? 1u : 0u);
            umma_commit_pair(&empty_bar[stage], 0x3);
            if (kb + 1 == w.kb1) umma_commit_pair(&tfull_bar[buf], 0x3);
          }
          __syncwarp();
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // every MMA issued so far has completed (in both CTAs) before TMEM is freed
      if (elect_one()) umma_commit_pair(drain_bar, 0x3);
      __syncwarp();
    }
    volatile int never = 0;
    mbar_wait(drain_bar, 0, &never);
    __syncwarp();
  } else {
    const int q = warp & 3;           // TMEM lane quarter of this warp
    const int half = (warp - 2) >> 2;  // its half of the columns
    const uint32_t tempty0 = mapa_shared(smem_u32(&tempty_bar[0]), 0);
    auto release = [&](int buf) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty0 + buf * 8);
    };
    const WarpTile wt{smem + STAGES * Cfg::STAGE_BYTES + (warp - 2) * 2048, lane};
    int acc_i = 0;
    for (int u = unit0; u < p.num_units; u += unit_step, ++acc_i) {
      const FfnUnit w = ffn_unit<Cfg>(p, u);
      const int buf = acc_i & 1;
      const int row0 = w.tm * 256 + rank * 128 + q * 32;  // first row of this warp
      const bool split = p.splits > 1;
      // gradient of the gate: the pre-activations of a 32-column chunk, 64 bytes of 8 rows a load
      uint4 n1[4], n3[4];
      auto fetch_h = [&](int c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const long long at = warp_at<8>(i, lane, row0, p.M, w.tn * BN + half * (BN / 2) + c * 32, p.N, p.N);
          const uint16_t* h = reinterpret_cast<const uint16_t*>(p.H);
          n1[i] = at >= 0 ? __ldg(reinterpret_cast<const uint4*>(h + at)) : make_uint4(0, 0, 0, 0);
          n3[i] = at >= 0 ? __ldg(reinterpret_cast<const uint4*>(h + p.h_plane + at)) : make_uint4(0, 0, 0, 0);
        }
      };
      if (Cfg::kEpi == kFfnGateGrad && !split) fetch_h(0);
      const bool got = mbar_wait(&tfull_bar[buf], (acc_i >> 1) & 1, s_abort);
      if (!__all_sync(0xffffffffu, got)) break;  // the TMEM loads are warp-collective
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BN;
      if constexpr (Cfg::kEpi == kFfnGate) {
#pragma unroll 1
        for (int c = 0; c < BN / 128; ++c) {
          const int f0 = half * (BN / 4) + c * 32;  // feature within the tile's BN / 2
          uint32_t rg[32], ru[32];
          tmem_ld32(t_row + f0, rg);
          tmem_ld32(t_row + BN / 2 + f0, ru);
          tmem_ld_wait(rg);
          reg_dep(ru);
          if (c == BN / 128 - 1) release(buf);
          const int col = w.tn * (BN / 2) + f0;
          if (split) {
            float* out = p.ws + (size_t)w.split * p.M * (2ll * p.N);
            store_warp32(wt, rg, out, row0, p.M, col, p.N, 2ll * p.N);
            store_warp32(wt, ru, out + p.N, row0, p.M, col, p.N, 2ll * p.N);
            continue;
          }
          uint4 v[4];
          if (p.H != nullptr) {
            pack32<Cfg::kElem>(rg, v);
            store_warp<8>(wt, v, p.H, row0, p.M, col, p.N);
            pack32<Cfg::kElem>(ru, v);
            store_warp<8>(wt, v, reinterpret_cast<uint16_t*>(p.H) + p.h_plane, row0, p.M, col, p.N);
          }
          with_gate(p.gate, [&](auto fn) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              rg[j] = __float_as_uint(gate_f<decltype(fn)::value>(__uint_as_float(rg[j])) * __uint_as_float(ru[j]));
          });
          pack32<Cfg::kElem>(rg, v);
          store_warp<8>(wt, v, p.C, row0, p.M, col, p.N);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < BN / 64; ++c) {
          const int c0 = half * (BN / 2) + c * 32, col = w.tn * BN + c0;
          uint32_t r[32];
          tmem_ld32(t_row + c0, r);
          tmem_ld_wait(r);
          if (c == BN / 64 - 1) release(buf);
          if (split) {
            store_warp32(wt, r, p.ws + (size_t)w.split * p.M * p.N, row0, p.M, col, p.N, p.N);
            continue;
          }
          uint4 v[4];
          if constexpr (Cfg::kEpi == kFfnGateGrad) {
            uint4 h1[4], h3[4], va[4];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) wt.across(i) = n1[i];
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) h1[j] = wt.own(j);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) wt.across(i) = n3[i];
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) h3[j] = wt.own(j);
            if (c + 1 < BN / 64) fetch_h(c + 1);
            with_gate(p.gate, [&](auto fn) {
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                float z1[8], z3[8], d1[8], d3[8], a[8];
                unpack8<Cfg::kElem>(h1[g], z1);
                unpack8<Cfg::kElem>(h3[g], z3);
                gate_grad8<decltype(fn)::value>(reinterpret_cast<const float*>(r) + g * 8, z1, z3, d1, d3, a);
                v[g] = pack8<Cfg::kElem>(d1);
                h3[g] = pack8<Cfg::kElem>(d3);
                va[g] = pack8<Cfg::kElem>(a);
              }
            });
            store_warp<8>(wt, v, p.C, row0, p.M, col, p.N);
            store_warp<8>(wt, h3, reinterpret_cast<uint16_t*>(p.C) + p.c_plane, row0, p.M, col, p.N);
            store_warp<8>(wt, va, p.Act, row0, p.M, col, p.N);
          } else {
            pack32<Cfg::kElem>(r, v);
            store_warp<8>(wt, v, p.C, row0, p.M, col, p.N);
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
    tmem_dealloc<2>(tmem_base, 2 * BN);
  }
}

// ------------------------------------------------------------ the three products of a gradient
// dx = dh1 W1 + dh3 W3 (A K-major, two planes in K, `splits` slices), dW1 and dW3 = dh^T x
// (two planes in M) and dW2 = dy^T a in one launch: they wait for the same thing, and the
// pairs that a product's last round leaves idle go on with the next product's tiles. dx's
// units come first, pair by pair; then the weights' tiles, all of one length, of which the
// pairs without a unit in dx's last round take `lead` rounds more. 333 x 1032 x 2760 takes
// 27 us so and 35 in a launch each; at 2048 x 4096 x 4736 the tensor pipe is busy in 95 % of
// the active cycles.
struct FfnGradMaps {
  CUtensorMap dh[2], w[2];    // dx: dh's planes K-major, W1 and W3
  CUtensorMap dht[2], x;      // dW1, dW3: dh's planes and x, T outermost
  CUtensorMap dyt, a;         // dW2: dy and a
  CUtensorMap w2d[2], dht2d[2], x2d, dyt2d, a2d;  // 2-D maps of the MN-major ones (load_half)
};
struct FfnGradParams {
  int T, H, I;
  int tm_x, tn_x, kb_x, kb_plane, splits, n_x;  // dx: tiles, K blocks, units
  int tm_13, tn_13, n_13;                       // dW1 and dW3: row tiles of a plane, column tiles, tiles in all
  int tm_2, tn_2, n_2;                          // dW2
  int kb_w;                                     // K blocks of a weight's tile
  int lead;
  int full_h, full_i;                           // columns of H and I in whole chunks (load_half)
  void *dx, *dw13, *dw2;
  float* ws;
};
struct FfnGradUnit {
  int job, tm, tn, plane, split, kb0, kb1;
};

// The k-th unit of pair c out of n; false past the last
__device__ __forceinline__ bool ffn_grad_unit(const FfnGradParams& p, int c, int n, int k, FfnGradUnit& w) {
  const int mine = c < p.n_x ? (p.n_x - 1 - c) / n + 1 : 0;
  w.plane = w.split = 0;
  if (k < mine) {
    const int u = c + k * n, tile = u / p.splits;
    w.job = 0;
    w.split = u - tile * p.splits;
    raster(tile, p.tm_x, p.tn_x, 8, w.tm, w.tn);
    w.kb0 = (int)((long long)w.split * p.kb_x / p.splits);
    w.kb1 = (int)((long long)(w.split + 1) * p.kb_x / p.splits);
    return true;
  }
  const int k2 = k - mine, busy = p.n_x % n;  // pairs with a unit in dx's last round
  const int idle = busy ? n - busy : 0, lead = busy ? p.lead : 0;
  long long t;
  if (c < busy)
    t = (long long)lead * idle + (long long)k2 * n + c;
  else if (k2 < lead)
    t = (long long)k2 * idle + c - busy;
  else
    t = (long long)lead * idle + (long long)(k2 - lead) * n + c;
  if (t >= p.n_13 + p.n_2) return false;
  w.kb0 = 0;
  w.kb1 = p.kb_w;
  w.job = t < p.n_13 ? 1 : 2;
  if (w.job == 1) {
    raster((int)t, 2 * p.tm_13, p.tn_13, 8, w.tm, w.tn);
    w.plane = w.tm >= p.tm_13;
    w.tm -= w.plane * p.tm_13;
  } else {
    raster((int)t - p.n_13, p.tm_2, p.tn_2, 8, w.tm, w.tn);
  }
  return true;
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
    ffn_grad_kernel(const __grid_constant__ FfnGradMaps maps, const FfnGradParams p) {
  constexpr int STAGES = Cfg::STAGES, BN = Cfg::BN, BK = Cfg::BK, AB = Cfg::A_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES + Cfg::EPI_WARPS * 2048);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* drain_bar = tempty_bar + 2;
  uint32_t* s_tmem_base = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem_base + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = (int)cluster_id_x(), pairs = (int)nclusters_x();

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], Cfg::EPI_WARPS * 2);
    }
    mbar_init(drain_bar, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<2>(s_tmem_base, 2 * BN);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers exist before anyone signals them
  tc_fence_after();
  const uint32_t tmem_base = *s_tmem_base;
  pdl_wait();
  pdl_launch();

  FfnGradUnit w;
  if (warp == 0) {
    if (elect_one()) {
      const CUtensorMap* m = maps.dh;
      for (int i = 0; i < 16; ++i) tma_prefetch_desc(m + i);
    }
    __syncwarp();
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full0 = mapa_shared(smem_u32(&full_bar[0]), 0);  // both CTAs' loads complete on the leader's
    // K blocks [kb0, kb1) of a unit through one set of maps, K counted from block `from`
    auto blocks = [&](auto a_mn_major, const CUtensorMap* ta, const CUtensorMap* ta2, int a_full, const CUtensorMap* tb,
                      const CUtensorMap* tb2, int b_full, int kb0, int kb1, int from) {
      const int a_mn = w.tm * 256 + rank * 128, b_mn = w.tn * BN + rank * (BN / 2);
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait(&empty_bar[stage], phase ^ 1, s_abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        if (elect_one()) {
          uint8_t* a_dst = smem + stage * Cfg::STAGE_BYTES;
          const uint32_t fb = full0 + stage * 8;
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * Cfg::STAGE_BYTES);
          load_half<decltype(a_mn_major)::value, 128>(a_dst, ta, ta2, fb, a_full, a_mn, (kb - from) * BK);
          load_half<true, BN / 2>(a_dst + AB, tb, tb2, fb, b_full, b_mn, (kb - from) * BK);
        }
        __syncwarp();
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    };
    for (int k = 0; ok && ffn_grad_unit(p, pair, pairs, k, w); ++k) {
      if (w.job == 0) {
        const int mid = p.kb_plane;
        blocks(std::false_type{}, &maps.dh[0], nullptr, 0, &maps.w[0], &maps.w2d[0], p.full_h, w.kb0, min(w.kb1, mid), 0);
        if (ok)
          blocks(std::false_type{}, &maps.dh[1], nullptr, 0, &maps.w[1], &maps.w2d[1], p.full_h, max(w.kb0, mid), w.kb1, mid);
      } else if (w.job == 1) {
        blocks(std::true_type{}, &maps.dht[w.plane], &maps.dht2d[w.plane], p.full_i, &maps.x, &maps.x2d, p.full_h, w.kb0,
               w.kb1, 0);
      } else {
        blocks(std::true_type{}, &maps.dyt, &maps.dyt2d, p.full_h, &maps.a, &maps.a2d, p.full_i, w.kb0, w.kb1, 0);
      }
    }
    if (!ok && leader) wait_copies<STAGES>(full_bar, issued);
    __syncwarp();
  } else if (warp == 1) {
    if (leader) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t b_desc = umma_desc_sw128(smem_u32(smem) + AB, BK * 128, 1024);
      // One loop for each form of A: what the MMA reads then stays uniform (elect_one).
      auto blocks = [&](auto a_mn, const FfnGradUnit& w, int buf) {
        constexpr bool kAMN = decltype(a_mn)::value;
        constexpr uint32_t a_step = kAMN ? 2048 >> 4 : 32 >> 4, idesc = Cfg::IDESC | (kAMN ? 1u << 15 : 0u);
        const uint64_t a_desc = umma_desc_sw128(smem_u32(smem), kAMN ? BK * 128 : 16, 1024);
        const uint32_t d_tmem = tmem_base + buf * BN;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          ok = mbar_wait(&full_bar[stage], phase, s_abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) return;
          tc_fence_after();
          const uint32_t off = stage * (Cfg::STAGE_BYTES >> 4);
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < BK / 16; ++i)
              umma_pair<false>(d_tmem, a_desc + off + i * a_step, b_desc + off + i * (2048 >> 4), idesc,
                               (kb > w.kb0 || i > 0) ? 1u : 0u);
            umma_commit_pair(&empty_bar[stage], 0x3);
            if (kb + 1 == w.kb1) umma_commit_pair(&tfull_bar[buf], 0x3);
          }
          __syncwarp();
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      };
      for (int k = 0; ok && ffn_grad_unit(p, pair, pairs, k, w); ++k) {
        const int buf = k & 1;
        ok = mbar_wait(&tempty_bar[buf], ((k >> 1) & 1) ^ 1, s_abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (w.job == 0)
          blocks(std::false_type{}, w, buf);
        else
          blocks(std::true_type{}, w, buf);
      }
      if (elect_one()) umma_commit_pair(drain_bar, 0x3);  // every MMA has completed (in both CTAs) before TMEM is freed
      __syncwarp();
    }
    volatile int never = 0;
    mbar_wait(drain_bar, 0, &never);
    __syncwarp();
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t tempty0 = mapa_shared(smem_u32(&tempty_bar[0]), 0);
    const WarpTile wt{smem + STAGES * Cfg::STAGE_BYTES + (warp - 2) * 2048, lane};
    for (int k = 0; ffn_grad_unit(p, pair, pairs, k, w); ++k) {
      const int buf = k & 1, row0 = w.tm * 256 + rank * 128 + q * 32;
      const bool got = mbar_wait(&tfull_bar[buf], (k >> 1) & 1, s_abort);
      if (!__all_sync(0xffffffffu, got)) break;  // the TMEM loads are warp-collective
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BN;
      const int M = w.job == 0 ? p.T : w.job == 1 ? p.I : p.H, N = w.job == 2 ? p.I : p.H;
      uint16_t* out = reinterpret_cast<uint16_t*>(w.job == 0 ? p.dx : w.job == 1 ? p.dw13 : p.dw2) +
                      (size_t)w.plane * p.I * p.H;
#pragma unroll 1
      for (int c = 0; c < BN / 64; ++c) {
        const int c0 = half * (BN / 2) + c * 32, col = w.tn * BN + c0;
        uint32_t r[32];
        tmem_ld32(t_row + c0, r);
        tmem_ld_wait(r);
        if (c == BN / 64 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(tempty0 + buf * 8);
        }
        if (w.job == 0 && p.splits > 1) {
          store_warp32(wt, r, p.ws + (size_t)w.split * M * N, row0, M, col, N, N);
        } else {
          uint4 v[4];
          pack32<Cfg::kElem>(r, v);
          store_warp<8>(wt, v, out, row0, M, col, N);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem_base, 2 * BN);
  }
}

// The sum over the slices, in slice order, of 8 elements that lie `at` floats into
// each slice of `stride` floats.
__device__ __forceinline__ void sum_slices8(const float* __restrict__ ws, int splits, size_t stride, size_t at,
                                            float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float4* src = reinterpret_cast<const float4*>(ws + s * stride + at);
    const float4 a = __ldcg(src), b = __ldcg(src + 1);
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
  }
}

// out[i] = sum of the slices, rounded once; n8: groups of 8 elements of the result, which
// lie end to end in it and in each slice
template <int kElem>
__global__ void __launch_bounds__(256) ffn_reduce_kernel(const float* __restrict__ ws, int splits, long long n8,
                                                         void* __restrict__ out) {
  pdl_wait();
  pdl_launch();
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n8; i += gridDim.x * 256ll) {
    float v[8];
    sum_slices8(ws, splits, n8 * 8, i * 8, v);
    store8<kElem>(out, (size_t)i * 8, v);
  }
}

// a = f(h1) h3 and on request h1 and h3, from slices of [T][h1 | h3]
template <int kElem>
__global__ void __launch_bounds__(256) ffn_gate_reduce_kernel(const float* __restrict__ ws, int splits, int T, int I,
                                                              int gate, void* __restrict__ a, void* __restrict__ h) {
  pdl_wait();
  pdl_launch();
  const long long n8 = (long long)T * I / 8;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n8; i += gridDim.x * 256ll) {
    const long long row = i * 8 / I, at = row * 2 * I + (i * 8 - row * I);
    float g[8], u[8];
    sum_slices8(ws, splits, 2ll * T * I, at, g);
    sum_slices8(ws, splits, 2ll * T * I, at + I, u);
    if (h != nullptr) {
      store8<kElem>(h, i * 8, g);
      store8<kElem>(h, (size_t)T * I + i * 8, u);
    }
    with_gate(gate, [&](auto fn) {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = gate_f<decltype(fn)::value>(g[j]) * u[j];
    });
    store8<kElem>(a, i * 8, g);
  }
}

// dh1, dh3 and a from slices of da [T][I] and the pre-activations
template <int kElem>
__global__ void __launch_bounds__(256)
    ffn_gate_grad_reduce_kernel(const float* __restrict__ ws, int splits, int T, int I, int gate,
                                const void* __restrict__ h, void* __restrict__ dh, void* __restrict__ act) {
  pdl_wait();
  pdl_launch();
  const long long n8 = (long long)T * I / 8;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n8; i += gridDim.x * 256ll) {
    const uint4* src = reinterpret_cast<const uint4*>(h) + i;
    float da[8], h1[8], h3[8], d1[8], d3[8], a[8];
    unpack8<kElem>(__ldg(src), h1);
    unpack8<kElem>(__ldg(src + n8), h3);
    sum_slices8(ws, splits, n8 * 8, i * 8, da);
    with_gate(gate, [&](auto fn) { gate_grad8<decltype(fn)::value>(da, h1, h3, d1, d3, a); });
    store8<kElem>(dh, i * 8, d1);
    store8<kElem>(dh, (size_t)(n8 + i) * 8, d3);
    store8<kElem>(act, i * 8, a);
  }
}

}  // namespace ek
