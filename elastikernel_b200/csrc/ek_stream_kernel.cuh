// Products of up to 128 tokens with a weight matrix, bound by the weight's bytes:
// D[n, t] = sum_k W[n, k] x[t, k] for bf16, fp16 and block-scaled e4m3, and for the
// gate/up pair D1 = W1 x, D3 = W3 x.
//
// The operands are swapped: weight rows are the MMA's 128-row side, tokens its N
// side, so a stage is 256 weight rows x 128 bytes of K (32 KB; for gate/up 128 rows
// of W1 and 128 of W3) and the few token rows beside them. The work is the sequence
// of (row tile, K block) units, tile by tile, and CTA c takes the same number of
// consecutive units whatever the matrix: every SM streams the same bytes. What a
// CTA has of one tile is a segment; its fp32 sums go to the segment's slot of the
// workspace, [token][256 rows], and the following launch (stream_*_reduce_kernel)
// adds a tile's segments in K order and applies what follows: the rounding, or the
// gate function and its rounding or quantisation. No atomics, no tickets.
//
// Block-scaled e4m3: a 128-byte stage is one scale block. Each K block is
// multiplied into its own TMEM buffer, and the epilogue adds (product x weight-block
// scale) x token scale to fp32 registers while the next block's MMA runs (see
// scale_pair for the order).
//
//   warp 0  TMA producer; warp 1  TMEM and MMA; warp 2  scales (e4m3)
//   warps 3..10  epilogue: two per TMEM lane quarter, one 128-row block each
//
// Measured (calls back to back in a graph): one token through the bf16 block of 4096 x
// 14336 61.5 us, 5.7 TB/s of weights; 14336 x 4096 in 8 bits 11, 12.2, 13.9 and 18.7 us for
// 1, 16, 32 and 64 tokens (bound at 64 by the epilogue's chain of waits per K block and the
// token rows beside the weights, 40 KB a unit).
//
// A tile cut over a cluster instead, its parts added over distributed shared memory in the
// same launch, was tried and left out: an SM draws about 46 GB/s, so what counts is that
// all of them stream, and whole tiles over clusters of 4 and 8 leave too many without work
// (16 tokens through 7168 x 2048 in 8 bits 22.4 us, 64 through 4096 x 14336 23.7 us, against
// 18.4 and 19.3).
//
// Launches overlap (programmatic dependent launch): within a call a CTA fills its
// stages with weights before it waits; everything else is read and written after.
#pragma once
#include <cuda_fp8.h>

#include "ek_ffn_kernel.cuh"

namespace ek {

template <int kElem_, int NT_, bool kGate_>
struct StreamCfg {
  static constexpr int kElem = kElem_, NT = NT_;
  static constexpr bool kGate = kGate_, kF8 = kElem == kE4M3;
  static constexpr int BK = kF8 ? 128 : 64, KSTEPS = 4;
  static constexpr int A_BYTES = 256 * 128, B_BYTES = NT * 128, STAGE_BYTES = A_BYTES + B_BYTES;
  // scales: slots of SGROUP K blocks, each the tokens' scales and then the two row blocks'
  static constexpr int SLOTS = 3, SGROUP = 4, SLOT_STRIDE = NT + 4;
  static constexpr int SCALE_BYTES = kF8 ? SLOTS * SGROUP * SLOT_STRIDE * 4 : 0;
  static constexpr int STAGES_FIT = (224 * 1024 - SCALE_BYTES - 512) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_FIT > 6 ? 6 : STAGES_FIT;
  static constexpr int TMEM_COLS = 4 * NT;  // two buffers of two accumulators
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 96 + 32 * EPI_WARPS;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + SCALE_BYTES + 512 + 1024;
  static constexpr uint32_t IDESC = umma_idesc(kElem == kBF16 ? 1u : 0u, false, 128, 0);  // N is the launch's
  static constexpr int CHUNK = NT < 32 || (kF8 && NT == 128) ? 16 : 32;  // 128 accumulators leave room for 16
  static_assert(NT == 16 || NT == 32 || NT == 64 || NT == 128, "token tile");
};

enum OutType : int { kOutBF16 = 0, kOutFP16 = 1, kOutFP32 = 3 };

__device__ __forceinline__ void store_out(void* out, int type, size_t at, float v) {
  if (type == kOutBF16)
    reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else if (type == kOutFP16)
    reinterpret_cast<__half*>(out)[at] = __float2half_rn(v);
  else
    reinterpret_cast<float*>(out)[at] = v;
}

// 4 consecutive values, `n` of them inside the row; wide: whole and aligned
__device__ __forceinline__ void store_out4(void* out, int type, size_t at, const float4& v, int n, bool wide) {
  if (wide && n >= 4) {
    if (type == kOutFP32) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at) = v;
    } else {
      uint2 pk;
      pk.x = type == kOutBF16 ? Elem16<kBF16>::pack(v.x, v.y) : Elem16<kFP16>::pack(v.x, v.y);
      pk.y = type == kOutBF16 ? Elem16<kBF16>::pack(v.z, v.w) : Elem16<kFP16>::pack(v.z, v.w);
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + at) = pk;
    }
    return;
  }
  const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) store_out(out, type, at + i, e[i]);
}

__device__ __forceinline__ void add4(float4& a, const float4& b) {
  a.x += b.x;
  a.y += b.y;
  a.z += b.z;
  a.w += b.w;
}

// What follows the sums. Plain: 4 values of token t from row n on.
struct StreamOut {
  int T, N;            // tokens; rows of the weight (gate: features)
  void* out;           // plain: the result; gate: a (or null)
  int type, wide;      // OutType; rows of the result take whole 16-byte stores
  int gate;            // GateFn
  void* h;             // gate: the pre-activations (or null)
  uint8_t* codes;      // gate: a in e4m3 and its scales instead of a
  float* scales;
};

// The scale of a group of activations whose largest magnitude is m: m / 448, 1 for zeros.
// Not below 2^-126: under that its reciprocal overflows, further down it is zero itself, and
// a zero beside such values would become NaN.
__device__ __forceinline__ float act_scale(float m) { return m > 0.f ? fmaxf(m / 448.0f, 0x1p-126f) : 1.0f; }

// Four values' e4m3 codes
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
         ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16);
}

// a[t, f] = f(h1) h3 for 4 features a lane, from feature f on, and h1 and h3 on request;
// with codes, a in e4m3 with the scale of the warp's 128 features (act_scale). Rows past the weight's hold zeros.
__device__ __forceinline__ void finish_gate(const StreamOut& o, int t, int tile, const float4& h1, const float4& h3) {
  const int f = tile * 128 + (threadIdx.x & 31) * 4, I = o.N;
  float4 act;
  with_gate(o.gate, [&](auto fn) {
    constexpr int F = decltype(fn)::value;
    act = make_float4(gate_f<F>(h1.x) * h3.x, gate_f<F>(h1.y) * h3.y, gate_f<F>(h1.z) * h3.z, gate_f<F>(h1.w) * h3.w);
  });
  const size_t at = (size_t)t * I + f;
  if (o.codes == nullptr) {
    store_out4(o.out, o.type, at, act, I - f, true);
    if (o.h != nullptr) {
      store_out4(o.h, o.type, at, h1, I - f, true);
      store_out4(o.h, o.type, (size_t)o.T * I + at, h3, I - f, true);
    }
    return;
  }
  float m = fmaxf(fmaxf(fabsf(act.x), fabsf(act.y)), fmaxf(fabsf(act.z), fabsf(act.w)));  // zeros past I
#pragma unroll
  for (int i = 16; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  const float s = act_scale(m);
  if (f < I) *reinterpret_cast<uint32_t*>(o.codes + at) = e4m3x4(act.x / s, act.y / s, act.z / s, act.w / s);
  if ((threadIdx.x & 31) == 0) o.scales[(size_t)t * ((I + 127) / 128) + tile] = s;
}

// Scales are fp32 of any finite value: the product of two of them may overflow where the
// scaled sum does not (0 * inf is no zero), or be a denormal of a few bits where the
// scaled sum is an ordinary number. A block's sum r of e4m3 products is 0 or has a
// magnitude in [2^-18, 2^25], so it comes between the two that would leave fp32's range:
// r * first * second, first the smaller one where their product is too large, the larger
// one where it is too small, never leaves it before the result does. Where the product is
// normal it comes second and 1 first.
__device__ __forceinline__ bool normal_f(float v) { return fabsf(v) >= 0x1p-126f && fabsf(v) < __int_as_float(0x7f800000); }
__device__ __forceinline__ void scale_pair(float& second, float& first) {
  const float a = second, b = first, p = a * b;
  const bool swap = (fabsf(a) > fabsf(b)) == (fabsf(p) < 1.0f && p != 0.0f);  // a zero comes first
  first = normal_f(p) ? 1.0f : swap ? a : b;
  second = normal_f(p) ? p : swap ? b : a;
}

// How the units are dealt out; the reducing launch reads it too.
struct StreamSplit {
  int tiles, k_blocks;  // row tiles (256 rows, or 128 gate features), K blocks
  int per_cta, ctas;    // consecutive units of a CTA
  int max_segs;         // slots per CTA: the tiles that per_cta units can touch
};

struct StreamParams {
  StreamSplit sp;
  int T;
  int early;               // a later launch of its call: the weights may be fetched before the wait
  int n;                   // tokens per MMA: T rounded up to 16 (the box's rows)
  const float* tok_scale;  // e4m3: [T][k_blocks]
  const float* w_scale;    // [rows / 128][k_blocks]; gate: W1's
  const float* w_scale2;   // gate: W3's
  int w_blocks;            // rows of w_scale
  float* ws;               // [ctas * max_segs][T][256]
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
    stream_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmW2,
                  const __grid_constant__ CUtensorMap tmX, const StreamParams p) {
  constexpr int STAGES = Cfg::STAGES, NT = Cfg::NT, CH = Cfg::CHUNK, NS = Cfg::SLOTS, SG = Cfg::SGROUP, RS = Cfg::SLOT_STRIDE;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_scale = reinterpret_cast<float*>(smem + STAGES * Cfg::STAGE_BYTES);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES + Cfg::SCALE_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* drain_bar = tempty_bar + 2;
  uint64_t* sfull_bar = drain_bar + 1;
  uint64_t* sempty_bar = sfull_bar + NS;
  uint32_t* s_tmem_base = reinterpret_cast<uint32_t*>(sempty_bar + NS);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem_base + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int KB = p.sp.k_blocks;
  const int u0 = blockIdx.x * p.sp.per_cta;
  const int u1 = min(u0 + p.sp.per_cta, p.sp.tiles * KB);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], Cfg::EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&sfull_bar[s], 32);
      mbar_init(&sempty_bar[s], Cfg::EPI_WARPS);
    }
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<1>(s_tmem_base, Cfg::TMEM_COLS);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *s_tmem_base;
  if (!p.early) pdl_wait();
  pdl_launch();

  if (warp == 0) {
    auto load_w = [&](int u, int stage) {
      const int tile = u / KB, k0 = (u - tile * KB) * Cfg::BK;
      if (elect_one()) {
        uint8_t* dst = smem + stage * Cfg::STAGE_BYTES;
        mbar_arrive_expect_tx(&full_bar[stage], Cfg::A_BYTES + p.n * 128);
        if constexpr (Cfg::kGate) {
          tma_load_2d(dst, &tmW, &full_bar[stage], k0, tile * 128);
          tma_load_2d(dst + 128 * 128, &tmW2, &full_bar[stage], k0, tile * 128);
        } else {
          tma_load_2d(dst, &tmW, &full_bar[stage], k0, tile * 256);
        }
      }
      __syncwarp();
    };
    auto load_x = [&](int u, int stage) {
      if (elect_one())
        tma_load_2d(smem + stage * Cfg::STAGE_BYTES + Cfg::A_BYTES, &tmX, &full_bar[stage], (u % KB) * Cfg::BK, 0);
      __syncwarp();
    };
    // the stages' first fill: the weights before the wait, the tokens after it
    const int first = min(u1 - u0, STAGES);
    for (int i = 0; i < first; ++i) load_w(u0 + i, i);
    pdl_wait();
    for (int i = 0; i < first; ++i) load_x(u0 + i, i);
    int stage = 0;
    uint32_t phase = 0;
    for (int u = u0 + STAGES; u < u1; ++u) {
      const bool ok = mbar_wait(&empty_bar[stage], phase, s_abort);
      if (!__all_sync(0xffffffffu, ok)) {
        wait_copies<STAGES>(full_bar, u - u0);
        break;
      }
      load_w(u, stage);
      load_x(u, stage);
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
    }
    __syncwarp();
  } else if (warp == 1) {
    int stage = 0, flush = 0;
    uint32_t phase = 0;
    bool fresh = true;  // the next MMA starts a sum
    const uint32_t idesc = Cfg::IDESC | ((uint32_t)(p.n >> 3) << 17);
    const uint64_t a_desc = umma_desc_sw128(smem_u32(smem), 16, 1024);
    const uint64_t b_desc = umma_desc_sw128(smem_u32(smem) + Cfg::A_BYTES, 16, 1024);
    for (int u = u0; u < u1; ++u) {
      const int buf = flush & 1;
      bool ok = !fresh || mbar_wait(&tempty_bar[buf], ((flush >> 1) & 1) ^ 1, s_abort);
      ok = ok && mbar_wait(&full_bar[stage], phase, s_abort);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t off = stage * (Cfg::STAGE_BYTES >> 4);
      const uint32_t d = tmem_base + buf * 2 * NT;
      const bool last = Cfg::kF8 || (u + 1) % KB == 0 || u + 1 == u1;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < Cfg::KSTEPS; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            umma<Cfg::kF8>(d + h * NT, a_desc + off + h * (128 * 128 >> 4) + 2 * k, b_desc + off + 2 * k, idesc,
                           (!fresh || k > 0) ? 1u : 0u);
        umma_commit(&empty_bar[stage]);
        if (last) umma_commit(&tfull_bar[buf]);
      }
      __syncwarp();
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
      fresh = last;
      flush += last;
    }
    if (elect_one()) umma_commit(drain_bar);  // every MMA has completed before TMEM is freed
    __syncwarp();
    volatile int never = 0;
    mbar_wait(drain_bar, 0, &never);
    __syncwarp();
  } else if (warp == 2) {
    if constexpr (Cfg::kF8) {
      pdl_wait();
      for (int u = u0, g = 0; u < u1; u += SG, ++g) {
        const int slot = g % NS;
        const bool ok = mbar_wait(&sempty_bar[slot], ((g / NS) & 1) ^ 1, s_abort);
        if (__any_sync(0xffffffffu, !ok)) break;
        for (int j = 0; j < SG && u + j < u1; ++j) {
          const int tile = (u + j) / KB, kb = u + j - tile * KB;
          float* dst = s_scale + (slot * SG + j) * RS;
          for (int t = lane; t < NT; t += 32)
            cp_async_4_zfill(dst + t, t < p.T ? p.tok_scale + (size_t)t * KB + kb : p.tok_scale, t < p.T ? 4 : 0);
          if (lane < 2) {
            const int blk = Cfg::kGate ? tile : 2 * tile + lane;
            const float* src = Cfg::kGate && lane ? p.w_scale2 : p.w_scale;
            cp_async_4_zfill(dst + NT + lane, blk < p.w_blocks ? src + (size_t)blk * KB + kb : src,
                             blk < p.w_blocks ? 4 : 0);
          }
        }
        cp_async_mbar_arrive(&sfull_bar[slot]);
      }
      cp_async_wait<0>();  // no copy into shared memory outlives the CTA
    }
    __syncwarp();
  } else {
    pdl_wait();
    const int q = warp & 3, rb = (warp - 3) >> 2;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + rb * NT;
    const int n0 = rb * 128 + q * 32 + lane;  // row within the tile's 256
    auto release = [&](int buf) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty_bar[buf]);
    };
    auto load = [](uint32_t(&r)[32], uint32_t at) {
      if constexpr (CH == 32)
        tmem_ld32(at, r);
      else
        tmem_ld16(at, r);
    };
    int flush = 0, seg = 0, slot = 0;
    uint32_t sphase = 0;
    for (int u = u0; u < u1;) {
      const int tile_end = min(u1, (u / KB + 1) * KB);
      float* out = p.ws + ((size_t)(blockIdx.x * p.sp.max_segs + seg) * p.T) * 256 + n0;
      bool good = true;
      if constexpr (Cfg::kF8) {
        float2 acc[NT / 2];
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) acc[j] = make_float2(0.f, 0.f);
        // Product x weight scale is 0 or in [2^-118, 2^125] where the weight's is in
        // [2^-100, 2^100], whatever the token's that follows; a segment with another one
        // takes the scales pair by pair (a loop of its own: a branch in one loop spills).
        const int nb = tile_end - u, tile = u / KB, blk = Cfg::kGate ? tile : 2 * tile + rb;
        const float* wsc = (Cfg::kGate && rb ? p.w_scale2 : p.w_scale) + (size_t)min(blk, p.w_blocks - 1) * KB + (u - tile * KB);
        bool far = false;
        for (int i = lane; i < nb; i += 32) {
          const float w = fabsf(__ldg(wsc + i));
          far |= !(w >= 0x1p-100f && w <= 0x1p100f);
        }
        // A failed wait has raised the abort flag: the loop then runs out without waiting and
        // nothing is written. A chunk of columns is in flight while the one before is added;
        // columns past the tokens are added too, and never used.
        auto blocks = [&](auto pairs) {
          for (; u < tile_end; ++u, ++flush) {
            const int buf = flush & 1, j = (u - u0) % SG;
            if (j == 0) mbar_wait_soon(&sfull_bar[slot], sphase, s_abort);
            const float* xs = s_scale + (slot * SG + j) * RS;
            const float ws = xs[NT + rb];
            mbar_wait_soon(&tfull_bar[buf], (flush >> 1) & 1, s_abort);
            __syncwarp();
            tc_fence_after();
            constexpr int C = NT / CH;
            uint32_t r[2][32];
            load(r[0], lane_base + buf * 2 * NT);
#pragma unroll
            for (int c = 0; c < C; ++c) {
              tmem_ld_wait(r[c & 1]);
              if (c + 1 < C)
                load(r[(c + 1) & 1], lane_base + buf * 2 * NT + (c + 1) * CH);
              else
                release(buf);
              const float4* xs4 = reinterpret_cast<const float4*>(xs + c * CH);
              const uint32_t(&v)[32] = r[c & 1];
#pragma unroll
              for (int i = 0; i < CH / 4; ++i) {
                const float4 x = xs4[i];
                float2* a = acc + (c * CH + 4 * i) / 2;
                float2 f0 = make_float2(ws, ws), f1 = f0, s0 = make_float2(x.x, x.y), s1 = make_float2(x.z, x.w);
                if constexpr (decltype(pairs)::value) {
                  scale_pair(s0.x, f0.x);
                  scale_pair(s0.y, f0.y);
                  scale_pair(s1.x, f1.x);
                  scale_pair(s1.y, f1.y);
                }
                a[0] = fma2(mul2(make_float2(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1])), f0), s0, a[0]);
                a[1] = fma2(mul2(make_float2(__uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3])), f1), s1, a[1]);
              }
            }
            if (j == SG - 1 || u + 1 == u1) {
              __syncwarp();
              if (lane == 0) mbar_arrive(&sempty_bar[slot]);
              if (++slot == NS) { slot = 0; sphase ^= 1; }
            }
          }
        };
        if (__any_sync(0xffffffffu, far))
          blocks(std::true_type{});
        else
          blocks(std::false_type{});
        good = !__any_sync(0xffffffffu, *s_abort);
        if (!good) break;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (t < p.T) __stcg(out + (size_t)t * 256, (t & 1) ? acc[t >> 1].y : acc[t >> 1].x);
      } else {
        const int buf = flush & 1;
        good = mbar_wait(&tfull_bar[buf], (flush >> 1) & 1, s_abort);
        if (!__all_sync(0xffffffffu, good)) break;
        tc_fence_after();
        const int chunks = (p.n + CH - 1) / CH;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          uint32_t r[32];
          load(r, lane_base + buf * 2 * NT + c * CH);
          tmem_ld_wait(r);
          if (c == chunks - 1) release(buf);
#pragma unroll
          for (int j = 0; j < CH; ++j)
            if (c * CH + j < p.T) __stcg(out + (size_t)(c * CH + j) * 256, __uint_as_float(r[j]));
        }
        ++flush;
        u = tile_end;
      }
      ++seg;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, Cfg::TMEM_COLS);
  }
}

// ------------------------------------------------------------ adding the segments
// A warp of a block of 8 sums 128 rows of a tile for one token, four rows a lane
// (kN = 2: a second 128 rows beside them, the up rows of a gate tile). `ways` warps
// share a token's segments, each taking every ways-th; their sums are added in
// order by the first of them. So the block covers 8 / ways tokens, and a tile cut
// into many segments has all its loads in flight at once. Returns whether this warp
// holds the result.
template <int kN>
__device__ __forceinline__ bool stream_sum(const StreamSplit& sp, const float* __restrict__ ws, int T, int tile, int t,
                                           int row, int ways, float4 (&v)[kN]) {
  __shared__ float4 s_part[8][32][kN];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, way = warp % ways;
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (t < T) {
    const int c0 = (int)((long long)tile * sp.k_blocks / sp.per_cta);
    const int c1 = (int)(((long long)(tile + 1) * sp.k_blocks - 1) / sp.per_cta);
    constexpr int U = 4;  // segments with their loads in flight
    for (int c = c0 + way; c <= c1; c += U * ways) {
      float4 x[U][kN];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int cj = c + j * ways;
        if (cj <= c1) {
          const int seg = tile - (int)((long long)cj * sp.per_cta / sp.k_blocks);
          const float* src = ws + ((size_t)(cj * sp.max_segs + seg) * T + t) * 256 + row + lane * 4;
#pragma unroll
          for (int i = 0; i < kN; ++i) x[j][i] = __ldcg(reinterpret_cast<const float4*>(src + i * 128));
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (c + j * ways <= c1) {
#pragma unroll
          for (int i = 0; i < kN; ++i) add4(v[i], x[j][i]);
        }
    }
  }
  if (ways > 1) {
#pragma unroll
    for (int i = 0; i < kN; ++i) s_part[warp][lane][i] = v[i];
    __syncthreads();
    if (way == 0)
      for (int w = 1; w < ways; ++w)
#pragma unroll
        for (int i = 0; i < kN; ++i) add4(v[i], s_part[warp + w][lane][i]);
  }
  return way == 0 && t < T;
}

// A plain product's result; blockIdx.x: half tiles of 128 rows
__global__ void __launch_bounds__(256)
    stream_store_reduce_kernel(const StreamSplit sp, const float* __restrict__ ws, const StreamOut o, int ways) {
  pdl_launch();
  pdl_wait();
  const int tile = blockIdx.x >> 1, row = (blockIdx.x & 1) * 128;
  const int t = blockIdx.y * (8 / ways) + (threadIdx.x >> 5) / ways;
  const int n = tile * 256 + row + (threadIdx.x & 31) * 4;
  float4 v[1];
  if (stream_sum<1>(sp, ws, o.T, tile, t, row, ways, v))
    store_out4(o.out, o.type, (size_t)t * o.N + n, v[0], o.N - n, o.wide);
}

// A gate/up pair's
__global__ void __launch_bounds__(256)
    stream_gate_reduce_kernel(const StreamSplit sp, const float* __restrict__ ws, const StreamOut o, int ways) {
  pdl_launch();
  pdl_wait();
  const int t = blockIdx.y * (8 / ways) + (threadIdx.x >> 5) / ways;
  float4 v[2];
  if (stream_sum<2>(sp, ws, o.T, blockIdx.x, t, 0, ways, v)) finish_gate(o, t, blockIdx.x, v[0], v[1]);
}

// e4m3 codes [T][H] and scales [T][ceil(H / 128)] of bf16 rows: a scale per 128 elements
// (largest magnitude / 448, 1 for zeros; of bf16 values never zero itself), IEEE quotients,
// as the row quantisation of the library. A half warp per group, 8 elements a lane, the loads of kU pairs of groups in
// flight; H a multiple of 8. Memory bound at many tokens, a launch at few: it lets the
// product after it fetch weights meanwhile.
template <int kU>
__global__ void __launch_bounds__(256) ffn_quant_kernel(const __nv_bfloat16* __restrict__ x, long long groups, int H,
                                                        uint8_t* __restrict__ codes, float* __restrict__ scales) {
  pdl_wait();
  pdl_launch();
  const int per_row = (H + 127) / 128, hl = threadIdx.x & 15;
  // the bound is uniform over the warp, so that every lane reaches the exchanges
  for (long long g0 = (blockIdx.x * 256ll + threadIdx.x) / 32 * (2 * kU); g0 < groups; g0 += gridDim.x * (16ll * kU)) {
    uint4 raw[kU];
    long long at[kU];
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      const long long g = g0 + 2 * i + ((threadIdx.x >> 4) & 1), row = g / per_row;
      const int c = (int)(g - row * per_row) * 128 + hl * 8;
      at[i] = g < groups && c < H ? row * H + c : -1;
      raw[i] = at[i] >= 0 ? __ldg(reinterpret_cast<const uint4*>(x + at[i])) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      float v[8];
      unpack8<kBF16>(raw[i], v);
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
#pragma unroll
      for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float s = m > 0.f ? m / 448.0f : 1.0f;
      if (at[i] < 0) continue;
      uint32_t pk[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) pk[j] = e4m3x4(v[4 * j] / s, v[4 * j + 1] / s, v[4 * j + 2] / s, v[4 * j + 3] / s);
      *reinterpret_cast<uint2*>(codes + at[i]) = make_uint2(pk[0], pk[1]);
      if (hl == 0) scales[g0 + 2 * i + ((threadIdx.x >> 4) & 1)] = s;
    }
  }
}

}  // namespace ek
