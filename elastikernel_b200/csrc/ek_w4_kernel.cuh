// Products of a few token rows with 4-bit weights on the tensor cores.
//
// out[tok, n] = sum_k x[tok, k] w[n, k], w = s (q - 8) or s q + m per group of
// 32, 64 or 128 k. The codes are streamed once from HBM, so the aim is to keep
// the memory system full while the SM converts: at 6.5 TB/s an SM receives 23
// bytes (46 weights) per clock, and its integer pipe does 64 operations per
// clock, so a weight may cost about one. Neither fp32 FMAs (one per weight and
// token) nor byte-wise unpacking keep up. Hence
//   * mma.sync m16n8k16 with 16 weight rows as the M side and 8 tokens as the N
//     side. A code word (8 weights) becomes four half2 registers of exact
//     integers with one shift, four and/ors (the nibbles over the exponent of
//     1024) and four half2 operations (which run on the floating-point pipe).
//     tcgen05 would need the converted tile in shared memory (its M side is 128
//     rows and it reads no registers), which costs more than the product
//     itself at these token counts;
//   * the tokens as fp16 too, whatever their type: a small kernel scales each
//     run of 256 elements by a power of two so that its largest magnitude lies
//     in [2^14, 2^15) and writes it in the order the nibbles come out. bf16 has
//     8 significant bits to fp16's 11: exact down to 2^-31 of the run's largest
//     (2^-17 scaled, seven bits above fp16's smallest step of 2^-24), and below
//     that off by half such a step, at most 2^-39 of the largest and less than
//     the fp32 sums are. fp16 rows go in as they are. fp32 rows (the experts'
//     activations) are rounded to 11 bits: more would need a second operand for
//     the low bits and twice the products, and three bits below a bf16
//     activation they hardly show beside the outputs' one rounding to 8 (error of
//     a layer's outputs against 64 bits 1.674e-3, with fp32 activations 1.661e-3);
//   * sums of one group in fp32 accumulators, then multiplied by the group's
//     fp32 scale: both operands are exact, so no weight is ever rounded. With
//     minima w = s (q - 8) + (m + 8 s), and the second term meets the sum of the
//     group's tokens, which the token kernel has left beside them;
//   * codes by TMA, 32 KB a stage (16 KB boxes and up are what the TMA engine
//     streams at full bandwidth), from one producer warp to eight consumer
//     warps of 32 weight rows each;
//   * the stages of all tiles, laid end to end, are cut into equal runs, one per
//     CTA, so that a few tiles fill every SM. A CTA leaves its fp32 sums of each
//     tile, or part of a tile, in the workspace; the launch that follows (the
//     one that rounds, applies SwiGLU or combines the experts' rows) adds the
//     parts in K order. An epilogue in the kernel itself cost more: its
//     registers spill in the main loop, and the last CTA's fence, ticket and
//     loads lie bare at the end.
//
// Measured, gate/up product of 32 experts of 7168 x 2048 (484 MB with scales; 74 us at
// the 6.5 TB/s of a copy): 8 tokens each 101 us (4.8 TB/s), 16 each 133, random
// choices of 64 tokens (8 to 24 each) 182. With one block of 8 tokens HBM and the SM's
// issue slots are about equally busy; a second block adds its products (a fifth
// of the time without them), token reads and scaling, and experts past 16 tokens
// stream their codes twice: there the ALU and tensor pipes are 41 % busy each, the
// issue slots 54 %, and the four warps a scheduler holds do not cover the latencies
// (96 registers a thread allow no more). Tried without gain: the tiles on tcgen05
// with the converted weights in tensor memory (187 us at 64 tokens), 16 warps of 16
// rows (209), runs cut by cost instead of stages (within 2 %), a deeper ring.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "ek_internal.h"
#include "ek_ptx.cuh"

namespace ek {
namespace w4 {

constexpr int kPiece = 32;       // elements per 16-byte piece of a code row; divides every group
constexpr int kStagePieces = 8;  // pieces per pipeline stage: 128 bytes of each row
constexpr int kStageElems = kStagePieces * kPiece;
constexpr int kWarps = 8;                    // consumer warps
constexpr int kThreads = 32 * (kWarps + 1);  // and the producer
constexpr int kRows = 32 * kWarps;           // weight rows per tile (gate/up: half of each matrix)
constexpr int kStageBytes = kRows * 128;
constexpr int kStages = 2;  // ring depth (two CTAs per SM; more stages of one CTA were no faster)
// Bytes of a token's record of a stage: 256 halfs, then its scale and the sums
// of its groups (fp32; at most 8). 64 more than 512 also keeps the reads of
// eight tokens free of bank conflicts; in shared memory the scales and sums stand
// behind the records, 48 bytes a token, for the same reason (read from the records
// themselves, four of them collide: 3 to 7 % more time with minima).
constexpr int kRecord = kStageElems * 2 + 64;
constexpr int kTail = 48;

__host__ __device__ inline int pieces(int K) { return (K + kPiece - 1) / kPiece; }
__host__ __device__ inline int groups(int K, int group) { return (K + group - 1) / group; }

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }

__device__ __forceinline__ uint32_t pack2(__half a, __half b) {
  const __half2 r = __halves2half2(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16 a, __nv_bfloat16 b) {
  const __nv_bfloat162 r = __halves2bfloat162(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// (w & mask) | 0x6400 6400: the masked nibbles over the exponent of 1024, whose
// last mantissa bit is worth 1, so that they are integers without a conversion (a
// published way: Kim et al., "Who Says Elephants Can't Run", 2022; the constants
// follow from the format).
__device__ __forceinline__ uint32_t nibbles(uint32_t w, uint32_t mask) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(0x64006400u));
  return r;
}

// Pairs (k = c, c + 4), c = 2 h and 2 h + 1, of a code word as exact fp16
// integers q - 8. The low nibble gives 1024 + q, the high one 1024 + 16 q.
__device__ __forceinline__ void code_pairs(uint32_t w, int h, uint32_t& lo, uint32_t& hi) {
  const uint32_t v = h ? w >> 8 : w;
  const uint32_t a = nibbles(v, 0x000f000fu), b = nibbles(v, 0x00f000f0u);
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0xe408e408u));                        // - 1032
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(hi) : "r"(b), "r"(0x2c002c00u), "r"(0xd480d480u));  // / 16 - 72
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same with a zero accumulator.
__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ float lds32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// ------------------------------------------------------------------ tokens
// A token row of K elements is stages(K) records, zero past K.
__host__ __device__ inline int stages(int K) { return (K + kStageElems - 1) / kStageElems; }

// [rows][stages(K)] records; each run of 8 halfs in the order 0 4 1 5 2 6 3 7.
struct Tokens {
  uint8_t* rec;
};
__device__ __forceinline__ float* tail_of(uint8_t* rec) { return reinterpret_cast<float*>(rec + kStageElems * 2); }

// The workspace of one product: the token records and the CTAs' sums.
struct Layout {
  size_t parts, bytes;
};
inline Layout layout(long long rows, int K, long long tiles, int ctas, int tok) {
  Layout l;
  l.parts = ((size_t)rows * stages(K) * kRecord + 255) / 256 * 256;
  l.bytes = l.parts + ((size_t)tiles + ctas) * kRows * tok * 4;
  return l;
}

__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A warp writes a record and its tail: eight elements v per lane. The scale comes from the
// largest finite magnitude, so an infinity or a NaN stays what it is and its
// neighbours stay finite. kScaled = false (fp16 rows): as they are. The sums are
// those of the rounded halfs, per `group` elements.
template <bool kScaled>
__device__ __forceinline__ void write_run(uint8_t* rec, float* tail, int group, const float (&v)[8]) {
  const int lane = threadIdx.x & 31;
  float f = 1.f, inv = 1.f;
  if constexpr (kScaled) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(v[i]) < INFINITY) m = fmaxf(m, fabsf(v[i]));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // m in [2^(b - 127), 2^(b - 126)) -> factor 2^(14 + 127 - b), kept normal
    const int b = (int)(__float_as_uint(m) >> 23);
    const int up = m > 0.f ? max(-113, min(126, 14 + 127 - b)) : 0;
    f = __uint_as_float((uint32_t)(127 + up) << 23);
    inv = __uint_as_float((uint32_t)(127 - up) << 23);
  }
  __half2 h[4];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = __floats2half2_rn(v[i] * f, v[i + 4] * f);
    const float2 r = __half22float2(h[i]);
    sum += r.x + r.y;
  }
  for (int o = group / 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);  // lanes of one group
  *reinterpret_cast<uint4*>(rec + lane * 16) = *reinterpret_cast<const uint4*>(h);
  if (lane == 0) tail[0] = inv;
  if (lane % (group / 8) == 0) tail[4 + lane / (group / 8)] = sum;
}

// A lane's eight elements of a row at k, zero past K. vec: rows of a multiple
// of 8 elements on a 16-byte base.
template <class T>
__device__ __forceinline__ void load_run(const T* __restrict__ src, int k, int K, bool vec, float (&v)[8]) {
  if (vec && k < K) {
    uint4 raw[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(src + k) + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f(reinterpret_cast<const T*>(raw)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f(src[k + i]) : 0.f;
  }
}

// Rows of x [rows, K] into tokens, a warp per run (runs first, first + step, ...).
template <class T>
__device__ __forceinline__ void write_tokens(const T* __restrict__ x, int rows, int K, int group, bool vec, const Tokens& out,
                                             long long first, long long step) {
  const int lane = threadIdx.x & 31, nst = stages(K);
  for (long long u = first; u < (long long)rows * nst; u += step) {
    const int row = (int)(u / nst), st = (int)(u - (long long)row * nst);
    float v[8];
    load_run(x + (size_t)row * K, st * kStageElems + lane * 8, K, vec, v);
    uint8_t* rec = out.rec + u * kRecord;
    write_run<!std::is_same<T, __half>::value>(rec, tail_of(rec), group, v);
  }
}

template <class T>
__global__ void __launch_bounds__(256)
    tokens_kernel(const T* __restrict__ x, int rows, int K, int group, bool vec, Tokens out) {
  griddep_launch();
  griddep_wait();
  write_tokens(x, rows, K, group, vec, out, ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5,
               ((long long)gridDim.x * blockDim.x) >> 5);
}

// ------------------------------------------------------------------ products
enum Mode { kDense, kGateUp, kDown };

// Scales and minima [rows, G] of one weight matrix.
template <class T>
struct Scales {
  const T* s;
  const T* m;  // null: symmetric
};

template <class T>
struct Params {
  Scales<T> w[2];            // gate/up: w1 and w3
  const uint8_t* codes[2];   // theirs, for the sums (the product has them by TMA)
  int group;
  int K, N;                  // N: weight rows (of an expert; of one matrix)
  int feature_tiles;         // tiles along N
  Tokens x;
  const T* rows;             // the rows themselves, where the kernel makes the records (Shape::kMakes); else null
  bool vec;                  // wide loads can read them
  int n_rows;                // token rows: M, or the packed rows
  int max_y;                 // token tiles there is room for
  const int* counts;         // rows per expert (null: dense)
  int E;
  const int* sorted_slots;   // fetch x through the permutation (null: x holds the rows)
  int n_slots;
  int topk;
  float* parts;
  bool wait_first;           // the predecessor makes the counts and the order too
};

// NT: 8 NT tokens a tile; FL: pieces per group (1, 2 or 4); kMin: minima.
// kMakes: the producer warp makes the token records itself, from the rows (a
// dense product of up to 8 tokens: one launch less, and the work is small enough
// to repeat per CTA).
template <int NT_, int FL_, bool kMin_, bool kMakes_>
struct Shape {
  static constexpr int NT = NT_, FL = FL_;
  static constexpr bool kMin = kMin_, kMakes = kMakes_;
  static constexpr int kTokens = 8 * NT;
  static constexpr int kTokenBytes = kTokens * (kRecord + kTail);  // of a stage
  static constexpr int kSmem = kStages * (kStageBytes + kTokenBytes) + 1024;  // + alignment of the swizzled stages
};

// A token tile: rows [r0, r0 + m) of expert e.
struct TokenTile {
  int e, r0, m;
};

// The packed layout's token tiles of `tok` rows: s_end[e] = tiles of experts
// 0..e, s_row[e] = first row of expert e, s_row[E] the rows in all (2 E + 1
// ints of shared memory); returns the tiles in all. Called by one warp.
__device__ __forceinline__ int expert_tiles(const int* __restrict__ counts, int E, int tok, int* s_end, int* s_row) {
  const int lane = threadIdx.x & 31;
  int row = 0, end = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int c = e0 + lane < E ? max(0, __ldcg(counts + e0 + lane)) : 0;
    const int k = (c + tok - 1) / tok;
    int ci = c, ki = k;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, ci, o), b = __shfl_up_sync(0xffffffffu, ki, o);
      if (lane >= o) {
        ci += a;
        ki += b;
      }
    }
    if (e0 + lane < E) {
      s_end[e0 + lane] = end + ki;
      s_row[e0 + lane] = row + ci - c;
    }
    row += __shfl_sync(0xffffffffu, ci, 31);
    end += __shfl_sync(0xffffffffu, ki, 31);
  }
  if (lane == 0) s_row[E] = row;
  return end;
}

template <Mode kMode, int TOK, class T>
__device__ __forceinline__ TokenTile open_tile(const Params<T>& p, int y, const int* s_end, const int* s_row) {
  if constexpr (kMode == kDense) {
    const int r0 = y * TOK;
    return {0, r0, min(TOK, p.n_rows - r0)};
  } else {
    int lo = 0, hi = p.E - 1;  // the first expert whose tiles end past y
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_end[mid] > y) hi = mid; else lo = mid + 1;
    }
    const int at = (y - (lo ? s_end[lo - 1] : 0)) * TOK, r0 = min(s_row[lo] + at, p.n_rows - 1);
    return {lo, r0, max(1, min(min(s_row[lo + 1] - s_row[lo] - at, TOK), p.n_rows - r0))};
  }
}

// The Tokens row of token i of a tile (the last one where there is none: the
// columns of a product do not mix, and what has no token is not stored).
template <class T>
__device__ __forceinline__ int token_row(const Params<T>& p, const TokenTile& t, int i) {
  const int r = t.r0 + min(i, t.m - 1);
  return p.sorted_slots ? min(max(__ldcg(p.sorted_slots + r), 0), p.n_slots - 1) / p.topk : r;
}

// The runs of stages: U stages of tiles of nst, cut for `ctas` CTAs (at most U,
// so that none is empty).
struct Runs {
  long long U;
  int ctas, nst;

  __device__ __forceinline__ long long begin(int cta) const { return U * cta / ctas; }
  // The CTA whose run holds stage u: the last one that begins at u or before.
  __device__ __forceinline__ int owner(long long u) const {
    const long long a = (u + 1) * ctas - 1;  // < U * ctas; a 64-bit division costs some 100 instructions
    return U * ctas < (1ll << 31) ? (int)((uint32_t)a / (uint32_t)U) : (int)(a / U);
  }
  // Where CTA `cta` leaves its sums of a tile, [token][kRows] floats. Along the
  // stages each new (tile, CTA) pair raises tile + cta, so the slots are distinct
  // and there are fewer than tiles + CTAs.
  template <int TOK>
  __device__ __forceinline__ float* part(float* parts, int cta, int tile) const {
    return parts + (size_t)(tile + cta) * (kRows * TOK);
  }
};

// The product: a CTA's run of stages, sums left in the workspace. Alone (cold
// caches): one token through 4096 x 4096 6 us, 16 tokens through 14336 x 4096 with
// minima per 64 21 us, gate/up of 2 experts of 4096 x 14336 for one token 29 us (4.1
// TB/s), their down projection 19 us.
template <class T, class S, Mode kMode>
__global__ void __launch_bounds__(kThreads, 2)
    w4_kernel(const __grid_constant__ CUtensorMap map0, const __grid_constant__ CUtensorMap map1,
              const __grid_constant__ Params<T> p) {
  constexpr int NT = S::NT, FL = S::FL;
  constexpr int kFeatures = kMode == kGateUp ? kRows / 2 : kRows;  // output features per tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_full[kStages], s_empty[kStages];
  __shared__ int s_abort, s_y;
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* smem_x = smem + kStages * kStageBytes;
  int* s_end = reinterpret_cast<int*>(smem_x + kStages * S::kTokenBytes);
  int* s_row = s_end + p.E;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  // The next launch may start from here on. What this one reads of the counts
  // and the order is older than its predecessor (or waited for), and so than
  // everything that can run beside it.
  if (p.wait_first) griddep_wait();
  griddep_launch();
  if (warp == 0) {
    int y = p.max_y;
    if (kMode != kDense) y = min(y, expert_tiles(p.counts, p.E, S::kTokens, s_end, s_row));
    if (lane == 0) {
      s_y = y;
      s_abort = 0;
    }
  } else if (warp == kWarps && lane == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s_full[i], 1 + 32);
      mbar_init(&s_empty[i], kWarps);
    }
    fence_mbar_init();
    tma_prefetch_desc(&map0);
    if (kMode == kGateUp) tma_prefetch_desc(&map1);
  }
  __syncthreads();

  // This CTA's run of the stages: [u0, u1) of the tiles' stages laid end to end.
  const int np = pieces(p.K), nst = (np + kStagePieces - 1) / kStagePieces;
  const long long U = (long long)s_y * p.feature_tiles * nst;
  const Runs run{U, (int)min((long long)gridDim.x, U), nst};
  if (blockIdx.x >= run.ctas) {
    // Not before its predecessor either: where no CTA has a stage (every slot
    // dropped), this grid's end must still mean that the tokens are written.
    griddep_wait();
    return;
  }
  const long long u0 = run.begin(blockIdx.x), u1 = run.begin(blockIdx.x + 1);
  int tile = (int)(u0 / nst), st = (int)(u0 - (long long)tile * nst);
  int y = tile / p.feature_tiles, f = tile - y * p.feature_tiles;
  int n_units = (int)(u1 - u0);

  if (warp == kWarps) {  // ---------------------------------------------- producer
    // Two cursors: the codes' (lane 0, by TMA), which starts on the first
    // stages before the tokens are ready, and the tokens' (all lanes, 16 bytes
    // of a token's run each).
    struct Cursor {
      int st, f, y;
      TokenTile tl;
    };
    auto next = [&](Cursor& c) {
      if (++c.st == nst) {
        c.st = 0;
        if (++c.f == p.feature_tiles) {
          c.f = 0;
          if (++c.y < s_y) c.tl = open_tile<kMode, S::kTokens>(p, c.y, s_end, s_row);
        }
      }
    };
    Cursor cw{st, f, y, open_tile<kMode, S::kTokens>(p, y, s_end, s_row)}, cx = cw;
    auto copy_codes = [&](int slot) {
      if (lane == 0) {
        uint8_t* dst = smem + slot * kStageBytes;
        mbar_arrive_expect_tx(&s_full[slot], kStageBytes);
        const int row = cw.tl.e * p.N + cw.f * kFeatures;
        tma_load_2d(dst, &map0, &s_full[slot], cw.st * 128, row);
        if (kMode == kGateUp) tma_load_2d(dst + kStageBytes / 2, &map1, &s_full[slot], cw.st * 128, row);
      }
      next(cw);
    };
    const int ahead = min(kStages, n_units);
    for (int i = 0; i < ahead; ++i) copy_codes(i);
    griddep_wait();
    constexpr int kTailUnits = S::kMin ? 1 + (kStagePieces / FL + 3) / 4 : 1;  // 16 bytes each: scale, sums
    int slot = 0, my_row = token_row(p, cx.tl, lane);  // lane j: the row of the tile's token j
    uint32_t parity = 1;
    for (int i = 0; i < n_units; ++i) {
      if (i >= ahead) {
        if (!mbar_wait(&s_empty[slot], parity, &s_abort)) {
          // given up: let the copies in flight land (the last kStages stages', all issued) before the CTA ends
          int never = 0;
          for (int j = i - kStages; j < i; ++j) mbar_wait(&s_full[j % kStages], j / kStages & 1, &never);
          break;
        }
        copy_codes(slot);
      }
      if constexpr (S::kMakes) {
        uint8_t* rec = smem_x + slot * S::kTokenBytes;
        for (int j = 0; j < cx.tl.m; ++j) {
          float v[8];
          load_run(p.rows + (size_t)(cx.tl.r0 + j) * p.K, cx.st * kStageElems + lane * 8, p.K, p.vec, v);
          write_run<!std::is_same<T, __half>::value>(
              rec + j * kRecord, reinterpret_cast<float*>(rec + S::kTokens * kRecord + j * kTail), FL * kPiece, v);
        }
        mbar_arrive(&s_full[slot]);
        next(cx);
        if (++slot == kStages) {
          slot = 0;
          parity ^= 1;
        }
        continue;
      }
      const uint32_t dst = smem_u32(smem_x + slot * S::kTokenBytes) + lane * 16;
      const uint8_t* src = p.x.rec + (size_t)cx.st * kRecord + lane * 16;
      for (int j = 0; j < cx.tl.m; ++j) {
        const uint8_t* rec = src + (size_t)__shfl_sync(0xffffffffu, my_row, j) * (nst * kRecord);
        cp_async16(dst + j * kRecord, rec);
        if (lane < kTailUnits) cp_async16(dst + S::kTokens * kRecord + j * kTail, rec + kStageElems * 2);
      }
      cp_async_mbar_arrive(&s_full[slot]);
      const int y0 = cx.y;
      next(cx);
      if (cx.y != y0) my_row = token_row(p, cx.tl, lane);
      if (++slot == kStages) {
        slot = 0;
        parity ^= 1;
      }
    }
    cp_async_commit();
    cp_async_wait<0>();
    return;
  }

  // ------------------------------------------------------------------ consumers
  constexpr int kSG = kStagePieces / FL;             // groups per stage
  constexpr int kSR = (kSG + 3) / 4;                 // of which lane t holds t, t + 4
  const int g = lane >> 2, t = lane & 3;
  const int G = groups(p.K, FL * kPiece);
  // Set s, row i of this warp: gate/up, matrix s, feature 16 warp + i; else
  // feature 32 warp + 16 s + i. In shared memory, 128 bytes a row, 16-byte unit
  // u at u ^ (row % 8) (TMA's 128-byte swizzle).
  const int set_row = kMode == kGateUp ? warp * 16 : warp * 32;
  const int set_step = kMode == kGateUp ? kRows / 2 : 16;
  const uint32_t base = smem_u32(smem);
  const int lrow = lane & 15, lpiece = lane >> 4;
  const uint32_t lm = base + (set_row + lrow) * 128 + ((lpiece ^ (lrow & 7)) << 4);

  TokenTile tl = open_tile<kMode, S::kTokens>(p, y, s_end, s_row);
  // Scales run one stage ahead. row0: this lane's first weight row, counted over
  // all experts; rows past the last are read as the last (nothing of them is used).
  const uint32_t last_row = (uint32_t)(kMode == kDense ? 1 : p.E) * (uint32_t)p.N - 1;
  uint32_t row0 = 0;
  auto open_scales = [&](int e, int ft) { row0 = (uint32_t)(e * p.N + ft * kFeatures + set_row + g); };
  uint32_t s_next[2][kSR], m_next[2][kSR];  // of rows g (low half) and g + 8
  auto load_scales = [&](int stage) {
#pragma unroll
    for (int i = 0; i < kSR; ++i) {
      const uint32_t gi = min(stage * kSG + (t + 4 * i) % kSG, G - 1);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Scales<T>& w = p.w[kMode == kGateUp ? s : 0];
        const uint32_t r = row0 + (kMode == kGateUp ? 0 : 16 * s);
        const uint32_t lo = min(r, last_row) * (uint32_t)G + gi, hi = min(r + 8, last_row) * (uint32_t)G + gi;
        s_next[s][i] = pack2(__ldg(w.s + lo), __ldg(w.s + hi));
        if constexpr (S::kMin) m_next[s][i] = pack2(__ldg(w.m + lo), __ldg(w.m + hi));
      }
    }
  };
  open_scales(tl.e, f);
  load_scales(st);

  // the weights are older than this launch's predecessor, the tokens are its
  // output; the consumers see them through the producer's copies
  // this lane's run of 8 of token g, and the tail of token 2 t
  const uint32_t xs = smem_u32(smem_x) + g * kRecord + t * 16;
  const uint32_t xt = smem_u32(smem_x) + S::kTokens * kRecord + t * 2 * kTail;

  float tot[2][NT][4] = {};
  int slot = 0;
  uint32_t parity = 0;
  for (; n_units > 0; --n_units) {
    // What comes after this stage: the next one of the tile, or the next tile's
    // first (found again at the end, so that it takes no registers meanwhile).
    const bool tile_end = st + 1 == nst;
    if (tile_end && n_units > 1) {
      const bool wrap = f + 1 == p.feature_tiles;
      open_scales(wrap ? open_tile<kMode, S::kTokens>(p, y + 1, s_end, s_row).e : tl.e, wrap ? 0 : f + 1);
    }
    uint32_t s_cur[2][kSR], m_cur[2][kSR];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < kSR; ++i) {
        s_cur[s][i] = s_next[s][i];
        if constexpr (S::kMin) m_cur[s][i] = m_next[s][i];
      }
    load_scales(tile_end ? 0 : st + 1);

    // A wait that ran out has raised the status word; the sums are then of no
    // use, but every warp goes on to the end of its run.
    mbar_wait(&s_full[slot], parity, &s_abort);
    auto stage = [&](auto blocks) {
      constexpr int NB = decltype(blocks)::value;  // blocks of 8 tokens there are
      float part[2][NB][4];
      uint32_t code[2][4];
#pragma unroll
      for (int pp = 0; pp < kStagePieces; ++pp) {
        if (pp % 2 == 0) {
#pragma unroll
          for (int s = 0; s < 2; ++s) ldmatrix4(code[s], (lm ^ (pp << 4)) + slot * kStageBytes + s * set_step * 128);
        }
        uint4 xb[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) xb[n] = lds128(xs + slot * S::kTokenBytes + n * 8 * kRecord + pp * 64);
        // the four products of a piece: both sets, then their second halves, so
        // that the two that share accumulators are as far apart as they can be
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint32_t wa = code[s][2 * (pp % 2)], wb = code[s][2 * (pp % 2) + 1];
            uint32_t a[4];
            code_pairs(wa, h, a[0], a[2]);
            code_pairs(wb, h, a[1], a[3]);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              const uint32_t b0 = h ? xb[n].z : xb[n].x, b1 = h ? xb[n].w : xb[n].y;
              if (pp % FL == 0 && h == 0) mma16816_first(part[s][n], a, b0, b1);
              else mma16816(part[s][n], a, b0, b1);
            }
          }
        if ((pp + 1) % FL == 0) {
          const int gi = pp / FL, from = (lane & ~3) + gi % 4;
          float xscale[NB][2], xsum[NB][2];
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t tail = xt + slot * S::kTokenBytes + (n * 8 + c) * kTail;
              xscale[n][c] = lds32(tail);
              if constexpr (S::kMin) xsum[n][c] = lds32(tail + 16 + gi * 4);
            }
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const float2 sv = unpack2<T>(__shfl_sync(0xffffffffu, s_cur[s][gi / 4], from));
            float2 mv = sv;
            if constexpr (S::kMin) {
              mv = unpack2<T>(__shfl_sync(0xffffffffu, m_cur[s][gi / 4], from));
              mv = make_float2(fmaf(8.f, sv.x, mv.x), fmaf(8.f, sv.y, mv.y));
            }
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float a = sv.x * part[s][n][c], b = sv.y * part[s][n][2 + c];
                if constexpr (S::kMin) {
                  a = fmaf(mv.x, xsum[n][c], a);
                  b = fmaf(mv.y, xsum[n][c], b);
                }
                tot[s][n][c] = fmaf(xscale[n][c], a, tot[s][n][c]);
                tot[s][n][2 + c] = fmaf(xscale[n][c], b, tot[s][n][2 + c]);
              }
          }
        }
      }
    };
    if (NT == 1 || tl.m <= 8) stage(std::integral_constant<int, 1>{});
    else stage(std::integral_constant<int, NT>{});
    __syncwarp();
    if (lane == 0) mbar_arrive(&s_empty[slot]);
    if (++slot == kStages) {
      slot = 0;
      parity ^= 1;
    }

    // ---- the tile, or this CTA's part of it, is done
    if (tile_end || n_units == 1) {
      float* mine = run.part<S::kTokens>(p.parts, blockIdx.x, y * p.feature_tiles + f) + set_row + g;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int tok = n * 8 + t * 2 + (c & 1);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (tok < tl.m) mine[tok * kRows + s * set_step + (c >> 1) * 8] = tot[s][n][c];
            tot[s][n][c] = 0.f;
          }
        }
    }
    if (!tile_end) {
      ++st;
    } else if (n_units > 1) {
      st = 0;
      if (++f == p.feature_tiles) {
        f = 0;
        tl = open_tile<kMode, S::kTokens>(p, ++y, s_end, s_row);
      }
    }
  }
}

// ------------------------------------------------------------------ sums
// These launches set up the tiles before they wait for the product: the counts
// and the order are older than it.

// *p where `on`, else zero, from L2 (the product before has just written it; an
// older launch on this SM may have left the last one's sums in L1). Predicated,
// since behind branches the compiler does not keep the loads in flight together.
__device__ __forceinline__ float load_if(const float* p, bool on) {
  float v = 0.f;
  asm volatile("{.reg .pred q; setp.ne.b32 q, %2, 0; @q ld.global.cg.f32 %0, [%1];}" : "+f"(v) : "l"(p), "r"((int)on));
  return v;
}
__device__ __forceinline__ void load4_if(float* v, const float* p, bool on) {
  v[0] = v[1] = v[2] = v[3] = 0.f;
  asm volatile("{.reg .pred q; setp.ne.b32 q, %5, 0; @q ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];}"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3])
               : "l"(p), "r"((int)on));
}

// The token tiles, set up by every thread of a CTA that reads the parts.
template <Mode kMode, int TOK, class T>
__device__ __forceinline__ Runs open_runs(const Params<T>& p, int grid, int* s_end, int* s_row, int* s_y) {
  if (threadIdx.x < 32) {
    int y = p.max_y;
    if (kMode != kDense) y = min(y, expert_tiles(p.counts, p.E, TOK, s_end, s_row));
    if (threadIdx.x == 0) *s_y = y;
  }
  __syncthreads();
  const int nst = stages(p.K);
  const long long U = (long long)*s_y * p.feature_tiles * nst;
  return {U, (int)min((long long)grid, U), nst};
}

// Sums of the parts of `tile` at [token][row .. row + kV) and, kN = 2, at
// kRows / 2 rows on, in K order (kV = 1, or 8 with row a multiple of 8).
template <int TOK, int kV, int kN>
__device__ __forceinline__ void sum_parts(const Runs& run, const float* parts, int tile, int tok, int row,
                                          float (&v)[kN][kV]) {
  const int c0 = run.owner((long long)tile * run.nst), c1 = run.owner((long long)(tile + 1) * run.nst - 1);
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int i = 0; i < kV; ++i) v[n][i] = 0.f;
  constexpr int kB = kV == 1 ? 8 : 2;  // parts whose loads are in flight together
  const float* q = parts + (size_t)(tile + c0) * (kRows * TOK) + tok * kRows + row;
  for (int c = c0; c <= c1; c += kB, q += (size_t)kB * (kRows * TOK)) {
    float b[kB][kN][kV];
#pragma unroll
    for (int j = 0; j < kB; ++j)
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const float* at = q + (size_t)j * (kRows * TOK) + n * (kRows / 2);
        if constexpr (kV == 1) {
          b[j][n][0] = load_if(at, c + j <= c1);
        } else {
#pragma unroll
          for (int i = 0; i < kV; i += 4) load4_if(&b[j][n][i], at + i, c + j <= c1);
        }
      }
#pragma unroll
    for (int j = 0; j < kB; ++j)
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kV; ++i) v[n][i] += b[j][n][i];
  }
}

__device__ __forceinline__ float swiglu(float h, float u) { return h / (1.f + expf(-h)) * u; }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

// With minima the product adds two terms, s (q - 8) x and (m + 8 s) x, which for an
// infinite x can be infinities of opposite signs, or 0 * inf beside an infinity,
// where (s q + m) x is one infinity. So a result that is not finite is made again:
// where the token row has infinite or NaN elements, the sum is theirs alone, against
// the weights themselves (n: weight row over all experts); the overflow of a
// finite row stays as it is. That is done in a second pass after a launch's own
// work, kept small for the sake of the first one: calls (a stack) cost every
// launch 0.6 us, 47 registers for 32 a tenth of a stage of 256 tokens, and as it
// is a layer with minima takes 0.7 to 3 us longer (one token 68.4 to 69.1, 64 tokens
// of 32 experts 380.6 to 383.5). What is made again is never finite: w * inf is an
// infinity or NaN. 16 tokens with an infinity each through 14336 x 4096: 403 us
// instead of 29.
template <class T>
__device__ __forceinline__ float sum_by_weights(const Params<T>& p, int matrix, size_t n, size_t row, float sum) {
  const int G = groups(p.K, p.group);
  const uint8_t* code = p.codes[matrix] + n * (pieces(p.K) * (kPiece / 2));
  float exact = 0.f;
  bool any = false;
  auto meet = [&](int k, float x) {
    const size_t at = n * G + k / p.group;
    const float q = (float)(__ldg(code + k / 2) >> (k & 1 ? 4 : 0) & 15);
    exact += fmaf(to_f(__ldg(p.w[matrix].s + at)), q, to_f(__ldg(p.w[matrix].m + at))) * x;
    any = true;
  };
  if (p.rows) {  // no records in the workspace
#pragma unroll 1
    for (int k = 0; k < p.K && !isnan(exact); ++k) {
      const float x = to_f(__ldg(p.rows + row * p.K + k));
      if (!finite(x)) meet(k, x);
    }
  } else {
    const uint8_t* rec = p.x.rec + row * stages(p.K) * kRecord;
#pragma unroll 1
    for (int k = 0; k < p.K && !isnan(exact); k += 8) {  // a record is whole past K
      const uint4 run = __ldcg(reinterpret_cast<const uint4*>(rec + (size_t)(k / kStageElems) * kRecord + k % kStageElems * 2));
      const uint32_t pair[4] = {run.x, run.y, run.z, run.w};  // elements i and i + 4
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = unpack2<__half>(pair[i]);
        if (!finite(x.x)) meet(k + i, x.x);
        if (!finite(x.y)) meet(k + i + 4, x.y);
      }
    }
  }
  return any ? exact : sum;
}

// Output feature n of token `tok` of the tile (y, n's feature tile), sums and all,
// a part at a time: this must not take more registers than the first pass.
template <Mode kMode, int TOK, class T>
__device__ __forceinline__ float result_again(const Params<T>& p, const Runs& run, const TokenTile& tl, int y, int tok, int n) {
  constexpr int kFeatures = kMode == kGateUp ? kRows / 2 : kRows;
  const int tile = y * p.feature_tiles + n / kFeatures;
  const int c0 = run.owner((long long)tile * run.nst), c1 = run.owner((long long)(tile + 1) * run.nst - 1);
  float gate = 0.f, v = 0.f;
#pragma unroll 1
  for (int j = 0; j < (kMode == kGateUp ? 2 : 1); ++j) {
    gate = v;
    v = 0.f;
    const float* at = p.parts + (size_t)(tile + c0) * (kRows * TOK) + tok * kRows + j * (kRows / 2) + n % kFeatures;
#pragma unroll 1
    for (int c = c0; c <= c1; ++c, at += kRows * TOK) v += __ldcg(at);
    if (!finite(v)) v = sum_by_weights(p, j, (size_t)tl.e * p.N + n, token_row(p, tl, tok), v);
  }
  return kMode == kGateUp ? swiglu(gate, v) : v;
}

// out[r, n] of a dense product or a down projection, act[r, n] of a gate/up: a
// CTA per feature tile and token, a thread per feature. `grid`: the product's. Bound
// by latency: 4.6 us alone for 16 x 14336, most of it overlapping the product's end.
template <Mode kMode, int TOK, bool kMin, class T, class O>
__global__ void __launch_bounds__(kRows, 8) finish_kernel(const __grid_constant__ Params<T> p, int grid, O* __restrict__ out) {
  extern __shared__ int s_index[];
  __shared__ int s_y;
  griddep_launch();
  int *s_end = s_index, *s_row = s_index + p.E;
  const Runs run = open_runs<kMode, TOK>(p, grid, s_end, s_row, &s_y);
  griddep_wait();
  constexpr int kFeatures = kMode == kGateUp ? kRows / 2 : kRows;
  constexpr int kPer = kRows / kFeatures;  // tokens a CTA takes at a time
  const int f = blockIdx.x, r = threadIdx.x % kFeatures, n = f * kFeatures + r;
  if (n >= p.N) return;
  const int i0 = blockIdx.y * kPer + threadIdx.x / kFeatures, step = gridDim.y * kPer;
  bool odd = false;
  for (int i = i0; i < s_y * TOK; i += step) {
    const int y = i / TOK, tok = i - y * TOK, tile = y * p.feature_tiles + f;
    const TokenTile tl = open_tile<kMode, TOK>(p, y, s_end, s_row);
    if (tok >= tl.m) continue;
    constexpr int kN = kMode == kGateUp ? 2 : 1;
    float v[kN][1];
    sum_parts<TOK, 1, kN>(run, p.parts, tile, tok, r, v);
    const float o = kN == 2 ? swiglu(v[0][0], v[kN - 1][0]) : v[0][0];
    odd |= !finite(o);
    out[(size_t)(tl.r0 + tok) * p.N + n] = from_f<O>(o);
  }
  if (kMin && odd)
    for (int i = i0; i < s_y * TOK; i += step) {
      const int y = i / TOK, tok = i - y * TOK;
      const TokenTile tl = open_tile<kMode, TOK>(p, y, s_end, s_row);
      O* o = out + (size_t)(tl.r0 + tok) * p.N + n;
      if (tok < tl.m && !finite(to_f(*o))) *o = from_f<O>(result_again<kMode, TOK>(p, run, tl, y, tok, n));
    }
}

// The activations of a gate/up product straight into the tokens of the down
// projection: a warp per packed row and run of 256 features (two tiles). Bound by
// latency: 7 us alone for one token, 9 us for 512 rows of 2048. With minima the
// infinite and NaN elements of a record may be of the wrong kind at first; its
// scale is the finite ones', and what the down product makes of the row is not
// finite whatever they are.
template <int TOK, bool kMin, class T>
__global__ void __launch_bounds__(256, kMin ? 4 : 5) act_tokens_kernel(const __grid_constant__ Params<T> p, int grid, int group, Tokens act) {
  extern __shared__ int s_index[];
  __shared__ int s_y;
  griddep_launch();
  int *s_end = s_index, *s_row = s_index + p.E;
  const Runs run = open_runs<kGateUp, TOK>(p, grid, s_end, s_row, &s_y);
  griddep_wait();
  const int lane = threadIdx.x & 31, nst = stages(p.N);
  const long long w0 = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const long long warps = ((long long)gridDim.x * blockDim.x) >> 5, total = (long long)s_y * TOK * nst;
  bool odd = false;
  for (long long w = w0; w < total; w += warps) {
    const int st = (int)(w % nst), ty = (int)(w / nst), y = ty / TOK, tok = ty - y * TOK;
    const TokenTile tl = open_tile<kGateUp, TOK>(p, y, s_end, s_row);
    if (tok >= tl.m) continue;
    const int n = st * kStageElems + lane * 8, f = n / (kRows / 2);
    float v[2][8] = {}, a[8];
    if (f < p.feature_tiles)
      sum_parts<TOK, 8, 2>(run, p.parts, y * p.feature_tiles + f, tok, n % (kRows / 2), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = n + i < p.N ? swiglu(v[0][i], v[1][i]) : 0.f;
      odd |= !finite(a[i]);
    }
    uint8_t* rec = act.rec + ((size_t)(tl.r0 + tok) * nst + st) * kRecord;
    write_run<true>(rec, tail_of(rec), group, a);
  }
  if (kMin && odd)
    for (long long w = w0; w < total; w += warps) {
      const int st = (int)(w % nst), ty = (int)(w / nst), y = ty / TOK, tok = ty - y * TOK;
      const TokenTile tl = open_tile<kGateUp, TOK>(p, y, s_end, s_row);
      if (tok >= tl.m) continue;
      __half* rec = reinterpret_cast<__half*>(act.rec + ((size_t)(tl.r0 + tok) * nst + st) * kRecord) + lane * 8;
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        __half* h = rec + (i < 4 ? 2 * i : 2 * i - 7);
        if (!finite(to_f(*h))) *h = __float2half_rn(result_again<kGateUp, TOK>(p, run, tl, y, tok, st * kStageElems + lane * 8 + i));
      }
    }
}

// The outputs of feature n of combine_parts_kernel that are not finite, made again.
template <int TOK, class T>
__device__ __forceinline__ void combine_again(const Params<T>& p, const Runs& run, const int* s_end, int y_end, const int* slot_rows,
                                           const int* ids, const float* weights, int tokens, int topk, int n, T* out) {
  const int* s_row = s_end + p.E;
  for (int t = blockIdx.y; t < tokens; t += gridDim.y) {
    if (finite(to_f(out[(size_t)t * p.N + n]))) continue;
    float acc = 0.f;
    for (int j = 0; j < topk; ++j) {
      const long long s = (long long)t * topk + j;
      const int r = __ldcg(slot_rows + s), e = __ldcg(ids + s);
      if (r < 0 || r >= p.n_rows || e < 0 || e >= p.E) continue;
      const int at = r - s_row[e], y = (e ? s_end[e - 1] : 0) + at / TOK;
      if (at < 0 || y >= min(s_end[e], y_end)) continue;
      const TokenTile tl = open_tile<kDown, TOK>(p, y, s_end, s_row);
      acc = fmaf(__ldcg(weights + s), result_again<kDown, TOK>(p, run, tl, y, at % TOK, n), acc);
    }
    out[(size_t)t * p.N + n] = from_f<T>(acc);
  }
}

// out[t] = sum_j w[t, j] y[row of slot (t, j)] from the parts of the down
// projection, fp32 in j order, rounded once. A CTA per token and 256 features; bound
// by latency (64 tokens, 8 choices, 7168 wide: 17 us alone for 15 MB of parts), so
// six CTAs an SM (four or eight: 1 % of the layer more).
template <int TOK, bool kMin, class T>
__global__ void __launch_bounds__(kRows, 6)
    combine_parts_kernel(const __grid_constant__ Params<T> p, int grid, const int* __restrict__ slot_rows,
                         const int* __restrict__ ids, const float* __restrict__ weights, int tokens, int topk,
                         T* __restrict__ out) {
  extern __shared__ int s_index[];
  __shared__ int s_y;
  griddep_launch();
  int *s_end = s_index, *s_row = s_index + p.E;
  const Runs run = open_runs<kDown, TOK>(p, grid, s_end, s_row, &s_y);
  // The token's parts in order, listed by the first warp (a slot per lane): row of
  // 256 sums, and for the last part of a slot its weight.
  constexpr int kList = 256, kB = 8;  // kB: loads in flight together
  __shared__ uint32_t s_part[kList];  // top bit: the slot's last
  __shared__ float s_w[kList];
  __shared__ int s_n;
  const int lane = threadIdx.x & 31, f = blockIdx.x, n = f * kRows + threadIdx.x;
  bool waited = false, odd = false;
  for (int t = blockIdx.y; t < tokens; t += gridDim.y) {
    float acc = 0.f, v = 0.f;
    for (int j0 = 0; j0 < topk; j0 += 32) {
      uint32_t part = 0;
      int np = 0, begin = 0;
      float w = 0.f;
      if (threadIdx.x < 32) {
        if (j0 + lane < topk) {
          const long long s = (long long)t * topk + j0 + lane;
          const int r = __ldcg(slot_rows + s), e = __ldcg(ids + s);
          w = __ldcg(weights + s);
          if (r >= 0 && r < p.n_rows && e >= 0 && e < p.E) {  // else dropped
            const int at = r - s_row[e], y = (e ? s_end[e - 1] : 0) + at / TOK;
            if (at >= 0 && y < min(s_end[e], s_y)) {
              const int tile = y * p.feature_tiles + f;
              const int c0 = run.owner((long long)tile * run.nst), c1 = run.owner((long long)(tile + 1) * run.nst - 1);
              part = (uint32_t)(tile + c0) * TOK + at % TOK;
              np = c1 - c0 + 1;
            }
          }
        }
        int incl = np;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int a = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += a;
        }
        begin = incl - np;
        if (lane == 31) s_n = incl;
      }
      for (int base = 0;; base += kList) {
        if (threadIdx.x < 32)
          for (int c = max(0, base - begin); c < np && begin + c < base + kList; ++c) {
            s_part[begin + c - base] = part + c * TOK | (c + 1 == np ? 1u << 31 : 0u);
            s_w[begin + c - base] = w;
          }
        __syncthreads();
        const int total = s_n, count = min(kList, total - base);
        if (!waited) griddep_wait();
        waited = true;
        for (int i = 0; i < count; i += kB) {
          float b[kB];
#pragma unroll
          for (int u = 0; u < kB; ++u)
            b[u] = load_if(p.parts + (size_t)(s_part[min(i + u, kList - 1)] & 0x7fffffffu) * kRows + threadIdx.x, i + u < count);
#pragma unroll
          for (int u = 0; u < kB; ++u) {
            if (i + u >= count) break;
            v += b[u];
            if (s_part[i + u] >> 31) {
              acc = fmaf(s_w[i + u], v, acc);
              v = 0.f;
            }
          }
        }
        __syncthreads();
        if (base + kList >= total) break;
      }
    }
    if (n < p.N) {
      out[(size_t)t * p.N + n] = from_f<T>(acc);
      odd |= !finite(acc);
    }
  }
  if constexpr (kMin)
    if (odd) combine_again<TOK>(p, run, s_end, s_y, slot_rows, ids, weights, tokens, topk, n, out);
}

}  // namespace w4
}  // namespace ek
