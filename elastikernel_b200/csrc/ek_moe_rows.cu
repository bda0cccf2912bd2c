// Token rows to expert-major order and back, with their gradients, for sm_100a.
//
//   dispatch       the (token, choice) slots stably sorted by expert, the token
//                  rows copied into that order
//   sum_rows       out[t] = sum_j w[t,j] rows[slot_row[t,j]]: the weighted way
//                  back; without weights, the gradient of the dispatch
//   combine_grad   the gradient of the weighted way back: d_rows[r] = w d_out[t],
//                  d_w[t,j] = <d_out[t], rows[r]>
//   route_grad     gradient of the renormalised top-k softmax to the gate logits
//
// All of it is data movement, bound by HBM for long batches and by the launch for
// short ones: the token side of each copy (T rows) is read or written once and
// kept in registers across the token's k slots, so the bytes are T rows plus T*k
// rows, whatever k. Measured with 8192 tokens, 8 choices, 256 experts, 7168 bf16
// (HBM copies run at 6.5 TB/s): dispatch 178 us (10 of them the order), its
// gradient 169 us (6.3 TB/s), weighted sum 160 us (6.6 TB/s), its gradient 304 us
// (6.6 TB/s). Slots with a negative expert id are
// dropped: they have no row, weigh nothing and get no gradient; the rows past
// the last kept one are zero.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "ek_internal.h"
#include "ek_moe_order.cuh"

namespace ek {

int register_status_reader(int (*fn)(int, int*));

namespace {

int read_status(int clear, int* v) {
  int rc = check_cuda(cudaMemcpyFromSymbol(v, g_ek_status, sizeof(int)), "read status");
  if (rc) return rc;
  if (clear) {
    int z = 0;
    rc = check_cuda(cudaMemcpyToSymbol(g_ek_status, &z, sizeof(int)), "clear status");
  }
  return rc;
}
const int s_status_reg = register_status_reader(read_status);

constexpr int kChunk = kOrderThreads;  // slots per sorting CTA, one per thread
constexpr int kMaxE = kOrderMaxE;

// ------------------------------------------------------------------ dispatch: the order
// Chunks of 1024 slots, a CTA each: count, then place. 65536 slots, 256 experts: 3.2
// and 8.2 us, bound by the latency of their steps (0.8 MB in all).
__global__ void __launch_bounds__(kChunk) dispatch_count_kernel(const int* __restrict__ ids, int n_slots, int E,
                                                                int* __restrict__ chunk_counts) {
  __shared__ int cnt[kMaxE];
  for (int i = threadIdx.x; i < E; i += kChunk) cnt[i] = 0;
  __syncthreads();
  const int s = blockIdx.x * kChunk + threadIdx.x;
  if (s < n_slots) {
    const int e = ids[s];
    if (e >= 0 && e < E)
      atomicAdd(&cnt[e], 1);
    else if (e >= E)
      atomicOr(&g_ek_status, kStatusBadIndex);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < E; i += kChunk) chunk_counts[(size_t)blockIdx.x * E + i] = cnt[i];
}

// Place chunk blockIdx.x: first row of each expert = the slots of all experts
// before it + its own slots in earlier chunks; a slot's rank inside the chunk
// is its place among the equal ids of its warp plus the earlier warps' counts.
__global__ void __launch_bounds__(kChunk)
    dispatch_place_kernel(const int* __restrict__ ids, int n_slots, int E, const int* __restrict__ chunk_counts,
                          int n_chunks, int* __restrict__ sorted_slots, int* __restrict__ slot_rows,
                          int* __restrict__ expert_counts, int* __restrict__ num_rows) {
  extern __shared__ int s_wcnt[];  // [32][E] counts of each warp
  __shared__ int s_next[kMaxE];    // first row of the chunk's slots of each expert
  __shared__ int s_tot[kMaxE], s_before[kMaxE];
  __shared__ int s_wsum[32];
  __shared__ int s_total;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunk = blockIdx.x;
  if (tid < E) s_tot[tid] = s_before[tid] = 0;
  for (int i = tid; i < 32 * E; i += kChunk) s_wcnt[i] = 0;
  __syncthreads();
  // thread (group, e) adds every `groups`-th chunk's count of expert e
  const int ep = E <= 32 ? 32 : 1 << (32 - __clz(E - 1)), groups = kChunk / ep;
  const int e_of = tid & (ep - 1);
  if (e_of < E) {
    int sum = 0, pre = 0;
#pragma unroll 8
    for (int c = tid / ep; c < n_chunks; c += groups) {
      const int v = __ldg(chunk_counts + (size_t)c * E + e_of);
      sum += v;
      if (c < chunk) pre += v;
    }
    atomicAdd(&s_tot[e_of], sum);
    atomicAdd(&s_before[e_of], pre);
  }
  __syncthreads();
  const int total = tid < E ? s_tot[tid] : 0, before = tid < E ? s_before[tid] : 0;
  int incl = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_wsum[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int w = s_wsum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += v;
    }
    s_wsum[lane] = w;
    if (lane == 31) s_total = w;
  }
  __syncthreads();
  if (tid < E) s_next[tid] = (warp ? s_wsum[warp - 1] : 0) + incl - total + before;
  const int kept = s_total;
  if (chunk == 0) {
    if (tid < E) expert_counts[tid] = total;
    if (tid == 0) *num_rows = kept;
  }
  const int s = chunk * kChunk + tid;
  const int id = s < n_slots ? ids[s] : -1;
  const int e = id < E ? id : -1;
  const unsigned peers = __match_any_sync(0xffffffffu, e < 0 ? -1 : e);
  const int rank = __popc(peers & ((1u << lane) - 1u));
  if (e >= 0 && rank == 0) s_wcnt[warp * E + e] = __popc(peers);
  __syncthreads();
  if (s < n_slots) {
    if (e >= 0) {
      int row = s_next[e] + rank;
      for (int w = 0; w < warp; ++w) row += s_wcnt[w * E + e];
      sorted_slots[row] = s;
      slot_rows[s] = row;
    } else {
      slot_rows[s] = -1;
    }
    if (s >= kept) sorted_slots[s] = n_slots;  // rows past the last: row s, one per slot index
  }
}

// ------------------------------------------------------------------ rows
// One vector of V bytes of a row (V = 16, 8, 4 or 2 by the rows' alignment).
template <int V>
struct Vec;
template <>
struct Vec<16> { using type = uint4; };
template <>
struct Vec<8> { using type = uint2; };
template <>
struct Vec<4> { using type = uint32_t; };
template <>
struct Vec<2> { using type = uint16_t; };

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

// N = V / sizeof(T) elements of a row as fp32 and back.
template <class T, int V>
struct Elems {
  static constexpr int N = V / (int)sizeof(T);
  using Raw = typename Vec<V>::type;
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[N]) {
    const T* p = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f(p[i]);
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[N]) {
    Raw r;
    T* p = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_f<T>(f[i]);
    return r;
  }
};

// *p where `on`, else zero. A predicated instruction: behind branches the
// compiler does not keep a token's loads in flight together.
__device__ __forceinline__ uint4 load_if(const uint4* p, bool on) {
  uint4 v = {};
  asm volatile("{.reg .pred q; setp.ne.b32 q, %5, 0; @q ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];}"
               : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
               : "l"(p), "r"((int)on));
  return v;
}
__device__ __forceinline__ uint2 load_if(const uint2* p, bool on) {
  uint2 v = {};
  asm volatile("{.reg .pred q; setp.ne.b32 q, %3, 0; @q ld.global.nc.v2.u32 {%0, %1}, [%2];}"
               : "+r"(v.x), "+r"(v.y)
               : "l"(p), "r"((int)on));
  return v;
}
__device__ __forceinline__ uint32_t load_if(const uint32_t* p, bool on) {
  uint32_t v = 0;
  asm volatile("{.reg .pred q; setp.ne.b32 q, %2, 0; @q ld.global.nc.u32 %0, [%1];}" : "+r"(v) : "l"(p), "r"((int)on));
  return v;
}
__device__ __forceinline__ uint16_t load_if(const uint16_t* p, bool on) {
  uint16_t v = 0;
  asm volatile("{.reg .pred q; setp.ne.b32 q, %2, 0; @q ld.global.nc.u16 %0, [%1];}" : "+h"(v) : "l"(p), "r"((int)on));
  return v;
}

// Zero the rows past the last kept one ([kept, n_rows)).
template <class Raw>
__device__ __forceinline__ void zero_tail(Raw* __restrict__ rows, int kept, int n_rows, int nvec) {
  const long long first = (long long)max(0, min(kept, n_rows)) * nvec, end = (long long)n_rows * nvec;
  for (long long i = first + (long long)blockIdx.x * blockDim.x + threadIdx.x; i < end;
       i += (long long)gridDim.x * blockDim.x)
    rows[i] = Raw{};
}

// The unit of the copies and sums: a warp, one token and a run of kRun vectors
// per lane. The token's k rows are fetched once per unit (lane j holds slot j's)
// and the run's loads are all in flight together.
struct Unit {
  int t, c0;  // token, first vector of this lane
};
template <int kRun>
__device__ __forceinline__ Unit unit_of(long long u, int runs) {
  const int t = (int)(u / runs);
  return {t, (int)(u - (long long)t * runs) * (32 * kRun) + (int)(threadIdx.x & 31)};
}
template <int kRun>
__host__ __device__ inline int runs_per_row(int nvec) { return (nvec + 32 * kRun - 1) / (32 * kRun); }

// Vectors of a row per lane and unit, more where they are narrow (8192 tokens, 1111
// wide: fp32 and 8 choices 67 us against 71 with four, bf16 and 2 choices 18 against 22).
template <class Raw>
constexpr int kCopyRun = sizeof(Raw) < 16 ? 8 : 4;

// Copy x[t] to the rows of token t; row_of(s): the row of slot s (negative:
// dropped). Neighbouring units go to different CTAs, so that few of them still
// reach every SM.
template <class Raw, class RowOf>
__device__ __forceinline__ void copy_rows(const Raw* __restrict__ x, int T, int k, int nvec, const RowOf& row_of,
                                          Raw* __restrict__ rows) {
  const int lane = threadIdx.x & 31, runs = runs_per_row<kCopyRun<Raw>>(nvec);
  const long long warps = ((long long)gridDim.x * blockDim.x) >> 5, units = (long long)T * runs;
  for (long long u = (long long)(threadIdx.x >> 5) * gridDim.x + blockIdx.x; u < units; u += warps) {
    const Unit w = unit_of<kCopyRun<Raw>>(u, runs);
    Raw v[kCopyRun<Raw>];
#pragma unroll
    for (int i = 0; i < kCopyRun<Raw>; ++i)
      if (w.c0 + 32 * i < nvec) v[i] = __ldg(x + (long long)w.t * nvec + w.c0 + 32 * i);
    for (int j0 = 0; j0 < k; j0 += 32) {
      const int mine = j0 + lane < k ? row_of((long long)w.t * k + j0 + lane) : -1;
      const int kn = min(32, k - j0);
      for (int j = 0; j < kn; ++j) {
        const int r = __shfl_sync(0xffffffffu, mine, j);
        if (r < 0) continue;
        Raw* dst = rows + (long long)r * nvec + w.c0;
#pragma unroll
        for (int i = 0; i < kCopyRun<Raw>; ++i)
          if (w.c0 + 32 * i < nvec) dst[32 * i] = v[i];
      }
    }
  }
}

// rows[slot_rows[t*k + j]] = x[t] for the kept slots of each token. 8192 tokens, 8
// choices, 7168 bf16: 168 us, 6.3 TB/s.
template <int V>
__global__ void __launch_bounds__(256)
    dispatch_copy_kernel(const typename Vec<V>::type* __restrict__ x, const int* __restrict__ slot_rows,
                         const int* __restrict__ num_rows, int T, int k, int nvec,
                         typename Vec<V>::type* __restrict__ rows) {
  copy_rows(x, T, k, nvec, [&](long long s) { return __ldg(slot_rows + s); }, rows);
  zero_tail(rows, *num_rows, T * k, nvec);
}

// Small batches (T * k <= kOrderThreads) in one launch: every CTA works out the
// whole order and copies its share of the rows; the first one writes the maps.
// Against count, place and copy (bf16): 64 tokens, 8 choices, 256 experts, 7168 wide
// 4.6 against 9.4 us; 1024 slots of 1024 experts 7.8 against 11.6; the order alone
// of 512 slots 3.0 against 5.0.
template <int V>
__global__ void __launch_bounds__(kOrderThreads)
    dispatch_small_kernel(const int* __restrict__ ids, int T, int k, int E, const typename Vec<V>::type* __restrict__ x,
                          int nvec, int* __restrict__ sorted_slots, int* __restrict__ slot_rows,
                          int* __restrict__ expert_counts, int* __restrict__ num_rows,
                          typename Vec<V>::type* __restrict__ rows) {
  extern __shared__ int sm[];
  __shared__ int s_row[kOrderThreads];
  const int tid = threadIdx.x, n = T * k;
  int id = tid < n ? ids[tid] : -1;
  if (id >= E) {
    if (blockIdx.x == 0) atomicOr(&g_ek_status, kStatusBadIndex);
    id = -1;
  }
  int kept;
  const int row = order_slots(max(id, -1), n, E, sm, &kept);
  s_row[tid] = row;
  if (blockIdx.x == 0) {
    const int* start = sm + (n + 31) / 32 * E;
    if (tid < E) expert_counts[tid] = (tid + 1 < E ? start[tid + 1] : kept) - start[tid];
    if (tid == 0) *num_rows = kept;
    if (tid < n) {
      slot_rows[tid] = row;
      if (row >= 0) sorted_slots[row] = tid;
      if (tid >= kept) sorted_slots[tid] = n;
    }
  }
  if (x == nullptr) return;
  __syncthreads();
  copy_rows(x, T, k, nvec, [&](long long s) { return s_row[s]; }, rows);
  zero_tail(rows, kept, n, nvec);
}

// Vectors of each row that a lane of the sums has in flight; twice as many where
// the rows' alignment leaves them narrow. Measured, one against two for up to 4
// choices: 4096 tokens, 3 choices, 4096 fp32 54 against 47 us; and for 4- and 2-byte
// vectors, without and with the doubling: 8192 tokens, 8 choices, 1111 fp32 104
// against 87 us, 2 choices, 1111 bf16 28 against 19 (four times as many: 141 and 21).
template <int V, int kK>
constexpr int kSumRun = (kK <= 4 ? 2 : 1) * (V < 16 ? 2 : 1);

// out[t] = sum_j w[t,j] rows[slot_rows[t,j]] (w = 1 without weights), fp32 sum
// in j order, rounded once. kK: rows whose loads are in flight together (2, 4 or
// 8, the least that holds the choices).
template <class T, int V, bool kWeighted, int kK>
__global__ void __launch_bounds__(256)
    sum_rows_kernel(const typename Vec<V>::type* __restrict__ rows, const int* __restrict__ slot_rows,
                    const float* __restrict__ weights, int T_tokens, int k, int n_rows, int nvec,
                    typename Vec<V>::type* __restrict__ out) {
  using E = Elems<T, V>;
  constexpr int kRun = kSumRun<V, kK>;
  const int lane = threadIdx.x & 31, runs = runs_per_row<kRun>(nvec);
  const long long warps = ((long long)gridDim.x * blockDim.x) >> 5, units = (long long)T_tokens * runs;
  for (long long u = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; u < units; u += warps) {
    const Unit w = unit_of<kRun>(u, runs);
    float acc[kRun][E::N] = {};
    for (int j0 = 0; j0 < k; j0 += kK) {
      int mine = -1;
      float wt = 1.f;
      if (lane < kK && j0 + lane < k) {
        mine = __ldg(slot_rows + (long long)w.t * k + j0 + lane);
        if (kWeighted) wt = __ldg(weights + (long long)w.t * k + j0 + lane);
      }
      if (mine < 0 || mine >= n_rows) {  // dropped, or past k: nothing times nothing
        mine = -1;
        wt = 0.f;
      }
      typename E::Raw v[kK][kRun];
#pragma unroll
      for (int j = 0; j < kK; ++j) {
        const int r = __shfl_sync(0xffffffffu, mine, j);
#pragma unroll
        for (int i = 0; i < kRun; ++i)
          v[j][i] = load_if(rows + (long long)r * nvec + w.c0 + 32 * i, r >= 0 && w.c0 + 32 * i < nvec);
      }
#pragma unroll
      for (int j = 0; j < kK; ++j) {
        const float wj = kWeighted ? __shfl_sync(0xffffffffu, wt, j) : 1.f;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          float f[E::N];
          E::unpack(v[j][i], f);
#pragma unroll
          for (int e = 0; e < E::N; ++e) acc[i][e] = kWeighted ? fmaf(wj, f[e], acc[i][e]) : acc[i][e] + f[e];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (w.c0 + 32 * i < nvec)
        out[(long long)w.t * nvec + w.c0 + 32 * i] = E::pack(acc[i]);
  }
}

// d_rows[r] = w[s] d_out[t] and d_weights[s] = <d_out[t], rows[r]> (fp32). kTpt
// threads per token; d_out[t] is read once (per kK slots), the kK rows' loads
// are in flight together, and the kK dot products stay in registers until the
// row's end. 4096 tokens, 8 choices, 7168 bf16: 156 us, 6.4 TB/s.
template <class T, int V, int kK, int kTpt>
__global__ void __launch_bounds__(128)
    combine_grad_kernel(const typename Vec<V>::type* __restrict__ rows, const int* __restrict__ slot_rows,
                        const float* __restrict__ weights, const typename Vec<V>::type* __restrict__ d_out,
                        const int* __restrict__ num_rows, int T_tokens, int k, int n_rows, int nvec,
                        typename Vec<V>::type* __restrict__ d_rows, float* __restrict__ d_weights) {
  using E = Elems<T, V>;
  constexpr int kWarpsPer = kTpt / 32, kPer = 128 / kTpt;  // warps per token, tokens per CTA
  __shared__ float s_red[4][kK];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = threadIdx.x % kTpt;
  // every warp of a CTA takes the same number of turns (the barriers below)
  for (long long t0 = (long long)blockIdx.x * kPer; t0 < T_tokens; t0 += (long long)gridDim.x * kPer) {
    const long long t = t0 + warp / kWarpsPer;
    for (int j0 = 0; j0 < k; j0 += kK) {
      int mine = -1;
      float wt = 0.f;
      if (t < T_tokens && lane < kK && j0 + lane < k) {
        mine = __ldg(slot_rows + t * k + j0 + lane);
        wt = __ldg(weights + t * k + j0 + lane);
        if (mine >= n_rows) mine = -1;
      }
      int r[kK];
      float w[kK], dot[kK];
#pragma unroll
      for (int j = 0; j < kK; ++j) {
        r[j] = __shfl_sync(0xffffffffu, mine, j);
        w[j] = __shfl_sync(0xffffffffu, wt, j);
        dot[j] = 0.f;
      }
      if (t < T_tokens) {
        // vectors of each row in flight per lane, two where they are narrow (8192
        // tokens, 8 choices, 1111 fp32: 159 us against 176; 2 choices, bf16: 21 against 30)
        constexpr int kU = V < 16 ? 2 : 1;
        for (int c0 = at; c0 < nvec; c0 += kTpt * kU) {
          typename E::Raw y[kU][kK], g[kU];
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            const int c = c0 + u * kTpt;
#pragma unroll
            for (int j = 0; j < kK; ++j) y[u][j] = load_if(rows + (long long)r[j] * nvec + c, r[j] >= 0 && c < nvec);
            g[u] = load_if(d_out + t * nvec + c, c < nvec);
          }
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            const int c = c0 + u * kTpt;
            float d[E::N];
            E::unpack(g[u], d);
#pragma unroll
            for (int j = 0; j < kK; ++j)
              if (r[j] >= 0 && c < nvec) {
                float f[E::N];
                E::unpack(y[u][j], f);
#pragma unroll
                for (int e = 0; e < E::N; ++e) {
                  dot[j] = fmaf(d[e], f[e], dot[j]);
                  f[e] = w[j] * d[e];
                }
                d_rows[(long long)r[j] * nvec + c] = E::pack(f);
              }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kK; ++j) {
#pragma unroll
        for (int o = 16; o; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
      }
      if constexpr (kWarpsPer > 1) {
        if (lane == 0) {
#pragma unroll
          for (int j = 0; j < kK; ++j) s_red[warp][j] = dot[j];
        }
        __syncthreads();
        if (threadIdx.x < kK) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < kWarpsPer; ++i) sum += s_red[i][threadIdx.x];
          if (j0 + threadIdx.x < k && t < T_tokens) d_weights[t * k + j0 + threadIdx.x] = mine >= 0 ? sum : 0.f;
        }
        __syncthreads();
      } else {
#pragma unroll
        for (int j = 0; j < kK; ++j)
          if (lane == j && j0 + j < k && t < T_tokens) d_weights[t * k + j0 + j] = mine >= 0 ? dot[j] : 0.f;
      }
    }
  }
  zero_tail(d_rows, *num_rows, n_rows, nvec);
}

// ------------------------------------------------------------------ route gradient
// The renormalised weights are the softmax of the chosen logits alone, so
// d_logit[ids_j] += w_j (dw_j - sum_i w_i dw_i) and every other logit gets 0.
// kp lanes (a power of two >= k, up to 32) per token, 32 / kp tokens per warp:
// the warp clears its tokens' rows with wide stores, then each lane puts its
// slot's value where it belongs (the lowest lane, where an id repeats; the sum
// then is in lane order, so that it does not change between runs). 32768 tokens, 256
// experts: 9.5 us with a cold cache for 37 MB. The zeros stay in L2; bound by the
// latency of a warp's one turn, the loads and then the exchanges among its lanes
// (issue slots 34 % busy, most stalls on the exchanges).
__global__ void __launch_bounds__(256)
    route_grad_kernel(const int* __restrict__ ids, const float* __restrict__ weights,
                      const float* __restrict__ d_weights, int T, int E, int k, int kp, bool wide,
                      float* __restrict__ d_logits) {
  const int lane = threadIdx.x & 31, j = lane & (kp - 1), per = 32 / kp;
  const long long warps = ((long long)gridDim.x * blockDim.x) >> 5, groups = ((long long)T + per - 1) / per;
  for (long long u = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; u < groups; u += warps) {
    const long long t = u * per + lane / kp;
    const bool live = j < k && t < T;
    int id = -1;
    float w = 0.f, d = 0.f;
    if (live) {
      id = __ldg(ids + t * k + j);
      w = __ldg(weights + t * k + j);
      d = __ldg(d_weights + t * k + j);
    }
    const long long first = u * per * E, n = min((long long)per, T - u * per) * E;
    if (wide) {
      float4* dst = reinterpret_cast<float4*>(d_logits + first);
      for (long long i = lane; i < n / 4; i += 32) dst[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      for (long long i = lane; i < n; i += 32) d_logits[first + i] = 0.f;
    }
    float mean = w * d;
    for (int o = kp >> 1; o; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
    float g = w * (d - mean);
    // lanes with this token's same expert: their values go to the lowest one
    const unsigned same = __match_any_sync(0xffffffffu, id >= 0 ? (long long)(lane / kp) << 32 | id : (long long)-1 - lane);
    if (__any_sync(0xffffffffu, __popc(same) > 1)) {
      float sum = 0.f;
      for (int i = 0; i < 32; ++i) {
        const float v = __shfl_sync(0xffffffffu, g, i);
        if (same >> i & 1u) sum += v;
      }
      g = sum;
    }
    __syncwarp();  // the zeros above come first
    if (live && id >= 0 && id < E && __ffs(same) - 1 == lane) d_logits[t * E + id] = g;
    __syncwarp();
  }
}

// More than 32 choices: a warp per token, every logit looks through them.
__global__ void __launch_bounds__(256)
    route_grad_any_kernel(const int* __restrict__ ids, const float* __restrict__ weights,
                          const float* __restrict__ d_weights, int T, int E, int k, float* __restrict__ d_logits) {
  const int lane = threadIdx.x & 31;
  const int warps = (gridDim.x * blockDim.x) >> 5;
  for (int t = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; t < T; t += warps) {
    const long long s = (long long)t * k;
    float mean = 0.f;
    for (int j = 0; j < k; ++j) mean += weights[s + j] * d_weights[s + j];
    for (int e = lane; e < E; e += 32) {
      float g = 0.f;
      for (int j = 0; j < k; ++j)
        if (ids[s + j] == e) g += weights[s + j] * (d_weights[s + j] - mean);
      d_logits[(long long)t * E + e] = g;
    }
  }
}

// ------------------------------------------------------------------ launches
int elem_bytes(int dtype) {
  return dtype == EK_DTYPE_BF16 || dtype == EK_DTYPE_FP16 ? 2 : dtype == EK_DTYPE_FP32 ? 4 : 0;
}

// Vectors of a row and a run past its end are counted in ints; the bytes are not.
constexpr int kMaxH = 1 << 30;

template <class T, int V>
int vectors(int H) {
  return (int)((size_t)H * sizeof(T) / V);
}

// Widest vector that divides the row and every base address.
int vec_bytes(size_t row_bytes, std::initializer_list<const void*> ptrs) {
  uintptr_t a = row_bytes;
  for (const void* p : ptrs) a |= reinterpret_cast<uintptr_t>(p);
  return a % 16 == 0 ? 16 : a % 8 == 0 ? 8 : a % 4 == 0 ? 4 : 2;
}

int rows_grid(long long items) { return (int)std::max<long long>(1, std::min<long long>((items + 255) / 256, 148 * 64)); }

int check_rows(const char* what, int T, int k, int n_rows, int H, int dtype) {
  if (T < 0 || k < 1 || H < 1 || n_rows < 0 || !elem_bytes(dtype))
    return set_error(EK_ERR_INVALID, "%s: bad sizes or type (T=%d k=%d rows=%d H=%d dtype=%d)", what, T, k, n_rows, H,
                     dtype);
  if (H > kMaxH) return set_error(EK_ERR_INVALID, "%s: rows of more than 2^30 elements (H=%d)", what, H);
  if ((long long)T * k > (1ll << 30)) return set_error(EK_ERR_INVALID, "%s: too many slots", what);
  return EK_OK;
}

// Base addresses must be aligned to the element.
bool misaligned(int dtype, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % elem_bytes(dtype)) return true;
  return false;
}

struct Rows {  // what the sums take
  const void* rows;
  const int* slot_rows;
  const float* w;
  int T, k, n_rows, H;
  cudaStream_t s;
};

template <class T, int V, bool kWeighted, int kK>
int launch_sum_k(const Rows& a, void* dst) {
  const int nvec = vectors<T, V>(a.H);
  sum_rows_kernel<T, V, kWeighted, kK><<<rows_grid((long long)a.T * runs_per_row<kSumRun<V, kK>>(nvec) * 32), 256, 0, a.s>>>(
      static_cast<const typename Vec<V>::type*>(a.rows), a.slot_rows, a.w, a.T, a.k, a.n_rows, nvec,
      static_cast<typename Vec<V>::type*>(dst));
  return check_cuda(cudaGetLastError(), "sum rows launch");
}

template <class T, int V, bool kWeighted>
int launch_sum(const Rows& a, void* dst) {
  if (a.k <= 2) return launch_sum_k<T, V, kWeighted, 2>(a, dst);
  if (a.k <= 4) return launch_sum_k<T, V, kWeighted, 4>(a, dst);
  return launch_sum_k<T, V, kWeighted, 8>(a, dst);
}

template <class T, bool kWeighted>
int sum_rows(const Rows& a, void* out) {
  switch (vec_bytes((size_t)a.H * sizeof(T), {a.rows, out})) {
    case 16: return launch_sum<T, 16, kWeighted>(a, out);
    case 8: return launch_sum<T, 8, kWeighted>(a, out);
    case 4: return launch_sum<T, 4, kWeighted>(a, out);
    default: return launch_sum<T, (int)sizeof(T), kWeighted>(a, out);
  }
}

template <bool kWeighted>
int sum_rows(const Rows& a, int dtype, void* out) {
  if (dtype == EK_DTYPE_BF16) return sum_rows<__nv_bfloat16, kWeighted>(a, out);
  if (dtype == EK_DTYPE_FP16) return sum_rows<__half, kWeighted>(a, out);
  return sum_rows<float, kWeighted>(a, out);
}

template <class T, int V, int kK>
int launch_combine_grad(const Rows& a, const void* d_out, const int* num_rows, void* d_rows, float* d_w) {
  using Raw = typename Vec<V>::type;
  const int nvec = vectors<T, V>(a.H);
  const auto* rows = static_cast<const Raw*>(a.rows);
  const auto* d = static_cast<const Raw*>(d_out);
  auto* o = static_cast<Raw*>(d_rows);
  // Short rows of many tokens: a warp per token; else a CTA of four, whose lanes
  // each have a vector and which are enough for few tokens too. Measured (bf16),
  // a warp against a CTA: 8192 tokens, 8 choices, 128 wide 9.4 against 24.1 us,
  // 512 wide 26.7 against 41.1, 1024 wide 50.3 against 52.7, 2048 wide 95.4 against
  // 90.5; 64 tokens, 8 choices, 128 wide 3.0 against 2.8, 1024 wide 5.2 against 3.0.
  if (nvec <= 128 && a.T >= 148 * 8)
    combine_grad_kernel<T, V, kK, 32><<<std::max(1, std::min((a.T + 3) / 4, 148 * 64)), 128, 0, a.s>>>(
        rows, a.slot_rows, a.w, d, num_rows, a.T, a.k, a.n_rows, nvec, o, d_w);
  else
    combine_grad_kernel<T, V, kK, 128><<<std::max(1, std::min(a.T, 148 * 64)), 128, 0, a.s>>>(
        rows, a.slot_rows, a.w, d, num_rows, a.T, a.k, a.n_rows, nvec, o, d_w);
  return check_cuda(cudaGetLastError(), "combine gradient launch");
}

template <class T, int V>
int combine_grad_k(const Rows& a, const void* d_out, const int* num_rows, void* d_rows, float* d_w) {
  if (a.k <= 2) return launch_combine_grad<T, V, 2>(a, d_out, num_rows, d_rows, d_w);
  if (a.k <= 4) return launch_combine_grad<T, V, 4>(a, d_out, num_rows, d_rows, d_w);
  return launch_combine_grad<T, V, 8>(a, d_out, num_rows, d_rows, d_w);
}

template <class T>
int combine_grad(const Rows& a, const void* d_out, const int* num_rows, void* d_rows, float* d_w) {
  switch (vec_bytes((size_t)a.H * sizeof(T), {a.rows, d_out, d_rows})) {
    case 16: return combine_grad_k<T, 16>(a, d_out, num_rows, d_rows, d_w);
    case 8: return combine_grad_k<T, 8>(a, d_out, num_rows, d_rows, d_w);
    case 4: return combine_grad_k<T, 4>(a, d_out, num_rows, d_rows, d_w);
    default: return combine_grad_k<T, (int)sizeof(T)>(a, d_out, num_rows, d_rows, d_w);
  }
}

struct Dispatch {
  const int* ids;
  int T, k, E, H;
  const void* x;
  int *sorted_slots, *slot_rows, *counts, *num_rows;
  void* rows;
  cudaStream_t s;
};

template <int V>
int launch_small(const Dispatch& d, size_t row_bytes) {
  using Raw = typename Vec<V>::type;
  const int n = d.T * d.k, nvec = (int)(row_bytes / V);
  const size_t smem = order_smem_ints(n, d.E) * sizeof(int);
  static bool attr_done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    const int rc = check_cuda(cudaFuncSetAttribute(dispatch_small_kernel<V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   order_smem_ints(kOrderThreads, kMaxE) * (int)sizeof(int)),
                              "cudaFuncSetAttribute(dispatch)");
    if (rc) return rc;
    attr_done[dev] = true;
  }
  // the units of the copy over up to a CTA per SM
  const int grid = d.x ? std::max(1, std::min(148, d.T * runs_per_row<kCopyRun<Raw>>(nvec))) : 1;
  dispatch_small_kernel<V><<<grid, kOrderThreads, smem, d.s>>>(d.ids, d.T, d.k, d.E, static_cast<const Raw*>(d.x), nvec,
                                                             d.sorted_slots, d.slot_rows, d.counts, d.num_rows,
                                                             static_cast<Raw*>(d.rows));
  return check_cuda(cudaGetLastError(), "dispatch launch");
}

template <int V>
int launch_copy(const Dispatch& d, size_t row_bytes) {
  using Raw = typename Vec<V>::type;
  const int nvec = (int)(row_bytes / V);
  dispatch_copy_kernel<V><<<rows_grid((long long)d.T * runs_per_row<kCopyRun<Raw>>(nvec) * 32), 256, 0, d.s>>>(
      static_cast<const Raw*>(d.x), d.slot_rows, d.num_rows, d.T, d.k, nvec, static_cast<Raw*>(d.rows));
  return check_cuda(cudaGetLastError(), "dispatch copy launch");
}

}  // namespace
}  // namespace ek

using namespace ek;

extern "C" {

int ek_moe_dispatch(const int* topk_ids, int T, int topk, int E, const void* x, int H, int dtype, int* sorted_slots,
                    int* slot_rows, int* expert_counts, int* num_rows, void* x_rows, void* scratch, void* stream) {
  clear_error();
  if (E < 1 || E > kMaxE) return set_error(EK_ERR_INVALID, "dispatch: need 1 <= E <= %d (got %d)", kMaxE, E);
  int rc = check_rows("dispatch", T, topk, 0, x ? H : 1, x ? dtype : EK_DTYPE_BF16);
  if (rc) return rc;
  if (!expert_counts || !num_rows || !scratch || (T > 0 && (!topk_ids || !sorted_slots || !slot_rows)) ||
      (T > 0 && x && !x_rows))
    return set_error(EK_ERR_INVALID, "dispatch: null pointer");
  if (x && misaligned(dtype, {x, x_rows}))
    return set_error(EK_ERR_INVALID, "dispatch: rows must be aligned to their elements");
  const int n_slots = T * topk;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Dispatch d{topk_ids, T, topk, E, H, x, sorted_slots, slot_rows, expert_counts, num_rows, x_rows, s};
  const size_t row_bytes = x ? (size_t)H * elem_bytes(dtype) : 16;
  const int v = x ? vec_bytes(row_bytes, {x, x_rows}) : 16;
  if (n_slots <= kOrderThreads) {
    if (v == 16) return launch_small<16>(d, row_bytes);
    if (v == 8) return launch_small<8>(d, row_bytes);
    if (v == 4) return launch_small<4>(d, row_bytes);
    return launch_small<2>(d, row_bytes);
  }
  const int n_chunks = (n_slots + kChunk - 1) / kChunk;
  int* chunk_counts = static_cast<int*>(scratch);
  static bool attr_done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    rc = check_cuda(cudaFuncSetAttribute(dispatch_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         32 * kMaxE * (int)sizeof(int)),
                    "cudaFuncSetAttribute(dispatch)");
    if (rc) return rc;
    attr_done[dev] = true;
  }
  dispatch_count_kernel<<<n_chunks, kChunk, 0, s>>>(topk_ids, n_slots, E, chunk_counts);
  dispatch_place_kernel<<<n_chunks, kChunk, 32 * E * sizeof(int), s>>>(topk_ids, n_slots, E, chunk_counts, n_chunks,
                                                                      sorted_slots, slot_rows, expert_counts, num_rows);
  rc = check_cuda(cudaGetLastError(), "dispatch order launch");
  if (rc || !x) return rc;
  if (v == 16) return launch_copy<16>(d, row_bytes);
  if (v == 8) return launch_copy<8>(d, row_bytes);
  if (v == 4) return launch_copy<4>(d, row_bytes);
  return launch_copy<2>(d, row_bytes);
}

int ek_moe_dispatch_grad(const void* d_rows, const int* slot_rows, int T, int topk, int n_rows, int H, int dtype,
                         void* d_x, void* stream) {
  clear_error();
  int rc = check_rows("dispatch gradient", T, topk, n_rows, H, dtype);
  if (rc || T == 0) return rc;
  if (!slot_rows || !d_x || (n_rows > 0 && !d_rows)) return set_error(EK_ERR_INVALID, "dispatch gradient: null pointer");
  if (misaligned(dtype, {d_rows, d_x}))
    return set_error(EK_ERR_INVALID, "dispatch gradient: rows must be aligned to their elements");
  return sum_rows<false>({d_rows, slot_rows, nullptr, T, topk, n_rows, H, static_cast<cudaStream_t>(stream)}, dtype, d_x);
}

int ek_moe_combine_weighted(const void* rows, const int* slot_rows, const float* weights, int T, int topk, int n_rows,
                            int H, int dtype, void* out, void* stream) {
  clear_error();
  int rc = check_rows("weighted combine", T, topk, n_rows, H, dtype);
  if (rc || T == 0) return rc;
  if (!slot_rows || !weights || !out || (n_rows > 0 && !rows))
    return set_error(EK_ERR_INVALID, "weighted combine: null pointer");
  if (misaligned(dtype, {rows, out}))
    return set_error(EK_ERR_INVALID, "weighted combine: rows must be aligned to their elements");
  return sum_rows<true>({rows, slot_rows, weights, T, topk, n_rows, H, static_cast<cudaStream_t>(stream)}, dtype, out);
}

int ek_moe_combine_weighted_grad(const void* rows, const int* slot_rows, const float* weights, const void* d_out,
                                 const int* num_rows, int T, int topk, int n_rows, int H, int dtype, void* d_rows,
                                 float* d_weights, void* stream) {
  clear_error();
  int rc = check_rows("weighted combine gradient", T, topk, n_rows, H, dtype);
  if (rc || T == 0) return rc;
  if (!slot_rows || !weights || !d_out || !num_rows || !d_weights || (n_rows > 0 && (!rows || !d_rows)))
    return set_error(EK_ERR_INVALID, "weighted combine gradient: null pointer");
  if (misaligned(dtype, {rows, d_out, d_rows}))
    return set_error(EK_ERR_INVALID, "weighted combine gradient: rows must be aligned to their elements");
  const Rows a{rows, slot_rows, weights, T, topk, n_rows, H, static_cast<cudaStream_t>(stream)};
  if (dtype == EK_DTYPE_BF16) return combine_grad<__nv_bfloat16>(a, d_out, num_rows, d_rows, d_weights);
  if (dtype == EK_DTYPE_FP16) return combine_grad<__half>(a, d_out, num_rows, d_rows, d_weights);
  return combine_grad<float>(a, d_out, num_rows, d_rows, d_weights);
}

int ek_moe_route_grad(const int* topk_ids, const float* topk_weights, const float* d_weights, int T, int E, int topk,
                      float* d_logits, void* stream) {
  clear_error();
  if (T < 0 || E < 1 || topk < 1) return set_error(EK_ERR_INVALID, "route gradient: bad sizes (T=%d E=%d k=%d)", T, E, topk);
  if (E > (1 << 30)) return set_error(EK_ERR_INVALID, "route gradient: more than 2^30 experts (%d)", E);
  if (T == 0) return EK_OK;
  if (!topk_ids || !topk_weights || !d_weights || !d_logits)
    return set_error(EK_ERR_INVALID, "route gradient: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (topk > 32) {
    route_grad_any_kernel<<<rows_grid((long long)T * 32), 256, 0, s>>>(topk_ids, topk_weights, d_weights, T, E, topk,
                                                                      d_logits);
  } else {
    int kp = 1;
    while (kp < topk) kp *= 2;
    route_grad_kernel<<<rows_grid((long long)T * kp), 256, 0, s>>>(topk_ids, topk_weights, d_weights, T, E, topk, kp,
                                                                  E % 4 == 0 && aligned16(d_logits), d_logits);
  }
  return check_cuda(cudaGetLastError(), "route gradient launch");
}

}  // extern "C"
