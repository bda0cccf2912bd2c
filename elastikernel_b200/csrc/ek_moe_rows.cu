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
// All of it is data movement: the token side of each copy (T rows) is read or
// written once and kept in registers across the token's k slots, so the bytes
// are T rows plus T*k rows, whatever k. Slots with a negative expert id are
// dropped: they have no row, weigh nothing and get no gradient; the rows past
// the last kept one are zero.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "ek_internal.h"
#include "ek_ptx.cuh"

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

constexpr int kChunk = 1024;  // slots per sorting CTA, one per thread
constexpr int kMaxE = 1024;

// ------------------------------------------------------------------ dispatch: the order
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
  __shared__ int s_wsum[32];
  __shared__ int s_total;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunk = blockIdx.x;
  int total = 0, before = 0;
  if (tid < E) {
    for (int c = 0; c < n_chunks; ++c) {
      const int v = __ldg(chunk_counts + (size_t)c * E + tid);
      total += v;
      if (c < chunk) before += v;
    }
  }
  for (int i = tid; i < 32 * E; i += kChunk) s_wcnt[i] = 0;
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

// Zero the rows past the last kept one ([*num_rows, n_rows)).
template <class Raw>
__device__ __forceinline__ void zero_tail(Raw* __restrict__ rows, const int* __restrict__ num_rows, int n_rows,
                                          int nvec) {
  const long long first = (long long)max(0, min(*num_rows, n_rows)) * nvec, end = (long long)n_rows * nvec;
  for (long long i = first + (long long)blockIdx.x * blockDim.x + threadIdx.x; i < end;
       i += (long long)gridDim.x * blockDim.x)
    rows[i] = Raw{};
}

// rows[slot_rows[t*k + j]] = x[t] for the kept slots of each token. A thread
// takes one vector of a token and stores it to the token's k rows.
template <int V>
__global__ void __launch_bounds__(256)
    dispatch_copy_kernel(const typename Vec<V>::type* __restrict__ x, const int* __restrict__ slot_rows,
                         const int* __restrict__ num_rows, int T, int k, int nvec,
                         typename Vec<V>::type* __restrict__ rows) {
  using Raw = typename Vec<V>::type;
  const long long items = (long long)T * nvec;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < items;
       i += (long long)gridDim.x * blockDim.x) {
    const int t = (int)(i / nvec), c = (int)(i - (long long)t * nvec);
    const Raw v = x[i];
    for (int j = 0; j < k; ++j) {
      const int r = __ldg(slot_rows + (long long)t * k + j);
      if (r >= 0) rows[(long long)r * nvec + c] = v;
    }
  }
  zero_tail(rows, num_rows, T * k, nvec);
}

// out[t] = sum_j w[t,j] rows[slot_rows[t,j]] (w = 1 without weights), fp32 sum
// in j order, rounded once to T.
template <class T, int V, bool kWeighted>
__global__ void __launch_bounds__(256)
    sum_rows_kernel(const typename Vec<V>::type* __restrict__ rows, const int* __restrict__ slot_rows,
                    const float* __restrict__ weights, int T_tokens, int k, int n_rows, int nvec,
                    typename Vec<V>::type* __restrict__ out) {
  using E = Elems<T, V>;
  const long long items = (long long)T_tokens * nvec;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < items;
       i += (long long)gridDim.x * blockDim.x) {
    const int t = (int)(i / nvec), c = (int)(i - (long long)t * nvec);
    float acc[E::N] = {};
    for (int j = 0; j < k; ++j) {
      const int r = __ldg(slot_rows + (long long)t * k + j);
      if (r < 0 || r >= n_rows) continue;
      const float w = kWeighted ? __ldg(weights + (long long)t * k + j) : 1.f;
      float f[E::N];
      E::unpack(rows[(long long)r * nvec + c], f);
#pragma unroll
      for (int e = 0; e < E::N; ++e) acc[e] += w * f[e];
    }
    out[i] = E::pack(acc);
  }
}

// d_rows[r] = w[s] d_out[t] and d_weights[s] = <d_out[t], rows[r]> (fp32), one
// CTA per token.
template <class T, int V>
__global__ void __launch_bounds__(256)
    combine_grad_kernel(const typename Vec<V>::type* __restrict__ rows, const int* __restrict__ slot_rows,
                        const float* __restrict__ weights, const typename Vec<V>::type* __restrict__ d_out,
                        const int* __restrict__ num_rows, int T_tokens, int k, int n_rows, int nvec,
                        typename Vec<V>::type* __restrict__ d_rows, float* __restrict__ d_weights) {
  using E = Elems<T, V>;
  __shared__ float s_red[8];
  for (int t = blockIdx.x; t < T_tokens; t += gridDim.x) {
    for (int j = 0; j < k; ++j) {
      const long long s = (long long)t * k + j;
      const int r = __ldg(slot_rows + s);
      const bool live = r >= 0 && r < n_rows;
      float dot = 0.f;
      if (live) {
        const float w = __ldg(weights + s);
        for (int c = threadIdx.x; c < nvec; c += blockDim.x) {
          float d[E::N], y[E::N];
          E::unpack(d_out[(long long)t * nvec + c], d);
          E::unpack(rows[(long long)r * nvec + c], y);
#pragma unroll
          for (int e = 0; e < E::N; ++e) {
            dot += d[e] * y[e];
            d[e] *= w;
          }
          d_rows[(long long)r * nvec + c] = E::pack(d);
        }
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = dot;
      __syncthreads();
      if (threadIdx.x == 0) {
        float sum = 0.f;
        for (int w = 0; w < 8; ++w) sum += s_red[w];
        d_weights[s] = live ? sum : 0.f;
      }
      __syncthreads();
    }
  }
  zero_tail(d_rows, num_rows, n_rows, nvec);
}

// ------------------------------------------------------------------ route gradient
// The renormalised weights are the softmax of the chosen logits alone, so
// d_logit[ids_j] += w_j (dw_j - sum_i w_i dw_i) and every other logit gets 0.
__global__ void __launch_bounds__(256)
    route_grad_kernel(const int* __restrict__ ids, const float* __restrict__ weights,
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
  if ((long long)T * k > (1ll << 30)) return set_error(EK_ERR_INVALID, "%s: too many slots", what);
  return EK_OK;
}

// Base addresses must be aligned to the element.
bool misaligned(int dtype, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % elem_bytes(dtype)) return true;
  return false;
}

template <class T, int V, bool kWeighted>
int launch_sum(const void* rows, const int* slot_rows, const float* w, int Tt, int k, int n_rows, int H, void* out,
               cudaStream_t s) {
  using Raw = typename Vec<V>::type;
  const int nvec = H * (int)sizeof(T) / V;
  sum_rows_kernel<T, V, kWeighted><<<rows_grid((long long)Tt * nvec), 256, 0, s>>>(
      static_cast<const Raw*>(rows), slot_rows, w, Tt, k, n_rows, nvec, static_cast<Raw*>(out));
  return check_cuda(cudaGetLastError(), "sum rows launch");
}

template <class T, bool kWeighted>
int sum_vec(int v, const void* rows, const int* slot_rows, const float* w, int Tt, int k, int n_rows, int H, void* out,
            cudaStream_t s) {
  if (v == 16) return launch_sum<T, 16, kWeighted>(rows, slot_rows, w, Tt, k, n_rows, H, out, s);
  if (v == 8) return launch_sum<T, 8, kWeighted>(rows, slot_rows, w, Tt, k, n_rows, H, out, s);
  if (v == 4) return launch_sum<T, 4, kWeighted>(rows, slot_rows, w, Tt, k, n_rows, H, out, s);
  return launch_sum<T, (int)sizeof(T), kWeighted>(rows, slot_rows, w, Tt, k, n_rows, H, out, s);
}

template <bool kWeighted>
int sum_rows(const void* rows, const int* slot_rows, const float* w, int Tt, int k, int n_rows, int H, int dtype,
             void* out, cudaStream_t s) {
  const int v = vec_bytes((size_t)H * elem_bytes(dtype), {rows, out});
  if (dtype == EK_DTYPE_BF16) return sum_vec<__nv_bfloat16, kWeighted>(v, rows, slot_rows, w, Tt, k, n_rows, H, out, s);
  if (dtype == EK_DTYPE_FP16) return sum_vec<__half, kWeighted>(v, rows, slot_rows, w, Tt, k, n_rows, H, out, s);
  return sum_vec<float, kWeighted>(v, rows, slot_rows, w, Tt, k, n_rows, H, out, s);
}

template <class T, int V>
int launch_combine_grad(const void* rows, const int* slot_rows, const float* w, const void* d_out, const int* num_rows,
                        int Tt, int k, int n_rows, int H, void* d_rows, float* d_w, cudaStream_t s) {
  using Raw = typename Vec<V>::type;
  const int nvec = H * (int)sizeof(T) / V;
  combine_grad_kernel<T, V><<<std::max(1, std::min(Tt, 148 * 64)), 256, 0, s>>>(
      static_cast<const Raw*>(rows), slot_rows, w, static_cast<const Raw*>(d_out), num_rows, Tt, k, n_rows, nvec,
      static_cast<Raw*>(d_rows), d_w);
  return check_cuda(cudaGetLastError(), "combine gradient launch");
}

template <class T>
int combine_grad_vec(int v, const void* rows, const int* slot_rows, const float* w, const void* d_out,
                     const int* num_rows, int Tt, int k, int n_rows, int H, void* d_rows, float* d_w, cudaStream_t s) {
  if (v == 16) return launch_combine_grad<T, 16>(rows, slot_rows, w, d_out, num_rows, Tt, k, n_rows, H, d_rows, d_w, s);
  if (v == 8) return launch_combine_grad<T, 8>(rows, slot_rows, w, d_out, num_rows, Tt, k, n_rows, H, d_rows, d_w, s);
  if (v == 4) return launch_combine_grad<T, 4>(rows, slot_rows, w, d_out, num_rows, Tt, k, n_rows, H, d_rows, d_w, s);
  return launch_combine_grad<T, (int)sizeof(T)>(rows, slot_rows, w, d_out, num_rows, Tt, k, n_rows, H, d_rows, d_w, s);
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
  const int n_chunks = std::max((n_slots + kChunk - 1) / kChunk, 1);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
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
  if (rc || !x || T == 0) return rc;
  const size_t row_bytes = (size_t)H * elem_bytes(dtype);
  const int v = vec_bytes(row_bytes, {x, x_rows});
  const int nvec = (int)(row_bytes / v);
  const int grid = rows_grid((long long)T * nvec);
  switch (v) {
    case 16:
      dispatch_copy_kernel<16><<<grid, 256, 0, s>>>(static_cast<const uint4*>(x), slot_rows, num_rows, T, topk, nvec,
                                                    static_cast<uint4*>(x_rows));
      break;
    case 8:
      dispatch_copy_kernel<8><<<grid, 256, 0, s>>>(static_cast<const uint2*>(x), slot_rows, num_rows, T, topk, nvec,
                                                   static_cast<uint2*>(x_rows));
      break;
    case 4:
      dispatch_copy_kernel<4><<<grid, 256, 0, s>>>(static_cast<const uint32_t*>(x), slot_rows, num_rows, T, topk, nvec,
                                                   static_cast<uint32_t*>(x_rows));
      break;
    default:
      dispatch_copy_kernel<2><<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(x), slot_rows, num_rows, T, topk, nvec,
                                                   static_cast<uint16_t*>(x_rows));
  }
  return check_cuda(cudaGetLastError(), "dispatch copy launch");
}

int ek_moe_dispatch_grad(const void* d_rows, const int* slot_rows, int T, int topk, int n_rows, int H, int dtype,
                         void* d_x, void* stream) {
  clear_error();
  int rc = check_rows("dispatch gradient", T, topk, n_rows, H, dtype);
  if (rc || T == 0) return rc;
  if (!slot_rows || !d_x || (n_rows > 0 && !d_rows)) return set_error(EK_ERR_INVALID, "dispatch gradient: null pointer");
  if (misaligned(dtype, {d_rows, d_x}))
    return set_error(EK_ERR_INVALID, "dispatch gradient: rows must be aligned to their elements");
  return sum_rows<false>(d_rows, slot_rows, nullptr, T, topk, n_rows, H, dtype, d_x, static_cast<cudaStream_t>(stream));
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
  return sum_rows<true>(rows, slot_rows, weights, T, topk, n_rows, H, dtype, out, static_cast<cudaStream_t>(stream));
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
  const int v = vec_bytes((size_t)H * elem_bytes(dtype), {rows, d_out, d_rows});
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == EK_DTYPE_BF16)
    return combine_grad_vec<__nv_bfloat16>(v, rows, slot_rows, weights, d_out, num_rows, T, topk, n_rows, H, d_rows,
                                           d_weights, s);
  if (dtype == EK_DTYPE_FP16)
    return combine_grad_vec<__half>(v, rows, slot_rows, weights, d_out, num_rows, T, topk, n_rows, H, d_rows, d_weights,
                                    s);
  return combine_grad_vec<float>(v, rows, slot_rows, weights, d_out, num_rows, T, topk, n_rows, H, d_rows, d_weights, s);
}

int ek_moe_route_grad(const int* topk_ids, const float* topk_weights, const float* d_weights, int T, int E, int topk,
                      float* d_logits, void* stream) {
  clear_error();
  if (T < 0 || E < 1 || topk < 1) return set_error(EK_ERR_INVALID, "route gradient: bad sizes (T=%d E=%d k=%d)", T, E, topk);
  if (T == 0) return EK_OK;
  if (!topk_ids || !topk_weights || !d_weights || !d_logits)
    return set_error(EK_ERR_INVALID, "route gradient: null pointer");
  route_grad_kernel<<<rows_grid((long long)T * 32), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      topk_ids, topk_weights, d_weights, T, E, topk, d_logits);
  return check_cuda(cudaGetLastError(), "route gradient launch");
}

}  // extern "C"
