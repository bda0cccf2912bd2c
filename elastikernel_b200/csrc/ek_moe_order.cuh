// Routing of one token and the expert-major order of a small batch's slots,
// shared by the kernels that start a MoE layer.
#pragma once
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "ek_ptx.cuh"

namespace ek {

constexpr int kRouteMaxE = 256;   // logits per token held in registers: up to 8 per lane
constexpr int kRouteMaxK = 8;

// One token's routing by one warp: logits row -> k expert ids and
// renormalised weights (written by lane 0); kRegs logits per lane, 32 kRegs >= E.
template <int kRegs>
__device__ __forceinline__ void route_token_regs(const float* __restrict__ row, int E, int k, int lane,
                                                 int* __restrict__ ids_out, float* __restrict__ wts_out) {
  float v[kRegs];
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int e = lane + 32 * i;
    v[i] = (e < E) ? row[e] : -INFINITY;
    mx = fmaxf(mx, v[i]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kRegs; ++i)
    if (lane + 32 * i < E) s += expf(v[i] - mx);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);

  // Selection on the logits (softmax is monotone): largest first, ties to the
  // lower expert id.
  uint32_t taken = 0;
  float p[kRouteMaxK];
  int sel[kRouteMaxK];
  float psum = 0.f;
#pragma unroll
  for (int j = 0; j < kRouteMaxK; ++j) {
    if (j >= k) break;
    float bv = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int e = lane + 32 * i;
      if (e < E && !(taken & (1u << i)) && (v[i] > bv || (v[i] == bv && e < bi))) {
        bv = v[i];
        bi = e;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (ov > bv || (ov == bv && oi < bi)) {
        bv = ov;
        bi = oi;
      }
    }
    if ((bi & 31) == lane) taken |= 1u << (bi >> 5);
    sel[j] = bi;
    p[j] = expf(bv - mx) / s;
    psum += p[j];
  }
  if (lane == 0) {
#pragma unroll
    for (int j = 0; j < kRouteMaxK; ++j) {
      if (j >= k) break;
      ids_out[j] = sel[j];
      wts_out[j] = p[j] / psum;
    }
  }
}

__device__ __forceinline__ void route_token(const float* __restrict__ row, int E, int k, int lane,
                                            int* __restrict__ ids_out, float* __restrict__ wts_out) {
  if (E <= 32) route_token_regs<1>(row, E, k, lane, ids_out, wts_out);
  else if (E <= 64) route_token_regs<2>(row, E, k, lane, ids_out, wts_out);
  else route_token_regs<kRouteMaxE / 32>(row, E, k, lane, ids_out, wts_out);
}

// ------------------------------------------------------------------ order
constexpr int kOrderThreads = 1024;  // also the slots one CTA orders
constexpr int kOrderMaxE = 1024;
// Shared memory of order_slots: the warps' counts of each expert, the experts'
// first rows, 33 ints of scan.
__host__ __device__ inline int order_smem_ints(int n, int E) { return ((n + 31) / 32 + 1) * E + 34; }

// Order n <= kOrderThreads slots stably by expert in one CTA (kOrderThreads
// threads, thread s holds id of slot s, negative: dropped). Returns the row of
// this thread's slot (-1: dropped or none); *kept = the rows in all, and after
// the call sm[(n + 31) / 32 * E + e] is the first row of expert e. sm: as
// order_smem_ints.
__device__ __forceinline__ int order_slots(int id, int n, int E, int* sm, int* kept) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = (n + 31) / 32;
  int *s_start = sm + warps * E, *s_scan = s_start + E;
  for (int i = tid; i < warps * E; i += kOrderThreads) sm[i] = 0;
  __syncthreads();
  int rank = 0;
  if (warp < warps) {
    const unsigned peers = __match_any_sync(0xffffffffu, id);
    rank = __popc(peers & ((1u << lane) - 1u));
    if (id >= 0 && rank == 0) sm[warp * E + id] = __popc(peers);
  }
  __syncthreads();
  // thread e: the warps' counts of expert e become its slots in earlier warps
  int total = 0;
  if (tid < E)
    for (int w = 0; w < warps; ++w) {
      const int c = sm[w * E + tid];
      sm[w * E + tid] = total;
      total += c;
    }
  int incl = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int w = s_scan[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += v;
    }
    s_scan[lane] = w;
  }
  __syncthreads();
  if (tid < E) s_start[tid] = (warp ? s_scan[warp - 1] : 0) + incl - total;
  *kept = s_scan[31];
  __syncthreads();
  return id >= 0 ? s_start[id] + sm[warp * E + id] + rank : -1;
}

}  // namespace ek
