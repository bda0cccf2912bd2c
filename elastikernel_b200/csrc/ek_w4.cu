// Products with 4-bit weights and group scales for sm_100a.
//
// A weight row of K elements is stored as ceil(K / 32) * 16 bytes of codes, two
// per byte, the even element in the low nibble (codes past K are ignored),
// and per `group` consecutive elements (32, 64 or 128) a 16-bit scale s and,
// for asymmetric weights, a 16-bit minimum m:
//   w = s (q - 8)        without minima
//   w = s q + m          with them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "ek_internal.h"

namespace ek {
namespace {

constexpr int kPiece = 32;  // elements per 16-byte piece of a code row; divides every group

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

__host__ __device__ inline int pieces(int K) { return (K + kPiece - 1) / kPiece; }
__host__ __device__ inline int groups(int K, int group) { return (K + group - 1) / group; }

// ------------------------------------------------------------------ quantise
__device__ __forceinline__ float load_f(const void* w, int dt, size_t i) {
  if (dt == EK_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  if (dt == EK_DTYPE_FP16) return __half2float(static_cast<const __half*>(w)[i]);
  return static_cast<const float*>(w)[i];
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// fp32 -> T, saturating at the largest finite value.
template <class T>
__device__ __forceinline__ float round_scale(float v) {
  constexpr float kTop = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;
  return to_f(from_f<T>(fminf(fmaxf(v, -kTop), kTop)));
}

// One warp per group of a row. The scale and the minimum are rounded to T
// first and the codes taken against the rounded values, so their rounding
// costs no accuracy; IEEE division and round-to-nearest-even define the codes.
template <class T>
__global__ void __launch_bounds__(256)
    quant_w4_kernel(const void* __restrict__ w, int w_dtype, long long rows, int K, int group, int symmetric,
                    uint8_t* __restrict__ codes, T* __restrict__ scales, T* __restrict__ mins) {
  const int lane = threadIdx.x & 31;
  const int G = groups(K, group), pitch = pieces(K) * (kPiece / 2);
  const long long warps = ((long long)gridDim.x * blockDim.x) >> 5;
  for (long long it = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; it < rows * G; it += warps) {
    const long long r = it / G;
    const int g = (int)(it - r * G);
    const int k0 = g * group, k1 = min(K, k0 + group);
    float hi = -INFINITY, lo = INFINITY;
    for (int c = k0 + lane; c < k1; c += 32) {
      const float v = load_f(w, w_dtype, (size_t)r * K + c);
      hi = fmaxf(hi, v);
      lo = fminf(lo, v);
    }
    hi = warp_max(hi);
    lo = -warp_max(-lo);
    float s, m = 0.f;
    if (symmetric) {
      s = round_scale<T>(fmaxf(fabsf(hi), fabsf(lo)) / 7.f);
    } else {
      m = round_scale<T>(lo);
      s = round_scale<T>((hi - m) / 15.f);
    }
    if (!(s > 0.f)) s = 1.f;  // a constant group (or one whose scale underflows T)
    if (lane == 0) {
      scales[it] = from_f<T>(s);
      if (!symmetric) mins[it] = from_f<T>(m);
    }
    const int pad1 = min(pieces(K) * kPiece, k0 + group);  // the last group also writes the row's padding
    for (int c = k0 + 2 * lane; c < pad1; c += 64) {
      uint32_t q[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = symmetric ? 8.f : 0.f;
        if (c + i < k1) {
          const float x = load_f(w, w_dtype, (size_t)r * K + c + i);
          v = symmetric ? rintf(x / s) + 8.f : rintf((x - m) / s);
        }
        q[i] = (uint32_t)fminf(fmaxf(v, 0.f), 15.f);
      }
      codes[(size_t)r * pitch + c / 2] = (uint8_t)(q[0] | (q[1] << 4));
    }
  }
}

template <class T>
__device__ __forceinline__ float code_value(int q, float s, const T* mins, size_t at) {
  return mins ? fmaf(s, (float)q, to_f(mins[at])) : s * (float)(q - 8);
}

// The weights the codes stand for, rounded once to T.
template <class T>
__global__ void __launch_bounds__(256)
    dequant_w4_kernel(const uint8_t* __restrict__ codes, const T* __restrict__ scales, const T* __restrict__ mins,
                      long long rows, int K, int group, T* __restrict__ out) {
  const int G = groups(K, group), pitch = pieces(K) * (kPiece / 2);
  const long long n = rows * K;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    const long long r = i / K;
    const int c = (int)(i - r * K);
    const int b = codes[(size_t)r * pitch + c / 2];
    const size_t at = (size_t)r * G + c / group;
    out[i] = from_f<T>(code_value(c & 1 ? b >> 4 : b & 15, to_f(scales[at]), mins, at));
  }
}

// ------------------------------------------------------------------ products
template <class T>
struct W4 {
  const uint8_t* codes;
  const T* scales;
  const T* mins;
  int K, group;
};

constexpr int kTok = 8;  // token rows per pass over a weight row

// One warp: the products of weight row `row` with `m` token rows (m <= kTok);
// x_of(i) is token i's row. The sums run over each piece in fp32, are scaled
// by the group and added across the lanes; every lane returns all of them.
template <class T, class RowOf>
__device__ __forceinline__ void dot_row(const W4<T>& w, long long row, int m, RowOf x_of, float (&acc)[kTok]) {
  const int lane = threadIdx.x & 31;
  const int np = pieces(w.K), G = groups(w.K, w.group);
#pragma unroll
  for (int i = 0; i < kTok; ++i) acc[i] = 0.f;
  for (int p = lane; p < np; p += 32) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(w.codes + ((size_t)row * np + p) * (kPiece / 2)));
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    const size_t at = (size_t)row * G + p * kPiece / w.group;
    const float s = to_f(w.scales[at]);
    const float mn = w.mins ? to_f(w.mins[at]) : 0.f;
    const int kn = min(kPiece, w.K - p * kPiece);
    for (int i = 0; i < m; ++i) {
      const T* x = x_of(i) + p * kPiece;
      float d = 0.f, sx = 0.f;
      for (int k = 0; k < kn; ++k) {
        const int q = (words[k >> 3] >> ((k & 7) * 4)) & 15;
        const float v = to_f(x[k]);
        d += v * (float)(w.mins ? q : q - 8);
        sx += v;
      }
      acc[i] += w.mins ? s * d + mn * sx : s * d;
    }
  }
#pragma unroll
  for (int i = 0; i < kTok; ++i)
#pragma unroll
    for (int o = 16; o; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
}

// C[m, n] = <x[m], w[n]>; one warp per weight row and kTok tokens.
template <class T>
__global__ void __launch_bounds__(256)
    gemm_w4_kernel(const T* __restrict__ x, W4<T> w, T* __restrict__ out, int M, int N) {
  const int lane = threadIdx.x & 31;
  const long long mt = (M + kTok - 1) / kTok;
  const long long u = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (u >= mt * N) return;
  const int n = (int)(u / mt), m0 = (int)(u - (long long)n * mt) * kTok;
  const int m = min(kTok, M - m0);
  float acc[kTok];
  dot_row(w, n, m, [&](int i) { return x + (size_t)(m0 + i) * w.K; }, acc);
#pragma unroll
  for (int i = 0; i < kTok; ++i)
    if (lane == i && i < m) out[(size_t)(m0 + i) * N + n] = from_f<T>(acc[i]);
}

// Expert of packed row r (-1 past the last routed row).
__device__ __forceinline__ int expert_of(const int* __restrict__ counts, int E, int r) {
  int end = 0;
  for (int e = 0; e < E; ++e) {
    end += max(0, __ldg(counts + e));
    if (r < end) return e;
  }
  return -1;
}

// act[r, n] = silu(<x, w1[e, n]>) * <x, w3[e, n]>, x the token of row r.
__global__ void __launch_bounds__(256)
    moe_gate_up_w4_kernel(const __nv_bfloat16* __restrict__ x, const int* __restrict__ sorted_slots, int topk,
                          int n_slots, W4<__nv_bfloat16> w1, W4<__nv_bfloat16> w3, const int* __restrict__ counts,
                          __nv_bfloat16* __restrict__ act, int rows, int E, int I) {
  const int lane = threadIdx.x & 31;
  const long long u = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (u >= (long long)rows * I) return;
  const int r = (int)(u / I), n = (int)(u - (long long)r * I);
  const int e = expert_of(counts, E, r);
  if (e < 0) return;
  long long xr = r;
  if (sorted_slots) {
    const int s = sorted_slots[r];
    if (s < 0 || s >= n_slots) return;
    xr = s / topk;
  }
  auto row = [&](int) { return x + (size_t)xr * w1.K; };
  float g[kTok], up[kTok];
  dot_row(w1, (long long)e * I + n, 1, row, g);
  dot_row(w3, (long long)e * I + n, 1, row, up);
  if (lane == 0) act[(size_t)r * I + n] = __float2bfloat16_rn(g[0] / (1.f + expf(-g[0])) * up[0]);
}

// y[r, n] = <act[r], w2[e, n]>.
__global__ void __launch_bounds__(256)
    moe_down_w4_kernel(const __nv_bfloat16* __restrict__ act, W4<__nv_bfloat16> w2, const int* __restrict__ counts,
                       __nv_bfloat16* __restrict__ y, int rows, int E, int H) {
  const int lane = threadIdx.x & 31;
  const long long u = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (u >= (long long)rows * H) return;
  const int r = (int)(u / H), n = (int)(u - (long long)r * H);
  const int e = expert_of(counts, E, r);
  if (e < 0) return;
  float acc[kTok];
  dot_row(w2, (long long)e * H + n, 1, [&](int) { return act + (size_t)r * w2.K; }, acc);
  if (lane == 0) y[(size_t)r * H + n] = __float2bfloat16_rn(acc[0]);
}

// ------------------------------------------------------------------ checks
int check_w4(const char* what, const void* codes, const void* scales, int K, int group) {
  if (K < 1 || (group != 32 && group != 64 && group != 128))
    return set_error(EK_ERR_INVALID, "%s: need K >= 1 and a group of 32, 64 or 128 (K=%d group=%d)", what, K, group);
  if (!codes || !scales) return set_error(EK_ERR_INVALID, "%s: null pointer", what);
  if (!aligned16(codes)) return set_error(EK_ERR_INVALID, "%s: codes must be 16-byte aligned", what);
  if (reinterpret_cast<uintptr_t>(scales) & 1u) return set_error(EK_ERR_INVALID, "%s: misaligned scales", what);
  return EK_OK;
}

template <class T>
W4<T> make_w4(const void* codes, const void* scales, const void* mins, int K, int group) {
  return {static_cast<const uint8_t*>(codes), static_cast<const T*>(scales), static_cast<const T*>(mins), K, group};
}

// Warps -> CTAs of 8 warps; the grid dimension holds 2^31 - 1 CTAs.
int warp_blocks(long long warps, unsigned* blocks) {
  const long long b = (warps + 7) / 8;
  if (b > 0x7fffffffll) return set_error(EK_ERR_INVALID, "4-bit products: too many outputs");
  *blocks = (unsigned)std::max<long long>(1, b);
  return EK_OK;
}

}  // namespace
}  // namespace ek

using namespace ek;

extern "C" {

int ek_quant_w4(const void* w, int w_dtype, long long rows, int K, int group, int symmetric, int dtype, void* codes,
                void* scales, void* mins, void* stream) {
  clear_error();
  if (rows < 0 || (w_dtype != EK_DTYPE_BF16 && w_dtype != EK_DTYPE_FP16 && w_dtype != EK_DTYPE_FP32) ||
      (dtype != EK_DTYPE_BF16 && dtype != EK_DTYPE_FP16))
    return set_error(EK_ERR_INVALID, "quant_w4: bad sizes or types (rows=%lld w_dtype=%d dtype=%d)", rows, w_dtype, dtype);
  if (rows == 0) return EK_OK;
  int rc = check_w4("quant_w4", codes, scales, K, group);
  if (rc) return rc;
  if (!w || (!symmetric && !mins)) return set_error(EK_ERR_INVALID, "quant_w4: null pointer");
  const unsigned grid = (unsigned)std::min<long long>((rows * groups(K, group) + 7) / 8, 148 * 64);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == EK_DTYPE_BF16)
    quant_w4_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(w, w_dtype, rows, K, group, symmetric,
                                                       static_cast<uint8_t*>(codes), static_cast<__nv_bfloat16*>(scales),
                                                       static_cast<__nv_bfloat16*>(mins));
  else
    quant_w4_kernel<__half><<<grid, 256, 0, s>>>(w, w_dtype, rows, K, group, symmetric, static_cast<uint8_t*>(codes),
                                                static_cast<__half*>(scales), static_cast<__half*>(mins));
  return check_cuda(cudaGetLastError(), "quant_w4 launch");
}

int ek_dequant_w4(const void* codes, const void* scales, const void* mins, long long rows, int K, int group, int dtype,
                  void* out, void* stream) {
  clear_error();
  if (rows < 0 || (dtype != EK_DTYPE_BF16 && dtype != EK_DTYPE_FP16))
    return set_error(EK_ERR_INVALID, "dequant_w4: bad sizes or type (rows=%lld dtype=%d)", rows, dtype);
  if (rows == 0) return EK_OK;
  int rc = check_w4("dequant_w4", codes, scales, K, group);
  if (rc) return rc;
  if (!out) return set_error(EK_ERR_INVALID, "dequant_w4: null pointer");
  const unsigned grid = (unsigned)std::min<long long>((rows * K + 255) / 256, 148 * 64);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == EK_DTYPE_BF16)
    dequant_w4_kernel<<<grid, 256, 0, s>>>(static_cast<const uint8_t*>(codes), static_cast<const __nv_bfloat16*>(scales),
                                           static_cast<const __nv_bfloat16*>(mins), rows, K, group,
                                           static_cast<__nv_bfloat16*>(out));
  else
    dequant_w4_kernel<<<grid, 256, 0, s>>>(static_cast<const uint8_t*>(codes), static_cast<const __half*>(scales),
                                           static_cast<const __half*>(mins), rows, K, group, static_cast<__half*>(out));
  return check_cuda(cudaGetLastError(), "dequant_w4 launch");
}

int ek_gemm_w4(const void* A, const void* codes, const void* scales, const void* mins, void* C, int M, int N, int K,
               int group, int dtype, int num_sms, void* stream) {
  clear_error();
  if (M < 0 || N < 0 || (dtype != EK_DTYPE_BF16 && dtype != EK_DTYPE_FP16))
    return set_error(EK_ERR_INVALID, "gemm_w4: bad sizes or type (M=%d N=%d dtype=%d)", M, N, dtype);
  if (M == 0 || N == 0) return EK_OK;
  int rc = check_w4("gemm_w4", codes, scales, K, group);
  if (rc) return rc;
  if (!A || !C) return set_error(EK_ERR_INVALID, "gemm_w4: null pointer");
  unsigned blocks = 0;
  rc = warp_blocks((long long)((M + kTok - 1) / kTok) * N, &blocks);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == EK_DTYPE_BF16)
    gemm_w4_kernel<<<blocks, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(A),
                                          make_w4<__nv_bfloat16>(codes, scales, mins, K, group),
                                          static_cast<__nv_bfloat16*>(C), M, N);
  else
    gemm_w4_kernel<<<blocks, 256, 0, s>>>(static_cast<const __half*>(A), make_w4<__half>(codes, scales, mins, K, group),
                                          static_cast<__half*>(C), M, N);
  return check_cuda(cudaGetLastError(), "gemm_w4 launch");
}

int ek_moe_gate_up_w4(const void* x, const int* sorted_slots, int topk, int n_slots, const void* w1_codes,
                      const void* w1_scales, const void* w1_mins, const void* w3_codes, const void* w3_scales,
                      const void* w3_mins, const int* expert_counts, void* act, int rows, int E, int H, int I,
                      int group, int num_sms, void* stream) {
  clear_error();
  if (rows < 0 || E < 1 || I < 1 || (sorted_slots && (topk < 1 || n_slots < 0)))
    return set_error(EK_ERR_INVALID, "gate_up_w4: bad sizes (rows=%d E=%d I=%d topk=%d)", rows, E, I, topk);
  if (rows == 0) return EK_OK;
  int rc = check_w4("gate_up_w4", w1_codes, w1_scales, H, group);
  if (!rc) rc = check_w4("gate_up_w4", w3_codes, w3_scales, H, group);
  if (rc) return rc;
  if (!x || !expert_counts || !act || !w1_mins != !w3_mins) return set_error(EK_ERR_INVALID, "gate_up_w4: null pointer");
  unsigned blocks = 0;
  rc = warp_blocks((long long)rows * I, &blocks);
  if (rc) return rc;
  moe_gate_up_w4_kernel<<<blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(x), sorted_slots, topk, n_slots,
      make_w4<__nv_bfloat16>(w1_codes, w1_scales, w1_mins, H, group),
      make_w4<__nv_bfloat16>(w3_codes, w3_scales, w3_mins, H, group), expert_counts, static_cast<__nv_bfloat16*>(act),
      rows, E, I);
  return check_cuda(cudaGetLastError(), "gate_up_w4 launch");
}

int ek_moe_down_w4(const void* act, const void* w2_codes, const void* w2_scales, const void* w2_mins,
                   const int* expert_counts, void* y, int rows, int E, int H, int I, int group, int num_sms,
                   void* stream) {
  clear_error();
  if (rows < 0 || E < 1 || H < 1) return set_error(EK_ERR_INVALID, "down_w4: bad sizes (rows=%d E=%d H=%d)", rows, E, H);
  if (rows == 0) return EK_OK;
  int rc = check_w4("down_w4", w2_codes, w2_scales, I, group);
  if (rc) return rc;
  if (!act || !expert_counts || !y) return set_error(EK_ERR_INVALID, "down_w4: null pointer");
  unsigned blocks = 0;
  rc = warp_blocks((long long)rows * H, &blocks);
  if (rc) return rc;
  moe_down_w4_kernel<<<blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(act), make_w4<__nv_bfloat16>(w2_codes, w2_scales, w2_mins, I, group),
      expert_counts, static_cast<__nv_bfloat16*>(y), rows, E, H);
  return check_cuda(cudaGetLastError(), "down_w4 launch");
}

}  // extern "C"
