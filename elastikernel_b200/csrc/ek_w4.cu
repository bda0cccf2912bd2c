// 4-bit weights with group scales for sm_100a: to codes and back.
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

#include "ek_w4_launch.cuh"

namespace ek {
namespace {

using namespace w4;

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

}  // namespace
}  // namespace ek

using namespace ek;
using namespace ek::w4;

extern "C" {

int ek_quant_w4(const void* w, int w_dtype, long long rows, int K, int group, int symmetric, int dtype, void* codes,
                void* scales, void* mins, void* stream) {
  clear_error();
  if (rows < 0 || (w_dtype != EK_DTYPE_BF16 && w_dtype != EK_DTYPE_FP16 && w_dtype != EK_DTYPE_FP32) ||
      (dtype != EK_DTYPE_BF16 && dtype != EK_DTYPE_FP16))
    return set_error(EK_ERR_INVALID, "quant_w4: bad sizes or types (rows=%lld w_dtype=%d dtype=%d)", rows, w_dtype, dtype);
  if (rows == 0) return EK_OK;
  int rc = check_w4("quant_w4", codes, scales, mins, K, group);
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
  int rc = check_w4("dequant_w4", codes, scales, mins, K, group);
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

}  // extern "C"
