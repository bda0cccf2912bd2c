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

// Both directions move 16-byte units of eight elements, lane by lane, so that
// a warp reads and writes whole lines. 14336 x 4096, bf16 (147 MB either way): back
// 34 us, 4.3 TB/s (a thread per element took 200), bound by instructions: issue
// slots 81 % busy, the integer pipe 78. To codes 105 us, bound by instructions too
// (issue slots 85 %, the pipe of the divisions' reciprocals and of the conversions
// 62); it runs once per weight.

// fp32 -> T, saturating at the largest finite value.
template <class T>
__device__ __forceinline__ float round_scale(float v) {
  constexpr float kTop = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;
  return to_f(from_f<T>(fminf(fmaxf(v, -kTop), kTop)));
}

// ------------------------------------------------------------------ quantise
// A warp per run of 256 elements of a row, group / 8 lanes per group. The scale
// and the minimum are rounded to T first and the codes taken against the
// rounded values, so their rounding costs no accuracy; IEEE division and
// round-to-nearest-even define the codes.
template <class W, class T>
__global__ void __launch_bounds__(256)
    quant_w4_kernel(const W* __restrict__ w, long long rows, int K, int group, bool symmetric, bool vec,
                    uint8_t* __restrict__ codes, T* __restrict__ scales, T* __restrict__ mins) {
  const int lane = threadIdx.x & 31;
  const int G = groups(K, group), pitch = pieces(K) * (kPiece / 2), runs = stages(K);
  const long long warps = ((long long)gridDim.x * blockDim.x) >> 5;
  for (long long it = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; it < rows * runs; it += warps) {
    const long long r = it / runs;
    const int k = (int)(it - r * runs) * kStageElems + lane * 8;
    float v[8];
    load_run(w + (size_t)r * K, k, K, vec, v);
    float hi = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) {
        hi = fmaxf(hi, v[i]);
        lo = fminf(lo, v[i]);
      }
    for (int o = group / 16; o; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    float s, m = 0.f;
    if (symmetric) {
      s = round_scale<T>(fmaxf(fabsf(hi), fabsf(lo)) / 7.f);
    } else {
      m = round_scale<T>(lo);
      s = round_scale<T>((hi - m) / 15.f);
    }
    if (!(s > 0.f)) s = 1.f;  // a constant group (or one whose scale underflows T)
    if (k < K && k % group == 0) {
      scales[(size_t)r * G + k / group] = from_f<T>(s);
      if (!symmetric) mins[(size_t)r * G + k / group] = from_f<T>(m);
    }
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float q = symmetric ? 8.f : 0.f;  // past K: the row's padding
      if (k + i < K) q = symmetric ? rintf(v[i] / s) + 8.f : rintf((v[i] - m) / s);
      word |= (uint32_t)fminf(fmaxf(q, 0.f), 15.f) << (4 * i);
    }
    if (k < pieces(K) * kPiece) *reinterpret_cast<uint32_t*>(codes + (size_t)r * pitch + k / 2) = word;
  }
}

// ------------------------------------------------------------------ dequantise
// The weights the codes stand for, rounded once to T; a warp per kDequantRuns
// runs of 256 elements of a row, all their loads in flight.
constexpr int kDequantRuns = 4;
template <class T>
__global__ void __launch_bounds__(256)
    dequant_w4_kernel(const uint8_t* __restrict__ codes, const T* __restrict__ scales, const T* __restrict__ mins,
                      long long rows, int K, int group, bool vec, T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int G = groups(K, group), pitch = pieces(K) * (kPiece / 2);
  const int per = (stages(K) + kDequantRuns - 1) / kDequantRuns, zero = mins ? 0 : 8;
  const long long warps = ((long long)gridDim.x * blockDim.x) >> 5;
  for (long long it = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; it < rows * per; it += warps) {
    const long long r = it / per;
    const int k0 = (int)(it - r * per) * (kDequantRuns * kStageElems) + lane * 8;
    uint32_t word[kDequantRuns];
    float s[kDequantRuns], m[kDequantRuns];
#pragma unroll
    for (int j = 0; j < kDequantRuns; ++j) {
      const int k = k0 + j * kStageElems;
      const size_t at = (size_t)r * G + k / group;
      word[j] = k < K ? __ldg(reinterpret_cast<const uint32_t*>(codes + (size_t)r * pitch + k / 2)) : 0u;
      s[j] = k < K ? to_f(scales[at]) : 0.f;
      m[j] = k < K && mins ? to_f(mins[at]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kDequantRuns; ++j) {
      const int k = k0 + j * kStageElems;
      alignas(16) T v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = from_f<T>(fmaf(s[j], (float)((int)(word[j] >> (4 * i) & 15u) - zero), m[j]));
      T* dst = out + (size_t)r * K + k;
      if (vec && k < K) {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i < K) dst[i] = v[i];
      }
    }
  }
}

template <class W>
int launch_quant(const void* w, long long rows, int K, int group, bool symmetric, int dtype, void* codes, void* scales,
                 void* mins, cudaStream_t stream) {
  const unsigned grid = (unsigned)std::min<long long>((rows * stages(K) + 7) / 8, 148 * 64);
  const W* src = static_cast<const W*>(w);
  const bool vec = K % 8 == 0 && aligned16(w);
  uint8_t* c = static_cast<uint8_t*>(codes);
  if (dtype == EK_DTYPE_BF16)
    quant_w4_kernel<<<grid, 256, 0, stream>>>(src, rows, K, group, symmetric, vec, c, static_cast<__nv_bfloat16*>(scales),
                                              static_cast<__nv_bfloat16*>(mins));
  else
    quant_w4_kernel<<<grid, 256, 0, stream>>>(src, rows, K, group, symmetric, vec, c, static_cast<__half*>(scales),
                                              static_cast<__half*>(mins));
  return check_cuda(cudaGetLastError(), "quant_w4 launch");
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
  int rc = check_w4("quant_w4", codes, scales, mins, 0, K, group);
  if (rc) return rc;
  if (!w || (!symmetric && !mins)) return set_error(EK_ERR_INVALID, "quant_w4: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (w_dtype == EK_DTYPE_BF16) return launch_quant<__nv_bfloat16>(w, rows, K, group, symmetric, dtype, codes, scales, mins, st);
  if (w_dtype == EK_DTYPE_FP16) return launch_quant<__half>(w, rows, K, group, symmetric, dtype, codes, scales, mins, st);
  return launch_quant<float>(w, rows, K, group, symmetric, dtype, codes, scales, mins, st);
}

int ek_dequant_w4(const void* codes, const void* scales, const void* mins, long long rows, int K, int group, int dtype,
                  void* out, void* stream) {
  clear_error();
  if (rows < 0 || (dtype != EK_DTYPE_BF16 && dtype != EK_DTYPE_FP16))
    return set_error(EK_ERR_INVALID, "dequant_w4: bad sizes or type (rows=%lld dtype=%d)", rows, dtype);
  if (rows == 0) return EK_OK;
  int rc = check_w4("dequant_w4", codes, scales, mins, 0, K, group);
  if (rc) return rc;
  if (!out) return set_error(EK_ERR_INVALID, "dequant_w4: null pointer");
  const long long warps = rows * ((stages(K) + kDequantRuns - 1) / kDequantRuns);
  const unsigned grid = (unsigned)std::min<long long>((warps + 7) / 8, 148 * 64);
  const bool vec = K % 8 == 0 && aligned16(out);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == EK_DTYPE_BF16)
    dequant_w4_kernel<<<grid, 256, 0, s>>>(static_cast<const uint8_t*>(codes), static_cast<const __nv_bfloat16*>(scales),
                                           static_cast<const __nv_bfloat16*>(mins), rows, K, group, vec,
                                           static_cast<__nv_bfloat16*>(out));
  else
    dequant_w4_kernel<<<grid, 256, 0, s>>>(static_cast<const uint8_t*>(codes), static_cast<const __half*>(scales),
                                           static_cast<const __half*>(mins), rows, K, group, vec,
                                           static_cast<__half*>(out));
  return check_cuda(cudaGetLastError(), "dequant_w4 launch");
}

}  // extern "C"
