// Launches of the 4-bit-weight kernels, shared by the dense product and the
// experts' products.
#pragma once
#include "ek_w4_kernel.cuh"

namespace ek {
namespace w4 {

// ------------------------------------------------------------------ launches
// One launch that may begin before its predecessor on the stream has ended (the
// kernels above wait for it themselves), or, with after = true, not.
template <class... P, class... A>
int launch(const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, bool after,
           A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after ? 0 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

// Blocks of 8 tokens per tile, 1 or 2, for `rows` token rows over `experts`
// weight matrices: to hold the mean and two standard deviations of an even
// spread, so that few experts need a second tile (which reads the codes again,
// from L2). Measured, the gate/up product of 32 experts of 7168 x 2048 with 8
// choices: 16 tokens 93 us with one block and 97 with two, 32 tokens 131 and 128,
// 64 tokens 214 and 184, 128 tokens 373 and 278; tiles of 24 and 32 tokens took
// 195 and 253 at 64 tokens (their accumulators leave fewer warps).
inline int pick_nt(long long rows, int experts) {
  const double used = (double)std::max<long long>(1, std::min<long long>(experts, rows));
  const double mean = rows / used, want = experts > 1 ? mean + 2.0 * std::sqrt(mean) : mean;
  return want <= 8 ? 1 : 2;
}
constexpr int kCtasPerSm = 2;

inline int max_token_tiles(long long rows, int experts, int nt) {
  const int tok = 8 * nt;
  if (experts <= 0) return (int)((rows + tok - 1) / tok);
  return (int)std::min<long long>(rows, std::min<long long>(experts, rows) + rows / tok);
}

template <class Kernel>
int allow_smem(Kernel kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(EK_ERR_CUDA, "device index out of range");
  if (done[dev]) return EK_OK;
  const int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                            "cudaFuncSetAttribute(w4)");
  done[dev] = rc == EK_OK;
  return rc;
}

constexpr int kIndexBytes = (2 * 1024 + 1) * (int)sizeof(int);  // of expert_tiles, at most

template <class T, Mode kMode, class S>
int launch_product_shape(const CUtensorMap& a, const CUtensorMap& b, const Params<T>& p, int grid, cudaStream_t stream) {
  static bool done[64] = {false};
  const int index = kMode == kDense ? 0 : (2 * p.E + 1) * (int)sizeof(int);
  const int rc = allow_smem(w4_kernel<T, S, kMode>, S::kSmem + (kMode == kDense ? 0 : kIndexBytes), done);
  return rc ? rc
            : launch("w4 product launch", w4_kernel<T, S, kMode>, dim3(grid), kThreads, S::kSmem + index, stream, S::kMakes,
                     a, b, p);
}

template <class T, Mode kMode, int FL, bool kMin>
int launch_product_nt(int nt, const CUtensorMap& a, const CUtensorMap& b, const Params<T>& p, int grid, cudaStream_t stream) {
  if constexpr (kMode == kDense)
    if (p.rows) return launch_product_shape<T, kMode, Shape<1, FL, kMin, true>>(a, b, p, grid, stream);
  return nt == 1 ? launch_product_shape<T, kMode, Shape<1, FL, kMin, false>>(a, b, p, grid, stream)
                 : launch_product_shape<T, kMode, Shape<2, FL, kMin, false>>(a, b, p, grid, stream);
}

// The product over the tokens p.x, its sums left in p.parts.
template <class T, Mode kMode>
int launch_product(int nt, int group, const CUtensorMap& a, const CUtensorMap& b, const Params<T>& p, int grid,
                   cudaStream_t stream) {
  const bool mins = p.w[0].m != nullptr;
  switch (group) {
    case 32:
      return mins ? launch_product_nt<T, kMode, 1, true>(nt, a, b, p, grid, stream)
                  : launch_product_nt<T, kMode, 1, false>(nt, a, b, p, grid, stream);
    case 64:
      return mins ? launch_product_nt<T, kMode, 2, true>(nt, a, b, p, grid, stream)
                  : launch_product_nt<T, kMode, 2, false>(nt, a, b, p, grid, stream);
    default:
      return mins ? launch_product_nt<T, kMode, 4, true>(nt, a, b, p, grid, stream)
                  : launch_product_nt<T, kMode, 4, false>(nt, a, b, p, grid, stream);
  }
}

template <class T>
int launch_tokens(const T* x, int rows, int K, int group, const Tokens& out, cudaStream_t stream) {
  const long long warps = (long long)rows * stages(K);
  const bool vec = K % 8 == 0 && aligned16(x);
  return launch("w4 tokens launch", tokens_kernel<T>, dim3((unsigned)std::min<long long>((warps + 7) / 8, 148 * 16)), 256, 0,
                stream, true, x, rows, K, group, vec, out);
}

// Codes [rows, K] as the TMA sees them: boxes of `box` rows x 128 bytes.
inline int codes_map(CUtensorMap* m, const void* codes, long long rows, int K, int box) {
  const uint64_t pitch = (uint64_t)pieces(K) * 16;
  return make_tmap_2d(m, codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, pitch, (uint64_t)rows, pitch, 128, box);
}

constexpr int kMaxK = 1 << 28;

// rows: of the whole weight, whose scales the products index in 32 bits (0: no
// matter); a token row's records are indexed in an int.
inline int check_w4(const char* what, const void* codes, const void* scales, const void* mins, long long rows, int K,
                    int group) {
  if (K < 1 || K > kMaxK || (group != 32 && group != 64 && group != 128))
    return set_error(EK_ERR_INVALID, "%s: need K >= 1 (at most 2^28) and a group of 32, 64 or 128 (K=%d group=%d)", what, K, group);
  if (rows * groups(K, group) > 0xffffffffll)
    return set_error(EK_ERR_INVALID, "%s: more than 2^32 scales (rows=%lld K=%d group=%d)", what, rows, K, group);
  if (!codes || !scales) return set_error(EK_ERR_INVALID, "%s: null pointer", what);
  if (!aligned16(codes)) return set_error(EK_ERR_INVALID, "%s: codes must be 16-byte aligned", what);
  if ((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(mins)) & 1u)
    return set_error(EK_ERR_INVALID, "%s: misaligned scales", what);
  return EK_OK;
}

}  // namespace w4
}  // namespace ek
