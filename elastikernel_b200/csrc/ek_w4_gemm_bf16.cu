// The dense 4-bit-weight product for bf16 and its entry points.
#include "ek_w4_gemm.cuh"

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

}  // namespace

int w4::gemm_bf16(const GemmArgs& a) { return gemm<__nv_bfloat16>(a); }

}  // namespace ek

using namespace ek;
using namespace ek::w4;

extern "C" {

size_t ek_gemm_w4_workspace_bytes(int M, int N, int K, int num_sms) {
  if (M < 0 || N < 0 || K < 1 || K > kMaxK || num_sms < 1) return (size_t)-1;
  if (M == 0 || N == 0) return 0;
  int nt = 0, grid = 0;
  return gemm_layout(M, N, K, num_sms, &nt, &grid).bytes;
}

int ek_gemm_w4(const void* A, const void* codes, const void* scales, const void* mins, void* C, int M, int N, int K,
               int group, int dtype, int num_sms, void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  if (M < 0 || N < 0 || (dtype != EK_DTYPE_BF16 && dtype != EK_DTYPE_FP16))
    return set_error(EK_ERR_INVALID, "gemm_w4: bad sizes or type (M=%d N=%d dtype=%d)", M, N, dtype);
  if (M == 0 || N == 0) return EK_OK;
  int rc = check_w4("gemm_w4", codes, scales, mins, N, K, group);
  if (rc) return rc;
  if (!A || !C || !workspace) return set_error(EK_ERR_INVALID, "gemm_w4: null pointer");
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(C)) & 1u)
    return set_error(EK_ERR_INVALID, "gemm_w4: A and C must be aligned to their elements");
  GemmArgs a{A, codes, scales, mins, C, M, N, K, group, 0, workspace, static_cast<cudaStream_t>(stream)};
  rc = resolve_num_sms(num_sms, stream, &a.sms);
  if (rc) return rc;
  const size_t need = ek_gemm_w4_workspace_bytes(M, N, K, a.sms);
  if (!aligned16(workspace) || ws_bytes < need)
    return set_error(EK_ERR_INVALID, "gemm_w4: workspace must be 16-byte aligned and hold %zu bytes (got %zu)", need,
                     ws_bytes);
  return dtype == EK_DTYPE_BF16 ? gemm_bf16(a) : gemm_fp16(a);
}

}  // extern "C"
