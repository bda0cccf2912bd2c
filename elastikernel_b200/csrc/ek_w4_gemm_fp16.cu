// The dense 4-bit-weight product for fp16.
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

int w4::gemm_fp16(const GemmArgs& a) { return gemm<__half>(a); }

}  // namespace ek
