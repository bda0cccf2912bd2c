// The dense product of one element type (a translation unit each).
#pragma once
#include "ek_w4_launch.cuh"

namespace ek {
namespace w4 {

struct GemmArgs {
  const void *A, *codes, *scales, *mins;
  void* C;
  int M, N, K, group, sms;
  void* workspace;
  cudaStream_t stream;
};

inline Layout gemm_layout(int M, int N, int K, int sms, int* nt, int* grid) {
  *nt = pick_nt(M, 1);
  *grid = sms * kCtasPerSm;
  const long long tiles = (long long)max_token_tiles(M, 0, *nt) * ((N + kRows - 1) / kRows);
  return layout(M, K, tiles, *grid, 8 * *nt);
}

// Whether each CTA makes the token records of its `units` / grid stages itself.
// A launch for them takes 1.4 us and 0.7 us pass for each record that a CTA
// makes. Measured, one launch less against one more: 4096 x 4096 (one stage per
// CTA) 6.9 against 8.3 us for one token, 8.4 against 8.5 for four, 11.6 against
// 9.0 for eight; 14336 x 4096 (four stages) 11.8 against 12.2 us for one, 13.4
// against 12.3 for two.
inline bool makes_records(int M, long long units, int grid) {
  return M <= 8 && M * ((units + grid - 1) / grid) <= 4;
}

int gemm_bf16(const GemmArgs& a);
int gemm_fp16(const GemmArgs& a);

// The sums of a product with minima may read the token rows again, so records
// are made where they are written over.
inline bool over_its_rows(const GemmArgs& a) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.A), c = reinterpret_cast<uintptr_t>(a.C);
  return a.mins && x < c + (size_t)a.M * a.N * 2 && c < x + (size_t)a.M * a.K * 2;
}

template <int TOK, bool kMin, class T>
int finish(const Params<T>& p, int grid, T* out, cudaStream_t stream) {
  const dim3 g(p.feature_tiles, std::min(p.max_y * TOK, 4096));
  return launch("w4 sums launch", finish_kernel<kDense, TOK, kMin, T, T>, g, kRows, 0, stream, false, p, grid, out);
}

template <class T>
int gemm(const GemmArgs& a) {
  int nt = 0, grid = 0;
  const Layout l = gemm_layout(a.M, a.N, a.K, a.sms, &nt, &grid);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  Params<T> p = {};
  p.w[0] = {static_cast<const T*>(a.scales), static_cast<const T*>(a.mins)};
  p.codes[0] = static_cast<const uint8_t*>(a.codes);
  p.group = a.group;
  p.K = a.K;
  p.N = a.N;
  p.feature_tiles = (a.N + kRows - 1) / kRows;
  p.x = {ws};
  p.n_rows = a.M;
  p.max_y = max_token_tiles(a.M, 0, nt);
  p.parts = reinterpret_cast<float*>(ws + l.parts);
  CUtensorMap map;
  int rc = codes_map(&map, a.codes, a.N, a.K, kRows);
  const T* x = static_cast<const T*>(a.A);
  if (makes_records(a.M, (long long)p.feature_tiles * stages(a.K), grid) && !over_its_rows(a)) {
    p.rows = x;
    p.vec = a.K % 8 == 0 && aligned16(x);
  } else if (!rc) {
    rc = launch_tokens(x, a.M, a.K, a.group, p.x, a.stream);
  }
  if (!rc) rc = launch_product<T, kDense>(nt, a.group, map, map, p, grid, a.stream);
  if (rc) return rc;
  T* out = static_cast<T*>(a.C);
  if (a.mins)
    return nt == 1 ? finish<8, true>(p, grid, out, a.stream) : finish<16, true>(p, grid, out, a.stream);
  return nt == 1 ? finish<8, false>(p, grid, out, a.stream) : finish<16, false>(p, grid, out, a.stream);
}

}  // namespace w4
}  // namespace ek
