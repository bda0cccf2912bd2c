// Entry points of the dense feed-forward operators: the block-scaled e4m3 product,
// the gated block in 16 bits and its gradients, and the gated block in 8 bits.
// Up to kStreamTokens tokens the forward products run in stream_kernel, whose time is the
// weights' bytes; past it, in 8 bits from 65 tokens on where they are the faster
// (fp8_streams), and for the gradients always, in the 256-row CTA-pair kernels.
#include <algorithm>
#include <cmath>

#include "ek_fp8_block_kernel.cuh"
#include "ek_internal.h"

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

constexpr int kStreamTokens = 128;
constexpr size_t kBad = (size_t)-1;

size_t round256(size_t x) { return (x + 255) / 256 * 256; }
int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

template <class Kernel>
int allow_smem(Kernel kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(EK_ERR_CUDA, "device index out of range");
  if (done[dev]) return EK_OK;
  const int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                            "cudaFuncSetAttribute(smem)");
  done[dev] = rc == EK_OK;
  return rc;
}

// Every kernel here waits for its predecessor itself (pdl_wait), so each launch may
// begin before that has ended. cluster: CTAs per cluster (0: none).
template <class... P, class... A>
int launch(const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, int cluster,
           const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n++].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == EK_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
         : dtype == EK_DTYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
}
int elem_size(int dtype) { return dtype == EK_DTYPE_E4M3 ? 1 : 2; }

// rows x k, the reduction axis contiguous: boxes of box_rows rows x 128 bytes
int map_k(CUtensorMap* m, const void* base, int dtype, int rows, int k, int box_rows) {
  const int es = elem_size(dtype);
  return make_tmap_2d(m, base, map_type(dtype), k, rows, (uint64_t)k * es, 128 / es, box_rows);
}
// k x cols, the reduction axis outermost (16 bits): the 3-D map of its whole 64-column
// chunks, two to a box, and the 2-D map of all columns (load_half); fewer than two whole
// chunks: the 2-D map twice.
int whole_chunks(int cols) { return cols >= 128 ? cols / 64 * 64 : 0; }
int map_mn(CUtensorMap* m, CUtensorMap* m2, const void* base, int dtype, int k, int cols) {
  int rc = make_tmap_2d(m2, base, map_type(dtype), cols, k, (uint64_t)cols * 2, 64, 64);
  if (rc) return rc;
  if (whole_chunks(cols))
    return make_tmap_3d(m, base, map_type(dtype), 64, k, cols / 64, (uint64_t)cols * 2, 128, 64, 64, 2);
  *m = *m2;
  return EK_OK;
}

int grid_for(long long work, int sms) { return (int)std::max<long long>(1, std::min<long long>(work, (long long)sms * 8)); }

// ------------------------------------------------------------------ splitting K
// The schedule of a pair kernel: tile columns and slices of K per tile. A pair runs
// ceil(tiles slices / pairs) units one after the other; a unit's blocks of K (t_kb each)
// run beside the epilogue of the unit before it (epi_us, kSliceUs for a slice), so it takes
// the longer of the two, and the last epilogue stands alone. Against that, the sums' way to
// memory and back and one more launch. A 128-column tile's block costs 0.7 of a 256-column
// one's (less to multiply, three quarters to load), its epilogue 0.8. Measured, launches of
// their own: 333 x 1032 over 5520 in 18 tiles of 128 columns cut in 4 takes 12 us, in 10 of
// 256 cut in 7 15 us; 5520 x 1032 over 333, 6 blocks of K, 11.7 us in tiles of 256 and 15.5
// in tiles of 128. cap: bytes the workspace has for the sums.
struct Plan {
  int bn, splits;
};
Plan pick_plan(long long rows, int cols, int k_blocks, int pairs, long long elems, double t_kb, double epi_us,
               bool narrow, size_t cap) {
  constexpr double kSliceUs = 4.0, kReduceUs = 3.0, kBytesPerUs = 4.0e6;
  Plan best{256, 1};
  double best_us = 1e30;
  for (int bn = 256; bn >= (narrow ? 128 : 256); bn /= 2) {
    const long long tiles = (long long)ceil_div(rows, 256) * ceil_div(cols, bn);
    const double kb_us = bn == 256 ? t_kb : 0.7 * t_kb;
    for (int s = 1; s <= 32 && (s == 1 || k_blocks / s >= 4); ++s) {
      const size_t bytes = (size_t)s * elems * 4;
      if (s > 1 && bytes > cap) break;
      const double epi = (s > 1 ? kSliceUs : epi_us) * (bn == 256 ? 1.0 : 0.8);
      double us = std::ceil((double)(tiles * s) / pairs) * std::max(std::ceil((double)k_blocks / s) * kb_us, epi) + epi;
      if (s > 1) us += kReduceUs + 2.0 * bytes / kBytesPerUs;
      if (us < 0.95 * best_us) {
        best_us = us;
        best = Plan{bn, s};
      }
    }
  }
  return best;
}
constexpr double kFfnBlockUs = 0.28, kFp8BlockUs = 0.5;
constexpr double kStoreUs = 4.0, kGateUs = 5.0;
// gelu's erfc makes the gradient's epilogue three times as long
constexpr double gate_grad_us(int gate) { return gate == kGateGelu ? 18.0 : 7.0; }
constexpr size_t kMostSplitBytes = 256u << 20;

// ------------------------------------------------------------------ few tokens
StreamSplit stream_split(int rows, int rows_per_tile, int k, int bk, int sms) {
  StreamSplit s;
  s.tiles = ceil_div(rows, rows_per_tile);
  s.k_blocks = ceil_div(k, bk);
  const long long units = (long long)s.tiles * s.k_blocks;
  s.per_cta = (int)std::max<long long>(2, (units + sms - 1) / sms);
  s.ctas = ceil_div(units, s.per_cta);
  s.max_segs = (s.per_cta - 1 + s.k_blocks - 1) / s.k_blocks + 1;
  return s;
}
size_t stream_bytes(const StreamSplit& s, int T) { return (size_t)s.ctas * s.max_segs * T * 256 * 4; }
// for any number of SMs up to sms (a smaller partition has fewer, longer runs)
size_t stream_bytes_most(int rows, int rows_per_tile, int T, int sms) {
  return ((size_t)ceil_div(rows, rows_per_tile) + 2 * (size_t)sms + 8) * T * 256 * 4;
}

template <class Cfg>
int launch_stream(const CUtensorMap& tw, const CUtensorMap& tw2, const CUtensorMap& tx, const StreamParams& p,
                  cudaStream_t s) {
  static bool done[64] = {false};
  const int rc = allow_smem(stream_kernel<Cfg>, Cfg::SMEM_BYTES, done);
  if (rc) return rc;
  return launch("stream product", stream_kernel<Cfg>, dim3(p.sp.ctas), Cfg::THREADS, Cfg::SMEM_BYTES, s, 0, tw, tw2, tx,
                p);
}

template <int kElem, bool kGate>
int launch_stream_nt(const void* w, const void* w2, const void* x, int rows, int K, StreamParams& p, cudaStream_t s) {
  const int nt = p.T <= 16 ? 16 : p.T <= 32 ? 32 : p.T <= 64 ? 64 : 128;
  p.n = (p.T + 15) / 16 * 16;
  CUtensorMap tw, tw2, tx;
  int rc = map_k(&tw, w, kElem, rows, K, kGate ? 128 : 256);
  if (rc) return rc;
  tw2 = tw;
  if (kGate && (rc = map_k(&tw2, w2, kElem, rows, K, 128))) return rc;
  if ((rc = map_k(&tx, x, kElem, p.T, K, p.n))) return rc;
  switch (nt) {
    case 16: return launch_stream<StreamCfg<kElem, 16, kGate>>(tw, tw2, tx, p, s);
    case 32: return launch_stream<StreamCfg<kElem, 32, kGate>>(tw, tw2, tx, p, s);
    case 64: return launch_stream<StreamCfg<kElem, 64, kGate>>(tw, tw2, tx, p, s);
    default: return launch_stream<StreamCfg<kElem, 128, kGate>>(tw, tw2, tx, p, s);
  }
}

// Warps that share a token's segments in the reducing launch: several where a tile
// has many and the blocks would leave SMs idle.
int stream_ways(const StreamSplit& sp, int T, int row_tiles, int sms) {
  const int segs = ceil_div(sp.k_blocks, sp.per_cta) + 1;
  int ways = 1;
  while (ways < 8 && 2 * ways <= segs && (long long)row_tiles * ceil_div(T, 8 / (2 * ways)) <= 4ll * sms) ways *= 2;
  return ways;
}

struct StreamScales {
  const float *tok = nullptr, *w = nullptr, *w2 = nullptr;
};

// The product of weight rows w (gate: w and w2) with the tokens x and what follows it, o.
template <bool kGate>
int stream_product(int dtype, const void* w, const void* w2, const void* x, const StreamScales& sc, int K,
                   const StreamOut& o, int sms, void* ws, size_t ws_bytes, cudaStream_t s, bool early) {
  StreamParams p{};
  p.sp = stream_split(o.N, kGate ? 128 : 256, K, 128 / elem_size(dtype), sms);
  if (ws_bytes < stream_bytes(p.sp, o.T)) return set_error(EK_ERR_INVALID, "workspace too small");
  p.early = early;
  p.T = o.T;
  p.tok_scale = sc.tok;
  p.w_scale = sc.w;
  p.w_scale2 = sc.w2;
  p.w_blocks = ceil_div(o.N, 128);
  p.ws = static_cast<float*>(ws);
  const int rc = dtype == EK_DTYPE_BF16 ? launch_stream_nt<kBF16, kGate>(w, w2, x, o.N, K, p, s)
                 : dtype == EK_DTYPE_FP16 ? launch_stream_nt<kFP16, kGate>(w, w2, x, o.N, K, p, s)
                                          : launch_stream_nt<kE4M3, kGate>(w, w2, x, o.N, K, p, s);
  if (rc) return rc;
  const int row_tiles = kGate ? p.sp.tiles : 2 * p.sp.tiles, ways = stream_ways(p.sp, o.T, row_tiles, sms);
  return launch("stream sums", kGate ? stream_gate_reduce_kernel : stream_store_reduce_kernel,
                dim3(row_tiles, ceil_div(o.T, 8 / ways)), 256, 0, s, 0, p.sp, (const float*)p.ws, o, ways);
}

// out[t, n] = x[t] . w[n]
int stream_store(int dtype, const void* w, const void* x, const StreamScales& sc, int T, int N, int K, void* out,
                 int out_type, int sms, void* ws, size_t ws_bytes, cudaStream_t s, bool early) {
  StreamOut o{};
  o.T = T;
  o.N = N;
  o.out = out;
  o.type = out_type;
  o.wide = aligned16(out) && N % 4 == 0;
  return stream_product<false>(dtype, w, w, x, sc, K, o, sms, ws, ws_bytes, s, early);
}

// a[t, i] = f(x[t] . w1[i]) (x[t] . w3[i]); with codes, those and scales of a
int stream_gate(int dtype, const void* w1, const void* w3, const void* x, const StreamScales& sc, int T, int I, int H,
                int gate, void* a, void* h, uint8_t* codes, float* scales, int sms, void* ws, size_t ws_bytes,
                cudaStream_t s, bool early) {
  StreamOut o{};
  o.T = T;
  o.N = I;
  o.out = a;
  o.type = dtype;
  o.gate = gate;
  o.h = h;
  o.codes = codes;
  o.scales = scales;
  return stream_product<true>(dtype, w1, w3, x, sc, H, o, sms, ws, ws_bytes, s, early);
}

// ------------------------------------------------------------------ 16-bit tiles
template <class Cfg>
int launch_ffn_cfg(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb2, FfnParams& p, int sms,
                   cudaStream_t s) {
  static bool done[64] = {false};
  const int rc = allow_smem(ffn_gemm_kernel<Cfg>, Cfg::SMEM_BYTES, done);
  if (rc) return rc;
  const long long units = (long long)p.tiles_m * p.tiles_n * p.splits;
  if (units > 0x3fffffff) return set_error(EK_ERR_INVALID, "too many tiles");
  p.num_units = (int)units;
  const int pairs = (int)std::min<long long>(std::max(1, sms / 2), units);
  return launch("feed-forward product", ffn_gemm_kernel<Cfg>, dim3(2 * pairs), Cfg::THREADS, Cfg::SMEM_BYTES, s, 2, ta, tb,
                tb2, p);
}

// Maps and launch of one product of p.M rows and p.N columns over k: A K-major, B K-major (b2
// the gate's second) or MN-major.
template <int kElem, bool kBMN, int kEpi>
int launch_ffn(const void* a, const void* b, const void* b2, int k, const Plan& plan, FfnParams& p, int sms, cudaStream_t s) {
  CUtensorMap ta, tb, tb2;
  int rc = map_k(&ta, a, kElem, p.M, k, 128);
  if (rc) return rc;
  if (kBMN) {
    rc = map_mn(&tb, &tb2, b, kElem, k, p.N);
    p.b_full = whole_chunks(p.N);
  } else {
    rc = map_k(&tb, b, kElem, p.N, k, plan.bn / 2);
    if (!rc) rc = map_k(&tb2, b2, kElem, p.N, k, plan.bn / 2);
  }
  if (rc) return rc;
  p.tiles_m = ceil_div(p.M, 256);
  p.tiles_n = ceil_div(p.N, kEpi == kFfnGate ? plan.bn / 2 : plan.bn);
  p.k_blocks = ceil_div(k, 64);
  p.splits = plan.splits;
  return plan.bn == 256 ? launch_ffn_cfg<FfnCfg<kElem, kBMN, kEpi, 256>>(ta, tb, tb2, p, sms, s)
                        : launch_ffn_cfg<FfnCfg<kElem, kBMN, kEpi, 128>>(ta, tb, tb2, p, sms, s);
}

Plan store_plan(int M, int N, int k, int sms, size_t cap) {
  return pick_plan(M, N, ceil_div(k, 64), std::max(1, sms / 2), (long long)M * N, kFfnBlockUs, kStoreUs, true, cap);
}
size_t ffn_store_bytes(int M, int N, int k, int sms) {
  const int s = store_plan(M, N, k, sms, kMostSplitBytes).splits;
  return s > 1 ? (size_t)s * M * N * 4 : 0;
}

// C [M, N] = a [M, k] . w [N, k]^T. ws holds the sums of a split.
template <int kElem>
int ffn_store(const void* a, const void* w, int M, int N, int k, void* C, int sms, void* ws, size_t ws_bytes,
              cudaStream_t s) {
  FfnParams p{};
  p.M = M;
  p.N = N;
  p.C = C;
  p.ws = static_cast<float*>(ws);
  const int rc = launch_ffn<kElem, false, kFfnStore>(a, w, w, k, store_plan(M, N, k, sms, ws_bytes), p, sms, s);
  if (rc || p.splits == 1) return rc;
  const long long n8 = (long long)M * N / 8;
  return launch("feed-forward sums", ffn_reduce_kernel<kElem>, dim3(grid_for((n8 + 255) / 256, sms)), 256, 0, s, 0,
                (const float*)p.ws, p.splits, n8, C);
}

// gate/up tiles hold half as many features as columns
Plan gate_plan(int T, int H, int I, int sms, size_t cap) {
  return pick_plan(T, 2 * I, ceil_div(H, 64), std::max(1, sms / 2), 2ll * T * I, kFfnBlockUs, kGateUs, true, cap);
}
size_t gate_bytes(int T, int H, int I, int sms) {
  const int s = gate_plan(T, H, I, sms, kMostSplitBytes).splits;
  return s > 1 ? (size_t)s * T * I * 8 : 0;
}
Plan gate_grad_plan(int T, int H, int I, int gate, int sms, size_t cap) {
  return pick_plan(T, I, ceil_div(H, 64), std::max(1, sms / 2), (long long)T * I, kFfnBlockUs,
                   gate_grad_us(gate), true, cap);
}
size_t gate_grad_bytes(int T, int H, int I, int sms) {  // of any gate function
  const int s = std::max(gate_grad_plan(T, H, I, kGateSilu, sms, kMostSplitBytes).splits,
                         gate_grad_plan(T, H, I, kGateGelu, sms, kMostSplitBytes).splits);
  return s > 1 ? (size_t)s * T * I * 4 : 0;
}

template <int kElem>
int ffn_gate(const void* x, const void* w1, const void* w3, void* a, void* h, int T, int H, int I, int gate, int sms,
             void* ws, size_t ws_bytes, cudaStream_t s) {
  FfnParams p{};
  p.M = T;
  p.N = I;
  p.gate = gate;
  p.C = a;
  p.H = h;
  p.h_plane = (long long)T * I;
  p.ws = static_cast<float*>(ws);
  const int rc = launch_ffn<kElem, false, kFfnGate>(x, w1, w3, H, gate_plan(T, H, I, sms, ws_bytes), p, sms, s);
  if (rc || p.splits == 1) return rc;
  return launch("feed-forward gate sums", ffn_gate_reduce_kernel<kElem>, dim3(grid_for(((long long)T * I / 8 + 255) / 256, sms)),
                256, 0, s, 0, (const float*)p.ws, p.splits, T, I, gate, a, h);
}

template <int kElem>
int gated_ffn(const void* x, const void* w1, const void* w2, const void* w3, void* y, void* h, int T, int H, int I,
              int gate, int sms, char* ws, size_t ws_bytes, cudaStream_t s) {
  const size_t a_bytes = round256((size_t)T * I * 2);
  if (ws_bytes < a_bytes) return set_error(EK_ERR_INVALID, "workspace of at least %zu bytes required", a_bytes);
  void* a = ws;
  char* rest = ws + a_bytes;
  const size_t rest_bytes = ws_bytes - a_bytes;
  int rc;
  if (T <= kStreamTokens) {
    rc = stream_gate(kElem, w1, w3, x, {}, T, I, H, gate, a, h, nullptr, nullptr, sms, rest, rest_bytes, s, false);
    if (rc) return rc;
    return stream_store(kElem, w2, a, {}, T, H, I, y, kElem, sms, rest, rest_bytes, s, true);
  }
  rc = ffn_gate<kElem>(x, w1, w3, a, h, T, H, I, gate, sms, rest, rest_bytes, s);
  if (rc) return rc;
  return ffn_store<kElem>(a, w2, T, H, I, y, sms, rest, rest_bytes, s);
}

// Tile columns and dx's slices for the gradient's three products in one launch: the pairs
// share the units' time (a unit: its blocks, or the epilogue beside them), but not less than
// dx's own rounds.
Plan grads_plan(int T, int H, int I, int sms, size_t cap) {
  const int pairs = std::max(1, sms / 2), kb_x = 2 * ceil_div(I, 64), kb_w = ceil_div(T, 64);
  Plan best{256, 1};
  double best_us = 1e30;
  for (int bn = 256; bn >= 128; bn /= 2) {
    const double kb_us = bn == 256 ? kFfnBlockUs : 0.7 * kFfnBlockUs, epi = bn == 256 ? kStoreUs : 0.8 * kStoreUs;
    const double n_w = 2.0 * ceil_div(I, 256) * ceil_div(H, bn) + (double)ceil_div(H, 256) * ceil_div(I, bn);
    const double t_w = std::max(kb_w * kb_us, epi);
    for (int s = 1; s <= 32 && (s == 1 || kb_x / s >= 4); ++s) {
      const size_t bytes = (size_t)s * T * H * 4;
      if (s > 1 && bytes > cap) break;
      const double n_x = (double)ceil_div(T, 256) * ceil_div(H, bn) * s, t_x = std::max(ceil_div(kb_x, s) * kb_us, epi);
      double us = std::max(std::ceil(n_x / pairs) * t_x, (n_x * t_x + n_w * t_w) / pairs + 0.5 * t_w) + epi;
      if (s > 1) us += 3.0 + 2.0 * bytes / 4.0e6;
      if (us < 0.97 * best_us) {
        best_us = us;
        best = Plan{bn, s};
      }
    }
  }
  return best;
}
size_t grads_bytes(int T, int H, int I, int sms) {
  const int s = grads_plan(T, H, I, sms, kMostSplitBytes).splits;
  return s > 1 ? (size_t)s * T * H * 4 : 0;
}

template <int kElem, int kBN>
int launch_grads(FfnGradMaps& m, FfnGradParams& p, int sms, cudaStream_t s) {
  using Cfg = FfnCfg<kElem, true, kFfnStore, kBN>;
  static bool done[64] = {false};
  const int rc = allow_smem(ffn_grad_kernel<Cfg>, Cfg::SMEM_BYTES, done);
  if (rc) return rc;
  const long long units = (long long)p.n_x + p.n_13 + p.n_2;
  const int pairs = (int)std::min<long long>(std::max(1, sms / 2), units);
  return launch("feed-forward gradients", ffn_grad_kernel<Cfg>, dim3(2 * pairs), Cfg::THREADS, Cfg::SMEM_BYTES, s, 2, m, p);
}

template <int kElem>
int gated_ffn_grad(const void* x, const void* w1, const void* w2, const void* w3, const void* h, const void* d_out,
                   void* d_x, void* d_w13, void* d_w2, int T, int H, int I, int gate, int sms, char* ws, size_t ws_bytes,
                   cudaStream_t s) {
  const size_t plane = (size_t)T * I * 2, dh_bytes = round256(2 * plane), a_bytes = round256(plane);
  if (ws_bytes < dh_bytes + a_bytes)
    return set_error(EK_ERR_INVALID, "workspace of at least %zu bytes required", dh_bytes + a_bytes);
  char* dh = ws;
  char* a = dh + dh_bytes;
  char* rest = a + a_bytes;
  const size_t rest_bytes = ws_bytes - dh_bytes - a_bytes;
  FfnParams p{};
  p.M = T;
  p.N = I;
  p.ws = reinterpret_cast<float*>(rest);
  p.gate = gate;
  p.C = dh;
  p.H = const_cast<void*>(h);
  p.c_plane = p.h_plane = (long long)T * I;
  p.Act = a;
  int rc = launch_ffn<kElem, true, kFfnGateGrad>(d_out, w2, nullptr, H, gate_grad_plan(T, H, I, gate, sms, rest_bytes), p,
                                                 sms, s);
  if (rc) return rc;
  if (p.splits > 1 &&
      (rc = launch("feed-forward gate gradient sums", ffn_gate_grad_reduce_kernel<kElem>,
                   dim3(grid_for(((long long)T * I / 8 + 255) / 256, sms)), 256, 0, s, 0, (const float*)p.ws,
                   p.splits, T, I, gate, h, (void*)dh, (void*)a)))
    return rc;
  // plane 1 of dh starts on a 16-byte boundary: a plane is T * I elements, I a multiple of 8
  const Plan plan = grads_plan(T, H, I, sms, rest_bytes);
  const int bn = plan.bn;
  FfnGradMaps m;
  const void* w13[2] = {w1, w3};
  for (int i = 0; i < 2; ++i) {
    const char* dh_i = dh + i * plane;
    if ((rc = map_k(&m.dh[i], dh_i, kElem, T, I, 128)) || (rc = map_mn(&m.w[i], &m.w2d[i], w13[i], kElem, I, H)) ||
        (rc = map_mn(&m.dht[i], &m.dht2d[i], dh_i, kElem, T, I)))
      return rc;
  }
  if ((rc = map_mn(&m.x, &m.x2d, x, kElem, T, H)) || (rc = map_mn(&m.dyt, &m.dyt2d, d_out, kElem, T, H)) ||
      (rc = map_mn(&m.a, &m.a2d, a, kElem, T, I)))
    return rc;
  FfnGradParams g{};
  g.T = T;
  g.H = H;
  g.I = I;
  g.tm_x = ceil_div(T, 256);
  g.tn_x = g.tn_13 = ceil_div(H, bn);
  g.kb_plane = ceil_div(I, 64);
  g.kb_x = 2 * g.kb_plane;
  g.splits = plan.splits;
  g.tm_13 = ceil_div(I, 256);
  g.tm_2 = ceil_div(H, 256);
  g.tn_2 = ceil_div(I, bn);
  g.kb_w = ceil_div(T, 64);
  const long long n_x = (long long)g.tm_x * g.tn_x * g.splits, n_13 = 2ll * g.tm_13 * g.tn_13, n_2 = (long long)g.tm_2 * g.tn_2;
  if (n_x + n_13 + n_2 > 0x3fffffff) return set_error(EK_ERR_INVALID, "too many tiles");
  g.n_x = (int)n_x;
  g.n_13 = (int)n_13;
  g.n_2 = (int)n_2;
  // in blocks of K alone, although grads_plan takes a weight's tile for its stores at least: while
  // dx's pairs multiply, the others' stores run faster than that. The ratio of the plan's own
  // times leaves tiles for after dx (64 x 4096 x 14336: 229 us for 204; 256 x 4096 x 4096: 81
  // for 69; 8 x 7168 x 2048: 62.6 for 56.8).
  g.lead = g.kb_x / g.splits / g.kb_w;
  g.full_h = whole_chunks(H);
  g.full_i = whole_chunks(I);
  g.dx = d_x;
  g.dw13 = d_w13;
  g.dw2 = d_w2;
  g.ws = reinterpret_cast<float*>(rest);
  rc = bn == 256 ? launch_grads<kElem, 256>(m, g, sms, s) : launch_grads<kElem, 128>(m, g, sms, s);
  if (rc || g.splits == 1) return rc;
  const long long n8 = (long long)T * H / 8;
  return launch("feed-forward sums", ffn_reduce_kernel<kElem>, dim3(grid_for((n8 + 255) / 256, sms)), 256, 0, s, 0,
                (const float*)g.ws, g.splits, n8, d_x);
}

// ------------------------------------------------------------------ 8-bit tiles
template <bool kGate>
int launch_fp8(const void* a, const void* w, const void* w2, int K, Fp8BlockParams& p, int sms, cudaStream_t s) {
  using Cfg = Fp8BlockCfg<kGate>;
  CUtensorMap ta, tb, tb2;
  int rc = map_k(&ta, a, EK_DTYPE_E4M3, p.M, K, 128);
  if (rc || (rc = map_k(&tb, w, EK_DTYPE_E4M3, p.N, K, 128))) return rc;
  tb2 = tb;
  if (kGate && (rc = map_k(&tb2, w2, EK_DTYPE_E4M3, p.N, K, 128))) return rc;
  static bool done[64] = {false};
  if ((rc = allow_smem(fp8_block_kernel<Cfg>, Cfg::SMEM_BYTES, done))) return rc;
  const long long units = (long long)p.tiles_m * p.tiles_n * p.splits;
  if (units > 0x3fffffff) return set_error(EK_ERR_INVALID, "too many tiles");
  p.num_units = (int)units;
  p.scale4 = p.k_blocks % 4 == 0 && aligned16(p.a_scale) && aligned16(p.w_scale) && aligned16(p.w_scale2);
  const int groups = (int)std::min<long long>(std::max(1, sms / 2), units);
  return launch("block-scaled product", fp8_block_kernel<Cfg>, dim3(2 * groups), Cfg::THREADS, Cfg::SMEM_BYTES, s,
                2, ta, tb, tb2, p);
}

int fp8_splits(int M, int N, int K, int sms, size_t cap) {
  return pick_plan(M, N, ceil_div(K, 128), std::max(1, sms / 2), (long long)M * N, kFp8BlockUs, kStoreUs, false, cap)
      .splits;
}

// of a gate/up pair, whose tiles hold 128 features
int fp8_gate_splits(int T, int I, int H, int sms, size_t cap) {
  if (T > 65535 * 8) return 1;  // the launch that adds the slices has a block for every 8 tokens
  return pick_plan(T, 2 * I, ceil_div(H, 128), std::max(1, sms / 2), 2ll * T * I, kFp8BlockUs, kGateUs, false, cap).splits;
}

// Whether an e4m3 product (gate: a gate/up pair of N features) of M tokens runs in
// stream_kernel. Up to 64 tokens it does. From there to kStreamTokens its unit of 32 KB
// takes 0.9 us and 9 ns a token (the sums of 128 tokens leave no registers to hide the loads
// behind), a block of the 256-row tiles 0.5 us whatever the tokens: 14336 x 4096 takes 18.7,
// 28 and 31 us for 64, 96 and 128 tokens in the one and 19 in the other, the 8-bit block of
// 7168 x 2048, with few tiles, 34 us for 128 tokens in the one and 41 in the other.
bool fp8_streams(int M, int N, int K, bool gate, int sms) {
  if (M <= 64) return true;
  if (M > kStreamTokens) return false;
  const int kb = ceil_div(K, 128), pairs = std::max(1, sms / 2);
  const double stream_us = stream_split(N, gate ? 128 : 256, K, 128, sms).per_cta * (0.9 + 0.009 * M) + 4.0;
  const int splits = (gate ? fp8_gate_splits : fp8_splits)(M, N, K, sms, kMostSplitBytes);
  const double rounds = std::ceil((double)ceil_div(N, gate ? 128 : 256) * splits / pairs);
  const double tile_us = rounds * ceil_div(kb, splits) * 0.5 + (splits > 1 ? 9.0 : 4.0);
  return stream_us < tile_us;
}

int fp8_store(const void* a, const void* w, const float* as, const float* wsc, void* C, int M, int N, int K, int out_type,
              int sms, void* ws, size_t ws_bytes, cudaStream_t s, bool early) {
  if (fp8_streams(M, N, K, false, sms))
    return stream_store(EK_DTYPE_E4M3, w, a, {as, wsc, nullptr}, M, N, K, C, out_type, sms, ws, ws_bytes, s, early);
  Fp8BlockParams p{};
  p.M = M;
  p.N = N;
  p.tiles_m = ceil_div(M, 256);
  p.tiles_n = ceil_div(N, 256);
  p.k_blocks = ceil_div(K, 128);
  p.splits = fp8_splits(M, N, K, sms, ws_bytes);
  p.a_scale = as;
  p.w_scale = wsc;
  p.w_blocks = ceil_div(N, 128);
  p.C = C;
  p.out_type = out_type;
  p.wide = aligned16(C) && (size_t)N * (out_type == kOutFP32 ? 4 : 2) % 16 == 0;
  p.ws = static_cast<float*>(ws);
  int rc = launch_fp8<false>(a, w, w, K, p, sms, s);
  if (rc || p.splits == 1) return rc;
  const long long n = (long long)M * N;
  return launch("block-scaled sums", fp8_block_reduce_kernel, dim3(grid_for((n + 255) / 256, sms)), 256, 0, s, 0,
                (const float*)p.ws, p.splits, n, C, out_type);
}

size_t fp8_store_bytes(int M, int N, int K, int sms) {
  // for either kernel: on a smaller partition the choice may be the other one
  const size_t stream = M <= kStreamTokens ? stream_bytes_most(N, 256, M, sms) : 0;
  const int s = M <= 64 ? 1 : fp8_splits(M, N, K, sms, kMostSplitBytes);
  return std::max(stream, s > 1 ? (size_t)s * M * N * 4 : 0);
}

struct Fp8FfnLayout {
  size_t xq, xs, aq, as, rest, total;
};
Fp8FfnLayout fp8_ffn_layout(int T, int H, int I, int sms) {
  Fp8FfnLayout L;
  L.xq = 0;
  L.xs = L.xq + round256((size_t)T * H);
  L.aq = L.xs + round256((size_t)T * ceil_div(H, 128) * 4);
  L.as = L.aq + round256((size_t)T * I);
  L.rest = L.as + round256((size_t)T * ceil_div(I, 128) * 4);
  const int splits = T <= 64 ? 1 : fp8_gate_splits(T, I, H, sms, kMostSplitBytes);
  const size_t gate = std::max(T <= kStreamTokens ? stream_bytes_most(I, 128, T, sms) : 0,
                               splits > 1 ? (size_t)splits * T * I * 8 : 0);
  L.total = L.rest + std::max(gate, fp8_store_bytes(T, H, I, sms));
  return L;
}

// ------------------------------------------------------------------ checks
constexpr int kMostRows = 0x7fffff00;  // a tile of 256 rows ends within an int
bool block_sizes_ok(int M, int N, int K) {
  return M >= 0 && M <= kMostRows && N >= 0 && N <= kMostRows && K > 0 && K % 16 == 0 && K <= (1 << 28);
}
bool sizes_ok(int T, int H, int I, int unit) {
  return T >= 0 && T <= kMostRows && H > 0 && I > 0 && H % unit == 0 && I % unit == 0 && H <= (1 << 28) && I <= (1 << 28);
}
bool sms_ok(int sms) { return sms > 0 && sms <= kGemmMaxSms; }

int check_ffn(int T, int H, int I, int unit, int gate) {
  if (!sizes_ok(T, H, I, unit))
    return set_error(EK_ERR_INVALID, "feed-forward: H and I must be positive multiples of %d up to 2^28, T up to 2^31 - 256 "
                     "(got T=%d H=%d I=%d)", unit, T, H, I);
  if (gate < kGateSilu || gate > kGateGeluTanh) return set_error(EK_ERR_INVALID, "unknown gate function %d", gate);
  return EK_OK;
}

template <class... P>
bool all_aligned(P... p) {
  return (aligned16(p) && ...);
}
template <class... P>
bool all_set(P... p) {
  return ((p != nullptr) && ...);
}

int resolve(int num_sms, void* stream, int* sms) {
  const int rc = resolve_num_sms(num_sms, stream, sms);
  if (rc) return rc;
  if (!sms_ok(*sms)) return set_error(EK_ERR_INVALID, "num_sms must be in [1, %d], got %d", kGemmMaxSms, *sms);
  return EK_OK;
}

}  // namespace
}  // namespace ek

using namespace ek;

extern "C" {

size_t ek_gemm_fp8_block_workspace_bytes(int M, int N, int K, int num_sms) {
  if (!block_sizes_ok(M, N, K) || !sms_ok(num_sms)) return kBad;
  return M == 0 || N == 0 ? 0 : fp8_store_bytes(M, N, K, num_sms);
}

int ek_gemm_fp8_block(const void* A, const void* W, const float* a_scale, const float* w_scale, void* C, int M, int N,
                      int K, int out_dtype, int num_sms, void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  if (!block_sizes_ok(M, N, K))
    return set_error(EK_ERR_INVALID, "block-scaled product: K must be a positive multiple of 16 up to 2^28, M and N up to "
                     "2^31 - 256 (got %d x %d x %d)", M, N, K);
  if (out_dtype != kOutBF16 && out_dtype != kOutFP16 && out_dtype != kOutFP32)
    return set_error(EK_ERR_INVALID, "block-scaled product: result in bf16, fp16 or fp32 (got dtype %d)", out_dtype);
  if (M == 0 || N == 0) return EK_OK;
  if (!all_set(A, W, a_scale, w_scale, C)) return set_error(EK_ERR_INVALID, "null operand");
  if (!all_aligned(A, W, workspace)) return set_error(EK_ERR_INVALID, "operands must be 16-byte aligned");
  int sms = 0;
  const int rc = resolve(num_sms, stream, &sms);
  if (rc) return rc;
  return fp8_store(A, W, a_scale, w_scale, C, M, N, K, out_dtype, sms, workspace, workspace ? ws_bytes : 0,
                   static_cast<cudaStream_t>(stream), false);
}

size_t ek_gated_ffn_workspace_bytes(int T, int H, int I, int num_sms) {
  if (!sizes_ok(T, H, I, 8) || !sms_ok(num_sms)) return kBad;
  if (T == 0) return 0;
  const size_t sums = T <= kStreamTokens
                          ? std::max(stream_bytes_most(I, 128, T, num_sms), stream_bytes_most(H, 256, T, num_sms))
                          : std::max(gate_bytes(T, H, I, num_sms), ffn_store_bytes(T, H, I, num_sms));
  return round256((size_t)T * I * 2) + sums;
}

int ek_gated_ffn(const void* x, const void* w1, const void* w2, const void* w3, void* y, void* h, int T, int H, int I,
                 int dtype, int gate, int num_sms, void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  int rc = check_ffn(T, H, I, 8, gate);
  if (rc) return rc;
  if (dtype != EK_DTYPE_BF16 && dtype != EK_DTYPE_FP16)
    return set_error(EK_ERR_INVALID, "feed-forward takes bf16 or fp16 (got dtype %d)", dtype);
  if (T == 0) return EK_OK;
  if (!all_set(x, w1, w2, w3, y, workspace)) return set_error(EK_ERR_INVALID, "null operand");
  if (!all_aligned(x, w1, w2, w3, y, h, workspace))
    return set_error(EK_ERR_INVALID, "operands must be 16-byte aligned");
  int sms = 0;
  if ((rc = resolve(num_sms, stream, &sms))) return rc;
  const auto f = dtype == EK_DTYPE_BF16 ? gated_ffn<kBF16> : gated_ffn<kFP16>;
  return f(x, w1, w2, w3, y, h, T, H, I, gate, sms, static_cast<char*>(workspace), ws_bytes,
           static_cast<cudaStream_t>(stream));
}

size_t ek_gated_ffn_grad_workspace_bytes(int T, int H, int I, int num_sms) {
  if (!sizes_ok(T, H, I, 8) || !sms_ok(num_sms)) return kBad;
  if (T == 0) return 0;
  const size_t sums = std::max(grads_bytes(T, H, I, num_sms), gate_grad_bytes(T, H, I, num_sms));
  return round256((size_t)T * I * 4) + round256((size_t)T * I * 2) + sums;
}

int ek_gated_ffn_grad(const void* x, const void* w1, const void* w2, const void* w3, const void* h, const void* d_out,
                      void* d_x, void* d_w13, void* d_w2, int T, int H, int I, int dtype, int gate, int num_sms,
                      void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  int rc = check_ffn(T, H, I, 8, gate);
  if (rc) return rc;
  if (dtype != EK_DTYPE_BF16 && dtype != EK_DTYPE_FP16)
    return set_error(EK_ERR_INVALID, "feed-forward takes bf16 or fp16 (got dtype %d)", dtype);
  if (!all_set(d_w13, d_w2)) return set_error(EK_ERR_INVALID, "null operand");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (T == 0) {  // sums over no token
    rc = check_cuda(cudaMemsetAsync(d_w13, 0, (size_t)I * H * 4, s), "feed-forward gradient");
    return rc ? rc : check_cuda(cudaMemsetAsync(d_w2, 0, (size_t)I * H * 2, s), "feed-forward gradient");
  }
  if (!all_set(x, w1, w2, w3, h, d_out, d_x, workspace)) return set_error(EK_ERR_INVALID, "null operand");
  if (!all_aligned(x, w1, w2, w3, h, d_out, d_x, d_w13, d_w2, workspace))
    return set_error(EK_ERR_INVALID, "operands must be 16-byte aligned");
  int sms = 0;
  if ((rc = resolve(num_sms, stream, &sms))) return rc;
  const auto f = dtype == EK_DTYPE_BF16 ? gated_ffn_grad<kBF16> : gated_ffn_grad<kFP16>;
  return f(x, w1, w2, w3, h, d_out, d_x, d_w13, d_w2, T, H, I, gate, sms, static_cast<char*>(workspace), ws_bytes, s);
}

size_t ek_gated_ffn_fp8_workspace_bytes(int T, int H, int I, int num_sms) {
  if (!sizes_ok(T, H, I, 16) || !sms_ok(num_sms)) return kBad;
  return T == 0 ? 0 : fp8_ffn_layout(T, H, I, num_sms).total;
}

int ek_gated_ffn_fp8(const void* x, const void* w1, const void* w2, const void* w3, const float* s1, const float* s2,
                     const float* s3, void* y, int T, int H, int I, int gate, int num_sms, void* workspace,
                     size_t ws_bytes, void* stream) {
  clear_error();
  int rc = check_ffn(T, H, I, 16, gate);
  if (rc) return rc;
  if (T == 0) return EK_OK;
  if (!all_set(x, w1, w2, w3, s1, s2, s3, y, workspace)) return set_error(EK_ERR_INVALID, "null operand");
  if (!all_aligned(x, w1, w2, w3, y, workspace)) return set_error(EK_ERR_INVALID, "operands must be 16-byte aligned");
  int sms = 0;
  if ((rc = resolve(num_sms, stream, &sms))) return rc;
  const Fp8FfnLayout L = fp8_ffn_layout(T, H, I, sms);
  if (ws_bytes < L.rest) return set_error(EK_ERR_INVALID, "workspace of at least %zu bytes required", L.rest);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  uint8_t *xq = reinterpret_cast<uint8_t*>(ws + L.xq), *aq = reinterpret_cast<uint8_t*>(ws + L.aq);
  float *xs = reinterpret_cast<float*>(ws + L.xs), *as = reinterpret_cast<float*>(ws + L.as);
  char* rest = ws + L.rest;
  const size_t rest_bytes = ws_bytes - L.rest;
  const long long groups = (long long)T * ceil_div(H, 128);
  // four pairs of groups a turn where every warp has several turns of one (8192 x 8192: 64 us, 71 with one)
  const bool many = groups >= 8ll * 2 * 64 * sms;
  rc = launch("feed-forward quantisation", many ? ffn_quant_kernel<4> : ffn_quant_kernel<1>,
              dim3(grid_for((groups + (many ? 63 : 15)) / (many ? 64 : 16), sms)), 256, 0, s, 0,
              static_cast<const __nv_bfloat16*>(x), groups, H, xq, xs);
  if (rc) return rc;
  if (fp8_streams(T, I, H, true, sms)) {
    rc = stream_gate(EK_DTYPE_E4M3, w1, w3, xq, {xs, s1, s3}, T, I, H, gate, nullptr, nullptr, aq, as, sms, rest,
                     rest_bytes, s, true);
  } else {
    Fp8BlockParams p{};
    p.M = T;
    p.N = I;
    p.tiles_m = ceil_div(T, 256);
    p.tiles_n = ceil_div(I, 128);
    p.k_blocks = ceil_div(H, 128);
    p.splits = fp8_gate_splits(T, I, H, sms, rest_bytes);
    p.ws = reinterpret_cast<float*>(rest);
    p.a_scale = xs;
    p.w_scale = s1;
    p.w_scale2 = s3;
    p.w_blocks = p.tiles_n;
    p.gate = gate;
    p.codes = aq;
    p.scales = as;
    rc = launch_fp8<true>(xq, w1, w3, H, p, sms, s);
    if (!rc && p.splits > 1) {
      StreamOut o{};
      o.T = T;
      o.N = I;
      o.gate = gate;
      o.codes = aq;
      o.scales = as;
      rc = launch("block-scaled gate sums", fp8_gate_reduce_kernel, dim3(p.tiles_n, ceil_div(T, 8)), 256, 0, s, 0,
                  (const float*)p.ws, p.splits, o);
    }
  }
  if (rc) return rc;
  return fp8_store(aq, w2, as, s2, y, T, H, I, kOutBF16, sms, rest, rest_bytes, s, true);
}

}  // extern "C"
