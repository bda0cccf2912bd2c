// The experts' products of a fused MoE layer with 4-bit weights.
#include "ek_moe_order.cuh"
#include "ek_w4_launch.cuh"

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
namespace {

using namespace w4;
using bf16 = __nv_bfloat16;

// Workspace: the tokens of both products and the sums of one (the down
// projection writes its sums after the gate/up's have been read).
struct MoeLayout {
  int nt, grid, max_y;
  size_t x, a, parts, bytes;
};
MoeLayout moe_layout(long long x_rows, int rows, int E, int H, int I, int sms) {
  MoeLayout l;
  l.nt = pick_nt(rows, E);
  l.grid = sms * kCtasPerSm;
  l.max_y = max_token_tiles(rows, E, l.nt);
  const int tok = 8 * l.nt;
  const long long ft1 = (I + kRows / 2 - 1) / (kRows / 2), ft2 = (H + kRows - 1) / kRows;
  const Layout x = layout(x_rows, H, l.max_y * ft1, l.grid, tok), a = layout(rows, I, l.max_y * ft2, l.grid, tok);
  l.x = 0;
  l.a = x.parts;
  l.parts = l.a + a.parts;
  l.bytes = l.parts + std::max(x.bytes - x.parts, a.bytes - a.parts);
  return l;
}

// The start of a layer in one launch, for up to kFrontSlots slots: the first
// CTA routes the tokens and orders their slots, the others write the tokens of
// the gate/up product, a warp per run. One CTA routes 32 tokens at a time and
// walks the warps' counts one after the other, so for more slots a launch for the
// routing and one for the order are sooner done. Measured, whole layers of
// 1024 x 512 in one launch against three: 2 slots, E = 8 15.8 against 17.5 us;
// 128 slots, E = 32 27.0 against 28.0, E = 8 25.8 against 24.8; 512 slots, E = 32
// 41.5 against 37.3, E = 256 85.7 against 70.9.
constexpr int kFrontSlots = 128;
struct Order {
  int *ids, *sorted_slots, *slot_rows, *counts;
  float* weights;
};
__global__ void __launch_bounds__(kOrderThreads)
    front_kernel(const float* __restrict__ logits, const bf16* __restrict__ x, int T, int k, int E, int H,
                 int group, bool vec, Order o, Tokens tokens) {
  extern __shared__ int sm[];
  griddep_launch();  // the next launch waits for the whole of this one
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = T * k;
  if (blockIdx.x > 0) {
    write_tokens(x, T, H, group, vec, tokens, (long long)(blockIdx.x - 1) * (kOrderThreads / 32) + warp,
                 (long long)(gridDim.x - 1) * (kOrderThreads / 32));
    return;
  }
  for (int t = warp; t < T; t += kOrderThreads / 32)
    route_token(logits + (size_t)t * E, E, k, lane, o.ids + (size_t)t * k, o.weights + (size_t)t * k);
  __syncthreads();
  int id = tid < n ? o.ids[tid] : -1;
  if (id >= E) {  // a row of NaN
    atomicOr(&g_ek_status, kStatusBadIndex);
    id = -1;
  }
  int kept;
  const int row = order_slots(id, n, E, sm, &kept);
  const int* start = sm + (n + 31) / 32 * E;
  if (tid < E) o.counts[tid] = (tid + 1 < E ? start[tid + 1] : kept) - start[tid];
  if (tid < n) {
    o.slot_rows[tid] = row;
    if (row >= 0) o.sorted_slots[row] = tid;
    if (tid >= kept) o.sorted_slots[tid] = n;
  }
}

struct Matrix {
  const void *codes, *scales, *mins;
};

const uint8_t* codes_of(const Matrix& m) { return static_cast<const uint8_t*>(m.codes); }
Scales<bf16> scales_of(const Matrix& m) { return {static_cast<const bf16*>(m.scales), static_cast<const bf16*>(m.mins)}; }

struct Moe {
  const int* counts;
  int rows, E, H, I, group;
  uint8_t* ws;
  MoeLayout l;
  cudaStream_t stream;
  size_t index_bytes() const { return (2 * E + 1) * sizeof(int); }
  Tokens x() const { return {ws + l.x}; }
  Tokens act() const { return {ws + l.a}; }

  Params<bf16> params(int K, int N, int features, const Tokens& tokens) const {
    Params<bf16> p = {};
    p.group = group;
    p.K = K;
    p.N = N;
    p.feature_tiles = (N + features - 1) / features;
    p.x = tokens;
    p.n_rows = rows;
    p.max_y = l.max_y;
    p.counts = counts;
    p.E = E;
    p.topk = 1;
    p.parts = reinterpret_cast<float*>(ws + l.parts);
    return p;
  }
  // x (x_rows of them; null: the tokens x() are being written by the launch
  // before, with the counts and the order) -> the sums of the gate/up product
  int gate_up(const bf16* xin, int x_rows, const int* sorted_slots, int topk, const Matrix& w1, const Matrix& w3,
              Params<bf16>* out) const {
    Params<bf16> p = params(H, I, kRows / 2, x());
    p.w[0] = scales_of(w1);
    p.w[1] = scales_of(w3);
    p.codes[0] = codes_of(w1);
    p.codes[1] = codes_of(w3);
    p.sorted_slots = sorted_slots;
    p.topk = topk;
    p.n_slots = rows;
    p.wait_first = xin == nullptr;
    *out = p;
    CUtensorMap m1, m3;
    int rc = codes_map(&m1, w1.codes, (long long)E * I, H, kRows / 2);
    if (!rc) rc = codes_map(&m3, w3.codes, (long long)E * I, H, kRows / 2);
    if (!rc && xin) rc = launch_tokens(xin, x_rows, H, group, p.x, stream);
    if (!rc) rc = launch_product<bf16, kGateUp>(l.nt, group, m1, m3, p, l.grid, stream);
    return rc;
  }
  // the tokens act() -> the sums of the down product
  int down(const Matrix& w2, Params<bf16>* out) const {
    Params<bf16> p = params(I, H, kRows, act());
    p.w[0] = scales_of(w2);
    p.codes[0] = codes_of(w2);
    *out = p;
    CUtensorMap m;
    const int rc = codes_map(&m, w2.codes, (long long)E * H, I, kRows);
    return rc ? rc : launch_product<bf16, kDown>(l.nt, group, m, m, p, l.grid, stream);
  }
  // One of the sums' launches: f(tokens per tile, minima) as constants.
  template <class F>
  int sums(const Params<bf16>& p, const F& f) const {
    using std::integral_constant;
    const integral_constant<int, 8> t8;
    const integral_constant<int, 16> t16;
    if (p.w[0].m) return l.nt == 1 ? f(t8, std::true_type{}) : f(t16, std::true_type{});
    return l.nt == 1 ? f(t8, std::false_type{}) : f(t16, std::false_type{});
  }
  template <Mode kMode, class O>
  int finish(const Params<bf16>& p, O* out) const {
    return sums(p, [&](auto tok, auto mins) {
      constexpr int TOK = decltype(tok)::value;
      const dim3 g(p.feature_tiles, std::min(l.max_y * TOK, 4096));
      return launch("w4 sums launch", finish_kernel<kMode, TOK, decltype(mins)::value, bf16, O>, g, kRows, index_bytes(),
                    stream, false, p, l.grid, out);
    });
  }
  // gate/up, down and combine, from an order of the slots
  int layer(const bf16* xin, const Order& o, int T, int topk, const Matrix& w1, const Matrix& w3, const Matrix& w2,
            bf16* out) const {
    Params<bf16> p;
    int rc = gate_up(xin, T, o.sorted_slots, topk, w1, w3, &p);
    if (!rc) rc = act_tokens(p);
    if (!rc) rc = down(w2, &p);
    return rc ? rc : combine(p, o.slot_rows, o.ids, o.weights, T, topk, out);
  }
  int act_tokens(const Params<bf16>& p) const {
    return sums(p, [&](auto tok, auto mins) {
      constexpr int TOK = decltype(tok)::value;
      const long long warps = (long long)l.max_y * TOK * stages(I);
      return launch("w4 act launch", act_tokens_kernel<TOK, decltype(mins)::value, bf16>,
                    dim3((unsigned)std::min<long long>((warps + 7) / 8, 148 * 8)), 256, index_bytes(), stream, false, p,
                    l.grid, group, act());
    });
  }
  int combine(const Params<bf16>& p, const int* slot_rows, const int* ids, const float* weights, int T, int topk,
              bf16* out) const {
    return sums(p, [&](auto tok, auto mins) {
      return launch("w4 combine launch", combine_parts_kernel<decltype(tok)::value, decltype(mins)::value, bf16>,
                    dim3(p.feature_tiles, std::min(T, 4096)), kRows, index_bytes(), stream, false, p, l.grid, slot_rows,
                    ids, weights, T, topk, out);
    });
  }
};

int open_moe(const char* what, Moe* m, long long x_rows, const int* counts, int rows, int E, int H, int I, int group,
             int num_sms, void* workspace, size_t ws_bytes, void* stream) {
  if (!counts || !workspace) return set_error(EK_ERR_INVALID, "%s: null pointer", what);
  int sms = 0;
  const int rc = resolve_num_sms(num_sms, stream, &sms);
  if (rc) return rc;
  *m = {counts, rows, E, H, I, group, static_cast<uint8_t*>(workspace), moe_layout(x_rows, rows, E, H, I, sms),
        static_cast<cudaStream_t>(stream)};
  if (!aligned16(workspace) || ws_bytes < m->l.bytes)
    return set_error(EK_ERR_INVALID, "%s: workspace must be 16-byte aligned and hold %zu bytes (got %zu)", what, m->l.bytes,
                     ws_bytes);
  return EK_OK;
}

int check_sizes(const char* what, long long x_rows, long long rows, int E, int H, int I) {
  if (x_rows < 0 || rows < 0 || E < 1 || E > 1024 || H < 1 || I < 1 || std::max(H, I) > kMaxK || (long long)E * std::max(H, I) > 0x7fffffffll)
    return set_error(EK_ERR_INVALID, "%s: bad sizes (rows=%lld E=%d H=%d I=%d)", what, rows, E, H, I);
  if (rows > (1ll << 24)) return set_error(EK_ERR_INVALID, "%s: too many rows", what);
  return EK_OK;
}

bool misaligned16bit(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 1u) return true;
  return false;
}

}  // namespace
}  // namespace ek

using namespace ek;

extern "C" {

size_t ek_moe_w4_workspace_bytes(int x_rows, int rows, int E, int H, int I, int num_sms) {
  if (num_sms < 1 || check_sizes("w4 workspace", x_rows, rows, E, H, I)) return (size_t)-1;
  return rows == 0 ? 0 : moe_layout(x_rows, rows, E, H, I, num_sms).bytes;
}

int ek_moe_gate_up_w4(const void* x, int x_rows, const int* sorted_slots, int topk, const void* w1_codes,
                      const void* w1_scales, const void* w1_mins, const void* w3_codes, const void* w3_scales,
                      const void* w3_mins, const int* expert_counts, void* act, int act_dtype, int rows, int E, int H,
                      int I, int group, int num_sms, void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  int rc = check_sizes("gate_up_w4", x_rows, rows, E, H, I);
  if (rc) return rc;
  if (act_dtype != EK_DTYPE_BF16 && act_dtype != EK_DTYPE_FP32)
    return set_error(EK_ERR_INVALID, "gate_up_w4: act must be bf16 or fp32 (dtype=%d)", act_dtype);
  if (topk < 1 || (long long)x_rows * (sorted_slots ? topk : 1) != rows)
    return set_error(EK_ERR_INVALID, "gate_up_w4: %d rows do not match %d of x (topk=%d)", rows, x_rows, topk);
  if (rows == 0) return EK_OK;
  rc = check_w4("gate_up_w4", w1_codes, w1_scales, w1_mins, (long long)E * I, H, group);
  if (!rc) rc = check_w4("gate_up_w4", w3_codes, w3_scales, w3_mins, (long long)E * I, H, group);
  if (rc) return rc;
  if (!x || !act || !w1_mins != !w3_mins) return set_error(EK_ERR_INVALID, "gate_up_w4: null pointer");
  if (misaligned16bit({x, act}) || (act_dtype == EK_DTYPE_FP32 && (reinterpret_cast<uintptr_t>(act) & 3u)))
    return set_error(EK_ERR_INVALID, "gate_up_w4: x and act must be aligned to their elements");
  Moe m;
  rc = open_moe("gate_up_w4", &m, x_rows, expert_counts, rows, E, H, I, group, num_sms, workspace, ws_bytes, stream);
  Params<bf16> p;
  if (!rc)
    rc = m.gate_up(static_cast<const bf16*>(x), x_rows, sorted_slots, topk, {w1_codes, w1_scales, w1_mins},
                   {w3_codes, w3_scales, w3_mins}, &p);
  if (rc) return rc;
  return act_dtype == EK_DTYPE_BF16 ? m.finish<kGateUp>(p, static_cast<bf16*>(act)) : m.finish<kGateUp>(p, static_cast<float*>(act));
}

int ek_moe_down_w4(const void* act, int act_dtype, const void* w2_codes, const void* w2_scales, const void* w2_mins,
                   const int* expert_counts, void* y, int y_dtype, int rows, int E, int H, int I, int group,
                   int num_sms, void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  int rc = check_sizes("down_w4", 0, rows, E, H, I);
  if (rc) return rc;
  if ((act_dtype != EK_DTYPE_BF16 && act_dtype != EK_DTYPE_FP32) || (y_dtype != EK_DTYPE_BF16 && y_dtype != EK_DTYPE_FP32))
    return set_error(EK_ERR_INVALID, "down_w4: act and y must be bf16 or fp32 (dtypes %d, %d)", act_dtype, y_dtype);
  if (rows == 0) return EK_OK;
  rc = check_w4("down_w4", w2_codes, w2_scales, w2_mins, (long long)E * H, I, group);
  if (rc) return rc;
  if (!act || !y) return set_error(EK_ERR_INVALID, "down_w4: null pointer");
  if (misaligned16bit({act, y}) || (act_dtype == EK_DTYPE_FP32 && (reinterpret_cast<uintptr_t>(act) & 3u)) ||
      (y_dtype == EK_DTYPE_FP32 && (reinterpret_cast<uintptr_t>(y) & 3u)))
    return set_error(EK_ERR_INVALID, "down_w4: act and y must be aligned to their elements");
  Moe m;
  rc = open_moe("down_w4", &m, 0, expert_counts, rows, E, H, I, group, num_sms, workspace, ws_bytes, stream);
  if (!rc)
    rc = act_dtype == EK_DTYPE_BF16 ? launch_tokens(static_cast<const bf16*>(act), rows, I, group, m.act(), m.stream)
                                    : launch_tokens(static_cast<const float*>(act), rows, I, group, m.act(), m.stream);
  Params<bf16> p;
  if (!rc) rc = m.down({w2_codes, w2_scales, w2_mins}, &p);
  if (rc) return rc;
  return y_dtype == EK_DTYPE_BF16 ? m.finish<kDown>(p, static_cast<bf16*>(y)) : m.finish<kDown>(p, static_cast<float*>(y));
}

int ek_moe_experts_w4(const void* x, int T, int topk, const int* topk_ids, const float* topk_weights,
                      const int* sorted_slots, const int* slot_rows, const int* expert_counts, const void* w1_codes,
                      const void* w1_scales, const void* w1_mins, const void* w3_codes, const void* w3_scales,
                      const void* w3_mins, const void* w2_codes, const void* w2_scales, const void* w2_mins, void* out,
                      int E, int H, int I, int group, int num_sms, void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  const long long rows = (long long)T * topk;
  int rc = topk < 1 ? set_error(EK_ERR_INVALID, "experts_w4: bad sizes (topk=%d)", topk)
                    : check_sizes("experts_w4", T, rows, E, H, I);
  if (rc || T == 0) return rc;
  rc = check_w4("experts_w4", w1_codes, w1_scales, w1_mins, (long long)E * I, H, group);
  if (!rc) rc = check_w4("experts_w4", w3_codes, w3_scales, w3_mins, (long long)E * I, H, group);
  if (!rc) rc = check_w4("experts_w4", w2_codes, w2_scales, w2_mins, (long long)E * H, I, group);
  if (rc) return rc;
  if (!x || !out || !topk_ids || !topk_weights || !sorted_slots || !slot_rows || !w1_mins != !w3_mins)
    return set_error(EK_ERR_INVALID, "experts_w4: null pointer");
  if (misaligned16bit({x, out})) return set_error(EK_ERR_INVALID, "experts_w4: x and out must be aligned to their elements");
  Moe m;
  rc = open_moe("experts_w4", &m, T, expert_counts, (int)rows, E, H, I, group, num_sms, workspace, ws_bytes, stream);
  if (rc) return rc;
  // the maps are read only
  const Order o{const_cast<int*>(topk_ids), const_cast<int*>(sorted_slots), const_cast<int*>(slot_rows),
                const_cast<int*>(expert_counts), const_cast<float*>(topk_weights)};
  return m.layer(static_cast<const bf16*>(x), o, T, topk, {w1_codes, w1_scales, w1_mins}, {w3_codes, w3_scales, w3_mins},
                 {w2_codes, w2_scales, w2_mins}, static_cast<bf16*>(out));
}

size_t ek_fused_moe_w4_workspace_bytes(int T, int topk, int E, int H, int I, int num_sms) {
  if (T < 0 || topk < 1 || topk > kRouteMaxK || E < 1 || E > kRouteMaxE) return (size_t)-1;
  const size_t experts = ek_moe_w4_workspace_bytes(T, (int)std::min<long long>((long long)T * topk, 0x7fffffff), E, H, I, num_sms);
  if (experts == (size_t)-1 || T == 0) return experts;
  return experts + 256 + ((size_t)4 * T * topk + E + 1) * sizeof(int) + ek_moe_permute_scratch_bytes(T, topk, E);
}

int ek_fused_moe_w4(const void* x, const float* logits, int T, int topk, const void* w1_codes, const void* w1_scales,
                    const void* w1_mins, const void* w3_codes, const void* w3_scales, const void* w3_mins,
                    const void* w2_codes, const void* w2_scales, const void* w2_mins, void* out, int E, int H, int I,
                    int group, int num_sms, void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  if (E < 1 || E > kRouteMaxE || topk < 1 || topk > kRouteMaxK || topk > E)
    return set_error(EK_ERR_INVALID, "fused_moe_w4: need 1 <= E <= %d and 1 <= k <= min(%d, E) (E=%d k=%d)", kRouteMaxE,
                     kRouteMaxK, E, topk);
  const long long rows = (long long)T * topk;
  int rc = check_sizes("fused_moe_w4", T, rows, E, H, I);
  if (rc || T == 0) return rc;
  rc = check_w4("fused_moe_w4", w1_codes, w1_scales, w1_mins, (long long)E * I, H, group);
  if (!rc) rc = check_w4("fused_moe_w4", w3_codes, w3_scales, w3_mins, (long long)E * I, H, group);
  if (!rc) rc = check_w4("fused_moe_w4", w2_codes, w2_scales, w2_mins, (long long)E * H, I, group);
  if (rc) return rc;
  if (!x || !logits || !out || !workspace || !w1_mins != !w3_mins)
    return set_error(EK_ERR_INVALID, "fused_moe_w4: null pointer");
  if (misaligned16bit({x, out}) || (reinterpret_cast<uintptr_t>(logits) & 3u))
    return set_error(EK_ERR_INVALID, "fused_moe_w4: x, logits and out must be aligned to their elements");
  int sms = 0;
  rc = resolve_num_sms(num_sms, stream, &sms);
  if (rc) return rc;
  const size_t need = ek_fused_moe_w4_workspace_bytes(T, topk, E, H, I, sms);
  if (!aligned16(workspace) || ws_bytes < need)
    return set_error(EK_ERR_INVALID, "fused_moe_w4: workspace must be 16-byte aligned and hold %zu bytes (got %zu)", need,
                     ws_bytes);
  const size_t experts = ek_moe_w4_workspace_bytes(T, (int)rows, E, H, I, sms);
  int* ints = reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + (experts + 255) / 256 * 256);
  const int n = (int)rows;
  const Order o{ints, ints + n, ints + 2 * n, ints + 4 * n, reinterpret_cast<float*>(ints + 3 * n)};
  Moe m;
  rc = open_moe("fused_moe_w4", &m, T, o.counts, n, E, H, I, group, sms, workspace, experts, stream);
  if (rc) return rc;
  const bf16* xin = static_cast<const bf16*>(x);
  if (n <= kFrontSlots) {
    const int warps = T * stages(H), per = kOrderThreads / 32;
    const int grid = 1 + std::min((warps + per - 1) / per, 147);
    rc = launch("w4 front launch", front_kernel, dim3(grid), kOrderThreads, order_smem_ints(n, E) * sizeof(int), m.stream,
                true, logits, xin, T, topk, E, H, group, H % 8 == 0 && aligned16(xin), o, m.x());
    xin = nullptr;
  } else {
    rc = ek_moe_route(logits, T, E, topk, o.ids, o.weights, stream);
    if (!rc)
      rc = ek_moe_dispatch(o.ids, T, topk, E, nullptr, 0, 0, o.sorted_slots, o.slot_rows, o.counts, o.counts + E, nullptr,
                           o.counts + E + 1, stream);
  }
  if (rc) return rc;
  return m.layer(xin, o, T, topk, {w1_codes, w1_scales, w1_mins}, {w3_codes, w3_scales, w3_mins},
                 {w2_codes, w2_scales, w2_mins}, static_cast<bf16*>(out));
}

}  // extern "C"
