// The experts' products of a fused MoE layer with 4-bit weights.
#include "ek_w4_kernel.cuh"

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
  size_t x, xs, a, as, parts, bytes;
};
MoeLayout moe_layout(long long x_rows, int rows, int E, int H, int I, int sms) {
  MoeLayout l;
  l.nt = pick_nt(rows, E);
  l.grid = sms * occupancy(l.nt);
  l.max_y = max_token_tiles(rows, E, l.nt);
  const int tok = 8 * l.nt;
  const long long ft1 = (I + kRows / 2 - 1) / (kRows / 2), ft2 = (H + kRows - 1) / kRows;
  const Layout x = layout(x_rows, H, l.max_y * ft1, l.grid, tok), a = layout(rows, I, l.max_y * ft2, l.grid, tok);
  l.x = 0;
  l.xs = x.scales;
  l.a = x.parts;
  l.as = l.a + a.scales;
  l.parts = l.a + a.parts;
  l.bytes = l.parts + std::max(x.bytes - x.parts, a.bytes - a.parts);
  return l;
}

struct Matrix {
  const void *codes, *scales, *mins;
};

Scales<bf16> scales_of(const Matrix& m) { return {static_cast<const bf16*>(m.scales), static_cast<const bf16*>(m.mins)}; }

struct Moe {
  const int* counts;
  int rows, E, H, I, group;
  uint8_t* ws;
  MoeLayout l;
  cudaStream_t stream;
  size_t index_bytes() const { return (2 * E + 1) * sizeof(int); }
  Tokens x() const { return {reinterpret_cast<__half*>(ws + l.x), reinterpret_cast<float*>(ws + l.xs)}; }
  Tokens act() const { return {reinterpret_cast<__half*>(ws + l.a), reinterpret_cast<float*>(ws + l.as)}; }

  Params<bf16> params(int K, int N, int features, const Tokens& tokens) const {
    Params<bf16> p = {};
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
  // x (x_rows of them) -> the sums of the gate/up product
  int gate_up(const bf16* xin, int x_rows, const int* sorted_slots, int topk, const Matrix& w1, const Matrix& w3,
              Params<bf16>* out) const {
    Params<bf16> p = params(H, I, kRows / 2, x());
    p.w[0] = scales_of(w1);
    p.w[1] = scales_of(w3);
    p.sorted_slots = sorted_slots;
    p.topk = topk;
    p.n_slots = rows;
    *out = p;
    CUtensorMap m1, m3;
    int rc = codes_map(&m1, w1.codes, (long long)E * I, H, kRows / 2);
    if (!rc) rc = codes_map(&m3, w3.codes, (long long)E * I, H, kRows / 2);
    if (!rc) rc = launch_tokens(xin, x_rows, H, p.x, stream, true);
    if (!rc) rc = launch_product<bf16, kGateUp>(l.nt, group, m1, m3, p, l.grid, stream);
    return rc;
  }
  // the tokens act() -> the sums of the down product
  int down(const Matrix& w2, Params<bf16>* out) const {
    Params<bf16> p = params(I, H, kRows, act());
    p.w[0] = scales_of(w2);
    *out = p;
    CUtensorMap m;
    const int rc = codes_map(&m, w2.codes, (long long)E * H, I, kRows);
    return rc ? rc : launch_product<bf16, kDown>(l.nt, group, m, m, p, l.grid, stream);
  }
  template <Mode kMode, int TOK, class O>
  int finish_tok(const Params<bf16>& p, O* out) const {
    const dim3 g(p.feature_tiles, std::min(l.max_y * TOK, 4096));
    return launch("w4 sums launch", finish_kernel<kMode, TOK, bf16, O>, g, kRows, index_bytes(), stream, false, p, l.grid, out);
  }
  template <Mode kMode, class O>
  int finish(const Params<bf16>& p, O* out) const {
    return l.nt == 1 ? finish_tok<kMode, 8>(p, out) : l.nt == 2 ? finish_tok<kMode, 16>(p, out) : finish_tok<kMode, 32>(p, out);
  }
  template <int TOK>
  int act_tokens(const Params<bf16>& p) const {
    const long long warps = (long long)l.max_y * TOK * stages(I);
    return launch("w4 act launch", act_tokens_kernel<TOK, bf16>, dim3((unsigned)std::min<long long>((warps + 7) / 8, 148 * 8)),
                  256, index_bytes(), stream, false, p, l.grid, act());
  }
  template <int TOK>
  int combine(const Params<bf16>& p, const int* slot_rows, const int* ids, const float* weights, int T, int topk,
              bf16* out) const {
    return launch("w4 combine launch", combine_parts_kernel<TOK, bf16>, dim3(p.feature_tiles, std::min(T, 4096)), kRows,
                  index_bytes(), stream, false, p, l.grid, slot_rows, ids, weights, T, topk, out);
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
  if (x_rows < 0 || rows < 0 || E < 1 || E > 1024 || H < 1 || I < 1 || (long long)E * std::max(H, I) > 0x7fffffffll)
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
  rc = check_w4("gate_up_w4", w1_codes, w1_scales, w1_mins, H, group);
  if (!rc) rc = check_w4("gate_up_w4", w3_codes, w3_scales, w3_mins, H, group);
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
  rc = check_w4("down_w4", w2_codes, w2_scales, w2_mins, I, group);
  if (rc) return rc;
  if (!act || !y) return set_error(EK_ERR_INVALID, "down_w4: null pointer");
  if (misaligned16bit({act, y}) || (act_dtype == EK_DTYPE_FP32 && (reinterpret_cast<uintptr_t>(act) & 3u)) ||
      (y_dtype == EK_DTYPE_FP32 && (reinterpret_cast<uintptr_t>(y) & 3u)))
    return set_error(EK_ERR_INVALID, "down_w4: act and y must be aligned to their elements");
  Moe m;
  rc = open_moe("down_w4", &m, 0, expert_counts, rows, E, H, I, group, num_sms, workspace, ws_bytes, stream);
  if (!rc)
    rc = act_dtype == EK_DTYPE_BF16 ? launch_tokens(static_cast<const bf16*>(act), rows, I, m.act(), m.stream, true)
                                    : launch_tokens(static_cast<const float*>(act), rows, I, m.act(), m.stream, true);
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
  rc = check_w4("experts_w4", w1_codes, w1_scales, w1_mins, H, group);
  if (!rc) rc = check_w4("experts_w4", w3_codes, w3_scales, w3_mins, H, group);
  if (!rc) rc = check_w4("experts_w4", w2_codes, w2_scales, w2_mins, I, group);
  if (rc) return rc;
  if (!x || !out || !topk_ids || !topk_weights || !sorted_slots || !slot_rows || !w1_mins != !w3_mins)
    return set_error(EK_ERR_INVALID, "experts_w4: null pointer");
  if (misaligned16bit({x, out})) return set_error(EK_ERR_INVALID, "experts_w4: x and out must be aligned to their elements");
  Moe m;
  rc = open_moe("experts_w4", &m, T, expert_counts, (int)rows, E, H, I, group, num_sms, workspace, ws_bytes, stream);
  Params<bf16> p;
  if (!rc)
    rc = m.gate_up(static_cast<const bf16*>(x), T, sorted_slots, topk, {w1_codes, w1_scales, w1_mins},
                   {w3_codes, w3_scales, w3_mins}, &p);
  if (!rc) rc = m.l.nt == 1 ? m.act_tokens<8>(p) : m.l.nt == 2 ? m.act_tokens<16>(p) : m.act_tokens<32>(p);
  if (!rc) rc = m.down({w2_codes, w2_scales, w2_mins}, &p);
  if (rc) return rc;
  bf16* o = static_cast<bf16*>(out);
  return m.l.nt == 1   ? m.combine<8>(p, slot_rows, topk_ids, topk_weights, T, topk, o)
         : m.l.nt == 2 ? m.combine<16>(p, slot_rows, topk_ids, topk_weights, T, topk, o)
                       : m.combine<32>(p, slot_rows, topk_ids, topk_weights, T, topk, o);
}

}  // extern "C"
