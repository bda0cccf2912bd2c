"""Torch-tensor front end of the C-ABI: argument checks, scratch management and
stream plumbing. Every launch goes to the *current* torch stream, which is
how a green-context partition stream reaches the kernels (the reference
relies on the same mechanism, sm_aware_matmul.py:270).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, _workspace
from ._lib import check, lib

_DTYPES = {torch.bfloat16: _lib.EK_DTYPE_BF16, torch.float16: _lib.EK_DTYPE_FP16}
_FP8 = getattr(torch, "float8_e4m3fn", None)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _require_cuda(*ts: torch.Tensor) -> torch.device:
    dev, index = None, -1
    for t in ts:
        if t is None:
            continue
        i = t.get_device()  # an int: cheaper than building and comparing devices
        if i < 0 or (dev is None and not t.is_cuda):
            raise RuntimeError("elastikernel_b200 operators take CUDA tensors only (no CPU path)")
        if dev is None:
            dev, index = t.device, i
        elif i != index or not t.is_cuda:
            raise RuntimeError(f"tensors on different devices: {dev} vs {t.device}")
    return dev


def _contig(name: str, t: torch.Tensor) -> None:
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def plan(M: int, N: int, K: int, num_sms: int, dtype=torch.bfloat16, b_layout: str = "kn", force_bn: int = 0,
         force_split: int = 0) -> dict:
    """Tile schedule the kernel would use for this shape on `num_sms` SMs (CPU-only call)."""
    p = _lib.GemmPlan()
    dt = _lib.EK_DTYPE_E4M3 if (_FP8 is not None and dtype == _FP8) else _DTYPES[dtype]
    bl = _lib.EK_B_KN if b_layout == "kn" else _lib.EK_B_NK
    check(lib().ek_gemm_plan_make(int(M), int(N), int(K), int(num_sms), dt, bl, int(force_bn), int(force_split),
                                  ctypes.byref(p)), "ek_gemm_plan_make")
    return p.as_dict()


# torch's own accessors of the current device and raw stream: the public ones
# build a Stream object per call (2-3 us, as much as a small launch)
_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_CURRENT_DEVICE = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def current_stream_handle(device: torch.device) -> int:
    if _RAW_STREAM is None or device.index is None:
        return _lib.stream_ptr(torch.cuda.current_stream(device))
    return _RAW_STREAM(device.index)


def gemm(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None, num_sms: int | None = None,
         b_layout: str = "kn", force_bn: int = 0, force_split: int = 0) -> torch.Tensor:
    """C = A @ B on the tcgen05 kernel.

    a: [M, K]; b: [K, N] (b_layout="kn", the reference's layout) or [N, K]
    (b_layout="nk"); bf16 or fp16; result in the input dtype.
    num_sms=None plans for the partition the current stream belongs to.
    """
    dev = _require_cuda(a, b, out)
    if a.dtype not in _DTYPES or b.dtype != a.dtype:
        raise RuntimeError(f"gemm takes bf16/fp16 operands of one dtype, got {a.dtype}, {b.dtype}")
    if a.dim() != 2 or b.dim() != 2:
        raise RuntimeError("gemm takes 2-D operands")
    _contig("a", a)
    _contig("b", b)
    M, K = a.shape
    if b_layout == "kn":
        K2, N = b.shape
        bl = _lib.EK_B_KN
    elif b_layout == "nk":
        N, K2 = b.shape
        bl = _lib.EK_B_NK
    else:
        raise ValueError(f"b_layout must be 'kn' or 'nk', got {b_layout!r}")
    if K2 != K:
        raise RuntimeError(f"inner dimensions differ: {K} vs {K2}")
    if out is None:
        out = torch.empty((M, N), device=dev, dtype=a.dtype)
    elif out.shape != (M, N) or out.dtype != a.dtype or not out.is_contiguous():
        raise RuntimeError("out must be a contiguous [M, N] tensor of the input dtype")
    if M == 0 or N == 0:
        return out
    if K == 0:
        return out.zero_()
    # the C-ABI takes 16-byte aligned operands (ragged shapes are padded
    # there); a view that starts mid-line is copied to a fresh device buffer
    if a.data_ptr() % 16:
        a = a.clone()
    if b.data_ptr() % 16:
        b = b.clone()
    if out.data_ptr() % 16:
        tmp = gemm(a, b, None, num_sms, b_layout, force_bn, force_split)
        return out.copy_(tmp)
    L = lib()
    stream = current_stream_handle(dev)
    sms = int(num_sms) if num_sms else _stream_sms(dev, stream)
    dt = _DTYPES[a.dtype]
    need = L.ek_gemm_workspace_bytes(M, N, K, sms, dt, bl, int(force_bn), int(force_split))
    if need == _SIZE_MAX:
        check(_lib.EK_ERR_INVALID, "ek_gemm_workspace_bytes")
    ws = _workspace.get(dev, stream, need)
    with _on_device(dev):
        check(L.ek_gemm(a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, dt, bl, sms, int(force_bn),
                        int(force_split), _ptr(ws), 0 if ws is None else ws.numel(), stream), "ek_gemm")
    return out


def gemm_fp8(a_q: torch.Tensor, w_q: torch.Tensor, a_scale: torch.Tensor, w_scale: torch.Tensor,
             out: torch.Tensor | None = None, num_sms: int | None = None, force_bn: int = 0,
             force_split: int = 0) -> torch.Tensor:
    """bf16 C[M,N] = (a_q * a_scale[:,None]) @ (w_q * w_scale[:,None])^T with e4m3 a_q [M,K], w_q [N,K]."""
    dev = _require_cuda(a_q, w_q, a_scale, w_scale, out)
    if _FP8 is None or a_q.dtype != _FP8 or w_q.dtype != _FP8:
        raise RuntimeError("gemm_fp8 takes float8_e4m3fn operands")
    for n, t in (("a_q", a_q), ("w_q", w_q), ("a_scale", a_scale), ("w_scale", w_scale)):
        _contig(n, t)
    if a_scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise RuntimeError("scales must be float32")
    M, K = a_q.shape
    N, K2 = w_q.shape
    if K2 != K or a_scale.numel() != M or w_scale.numel() != N:
        raise RuntimeError("shape mismatch in gemm_fp8")
    if out is None:
        out = torch.empty((M, N), device=dev, dtype=torch.bfloat16)
    stream = current_stream_handle(dev)
    sms = int(num_sms) if num_sms else _stream_sms(dev, stream)
    need = lib().ek_gemm_workspace_bytes(M, N, K, sms, _lib.EK_DTYPE_E4M3, _lib.EK_B_NK, int(force_bn),
                                         int(force_split))
    if need == _SIZE_MAX:
        check(_lib.EK_ERR_INVALID, "ek_gemm_workspace_bytes")
    ws = _workspace.get(dev, stream, need)
    with _on_device(dev):
        check(lib().ek_gemm_fp8(a_q.data_ptr(), w_q.data_ptr(), a_scale.data_ptr(), w_scale.data_ptr(),
                                out.data_ptr(), M, N, K, sms, int(force_bn), int(force_split), _ptr(ws),
                                0 if ws is None else ws.numel(), stream), "ek_gemm_fp8")
    return out


def quant_e4m3(x: torch.Tensor, block: tuple[int, int] = (1, 0), pow2: bool = False) -> tuple[torch.Tensor,
                                                                                              torch.Tensor]:
    """e4m3 codes and fp32 scales (amax / 448 per block) of a bf16/fp32 [rows, cols] tensor.

    block = (1, 0): one scale per row; (1, 128): per 1 x 128 group;
    (br, bc): per br x bc block. Scales come back shaped [ceil(rows/br), ceil(cols/bc)]
    (or [rows] for row-wise). pow2=True rounds every scale up to a power of
    two (the UE8M0 scale factors of the block-scaled GEMMs)."""
    dev = _require_cuda(x)
    if x.dtype not in (torch.bfloat16, torch.float32) or x.dim() != 2:
        raise RuntimeError("quant_e4m3 takes a 2-D bf16 or fp32 tensor")
    _contig("x", x)
    if _FP8 is None:
        raise RuntimeError("this torch has no float8_e4m3fn")
    rows, cols = x.shape
    br, bc = int(block[0]), int(block[1])
    q = torch.empty((rows, cols), dtype=_FP8, device=dev)
    if br == 1 and bc <= 0:
        scales = torch.empty(rows, dtype=torch.float32, device=dev)
    else:
        scales = torch.empty((-(-rows // br), -(-cols // bc)), dtype=torch.float32, device=dev)
    with _on_device(dev):
        check(lib().ek_quant_e4m3_ex(x.data_ptr(), 0 if x.dtype == torch.bfloat16 else 3, rows, cols, br, bc,
                                     _lib.EK_QUANT_POW2_SCALES if pow2 else 0, q.data_ptr(), scales.data_ptr(),
                                     current_stream_handle(dev)), "ek_quant_e4m3_ex")
    return q, scales


def quant_e4m3_kmajor(x: torch.Tensor, pow2: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes and 1 x 128 group scales of a bf16/fp32 [rows, cols] tensor, the
    scales K-block-major: [ceil(cols/128), rows] (the transpose of quant_e4m3's
    (1, 128) scales, bit for bit). The FP8 block-scaled MoE GEMMs take this layout.
    pow2=True: power-of-two scales, as quant_e4m3."""
    dev = _require_cuda(x)
    if x.dtype not in (torch.bfloat16, torch.float32) or x.dim() != 2:
        raise RuntimeError("quant_e4m3_kmajor takes a 2-D bf16 or fp32 tensor")
    _contig("x", x)
    if _FP8 is None:
        raise RuntimeError("this torch has no float8_e4m3fn")
    rows, cols = x.shape
    q = torch.empty((rows, cols), dtype=_FP8, device=dev)
    scales = torch.empty((-(-cols // 128), rows), dtype=torch.float32, device=dev)
    with _on_device(dev):
        check(lib().ek_quant_e4m3_kmajor_ex(x.data_ptr(), 0 if x.dtype == torch.bfloat16 else 3, rows, cols,
                                            _lib.EK_QUANT_POW2_SCALES if pow2 else 0, q.data_ptr(),
                                            scales.data_ptr(), current_stream_handle(dev)), "ek_quant_e4m3_kmajor_ex")
    return q, scales


def moe_gather_cols_f32(perm: dict, src: torch.Tensor) -> torch.Tensor:
    """[cols, max_rows] fp32: column c, row r = src[sorted_slots[r] // topk, c] (0 for
    unused rows) - per-row values such as received group scales, gathered in the
    permutation's order and transposed to the K-block-major layout."""
    dev = _require_cuda(src)
    if src.dtype != torch.float32 or src.dim() != 2:
        raise RuntimeError("moe_gather_cols_f32 takes a 2-D fp32 tensor")
    _contig("src", src)
    rows, cols = perm["max_rows"], src.shape[1]
    dst = torch.empty((cols, rows), dtype=torch.float32, device=dev)
    with _on_device(dev):
        check(lib().ek_moe_gather_cols_f32(perm["sorted_slots"].data_ptr(), perm["num_rows_padded"].data_ptr(), rows,
                                           perm["T"] * perm["topk"], perm["topk"], src.data_ptr(), cols,
                                           dst.data_ptr(), current_stream_handle(dev)), "ek_moe_gather_cols_f32")
    return dst


_SIZE_MAX = ctypes.c_size_t(-1).value
_DEV_SMS: dict[int, int] = {}


class _NullCtx:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_NULL = _NullCtx()


def _on_device(dev: torch.device):
    """Make `dev` current for a launch (a no-op when it already is)."""
    return _NULL if dev.index is None or dev.index == _CURRENT_DEVICE() else torch.cuda.device(dev)


def _stream_sms(dev: torch.device, stream: int) -> int:
    """SM count of the partition `stream` belongs to (registry), else the device's."""
    v = ctypes.c_int(0)
    check(lib().ek_gctx_stream_sm_count(ctypes.c_void_p(stream), ctypes.byref(v)), "ek_gctx_stream_sm_count")
    if v.value > 0:
        return v.value
    return _device_sms(dev)


def _device_sms(dev: torch.device) -> int:
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    n = _DEV_SMS.get(idx)
    if n is None:
        n = _DEV_SMS[idx] = torch.cuda.get_device_properties(idx).multi_processor_count
    return n


# ---------------------------------------------------------------------- MoE
BLOCK_M = 128


def moe_route(gate_logits: torch.Tensor, topk: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Softmax top-k routing (definition.py:152-153): int32 ids [T,k] and fp32
    renormalised weights [T,k]. Ties go to the lower expert id."""
    dev = _require_cuda(gate_logits)
    if gate_logits.dtype != torch.float32 or gate_logits.dim() != 2:
        raise RuntimeError("gate_logits must be a 2-D float32 tensor")
    _contig("gate_logits", gate_logits)
    T, E = gate_logits.shape
    ids = torch.empty((T, topk), dtype=torch.int32, device=dev)
    wts = torch.empty((T, topk), dtype=torch.float32, device=dev)
    with _on_device(dev):
        check(lib().ek_moe_route(gate_logits.data_ptr(), T, E, int(topk), ids.data_ptr(), wts.data_ptr(),
                                 current_stream_handle(dev)), "ek_moe_route")
    return ids, wts


def moe_permute(topk_ids: torch.Tensor, num_experts: int, x: torch.Tensor | None = None,
                block_m: int = BLOCK_M) -> dict:
    """Expert-sorted, block-padded layout of the (token, choice) slots, with the
    token rows of `x` gathered into it when given."""
    dev = _require_cuda(topk_ids, x)
    if topk_ids.dtype != torch.int32 or topk_ids.dim() != 2:
        raise RuntimeError("topk_ids must be a 2-D int32 tensor")
    _contig("topk_ids", topk_ids)
    T, k = topk_ids.shape
    E = int(num_experts)
    max_rows = int(lib().ek_moe_max_padded_rows(T, k, E, block_m))
    sorted_slots = torch.empty(max_rows, dtype=torch.int32, device=dev)
    block_expert = torch.empty(max_rows // block_m, dtype=torch.int32, device=dev)
    num_rows = torch.empty(1, dtype=torch.int32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    x_perm = None
    H = 0
    es = 0
    if x is not None:
        _contig("x", x)
        if x.dim() != 2 or x.shape[0] != T:
            raise RuntimeError("x must be [T, H]")
        H = x.shape[1]
        es = x.element_size()
        x_perm = torch.empty((max_rows, H), dtype=x.dtype, device=dev)
    scratch = torch.empty(int(lib().ek_moe_permute_scratch_bytes(T, k, E)), dtype=torch.uint8, device=dev)
    with _on_device(dev):
        check(lib().ek_moe_permute(topk_ids.data_ptr(), T, k, E, block_m, sorted_slots.data_ptr(),
                                   block_expert.data_ptr(), num_rows.data_ptr(), counts.data_ptr(), _ptr(x), H, es,
                                   _ptr(x_perm), scratch.data_ptr(), current_stream_handle(dev)), "ek_moe_permute")
    return {"sorted_slots": sorted_slots, "block_expert": block_expert, "num_rows_padded": num_rows,
            "expert_counts": counts, "x_perm": x_perm, "max_rows": max_rows, "T": T, "topk": k, "E": E,
            "block_m": block_m}


def moe_route_permute(gate_logits: torch.Tensor, topk: int, num_experts: int, x: torch.Tensor | None = None,
                      block_m: int = BLOCK_M) -> tuple[torch.Tensor, torch.Tensor, dict]:
    """moe_route then moe_permute (same outputs): ids, weights and the
    permutation dict. Up to 128 slots the routing, the permutation and a
    small row gather are one launch."""
    dev = _require_cuda(gate_logits, x)
    if gate_logits.dtype != torch.float32 or gate_logits.dim() != 2:
        raise RuntimeError("gate_logits must be a 2-D float32 tensor")
    _contig("gate_logits", gate_logits)
    T, E_logits = gate_logits.shape
    E = int(num_experts)
    if E_logits != E:
        raise RuntimeError("gate_logits must have one column per expert")
    k = int(topk)
    ids = torch.empty((T, k), dtype=torch.int32, device=dev)
    wts = torch.empty((T, k), dtype=torch.float32, device=dev)
    max_rows = int(lib().ek_moe_max_padded_rows(T, k, E, block_m))
    sorted_slots = torch.empty(max_rows, dtype=torch.int32, device=dev)
    block_expert = torch.empty(max_rows // block_m, dtype=torch.int32, device=dev)
    num_rows = torch.empty(1, dtype=torch.int32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    x_perm = None
    H = es = 0
    if x is not None:
        _contig("x", x)
        if x.dim() != 2 or x.shape[0] != T:
            raise RuntimeError("x must be [T, H]")
        H, es = x.shape[1], x.element_size()
        x_perm = torch.empty((max_rows, H), dtype=x.dtype, device=dev)
    scratch = torch.empty(int(lib().ek_moe_permute_scratch_bytes(T, k, E)), dtype=torch.uint8, device=dev)
    with _on_device(dev):
        check(lib().ek_moe_route_permute(gate_logits.data_ptr(), T, E, k, ids.data_ptr(), wts.data_ptr(), block_m,
                                         sorted_slots.data_ptr(), block_expert.data_ptr(), num_rows.data_ptr(),
                                         counts.data_ptr(), _ptr(x), H, es, _ptr(x_perm), scratch.data_ptr(),
                                         current_stream_handle(dev)), "ek_moe_route_permute")
    perm = {"sorted_slots": sorted_slots, "block_expert": block_expert, "num_rows_padded": num_rows,
            "expert_counts": counts, "x_perm": x_perm, "max_rows": max_rows, "T": T, "topk": k, "E": E,
            "block_m": block_m}
    return ids, wts, perm


def _check_bf16(name: str, t: torch.Tensor) -> None:
    if t.dtype != torch.bfloat16:
        raise RuntimeError(f"{name} must be bfloat16")
    _contig(name, t)


def _check_padded(perm: dict) -> None:
    if perm["block_expert"] is None:
        raise RuntimeError("the padded GEMMs take a moe_permute layout (moe_dispatch's is packed)")


def _slot_rows_out(perm: dict, H: int, dev: torch.device) -> torch.Tensor:
    """[T*k, H] bf16 for a product that scatters its rows to their slots. It writes
    the kept slots alone, so the others' rows are cleared where an order may
    have dropped some."""
    make = torch.empty if perm.get("slot_rows") is None else torch.zeros
    return make((perm["T"] * perm["topk"], H), dtype=torch.bfloat16, device=dev)


def moe_gate_up(perm: dict, w1: torch.Tensor, w3: torch.Tensor, num_sms: int | None = None,
                force_bn: int = 0) -> torch.Tensor:
    """act[r] = silu(x_perm[r] . w1[e]) * (x_perm[r] . w3[e]) over the padded rows
    (a layout padded to 256 rows per expert runs on CTA pairs)."""
    _check_padded(perm)
    x_perm = perm["x_perm"]
    dev = _require_cuda(x_perm, w1, w3)
    for n, t in (("x_perm", x_perm), ("w1", w1), ("w3", w3)):
        _check_bf16(n, t)
    E, I, H = w1.shape
    if w3.shape != w1.shape or x_perm.shape[1] != H or E != perm["E"]:
        raise RuntimeError("gate_up: shape mismatch")
    max_rows = perm["max_rows"]
    act = torch.empty((max_rows, I), dtype=torch.bfloat16, device=dev)
    stream = current_stream_handle(dev)
    with _on_device(dev):
        check(lib().ek_moe_gate_up(x_perm.data_ptr(), w1.data_ptr(), w3.data_ptr(), perm["block_expert"].data_ptr(),
                                   perm["num_rows_padded"].data_ptr(), act.data_ptr(), max_rows, E, H, I,
                                   perm["T"] * perm["topk"], int(num_sms or 0), int(force_bn), int(perm["block_m"]),
                                   stream), "ek_moe_gate_up")
    return act


def moe_down(perm: dict, act: torch.Tensor, w2: torch.Tensor, topk_weights: torch.Tensor,
             num_sms: int | None = None, force_bn: int = 0) -> torch.Tensor:
    """y[s] = topk_weight[s] * (act[r] @ w2[e]^T) for the slot s of each used row r."""
    _check_padded(perm)
    dev = _require_cuda(act, w2, topk_weights)
    _check_bf16("act", act)
    _check_bf16("w2", w2)
    _contig("topk_weights", topk_weights)
    if topk_weights.dtype != torch.float32:
        raise RuntimeError("topk_weights must be float32")
    E, H, I = w2.shape
    T, k = perm["T"], perm["topk"]
    if act.shape[1] != I or E != perm["E"] or topk_weights.numel() != T * k:
        raise RuntimeError("down: shape mismatch")
    y = torch.empty((T * k, H), dtype=torch.bfloat16, device=dev)
    with _on_device(dev):
        check(lib().ek_moe_down(act.data_ptr(), w2.data_ptr(), perm["block_expert"].data_ptr(),
                                perm["num_rows_padded"].data_ptr(), perm["sorted_slots"].data_ptr(),
                                topk_weights.data_ptr(), y.data_ptr(), perm["max_rows"], E, H, I, T, k,
                                int(num_sms or 0), int(force_bn), int(perm["block_m"]), current_stream_handle(dev)),
              "ek_moe_down")
    return y


def moe_gate_up_packed(perm: dict, w1: torch.Tensor, w3: torch.Tensor, num_sms: int | None = None,
                       tok_tile: int = 0, pair: int = -1, ksplit: bool = True) -> torch.Tensor:
    """Swapped-operand gate/up over the packed layout (permute with block_m=1).
    ksplit=False withholds the workspace, so K is never split."""
    x_perm = perm["x_perm"]
    dev = _require_cuda(x_perm, w1, w3)
    for n, t in (("x_perm", x_perm), ("w1", w1), ("w3", w3)):
        _check_bf16(n, t)
    if perm["block_m"] != 1:
        raise RuntimeError("the packed GEMMs take the packed layout (moe_permute(..., block_m=1))")
    E, I, H = w1.shape
    if w3.shape != w1.shape or x_perm.shape[1] != H or E != perm["E"]:
        raise RuntimeError("gate_up_packed: shape mismatch")
    rows = perm["max_rows"]
    act = torch.empty((rows, I), dtype=torch.bfloat16, device=dev)
    ws, nb = _packed_workspace(rows, H, I, dev) if ksplit else (None, 0)
    with _on_device(dev):
        check(lib().ek_moe_gate_up_packed(x_perm.data_ptr(), w1.data_ptr(), w3.data_ptr(),
                                          perm["expert_counts"].data_ptr(), act.data_ptr(), rows, E, H, I,
                                          int(tok_tile), int(pair), int(num_sms or 0), _ptr(ws), nb,
                                          current_stream_handle(dev)), "ek_moe_gate_up_packed")
    return act


def _packed_workspace(rows: int, H: int, I: int, dev: torch.device) -> tuple[torch.Tensor | None, int]:
    """Workspace of the packed GEMMs' K-split (None where the size never splits)."""
    nb = int(lib().ek_moe_packed_workspace_bytes(int(rows), int(H), int(I)))
    return (torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None), nb


def moe_down_packed(perm: dict, act: torch.Tensor, w2: torch.Tensor, topk_weights: torch.Tensor,
                    num_sms: int | None = None, tok_tile: int = 0, pair: int = -1,
                    ksplit: bool = True) -> torch.Tensor:
    """Swapped-operand down projection with the routing weight, scattered to slots
    (a slot that a moe_dispatch order dropped gets zeros). ksplit=False
    withholds the workspace, so K is never split."""
    dev = _require_cuda(act, w2, topk_weights)
    _check_bf16("act", act)
    _check_bf16("w2", w2)
    _contig("topk_weights", topk_weights)
    E, H, I = w2.shape
    T, k = perm["T"], perm["topk"]
    if act.shape[1] != I or E != perm["E"] or topk_weights.numel() != T * k or perm["block_m"] != 1:
        raise RuntimeError("down_packed: shape mismatch")
    y = _slot_rows_out(perm, H, dev)
    ws, nb = _packed_workspace(perm["max_rows"], H, I, dev) if ksplit else (None, 0)
    with _on_device(dev):
        check(lib().ek_moe_down_packed(act.data_ptr(), w2.data_ptr(), perm["expert_counts"].data_ptr(),
                                       perm["sorted_slots"].data_ptr(), topk_weights.data_ptr(), y.data_ptr(),
                                       perm["max_rows"], E, H, I, T, k, int(tok_tile), int(pair),
                                       int(num_sms or 0), _ptr(ws), nb, current_stream_handle(dev)),
              "ek_moe_down_packed")
    return y


def quant_moe_weights_fp8(w1: torch.Tensor, w2: torch.Tensor, w3: torch.Tensor, pow2: bool = False) -> dict:
    """e4m3 expert weights with 128 x 128 fp32 block scales (DeepSeek style).
    w1, w3 [E, I, H] and w2 [E, H, I] (bf16 or fp32); I and H multiples of 128.
    pow2=True: power-of-two block scales; the layer then quantises its tokens
    and activations the same way and runs the GEMMs whose tensor cores apply
    the scales (ek_moe_*_fp8mx)."""
    E, I, H = w1.shape
    if I % 128 or H % 128:
        raise RuntimeError("block-scaled FP8 needs I and H multiples of 128")
    out = {"E": E, "I": I, "H": H, "pow2": bool(pow2)}
    for name, w, rows, cols in (("w1", w1, I, H), ("w3", w3, I, H), ("w2", w2, H, I)):
        q, s = quant_e4m3(w.reshape(E * rows, cols).contiguous(), block=(128, 128), pow2=pow2)
        out[name + "q"] = q.view(E, rows, cols)
        out[name + "s"] = s
    return stack_gate_up_planes(out)


def stack_gate_up_planes(qw: dict) -> dict:
    """Store the e4m3 w1 and w3 codes as the two planes of one [2, E, I, H]
    buffer (w1q / w3q become views of it). The gate/up GEMMs then load a
    tile's [w1 rows | w3 rows] with one TMA box instead of two, which lets an
    SM draw about twice the HBM bandwidth (the TMA engine keeps only a few
    boxes in flight). Any layout stays correct; this one is faster. Call it
    again after concatenating the codes of several quantised shards."""
    w1q, w3q = qw["w1q"], qw["w3q"]
    if w1q.shape != w3q.shape:
        raise RuntimeError("w1q and w3q must have one shape")
    planes = torch.stack([w1q, w3q])
    qw = dict(qw)
    qw["w1q"], qw["w3q"] = planes[0], planes[1]
    return qw


def _mx(qw: dict, mx: bool | None) -> bool:
    """Whether the block-scaled GEMMs apply the scales in the tensor cores
    (power-of-two scales) or scale each K block's product in the epilogue."""
    pow2 = bool(qw.get("pow2", False))
    if mx is None:
        return pow2
    if mx and not pow2:
        raise RuntimeError("the tensor-core-scaled FP8 GEMMs need power-of-two scales (quant_moe_weights_fp8(pow2=True))")
    return bool(mx)


def moe_gate_up_fp8bs(perm: dict, xq: torch.Tensor, xs: torch.Tensor, qw: dict, num_sms: int | None = None,
                      tok_tile: int = 0, pair: int = -1, mx: bool | None = None) -> torch.Tensor:
    """Block-scaled FP8 gate/up (SwiGLU) over the packed layout; bf16 act [rows, I].
    xs: K-block-major token scales [H/128, rows] (quant_e4m3_kmajor).
    tok_tile 0 and pair -1 let the library choose (CTA pairs for tiles of 128/256).
    mx (default: the weights' scale form) picks ek_moe_gate_up_fp8mx, whose
    tensor cores apply power-of-two scales, over ek_moe_gate_up_fp8bs."""
    dev = _require_cuda(xq, xs)
    if perm["block_m"] != 1:
        raise RuntimeError("the FP8 block-scaled GEMMs take the packed layout (block_m=1)")
    rows, E, H, I = perm["max_rows"], qw["E"], qw["H"], qw["I"]
    if xq.shape != (rows, H) or xs.shape != (H // 128, rows):
        raise RuntimeError("gate_up_fp8bs: activation shape mismatch")
    act = torch.empty((rows, I), dtype=torch.bfloat16, device=dev)
    fn = lib().ek_moe_gate_up_fp8mx if _mx(qw, mx) else lib().ek_moe_gate_up_fp8bs
    with _on_device(dev):
        check(fn(xq.data_ptr(), xs.data_ptr(), qw["w1q"].data_ptr(), qw["w3q"].data_ptr(), qw["w1s"].data_ptr(),
                 qw["w3s"].data_ptr(), perm["expert_counts"].data_ptr(), act.data_ptr(), rows, E, H, I, int(tok_tile),
                 int(pair), int(num_sms or 0), current_stream_handle(dev)), fn.__name__)
    return act


def moe_down_fp8bs(perm: dict, aq: torch.Tensor, as_: torch.Tensor, qw: dict, topk_weights: torch.Tensor,
                   num_sms: int | None = None, tok_tile: int = 0, pair: int = -1, mx: bool | None = None) -> torch.Tensor:
    """Block-scaled FP8 down projection with the routing weight, scattered to slots (bf16 [T*k, H];
    zeros for a slot that a moe_dispatch order dropped).
    as_: K-block-major act scales [I/128, rows]. mx as for moe_gate_up_fp8bs."""
    dev = _require_cuda(aq, as_, topk_weights)
    rows, E, H, I = perm["max_rows"], qw["E"], qw["H"], qw["I"]
    T, k = perm["T"], perm["topk"]
    if aq.shape != (rows, I) or as_.shape != (I // 128, rows) or topk_weights.numel() != T * k:
        raise RuntimeError("down_fp8bs: shape mismatch")
    y = _slot_rows_out(perm, H, dev)
    fn = lib().ek_moe_down_fp8mx if _mx(qw, mx) else lib().ek_moe_down_fp8bs
    with _on_device(dev):
        check(fn(aq.data_ptr(), as_.data_ptr(), qw["w2q"].data_ptr(), qw["w2s"].data_ptr(),
                 perm["expert_counts"].data_ptr(), perm["sorted_slots"].data_ptr(), topk_weights.data_ptr(),
                 y.data_ptr(), rows, E, H, I, T, k, int(tok_tile), int(pair), int(num_sms or 0),
                 current_stream_handle(dev)), fn.__name__)
    return y


def fused_moe_fp8(hidden_states: torch.Tensor, gate_logits: torch.Tensor, qw: dict, topk: int,
                  out: torch.Tensor | None = None, num_sms: int | None = None) -> torch.Tensor:
    """MoE layer with e4m3 block-scaled experts: route -> quantise the token
    rows (1 x 128 groups; a group lies in one row, so quantising before the
    permutation gives the same codes and scales) -> permute + gather the e4m3
    rows (half the bytes of bf16) and their scales (K-block-major) -> FP8
    gate/up SwiGLU -> quantise act -> FP8 down (+weight) -> combine."""
    _require_cuda(hidden_states, gate_logits, out)
    _check_bf16("hidden_states", hidden_states)
    T = hidden_states.shape[0]
    if T == 0:
        return out if out is not None else torch.empty_like(hidden_states)
    pow2 = bool(qw.get("pow2", False))  # tokens and activations take the weights' scale form
    xq_tok, xs_tok = quant_e4m3(hidden_states, block=(1, 128), pow2=pow2)
    ids, wts, perm = moe_route_permute(gate_logits, topk, qw["E"], x=xq_tok, block_m=1)
    xs = moe_gather_cols_f32(perm, xs_tok)
    act = moe_gate_up_fp8bs(perm, perm["x_perm"], xs, qw, num_sms=num_sms)
    aq, as_ = quant_e4m3_kmajor(act, pow2=pow2)
    y = moe_down_fp8bs(perm, aq, as_, qw, wts, num_sms=num_sms)
    return moe_combine(y, T, topk, out=out)


def moe_combine(y: torch.Tensor, T: int, topk: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = sum_j y[t*k + j] (fp32 sum in j order), bf16."""
    dev = _require_cuda(y, out)
    _check_bf16("y", y)
    H = y.shape[1]
    if out is None:
        out = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
    else:
        _check_bf16("out", out)
    with _on_device(dev):
        check(lib().ek_moe_combine(y.data_ptr(), out.data_ptr(), int(T), int(topk), H, current_stream_handle(dev)),
              "ek_moe_combine")
    return out


PACKED_MIN_SMS = 112
PACKED_MAX_ROWS_PER_EXPERT = 288
# below PACKED_MIN_SMS the packed layout still wins at decode sizes (routed rows)
PACKED_DECODE_MIN_SMS = 64
PACKED_DECODE_ROWS = 2
PACKED_DECODE_WIDE_SMS = 96
PACKED_DECODE_ROWS_WIDE = 4


def moe_layout(num_sms: int, num_experts: int, rows: int | None = None) -> str:
    """Layout the fused MoE uses on a partition of `num_sms` SMs for `rows`
    routed rows (tokens x top-k; None: not known).

    Measured on B200 (Mixtral shapes, T = 1..4096): the packed layout with the
    swapped-operand GEMMs is faster on (nearly) the full device while experts
    get up to a few hundred rows -- T=128: 519 us packed vs 578 us padded,
    T=1024 (256 rows per expert): 861 vs 875 us on 148 SMs -- and the 128-row
    padded layout from 320 rows per expert (T=1280: 1029-1057 vs 1054-1206 us,
    T=1536: 1241 vs 1322 us, T=2048: 1393 vs 1631 us, T=4096: 2402 vs 2572
    us) and on small partitions (T=128 on 72 SMs: 632 us padded
    vs 833 us packed), except at decode sizes, where the packed GEMMs stream
    only the experts hit and split K over the idle SMs (96 SMs: T=1 202 vs
    245 us, T=2 254 vs 284 us, T=4 347 vs 325 us; 72 SMs: T=1 248 vs 254 us,
    T=2 339 vs 314 us)."""
    if num_experts > 256:
        return "padded"
    if num_sms < PACKED_MIN_SMS:
        decode_rows = (PACKED_DECODE_ROWS_WIDE if num_sms >= PACKED_DECODE_WIDE_SMS
                       else PACKED_DECODE_ROWS if num_sms >= PACKED_DECODE_MIN_SMS else 0)
        return "packed" if rows is not None and rows <= decode_rows else "padded"
    if rows is not None and rows > PACKED_MAX_ROWS_PER_EXPERT * num_experts:
        return "padded"
    return "packed"


PAIR_MIN_ROWS_PER_EXPERT = 768        # from PACKED_MIN_SMS SMs up
PAIR_MIN_ROWS_PER_EXPERT_SMALL = 256  # on smaller partitions


def padded_block_m(num_sms: int, num_experts: int, rows: int) -> int:
    """Row padding of the padded layout: 256 (2-SM CTA-pair tiles) from 768
    routed rows per expert on 112+ SMs and from 256 on 2..111 SMs, else 128.
    Measured on B200 (Mixtral shapes): on 148 SMs T=4096 (1024 rows per
    expert) gate/up 1751-1786 vs 1882 us and down 858-887 vs 957-969 us,
    T=2048 (512 rows per expert) no gain, the extra padding eats the pair's
    higher per-row rate; on 72 SMs the layer at T=1024 / 2048 / 4096 takes
    1280 / 1903-1987 / 3598-3731 us with pairs vs 1303-1316 / 2144 /
    4152-4257 us, at T=512 863-976 vs 859-884 us."""
    if num_sms < 2:
        return BLOCK_M
    per_expert = PAIR_MIN_ROWS_PER_EXPERT if num_sms >= PACKED_MIN_SMS else PAIR_MIN_ROWS_PER_EXPERT_SMALL
    return 256 if rows >= per_expert * num_experts else BLOCK_M


def fused_moe(hidden_states: torch.Tensor, gate_logits: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor,
              w3: torch.Tensor, topk: int, out: torch.Tensor | None = None, num_sms: int | None = None,
              layout: str = "auto") -> torch.Tensor:
    """The whole MoE layer: route -> permute(+gather) -> gate/up SwiGLU -> down(+weight) -> combine.

    layout="packed": expert-major rows without padding and the swapped-operand
    GEMMs; "padded": 128-row padded blocks and the token-major GEMMs; "auto"
    (default): moe_layout() for the partition of the current stream."""
    dev = _require_cuda(hidden_states, gate_logits, w1, w2, w3, out)
    _check_bf16("hidden_states", hidden_states)
    T = hidden_states.shape[0]
    if T == 0:
        return out if out is not None else torch.empty_like(hidden_states)
    sms = int(num_sms) if num_sms else _stream_sms(dev, current_stream_handle(dev))
    if layout == "auto":
        layout = moe_layout(sms, w1.shape[0], T * topk)
    if layout == "packed" and w1.shape[0] <= 256:
        ids, wts, perm = moe_route_permute(gate_logits, topk, w1.shape[0], x=hidden_states, block_m=1)
        act = moe_gate_up_packed(perm, w1, w3, num_sms=num_sms)
        y = moe_down_packed(perm, act, w2, wts, num_sms=num_sms)
    else:
        ids, wts, perm = moe_route_permute(gate_logits, topk, w1.shape[0], x=hidden_states,
                                           block_m=padded_block_m(sms, w1.shape[0], T * topk))
        act = moe_gate_up(perm, w1, w3, num_sms=num_sms)
        y = moe_down(perm, act, w2, wts, num_sms=num_sms)
    return moe_combine(y, T, topk, out=out)


# ------------------------------------------------- token rows to experts and back
_ROW_DTYPES = {torch.bfloat16: _lib.EK_DTYPE_BF16, torch.float16: _lib.EK_DTYPE_FP16,
               torch.float32: _lib.EK_DTYPE_FP32}


# The library's own limits, checked here too: a size past 32 bits would reach it
# as another one.
_MAX_SLOTS = _MAX_ROW = _MAX_EXPERTS = 1 << 30
_MAX_W4_K, _MAX_W4_ROWS = 1 << 28, 1 << 24


def _check_rows(name: str, t: torch.Tensor, rows: int | None = None) -> int:
    """dtype code of a contiguous bf16/fp16/fp32 row matrix (of `rows` rows)."""
    dt, shape = _ROW_DTYPES.get(t.dtype), t.shape
    if dt is None or len(shape) != 2:
        raise RuntimeError(f"{name} must be a 2-D bf16, fp16 or fp32 tensor")
    if rows is not None and shape[0] != rows:
        raise RuntimeError(f"{name} must have {rows} rows, got {shape[0]}")
    if not 0 < shape[1] <= _MAX_ROW or shape[0] > 0x7fffffff:
        raise RuntimeError(f"{name} has rows of no elements" if shape[1] == 0 else
                           f"{name}: rows of more than 2^30 elements, or more than 2^31 of them")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    return dt


def _check_slots(name: str, t: torch.Tensor, T: int, k: int, dtype: torch.dtype) -> None:
    if t.dtype is not dtype or t.shape != (T, k):
        raise RuntimeError(f"{name} must be a {dtype} tensor of shape {(T, k)}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    return a.data_ptr() < b.data_ptr() + b.nbytes and b.data_ptr() < a.data_ptr() + a.nbytes


def _slot_rows(perm: dict) -> torch.Tensor:
    if perm.get("slot_rows") is None:
        raise RuntimeError("the permutation has no slot_rows (make it with moe_dispatch)")
    return perm["slot_rows"]


def moe_dispatch(x: torch.Tensor | None, topk_ids: torch.Tensor, num_experts: int) -> dict:
    """Token rows in expert-major order, for training and for batches with padding.

    The (token, choice) slots are sorted stably by expert id and x's rows
    (bf16, fp16 or fp32, any width) copied into that order. A negative id
    drops its slot: a padding token, or a slot over its expert's capacity. An
    id past num_experts drops it too and raises EK_STATUS_BAD_INDEX. x=None
    makes the order alone.

    Returns the packed layout the *_packed and *_w4 products take (as
    moe_permute(..., block_m=1), without block_expert): x_perm [T*k, H] with
    zero rows past the last kept one, sorted_slots, expert_counts and
    num_rows_padded, plus slot_rows [T*k], the row of each slot (-1: dropped),
    which the way back and the gradients need."""
    dev = _require_cuda(topk_ids, x)
    if topk_ids.dtype != torch.int32 or topk_ids.dim() != 2:
        raise RuntimeError("topk_ids must be a 2-D int32 tensor")
    _contig("topk_ids", topk_ids)
    T, k = topk_ids.shape
    E, n = int(num_experts), T * k
    if n > _MAX_SLOTS or k > _MAX_SLOTS:
        raise RuntimeError(f"moe_dispatch: too many slots ({T} x {k})")
    if abs(E) > _MAX_EXPERTS:
        raise RuntimeError(f"moe_dispatch: need 1 <= E <= 1024 (got {E})")
    H = dt = 0
    x_perm = None
    if x is not None:
        dt = _check_rows("x", x, T)
        H = x.shape[1]
        x_perm = x.new_empty((n, H))
    L = lib()
    ints = int(L.ek_moe_permute_scratch_bytes(T, k, E)) // 4
    sorted_slots, slot_rows, counts, num_rows, scratch = topk_ids.new_empty(
        2 * n + max(E, 0) + 1 + ints).split_with_sizes([n, n, max(E, 0), 1, ints])
    with _on_device(dev):
        check(L.ek_moe_dispatch(topk_ids.data_ptr(), T, k, E, _ptr(x), H, dt, sorted_slots.data_ptr(),
                                slot_rows.data_ptr(), counts.data_ptr(), num_rows.data_ptr(), _ptr(x_perm),
                                scratch.data_ptr(), current_stream_handle(dev)), "ek_moe_dispatch")
    return {"sorted_slots": sorted_slots, "slot_rows": slot_rows, "block_expert": None, "num_rows_padded": num_rows,
            "expert_counts": counts, "x_perm": x_perm, "max_rows": n, "T": T, "topk": k, "E": E, "block_m": 1}


def moe_dispatch_grad(perm: dict, d_rows: torch.Tensor) -> torch.Tensor:
    """Gradient of moe_dispatch's copy: d_x[t] = the sum of the gradients of
    token t's rows (fp32 in choice order, rounded once), [T, H]."""
    slot_rows = _slot_rows(perm)
    dev = _require_cuda(d_rows, slot_rows)
    dt = _check_rows("d_rows", d_rows)
    T, k, (n, H) = perm["T"], perm["topk"], d_rows.shape
    d_x = d_rows.new_empty((T, H))
    with _on_device(dev):
        check(lib().ek_moe_dispatch_grad(d_rows.data_ptr(), slot_rows.data_ptr(), T, k, n, H, dt, d_x.data_ptr(),
                                         current_stream_handle(dev)), "ek_moe_dispatch_grad")
    return d_x


def moe_combine_weighted(perm: dict, rows: torch.Tensor, topk_weights: torch.Tensor,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = sum_j topk_weights[t, j] * (row of slot t, j) over the kept slots:
    expert-major rows back to the tokens (fp32 in choice order, rounded once)."""
    slot_rows = _slot_rows(perm)
    dev = _require_cuda(rows, topk_weights, slot_rows, out)
    dt = _check_rows("rows", rows)
    T, k, (n, H) = perm["T"], perm["topk"], rows.shape
    _check_slots("topk_weights", topk_weights, T, k, torch.float32)
    if out is None:
        out = rows.new_empty((T, H))
    elif out.dtype != rows.dtype or out.shape != (T, H) or not out.is_contiguous():
        raise RuntimeError("out must be a contiguous [T, H] tensor of the rows' dtype")
    elif _overlap(out, rows):
        raise RuntimeError("out must not overlap the rows (they are still read while it is written)")
    with _on_device(dev):
        check(lib().ek_moe_combine_weighted(rows.data_ptr(), slot_rows.data_ptr(), topk_weights.data_ptr(), T, k, n, H,
                                            dt, out.data_ptr(), current_stream_handle(dev)),
              "ek_moe_combine_weighted")
    return out


def moe_combine_weighted_grad(perm: dict, rows: torch.Tensor, topk_weights: torch.Tensor,
                              d_out: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradient of moe_combine_weighted: d_rows (the rows' dtype; zero past the
    last kept row) and d_weights [T, k] (fp32; zero for a dropped slot)."""
    slot_rows = _slot_rows(perm)
    dev = _require_cuda(rows, topk_weights, d_out, slot_rows)
    dt = _check_rows("rows", rows)
    T, k, (n, H) = perm["T"], perm["topk"], rows.shape
    _check_slots("topk_weights", topk_weights, T, k, torch.float32)
    if d_out.dtype != rows.dtype or d_out.shape != (T, H):
        raise RuntimeError(f"d_out must be a {rows.dtype} tensor of shape {(T, H)}")
    _contig("d_out", d_out)
    d_rows = torch.empty_like(rows)
    d_weights = torch.empty_like(topk_weights)
    with _on_device(dev):
        check(lib().ek_moe_combine_weighted_grad(rows.data_ptr(), slot_rows.data_ptr(), topk_weights.data_ptr(),
                                                 d_out.data_ptr(), perm["num_rows_padded"].data_ptr(), T, k, n, H, dt,
                                                 d_rows.data_ptr(), d_weights.data_ptr(), current_stream_handle(dev)),
              "ek_moe_combine_weighted_grad")
    return d_rows, d_weights


def moe_route_grad(topk_ids: torch.Tensor, topk_weights: torch.Tensor, d_weights: torch.Tensor,
                   num_experts: int) -> torch.Tensor:
    """Gradient of moe_route's weights with respect to the gate logits, fp32 [T, E].

    The renormalised weights are the softmax of the chosen logits, so
    d_logits[t, ids_j] = w_j (dw_j - sum_i w_i dw_i), and an expert that was not
    chosen gets 0. topk_ids are the ids as moe_route gave them, dropped slots'
    too: a choice dropped for capacity was in the softmax, so its logit has a
    gradient although its dw is 0. Ids masked to -1 (what moe_dispatch takes
    for a dropped slot) would lose it."""
    dev = _require_cuda(topk_ids, topk_weights, d_weights)
    if topk_ids.dim() != 2:
        raise RuntimeError("topk_ids must be a 2-D int32 tensor")
    T, k = topk_ids.shape
    _check_slots("topk_ids", topk_ids, T, k, torch.int32)
    _check_slots("topk_weights", topk_weights, T, k, torch.float32)
    _check_slots("d_weights", d_weights, T, k, torch.float32)
    E = int(num_experts)
    if not 1 <= E <= _MAX_EXPERTS or max(T, k) > 0x7fffffff:
        raise RuntimeError("num_experts must be positive, at most 2^30, and ids within 2^31 x 2^31")
    d_logits = d_weights.new_empty((T, E))
    with _on_device(dev):
        check(lib().ek_moe_route_grad(topk_ids.data_ptr(), topk_weights.data_ptr(), d_weights.data_ptr(), T, E, k,
                                      d_logits.data_ptr(), current_stream_handle(dev)), "ek_moe_route_grad")
    return d_logits


# ------------------------------------------------------------------ 4-bit weights
W4_GROUPS = (32, 64, 128)


def quant_w4(w: torch.Tensor, group: int = 128, symmetric: bool = True, dtype: torch.dtype | None = None) -> dict:
    """4-bit codes of weights w [..., N, K] (bf16, fp16 or fp32; finite) with a
    scale, and with symmetric=False a minimum, per `group` elements of a row.

    Returns {"codes": uint8 [..., N, ceil(K/32)*16], "scales": [..., N,
    ceil(K/group)], "mins": same or None, "K", "group"}; two codes per byte,
    the even element in the low nibble. Scales and minima are in `dtype` (bf16
    or fp16; default w's, bf16 for fp32 w), the type of the activations the
    products take. The weight is s * (q - 8), or s * q + m with minima; weights
    quantised elsewhere go in by building this dict."""
    dev = _require_cuda(w)
    if w.dtype not in _ROW_DTYPES or w.dim() < 2 or not 0 < w.shape[-1] <= _MAX_W4_K:
        raise RuntimeError("quant_w4 takes bf16, fp16 or fp32 weights [..., N, K] with K of 1 to 2^28")
    if dtype is None:
        dtype = w.dtype if w.dtype in _DTYPES else torch.bfloat16
    if dtype not in _DTYPES or group not in W4_GROUPS:
        raise RuntimeError(f"quant_w4: dtype must be bf16 or fp16 and group one of {W4_GROUPS}")
    _contig("w", w)
    K = w.shape[-1]
    lead = tuple(w.shape[:-1])
    rows = w.numel() // K
    codes = torch.empty(lead + (-(-K // 32) * 16,), dtype=torch.uint8, device=dev)
    scales = torch.empty(lead + (-(-K // group),), dtype=dtype, device=dev)
    mins = None if symmetric else torch.empty_like(scales)
    with _on_device(dev):
        check(lib().ek_quant_w4(w.data_ptr(), _ROW_DTYPES[w.dtype], rows, K, group, 1 if symmetric else 0,
                                _DTYPES[dtype], codes.data_ptr(), scales.data_ptr(), _ptr(mins),
                                current_stream_handle(dev)), "ek_quant_w4")
    return {"codes": codes, "scales": scales, "mins": mins, "K": K, "group": group}


def _check_w4(name: str, qw: dict, dtype: torch.dtype | None = None) -> tuple:
    """(codes, scales, mins, leading shape, K, group) of a 4-bit weight."""
    codes, scales, mins, K, group = qw["codes"], qw["scales"], qw.get("mins"), int(qw["K"]), int(qw["group"])
    if group not in W4_GROUPS or not 1 <= K <= _MAX_W4_K:
        raise RuntimeError(f"{name}: need K of 1 to 2^28 and a group out of {W4_GROUPS}")
    *lead, width = codes.shape
    lead, kind = tuple(lead), scales.dtype
    if codes.dtype != torch.uint8 or not lead or width != -(-K // 32) * 16:
        raise RuntimeError(f"{name}: codes must be uint8 [..., N, {-(-K // 32) * 16}]")
    if kind not in _DTYPES or scales.shape != (*lead, -(-K // group)):
        raise RuntimeError(f"{name}: scales must be bf16 or fp16 [..., N, {-(-K // group)}]")
    if dtype is not None and kind != dtype:
        raise RuntimeError(f"{name}: scales must be {dtype}, got {kind}")
    if mins is not None and (mins.dtype != kind or mins.shape != scales.shape or not mins.is_contiguous()):
        raise RuntimeError(f"{name}: mins must match the scales")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        raise RuntimeError(f"{name}: codes and scales must be contiguous")
    return codes, scales, mins, lead, K, group


def dequant_w4(qw: dict) -> torch.Tensor:
    """The weights a 4-bit dict stands for, rounded once to the scales' dtype."""
    codes, scales, mins, lead, K, group = _check_w4("dequant_w4", qw)
    dev = _require_cuda(codes, scales, mins)
    out = torch.empty(lead + (K,), dtype=scales.dtype, device=dev)
    with _on_device(dev):
        check(lib().ek_dequant_w4(codes.data_ptr(), scales.data_ptr(), _ptr(mins), out.numel() // K, K, group,
                                  _DTYPES[scales.dtype], out.data_ptr(), current_stream_handle(dev)), "ek_dequant_w4")
    return out


def gemm_w4(a: torch.Tensor, qw: dict, out: torch.Tensor | None = None, num_sms: int | None = None) -> torch.Tensor:
    """C = a @ W^T with a [M, K] (bf16 or fp16) and a 4-bit weight W [N, K]
    (quant_w4) whose scales have a's dtype; C [M, N] in that dtype, fp32 sums.

    Made for a few tokens; any M is right, but from about a hundred rows
    gemm(a, dequant_w4(qw), b_layout="nk") is faster (with the weights rounded
    to a's dtype, which this product does not do): 14336 x 4096 takes 17 against
    62 us for 16 rows, 45 against 62 for 64, 83 against 63 for 128."""
    codes, scales, mins, lead, K, group = _check_w4("gemm_w4", qw, a.dtype)
    dev = _require_cuda(a, codes, scales, mins, out)
    if a.dim() != 2 or a.shape[1] != K or len(lead) != 1:
        raise RuntimeError(f"gemm_w4 takes a [M, {K}] and a 2-D weight")
    _contig("a", a)
    M, N = a.shape[0], lead[0]
    if max(M, N) > 0x7fffffff:
        raise RuntimeError(f"gemm_w4: more than 2^31 rows ({M} x {N})")
    if out is None:
        out = a.new_empty((M, N))
    elif out.shape != (M, N) or out.dtype != a.dtype or not out.is_contiguous():
        raise RuntimeError("out must be a contiguous [M, N] tensor of the input dtype")
    if M == 0 or N == 0:
        return out
    L = lib()
    stream, sms = current_stream_handle(dev), int(num_sms or 0)
    ws = _scratch(L.ek_gemm_w4_workspace_bytes(M, N, K, _most_sms(dev, sms)), codes)
    with _on_device(dev):
        check(L.ek_gemm_w4(a.data_ptr(), codes.data_ptr(), scales.data_ptr(), _ptr(mins), out.data_ptr(), M, N, K,
                           group, _DTYPES[a.dtype], sms, ws.data_ptr(), ws.numel(), stream), "ek_gemm_w4")
    return out


def _most_sms(dev: torch.device, num_sms: int) -> int:
    """SMs to size a workspace for: num_sms, or with 0 (the library then asks the
    stream for its partition's) all of the device, which no partition exceeds."""
    if num_sms:
        return num_sms
    n = _DEV_SMS.get(dev.index)
    return n if n is not None else _device_sms(dev)


def _scratch(nbytes: int, codes: torch.Tensor) -> torch.Tensor:
    """Workspace of one call beside the codes (bytes too), from torch's allocator:
    nothing in it outlives the call, and a captured graph gets its own."""
    if nbytes == _SIZE_MAX:
        check(_lib.EK_ERR_INVALID, "workspace size")
    return codes.new_empty(nbytes)


def quant_moe_weights_w4(w1: torch.Tensor, w2: torch.Tensor, w3: torch.Tensor, group: int = 128,
                         symmetric: bool = True) -> dict:
    """4-bit expert weights (w1, w3 [E, I, H], w2 [E, H, I]) for fused_moe_w4."""
    E, I, H = w1.shape
    if w3.shape != w1.shape or tuple(w2.shape) != (E, H, I):
        raise RuntimeError("quant_moe_weights_w4: w1 and w3 must be [E, I, H] and w2 [E, H, I]")
    q = {n: quant_w4(w, group, symmetric, torch.bfloat16) for n, w in (("w1", w1), ("w3", w3), ("w2", w2))}
    return {"E": E, "H": H, "I": I, **q}


_ACT_DTYPES = {torch.bfloat16: _lib.EK_DTYPE_BF16, torch.float32: _lib.EK_DTYPE_FP32}


def _check_experts(qw: dict, *names: str) -> list:
    """(codes, scales, mins) of the named expert weights, checked against qw's E, H, I."""
    E, H, I = qw["E"], qw["H"], qw["I"]
    out, kinds = [], set()
    for name in names:
        c, s, m, lead, K, group = _check_w4(name, qw[name], torch.bfloat16)
        if lead != ((E, H) if name == "w2" else (E, I)) or K != (I if name == "w2" else H):
            raise RuntimeError(f"{name}: shape mismatch")
        kinds.add((group, m is None))
        out.append((c, s, m, group))
    if len(kinds) != 1:
        raise RuntimeError("the experts' weights must share one group and be all symmetric or all with minima")
    return out


def moe_gate_up_w4(perm: dict, qw: dict, x: torch.Tensor | None = None, num_sms: int | None = None,
                   dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """act[r] = silu(row . w1[e]) * (row . w3[e]) over the packed rows, 4-bit experts.
    The rows are perm["x_perm"], or with x (the tokens [T, H]) fetched through
    the permutation, so nothing has to be copied first. act in `dtype` (bf16
    or fp32). Rows past the last kept one are left unwritten."""
    E, H, I = qw["E"], qw["H"], qw["I"]
    (c1, s1, m1, group), (c3, s3, m3, _) = _check_experts(qw, "w1", "w3")
    src = perm["x_perm"] if x is None else x
    if src is None:
        raise RuntimeError("moe_gate_up_w4: the permutation has no rows; give x")
    dev = _require_cuda(src, c1, s1, m1, c3, s3, m3, perm["expert_counts"])
    _check_bf16("x", src)
    rows, x_rows = perm["max_rows"], perm["max_rows"] if x is None else perm["T"]
    if perm["E"] != E or tuple(src.shape) != (x_rows, H) or perm["block_m"] != 1 or dtype not in _ACT_DTYPES:
        raise RuntimeError("gate_up_w4: shape mismatch")
    act = torch.empty((rows, I), dtype=dtype, device=dev)
    L = lib()
    stream, sms = current_stream_handle(dev), int(num_sms or 0)
    ws = _scratch(L.ek_moe_w4_workspace_bytes(x_rows, rows, E, H, I, _most_sms(dev, sms)), c1)
    with _on_device(dev):
        check(L.ek_moe_gate_up_w4(src.data_ptr(), x_rows, None if x is None else perm["sorted_slots"].data_ptr(),
                                  1 if x is None else perm["topk"], c1.data_ptr(), s1.data_ptr(), _ptr(m1),
                                  c3.data_ptr(), s3.data_ptr(), _ptr(m3), perm["expert_counts"].data_ptr(),
                                  act.data_ptr(), _ACT_DTYPES[dtype], rows, E, H, I, group, sms, ws.data_ptr(),
                                  ws.numel(), stream), "ek_moe_gate_up_w4")
    return act


def moe_down_w4(perm: dict, act: torch.Tensor, qw: dict, num_sms: int | None = None,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y[r] = act[r] . w2[e] over the packed rows, 4-bit experts (no routing
    weight: moe_combine_weighted applies it), in `dtype` (bf16 or fp32); act is
    bf16 or fp32. Rows past the last are left unwritten."""
    E, H, I = qw["E"], qw["H"], qw["I"]
    ((c2, s2, m2, group),) = _check_experts(qw, "w2")
    dev = _require_cuda(act, c2, s2, m2, perm["expert_counts"])
    _contig("act", act)
    rows = perm["max_rows"]
    if perm["E"] != E or tuple(act.shape) != (rows, I) or perm["block_m"] != 1 or act.dtype not in _ACT_DTYPES or \
            dtype not in _ACT_DTYPES:
        raise RuntimeError("down_w4: shape mismatch")
    y = torch.empty((rows, H), dtype=dtype, device=dev)
    L = lib()
    stream, sms = current_stream_handle(dev), int(num_sms or 0)
    ws = _scratch(L.ek_moe_w4_workspace_bytes(0, rows, E, H, I, _most_sms(dev, sms)), c2)
    with _on_device(dev):
        check(L.ek_moe_down_w4(act.data_ptr(), _ACT_DTYPES[act.dtype], c2.data_ptr(), s2.data_ptr(), _ptr(m2),
                               perm["expert_counts"].data_ptr(), y.data_ptr(), _ACT_DTYPES[dtype], rows, E, H, I, group,
                               sms, ws.data_ptr(), ws.numel(), stream), "ek_moe_down_w4")
    return y


def moe_experts_w4(perm: dict, x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, qw: dict,
                   out: torch.Tensor | None = None, num_sms: int | None = None) -> torch.Tensor:
    """The experts' part of a layer over 4-bit weights: gate/up, down and the
    weighted combine for the tokens x [T, H] (bf16) and a moe_dispatch order of
    topk_ids. Activations and the experts' rows stay in the workspace (11
    significant bits and fp32); the output [T, H] is rounded once."""
    E, H, I = qw["E"], qw["H"], qw["I"]
    (c1, s1, m1, group), (c3, s3, m3, _), (c2, s2, m2, _) = _check_experts(qw, "w1", "w3", "w2")
    slot_rows = _slot_rows(perm)
    dev = _require_cuda(x, topk_ids, topk_weights, c1, s1, m1, c3, s3, m3, c2, s2, m2, slot_rows, out)
    _check_bf16("x", x)
    T, k = perm["T"], perm["topk"]
    _check_slots("topk_ids", topk_ids, T, k, torch.int32)
    _check_slots("topk_weights", topk_weights, T, k, torch.float32)
    if perm["E"] != E or tuple(x.shape) != (T, H):
        raise RuntimeError("experts_w4: shape mismatch")
    if out is None:
        out = torch.empty_like(x)
    else:
        _check_bf16("out", out)
        if out.shape != x.shape:
            raise RuntimeError("out must be a [T, H] tensor")
    if T == 0:
        return out
    L = lib()
    stream, sms = current_stream_handle(dev), int(num_sms or 0)
    ws = _scratch(L.ek_moe_w4_workspace_bytes(T, T * k, E, H, I, _most_sms(dev, sms)), c1)
    with _on_device(dev):
        check(L.ek_moe_experts_w4(x.data_ptr(), T, k, topk_ids.data_ptr(), topk_weights.data_ptr(),
                                  perm["sorted_slots"].data_ptr(), slot_rows.data_ptr(),
                                  perm["expert_counts"].data_ptr(), c1.data_ptr(), s1.data_ptr(), _ptr(m1),
                                  c3.data_ptr(), s3.data_ptr(), _ptr(m3), c2.data_ptr(), s2.data_ptr(), _ptr(m2),
                                  out.data_ptr(), E, H, I, group, sms, ws.data_ptr(), ws.numel(), stream),
              "ek_moe_experts_w4")
    return out


def fused_moe_w4(hidden_states: torch.Tensor, gate_logits: torch.Tensor, qw: dict, topk: int,
                 out: torch.Tensor | None = None, num_sms: int | None = None) -> torch.Tensor:
    """MoE layer over 4-bit experts (quant_moe_weights_w4), for batches of a few
    tokens per expert: moe_route -> moe_dispatch -> moe_experts_w4 in one call
    (five launches up to 128 slots)."""
    E, H, I = qw["E"], qw["H"], qw["I"]
    (c1, s1, m1, group), (c3, s3, m3, _), (c2, s2, m2, _) = _check_experts(qw, "w1", "w3", "w2")
    dev = _require_cuda(hidden_states, gate_logits, c1, s1, m1, c3, s3, m3, c2, s2, m2, out)
    _check_bf16("hidden_states", hidden_states)
    T = hidden_states.shape[0]
    if hidden_states.shape != (T, H):
        raise RuntimeError("fused_moe_w4: shape mismatch")
    if not 0 <= T * int(topk) <= _MAX_W4_ROWS:
        raise RuntimeError(f"fused_moe_w4: too many rows, or a negative number of them ({T} tokens x {topk})")
    if gate_logits.dtype != torch.float32 or gate_logits.shape != (T, E):
        raise RuntimeError("gate_logits must be float32 with one row per token and one column per expert")
    _contig("gate_logits", gate_logits)
    if out is None:
        out = torch.empty_like(hidden_states)
    else:
        _check_bf16("out", out)
        if out.shape != hidden_states.shape:
            raise RuntimeError("out must be a [T, H] tensor")
    L, k = lib(), int(topk)
    stream, sms = current_stream_handle(dev), int(num_sms or 0)
    ws = _scratch(L.ek_fused_moe_w4_workspace_bytes(T, k, E, H, I, _most_sms(dev, sms)), c1)
    with _on_device(dev):
        check(L.ek_fused_moe_w4(hidden_states.data_ptr(), gate_logits.data_ptr(), T, k, c1.data_ptr(), s1.data_ptr(),
                                _ptr(m1), c3.data_ptr(), s3.data_ptr(), _ptr(m3), c2.data_ptr(), s2.data_ptr(),
                                _ptr(m2), out.data_ptr(), E, H, I, group, sms, ws.data_ptr(), ws.numel(), stream),
              "ek_fused_moe_w4")
    return out


# ---------------------------------------------------- dense feed-forward blocks
GATES = {"silu": _lib.EK_GATE_SILU, "gelu": _lib.EK_GATE_GELU, "gelu_tanh": _lib.EK_GATE_GELU_TANH}
_MAX_FFN_DIM = 1 << 28  # of H and I, and _MAX_TOKENS of the rows: the library's ints
_MAX_TOKENS = (1 << 31) - 256


def _check_matrix(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> torch.Tensor:
    """t, checked and 16-byte aligned (a view that starts mid-line is copied)."""
    if t.dtype is not dtype or t.shape != shape:
        raise RuntimeError(f"{name} must be a {dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _gate(act: str) -> int:
    if act not in GATES:
        raise RuntimeError(f"act must be one of {tuple(GATES)}, got {act!r}")
    return GATES[act]


def _blocks128(n: int) -> int:
    return -(-n // 128)


def gemm_fp8_block(a_q: torch.Tensor, w_q: torch.Tensor, a_scale: torch.Tensor, w_scale: torch.Tensor,
                   out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
                   num_sms: int | None = None) -> torch.Tensor:
    """C[M, N] = A @ W^T for e4m3 a_q [M, K] and w_q [N, K] with block scales.

    a_scale [M, ceil(K/128)] holds a scale per 1 x 128 group of a row, w_scale
    [ceil(N/128), ceil(K/128)] one per 128 x 128 block, both fp32 of any finite value:
    what quant_e4m3(x, block=(1, 128)) and quant_e4m3(w, block=(128, 128)) give.
    K is a multiple of 16; M, N (up to 2^31 - 256) and the last block of each axis
    are any size. The sums are fp32; C is bf16, fp16 or fp32 (`dtype`, or out's),
    rounded once."""
    dev = _require_cuda(a_q, w_q, a_scale, w_scale, out)
    shape = a_q.shape
    if _FP8 is None or len(shape) != 2 or w_q.dim() != 2:
        raise RuntimeError("gemm_fp8_block takes 2-D float8_e4m3fn operands")
    (M, K), N = shape, w_q.shape[0]
    if K == 0 or K % 16 or K > _MAX_FFN_DIM or max(M, N) > _MAX_TOKENS:
        raise RuntimeError(f"gemm_fp8_block: K must be a positive multiple of 16 up to 2^28, M and N up to "
                           f"2^31 - 256 (got {M} x {N} x {K})")
    a_q = _check_matrix("a_q", a_q, _FP8, (M, K))
    w_q = _check_matrix("w_q", w_q, _FP8, (N, K))
    a_scale = _check_matrix("a_scale", a_scale, torch.float32, (M, _blocks128(K)))
    w_scale = _check_matrix("w_scale", w_scale, torch.float32, (_blocks128(N), _blocks128(K)))
    if out is not None:
        dtype = out.dtype
    if dtype not in _ROW_DTYPES:
        raise RuntimeError("gemm_fp8_block: the result is bf16, fp16 or fp32")
    if out is None:
        out = a_scale.new_empty((M, N), dtype=dtype)
    elif out.shape != (M, N) or not out.is_contiguous():
        raise RuntimeError("out must be a contiguous [M, N] tensor")
    if M == 0 or N == 0:
        return out
    L = lib()
    stream, sms = current_stream_handle(dev), int(num_sms or 0)
    need = L.ek_gemm_fp8_block_workspace_bytes(M, N, K, _most_sms(dev, sms))
    ws = _bytes(need, a_scale)
    with _on_device(dev):
        check(L.ek_gemm_fp8_block(a_q.data_ptr(), w_q.data_ptr(), a_scale.data_ptr(), w_scale.data_ptr(),
                                  out.data_ptr(), M, N, K, _ROW_DTYPES[dtype], sms, ws.data_ptr(), need, stream),
              "ek_gemm_fp8_block")
    return out


def _bytes(n: int, like: torch.Tensor) -> torch.Tensor:
    """Workspace of one call, as _scratch."""
    if n == _SIZE_MAX:
        check(_lib.EK_ERR_INVALID, "workspace size")
    return like.new_empty(n, dtype=torch.uint8)


def _check_ffn(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, w3: torch.Tensor, dtype: torch.dtype,
               unit: int) -> tuple:
    """(x, w1, w2, w3, T, H, I) of a feed-forward block, checked and aligned."""
    if x.dim() != 2 or w1.dim() != 2:
        raise RuntimeError("x must be [T, H] and w1 [I, H]")
    (T, H), I = x.shape, w1.shape[0]
    if not (0 < H <= _MAX_FFN_DIM and 0 < I <= _MAX_FFN_DIM) or H % unit or I % unit or T > _MAX_TOKENS:
        raise RuntimeError(f"H and I must be positive multiples of {unit} up to 2^28, T up to 2^31 - 256 "
                           f"(got T={T}, H={H}, I={I})")
    wt = dtype if unit == 8 else _FP8
    return (_check_matrix("x", x, dtype, (T, H)), _check_matrix("w1", w1, wt, (I, H)),
            _check_matrix("w2", w2, wt, (H, I)), _check_matrix("w3", w3, wt, (I, H)), T, H, I)


def gated_ffn(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, w3: torch.Tensor, act: str = "silu",
              out: torch.Tensor | None = None, save: bool = False, num_sms: int | None = None):
    """Dense gated feed-forward block: y = (f(x W1^T) * (x W3^T)) W2^T.

    x [T, H], w1 and w3 [I, H], w2 [H, I] in bf16 or fp16 (H and I multiples of 8,
    T up to 2^31 - 256); f is "silu", "gelu" or "gelu_tanh". Sums are fp32; the
    activations are rounded to x's dtype between the two products. With save=True
    returns (y, h), h [2, T, I] the rounded pre-activations x W1^T and x W3^T that
    gated_ffn_grad takes."""
    dev = _require_cuda(x, w1, w2, w3, out)
    if x.dtype not in _DTYPES:
        raise RuntimeError("gated_ffn takes bf16 or fp16")
    gate, dtype = _gate(act), x.dtype
    x, w1, w2, w3, T, H, I = _check_ffn(x, w1, w2, w3, dtype, 8)
    y = x.new_empty((T, H)) if out is None else out
    if out is not None and (out.dtype != dtype or out.shape != (T, H) or not out.is_contiguous()):
        raise RuntimeError("out must be a contiguous [T, H] tensor of x's dtype")
    if out is not None and out.data_ptr() % 16:
        y = x.new_empty((T, H))
    h = x.new_empty((2, T, I)) if save else None
    if T > 0:
        L = lib()
        stream, sms = current_stream_handle(dev), int(num_sms or 0)
        need = L.ek_gated_ffn_workspace_bytes(T, H, I, _most_sms(dev, sms))
        ws = _bytes(need, x)
        with _on_device(dev):
            check(L.ek_gated_ffn(x.data_ptr(), w1.data_ptr(), w2.data_ptr(), w3.data_ptr(), y.data_ptr(), _ptr(h), T, H,
                                 I, _DTYPES[dtype], gate, sms, ws.data_ptr(), need, stream), "ek_gated_ffn")
    if out is not None and y is not out:
        y = out.copy_(y)
    return (y, h) if save else y


def gated_ffn_grad(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, w3: torch.Tensor, h: torch.Tensor,
                   d_out: torch.Tensor, act: str = "silu", num_sms: int | None = None) -> tuple:
    """Gradients (d_x, d_w1, d_w2, d_w3) of gated_ffn from the h it saved and the
    gradient d_out [T, H] of its result, all in x's dtype.

    The gradients of the pre-activations and the activations (made again from h)
    are rounded to that dtype between the products; sums are fp32. d_w1 and d_w3
    are the two halves of one buffer."""
    dev = _require_cuda(x, w1, w2, w3, h, d_out)
    if x.dtype not in _DTYPES:
        raise RuntimeError("gated_ffn_grad takes bf16 or fp16")
    gate, dtype = _gate(act), x.dtype
    x, w1, w2, w3, T, H, I = _check_ffn(x, w1, w2, w3, dtype, 8)
    h = _check_matrix("h", h, dtype, (2, T, I))
    d_out = _check_matrix("d_out", d_out, dtype, (T, H))
    d_x, d_w13, d_w2 = x.new_empty((T, H)), x.new_empty((2, I, H)), x.new_empty((H, I))
    L = lib()
    stream, sms = current_stream_handle(dev), int(num_sms or 0)
    need = L.ek_gated_ffn_grad_workspace_bytes(T, H, I, _most_sms(dev, sms))
    ws = _bytes(need, x)
    with _on_device(dev):
        check(L.ek_gated_ffn_grad(x.data_ptr(), w1.data_ptr(), w2.data_ptr(), w3.data_ptr(), h.data_ptr(),
                                  d_out.data_ptr(), d_x.data_ptr(), d_w13.data_ptr(), d_w2.data_ptr(), T, H, I,
                                  _DTYPES[dtype], gate, sms, ws.data_ptr(), need, stream), "ek_gated_ffn_grad")
    return d_x, d_w13[0], d_w2, d_w13[1]


def quant_ffn_weights_fp8(w1: torch.Tensor, w2: torch.Tensor, w3: torch.Tensor) -> dict:
    """e4m3 weights of a gated block (w1, w3 [I, H], w2 [H, I]; bf16 or fp32) with
    128 x 128 fp32 block scales, for gated_ffn_fp8."""
    I, H = w1.shape
    if w3.shape != w1.shape or tuple(w2.shape) != (H, I):
        raise RuntimeError("quant_ffn_weights_fp8: w1 and w3 must be [I, H] and w2 [H, I]")
    out = {"H": H, "I": I}
    for name, w in (("w1", w1), ("w3", w3), ("w2", w2)):
        out[name + "q"], out[name + "s"] = quant_e4m3(w, block=(128, 128))
    return out


def gated_ffn_fp8(x: torch.Tensor, qw: dict, act: str = "silu", out: torch.Tensor | None = None,
                  num_sms: int | None = None) -> torch.Tensor:
    """gated_ffn over e4m3 weights with block scales (quant_ffn_weights_fp8), bf16 x
    and y [T, H], H and I multiples of 16.

    The tokens, and the activations from their fp32 sums, are quantised per 1 x 128
    group as quant_e4m3(x, block=(1, 128)) does (the activations' scales not below
    2^-126); both products are gemm_fp8_block's. The result is rounded once."""
    H, I = int(qw["H"]), int(qw["I"])
    w1, w3, w2, s1, s3, s2 = (qw[n] for n in ("w1q", "w3q", "w2q", "w1s", "w3s", "w2s"))
    dev = _require_cuda(x, w1, w2, w3, s1, s2, s3, out)
    if x.dtype != torch.bfloat16 or _FP8 is None:
        raise RuntimeError("gated_ffn_fp8 takes bfloat16 tokens")
    gate = _gate(act)
    x, w1, w2, w3, T, Hx, Iw = _check_ffn(x, w1, w2, w3, torch.bfloat16, 16)
    if (Hx, Iw) != (H, I):
        raise RuntimeError(f"gated_ffn_fp8: x and weights of H={Hx}, I={Iw}, the dict says H={H}, I={I}")
    bh, bi = _blocks128(H), _blocks128(I)
    s1 = _check_matrix("w1s", s1, torch.float32, (bi, bh))
    s3 = _check_matrix("w3s", s3, torch.float32, (bi, bh))
    s2 = _check_matrix("w2s", s2, torch.float32, (bh, bi))
    if out is None:
        out = x.new_empty((T, H))
    else:
        _check_bf16("out", out)
        if tuple(out.shape) != (T, H):
            raise RuntimeError("out must be a [T, H] tensor")
    if T == 0:
        return out
    y = out if out.data_ptr() % 16 == 0 else x.new_empty((T, H))
    L = lib()
    stream, sms = current_stream_handle(dev), int(num_sms or 0)
    need = L.ek_gated_ffn_fp8_workspace_bytes(T, H, I, _most_sms(dev, sms))
    ws = _bytes(need, x)
    with _on_device(dev):
        check(L.ek_gated_ffn_fp8(x.data_ptr(), w1.data_ptr(), w2.data_ptr(), w3.data_ptr(), s1.data_ptr(),
                                 s2.data_ptr(), s3.data_ptr(), y.data_ptr(), T, H, I, gate, sms, ws.data_ptr(),
                                 need, stream), "ek_gated_ffn_fp8")
    return out if y is out else out.copy_(y)


def moe_segment_gemm(hidden_states: torch.Tensor, weights: torch.Tensor, expert_offsets: torch.Tensor,
                     num_experts: int, N: int, K: int, num_sms: int | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Reference segment GEMM semantics (sm_aware_benchmark.py:228-290)."""
    dev = _require_cuda(hidden_states, weights, expert_offsets, out)
    if hidden_states.dtype not in _DTYPES or weights.dtype != hidden_states.dtype:
        raise RuntimeError("segment GEMM takes bf16/fp16 operands of one dtype")
    for n, t in (("hidden_states", hidden_states), ("weights", weights), ("expert_offsets", expert_offsets)):
        _contig(n, t)
    if expert_offsets.dtype != torch.int32 or expert_offsets.numel() != num_experts + 1:
        raise RuntimeError("expert_offsets must be int32 [num_experts + 1]")
    M = hidden_states.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=hidden_states.dtype, device=dev)
    with _on_device(dev):
        check(lib().ek_moe_segment_gemm(hidden_states.data_ptr(), weights.data_ptr(), expert_offsets.data_ptr(),
                                        out.data_ptr(), M, int(N), int(K), int(num_experts),
                                        _DTYPES[hidden_states.dtype], int(num_sms or 0),
                                        current_stream_handle(dev)), "ek_moe_segment_gemm")
    return out
