"""Operators of a dense feed-forward block and of its 8-bit products, with their plain forms.

* gemm_fp8_block: a product of e4m3 matrices with an fp32 scale per 1 x 128 group of
  the tokens and per 128 x 128 block of the weight;
* gated_ffn: y = (f(x W1^T) * (x W3^T)) W2^T in bf16 or fp16, f one of silu, gelu
  and gelu_tanh, with or without the pre-activations that a backward pass needs;
* gated_ffn_grad: its gradients with respect to x and the three weights;
* gated_ffn_fp8: the same block over e4m3 weights with block scales, tokens and
  activations quantised per 1 x 128 group on the way.

``listed()`` names the measured cases, ``draw(rng)`` makes further ones of the
same ranges, ``prepare(case, seed)`` makes the inputs on the GPU, ``run(state)``
is one pass (plain torch, or the package's operators when ``own`` is set) and
``exact(case, seed)`` the same outputs in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_G = 128  # elements of K under one scale
_E4M3_MAX = 448.0


# ------------------------------------------------------------------------ cases
def _gemm_case(M, N, K, out):
    return dict(op="gemm_fp8_block", M=M, N=N, K=K, out=out)


def _ffn_case(T, H, I, dtype, act, save):
    return dict(op="gated_ffn", T=T, H=H, I=I, dtype=dtype, act=act, save=save)


def _grad_case(T, H, I, dtype, act):
    return dict(op="gated_ffn_grad", T=T, H=H, I=I, dtype=dtype, act=act)


def _fp8_case(T, H, I, act):
    return dict(op="gated_ffn_fp8", T=T, H=H, I=I, act=act)


def listed():
    return [
        # one token through a DeepSeek-V3 expert's projection: latency of a small weight
        dict(name="fp8-token", **_gemm_case(1, 2048, 7168, "bf16")),
        # a decode batch through a Mixtral projection: the weight's bytes
        dict(name="fp8-batch", **_gemm_case(64, 14336, 4096, "bf16")),
        # odd sizes, a part of a block at every edge, fp32 out as for logits or an accumulated gradient
        dict(name="fp8-ragged", **_gemm_case(1111, 2113, 7184, "fp32")),
        # a prompt or training batch at the Mixtral projection
        dict(name="fp8-prompt", **_gemm_case(4096, 14336, 4096, "bf16")),
        # one token through a dense block of the Mixtral expert's shape
        dict(name="ffn-token", **_ffn_case(1, 4096, 14336, "bf16", "silu", False)),
        # a decode batch through a shared expert of the DeepSeek-V3 shape, fp16, the tanh form
        dict(name="ffn-batch", **_ffn_case(48, 7168, 2048, "fp16", "gelu_tanh", False)),
        # the forward pass of a training step, pre-activations kept
        dict(name="ffn-train", **_ffn_case(4096, 4096, 14336, "bf16", "silu", True)),
        # backward of a short ragged batch through a small block, fp16
        dict(name="ffn-grad-ragged", **_grad_case(333, 1032, 2760, "fp16", "gelu")),
        # backward of the training step above
        dict(name="ffn-grad-long", **_grad_case(4096, 4096, 14336, "bf16", "silu")),
        # a few tokens through the shared expert in 8 bits
        dict(name="ffn-fp8-decode", **_fp8_case(16, 7168, 2048, "silu")),
        # a prompt through the Mixtral shape in 8 bits
        dict(name="ffn-fp8-prompt", **_fp8_case(2048, 4096, 14336, "silu")),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST = 4096 * 4096 * 14336
_ACTS = ["silu", "silu", "gelu", "gelu_tanh"]


def draw(rng):
    op = rng.choice(["gemm_fp8_block", "gated_ffn", "gated_ffn_grad", "gated_ffn_fp8"])
    while True:
        if op == "gemm_fp8_block":
            M, N, K = _log_int(rng, 1, 8192), _log_int(rng, 64, 28672), 16 * _log_int(rng, 4, 1024)
            if M * N * K <= _MOST and N * K <= 28672 * 4096:
                return _gemm_case(M, N, K, rng.choice(["bf16", "bf16", "fp16", "fp32"]))
            continue
        T = _log_int(rng, 1, 8192)
        u = 16 if op == "gated_ffn_fp8" else 8
        H, I = u * _log_int(rng, 128 // u, 8192 // u), u * _log_int(rng, 128 // u, 16384 // u)
        if T * H * I > _MOST or H * I > 4096 * 14336:
            continue
        dtype, act = rng.choice(["bf16", "fp16"]), rng.choice(_ACTS)
        if op == "gated_ffn":
            return _ffn_case(T, H, I, dtype, act, rng.random() < 0.4)
        if op == "gated_ffn_grad":
            return _grad_case(T, H, I, dtype, act)
        return _fp8_case(T, H, I, act)


def _blocks(n):
    return -(-n // _G)


def work(case):
    op = case["op"]
    if op == "gemm_fp8_block":
        M, N, K = case["M"], case["N"], case["K"]
        scales = 4 * _blocks(K) * (M + _blocks(N))
        return {"bytes": M * K + N * K + scales + M * N * _BYTES[case["out"]], "flops": 2 * M * N * K}
    T, H, I = case["T"], case["H"], case["I"]
    if op == "gated_ffn_fp8":
        return {"bytes": 3 * H * I + 12 * _blocks(H) * _blocks(I) + 4 * T * H, "flops": 6 * T * H * I}
    if op == "gated_ffn":
        return {"bytes": 2 * (3 * H * I + 2 * T * H + (2 * T * I if case["save"] else 0)), "flops": 6 * T * H * I}
    # x, d_out, both pre-activations and the weights in; d_x and the weights' gradients out
    return {"bytes": 2 * (6 * H * I + 3 * T * H + 2 * T * I), "flops": 12 * T * H * I}


# ------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _quantise(x, rows_per_block):
    """e4m3 codes and fp32 scales (largest magnitude / 448, 1 for zeros) of x [R, K] fp32
    per block of rows_per_block x 128."""
    R, K = x.shape
    b, rb, kb = rows_per_block, -(-R // rows_per_block), _blocks(K)
    pad = torch.zeros((rb * b, kb * _G), device=x.device)
    pad[:R, :K] = x
    v = pad.view(rb, b, kb, _G)
    s = v.abs().amax(dim=3).amax(dim=1)
    s = s / torch.full_like(s, _E4M3_MAX)  # a tensor: by a number, torch multiplies with the reciprocal
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (v / s[:, None, :, None]).view(rb * b, kb * _G)[:R, :K]
    return q.to(torch.float8_e4m3fn).contiguous(), s.contiguous()


def _tokens(g, T, K):
    """Hidden states: normal values, a few channels much larger than the rest, as a trained model has them."""
    x = _randn(g, T, K)
    loud = torch.rand((K,), generator=g, device="cuda") < 0.004
    return torch.where(loud, x * 20.0, x)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    st = {"case": case, "op": op}
    if op == "gemm_fp8_block":
        M, N, K = case["M"], case["N"], case["K"]
        st["a_q"], st["a_scale"] = _quantise(_tokens(g, M, K), 1)
        st["w_q"], st["w_scale"] = _quantise(_randn(g, N, K) / math.sqrt(K), _G)
        return st
    T, H, I = case["T"], case["H"], case["I"]
    if op == "gated_ffn_fp8":
        st["x"] = _tokens(g, T, H).to(torch.bfloat16)
        st["qw"] = {"H": H, "I": I}
        for name, n, k in (("w1", I, H), ("w3", I, H), ("w2", H, I)):
            st["qw"][name + "q"], st["qw"][name + "s"] = _quantise(_randn(g, n, k) / math.sqrt(k), _G)
        return st
    dt = _DTYPES[case["dtype"]]
    st["x"] = _randn(g, T, H).to(dt)
    st["w1"] = (_randn(g, I, H) / math.sqrt(H)).to(dt)
    st["w3"] = (_randn(g, I, H) / math.sqrt(H)).to(dt)
    st["w2"] = (_randn(g, H, I) / math.sqrt(I)).to(dt)
    if op == "gated_ffn_grad":
        xf = st["x"].float()
        st["h"] = torch.stack([(xf @ st[n].float().t()).to(dt) for n in ("w1", "w3")])
        st["d_out"] = (0.1 * _randn(g, T, H)).to(dt)
    return st


# ------------------------------------------------------------------------ plain forms
_SQRT_HALF = math.sqrt(0.5)
_TANH_A, _TANH_B = math.sqrt(2.0 / math.pi), 0.044715


def _plain_act(z, act):
    """f(z) and f'(z)."""
    if act == "silu":
        s = 1.0 / (1.0 + (-z).exp())
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * _SQRT_HALF))
        return z * c, c + z * (-0.5 * z * z).exp() * (_TANH_A * 0.5)
    t = torch.tanh(_TANH_A * (z + _TANH_B * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * _TANH_A * (1.0 + 3.0 * _TANH_B * z * z)


def _dequantise(q, s, rows_per_block):
    """The fp32 matrix that codes and scales stand for."""
    full = s.repeat_interleave(rows_per_block, dim=0)[:q.shape[0]] if rows_per_block > 1 else s
    return q.float() * full.repeat_interleave(_G, dim=1)[:, :q.shape[1]]


def _run_plain(st):
    case, op = st["case"], st["op"]
    if op == "gemm_fp8_block":
        y = _dequantise(st["a_q"], st["a_scale"], 1) @ _dequantise(st["w_q"], st["w_scale"], _G).t()
        return y.to(_DTYPES[case["out"]])
    if op == "gated_ffn_fp8":
        qw = st["qw"]
        w1, w3, w2 = (_dequantise(qw[n + "q"], qw[n + "s"], _G) for n in ("w1", "w3", "w2"))
        x = _dequantise(*_quantise(st["x"].float(), 1), 1)
        act = _plain_act(x @ w1.t(), case["act"])[0] * (x @ w3.t())
        return (_dequantise(*_quantise(act, 1), 1) @ w2.t()).to(torch.bfloat16)
    dt = st["x"].dtype
    x, w1, w2, w3 = (st[n].float() for n in ("x", "w1", "w2", "w3"))
    if op == "gated_ffn":
        h1, h3 = x @ w1.t(), x @ w3.t()
        y = ((_plain_act(h1, case["act"])[0] * h3) @ w2.t()).to(dt)
        return (y, torch.stack([h1, h3]).to(dt)) if case["save"] else y
    h1, h3, d_out = st["h"][0].float(), st["h"][1].float(), st["d_out"].float()
    f, df = _plain_act(h1, case["act"])
    d_a = d_out @ w2
    d1, d3 = d_a * h3 * df, d_a * f
    return ((d1 @ w1 + d3 @ w3).to(dt), (d1.t() @ x).to(dt), (d_out.t() @ (f * h3)).to(dt), (d3.t() @ x).to(dt))


# ------------------------------------------------------------------------ the package's operators
def _run_own(st):
    from elastikernel_b200 import _ops

    case, op = st["case"], st["op"]
    if op == "gemm_fp8_block":
        return _ops.gemm_fp8_block(st["a_q"], st["w_q"], st["a_scale"], st["w_scale"], dtype=_DTYPES[case["out"]])
    if op == "gated_ffn_fp8":
        return _ops.gated_ffn_fp8(st["x"], st["qw"], act=case["act"])
    if op == "gated_ffn":
        return _ops.gated_ffn(st["x"], st["w1"], st["w2"], st["w3"], act=case["act"], save=case["save"])
    return _ops.gated_ffn_grad(st["x"], st["w1"], st["w2"], st["w3"], st["h"], st["d_out"], act=case["act"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------ 64-bit values
def _exact_values(q, s, rows_per_block):
    """Codes times scales in 64 bits, one column of blocks at a time."""
    v = q.to(torch.float64)
    row = torch.arange(q.shape[0], device=q.device) // rows_per_block
    for b in range(s.shape[1]):
        v[:, b * _G:(b + 1) * _G] *= s[:, b].double()[row][:, None]
    return v


def _exact_round(v):
    """v [R, K] in 64 bits through e4m3 with a scale per 1 x 128: the scale and the
    quotient are fp32 by definition (a 16-bit value's quotient is often on a border),
    then 3 bits of mantissa, exponents from -6, halves to even."""
    out = torch.empty_like(v)
    for b in range(_blocks(v.shape[1])):
        p = v[:, b * _G:(b + 1) * _G]
        top = p.abs().amax(dim=1, keepdim=True).float()
        s = torch.where(top == 0, torch.ones_like(top), top / torch.full_like(top, _E4M3_MAX))
        z = (p.float() / s).double()
        exponent = (torch.frexp(z).exponent - 1).clamp(min=-6).double()
        step = torch.exp2(exponent - 3.0)
        out[:, b * _G:(b + 1) * _G] = torch.round(z / step) * step * s.double()
    return out


def _exact_gate(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    u = math.sqrt(8.0 / math.pi) * (z + 0.044715 * z ** 3)  # (1 + tanh(u/2)) / 2 = sigmoid(u)
    return z * torch.sigmoid(u)


def _exact_slope(z, act):
    if act == "silu":
        s = torch.sigmoid(z)
        return s + z * s * torch.sigmoid(-z)
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
    k = math.sqrt(8.0 / math.pi)
    s = torch.sigmoid(k * (z + 0.044715 * z ** 3))
    return s + z * s * (1.0 - s) * k * (1.0 + 3.0 * 0.044715 * z ** 2)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "gemm_fp8_block":
        return _exact_values(st["a_q"], st["a_scale"], 1) @ _exact_values(st["w_q"], st["w_scale"], _G).T
    if op == "gated_ffn_fp8":
        qw = st["qw"]
        w = {n: _exact_values(qw[n + "q"], qw[n + "s"], _G) for n in ("w1", "w3", "w2")}
        x = _exact_round(st["x"].double())
        return _exact_round(_exact_gate(x @ w["w1"].T, case["act"]) * (x @ w["w3"].T)) @ w["w2"].T
    x, w1, w2, w3 = (st[n].double() for n in ("x", "w1", "w2", "w3"))
    if op == "gated_ffn":
        g, u = x @ w1.T, x @ w3.T
        y = (_exact_gate(g, case["act"]) * u) @ w2.T
        return (y, torch.stack([g, u])) if case["save"] else y
    g, u, d = st["h"][0].double(), st["h"][1].double(), st["d_out"].double()
    d_act = d @ w2
    f = _exact_gate(g, case["act"])
    d_g, d_u = d_act * u * _exact_slope(g, case["act"]), d_act * f
    return d_g @ w1 + d_u @ w3, d_g.T @ x, d.T @ (f * u), d_u.T @ x
