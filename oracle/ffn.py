"""Dense feed-forward operators in float64 (torch tensors on any device): the
block-scaled product, the gated block, its gradients and its 8-bit form, with the
magnitudes that bound their rounding errors."""
from __future__ import annotations

import math

import torch

G = 128  # elements of K under one scale


def expand(q: torch.Tensor, s: torch.Tensor, rows: int) -> torch.Tensor:
    """Codes q [R, K] times the scales s of their rows x 128 blocks."""
    r = torch.arange(q.shape[0], device=q.device) // rows
    k = torch.arange(q.shape[1], device=q.device) // G
    return q.double() * s.double()[r][:, k]


def normal_cdf(z: torch.Tensor) -> torch.Tensor:
    # torch.special.ndtr is (1 + erf) / 2: zero from -9 down, where this keeps its digits
    return torch.special.erfc(z * -math.sqrt(0.5)) / 2


def gate(z: torch.Tensor, act: str) -> torch.Tensor:
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * normal_cdf(z)
    return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))


def slope(z: torch.Tensor, act: str) -> torch.Tensor:
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return normal_cdf(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
    return s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z ** 2)


def forward(x, w1, w2, w3, act: str) -> dict:
    x, w1, w2, w3 = (t.double() for t in (x, w1, w2, w3))
    h1, h3 = x @ w1.T, x @ w3.T
    a = gate(h1, act) * h3
    return {"h": torch.stack([h1, h3]), "a": a, "y": a @ w2.T}


def backward(x, w1, w2, w3, h, d_out, act: str) -> dict:
    x, w1, w2, w3, h, d_out = (t.double() for t in (x, w1, w2, w3, h, d_out))
    da = d_out @ w2
    f = gate(h[0], act)
    d1, d3, a = da * h[1] * slope(h[0], act), da * f, f * h[1]
    return {"da": da, "d1": d1, "d3": d3, "a": a, "x": d1 @ w1 + d3 @ w3, "w1": d1.T @ x, "w2": d_out.T @ a,
            "w3": d3.T @ x}


def e4m3_groups(v: torch.Tensor) -> torch.Tensor:
    """v [R, K] as its e4m3 codes per 1 x 128 group stand for it: scale = largest / 448
    (1 for zeros) and quotient in fp32 as the quantisation defines them (16-bit values
    often have quotients on a border, where 64 bits would round to the other side), then
    3 bits of mantissa, exponents from -6, halves to even."""
    out = torch.empty_like(v)
    for k in range(0, v.shape[1], G):
        p = v[:, k:k + G]
        top = p.abs().amax(dim=1, keepdim=True).float()
        # a tensor below the bar: torch takes a number there as a product with its reciprocal
        s = torch.where(top > 0, top / torch.full_like(top, 448.0), torch.ones_like(top))
        z = (p.float() / s).double()
        step = torch.exp2((torch.frexp(z).exponent - 1).clamp(min=-6).double() - 3)
        out[:, k:k + G] = torch.round(z / step) * step * s.double()
    return out


def forward_fp8(x, w1, w2, w3, act: str) -> dict:
    """The 8-bit block over the float64 weights that the codes stand for."""
    xq = e4m3_groups(x.double())
    a = gate(xq @ w1.T, act) * (xq @ w3.T)
    aq = e4m3_groups(a)
    return {"x": xq, "a": a, "aq": aq, "y": aq @ w2.T}
