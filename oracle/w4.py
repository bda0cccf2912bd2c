"""4-bit weights with group scales: quantisation in float32 as the kernels
define it, and the weights and products in float64."""
from __future__ import annotations

import numpy as np
import torch


def quantise(w: torch.Tensor, group: int, symmetric: bool, dtype: torch.dtype):
    """(codes uint8 [N, ceil(K/32)*16], scales, mins | None) of w [N, K] on the CPU."""
    w = w.float()
    N, K = w.shape
    G, Kp = -(-K // group), -(-K // 32) * 32
    pad = torch.zeros((N, G * group))
    pad[:, :K] = w
    inside = torch.zeros(G * group, dtype=torch.bool)
    inside[:K] = True
    v, ok = pad.view(N, G, group), inside.view(1, G, group)
    hi = torch.where(ok, v, -torch.inf).amax(dim=2)
    lo = torch.where(ok, v, torch.inf).amin(dim=2)
    top = torch.finfo(dtype).max
    if symmetric:
        m = torch.zeros_like(lo)
        s = (torch.maximum(hi.abs(), lo.abs()) / 7).clamp(max=top).to(dtype)
    else:
        m = lo.clamp(-top, top).to(dtype)
        s = ((hi - m.float()) / 15).clamp(max=top).to(dtype)
    s = torch.where(s > 0, s, torch.ones_like(s))
    q = torch.round((v - m.float()[..., None]) / s.float()[..., None]) + (8 if symmetric else 0)
    q = torch.where(ok, q.clamp(0, 15), torch.tensor(8.0 if symmetric else 0.0))
    q = q.view(N, G * group).to(torch.uint8)
    q = q[:, :Kp] if G * group >= Kp else torch.nn.functional.pad(q, (0, Kp - G * group))
    return q[:, 0::2] | (q[:, 1::2] << 4), s, None if symmetric else m


def values(codes, scales, mins, K: int, group: int) -> np.ndarray:
    """Float64 weights [..., N, K] of packed codes (torch tensors on any device)."""
    c = codes.cpu().numpy()
    q = np.stack([c & 15, c >> 4], axis=-1).reshape(c.shape[:-1] + (-1,))[..., :K].astype(np.float64)
    at = np.arange(K) // group
    s = scales.double().cpu().numpy()[..., at]
    return s * (q - 8) if mins is None else s * q + mins.double().cpu().numpy()[..., at]


def abs_bound(codes, scales, mins, K: int, group: int) -> np.ndarray:
    """Float64 bound |s| q' + |m| of the magnitudes a product's partial sums add up."""
    if mins is None:
        return np.abs(values(codes, scales, None, K, group))
    return np.abs(values(codes, scales, torch.zeros_like(scales), K, group)) + \
        np.abs(mins.double().cpu().numpy()[..., np.arange(K) // group])
