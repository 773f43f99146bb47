"""Microscaled formats and products in 64 bits on the CPU -- TEST INFRASTRUCTURE, never the product path.

Written from the formats' definition (``include/ipc_b200.h``): a block of 32 numbers is kept as codes and one power
of two, the smallest that clips nothing.  Layout functions follow the same text.
"""
from __future__ import annotations

import torch

from . import ipc_oracle as O

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _blocks(v: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.pad(v.double(), (0, (-v.shape[1]) % 32)).reshape(v.shape[0], -1, 32)


def _scale_byte(m: torch.Tensor, top: float) -> torch.Tensor:
    """s + 127 for the smallest s >= -127 with m <= top * 2^s; 255 where m is not finite."""
    fin = torch.isfinite(m)
    frac, exp = torch.frexp(torch.where(fin, m, torch.zeros_like(m)) / top)
    s = torch.where(frac == 0.5, exp - 1, exp)
    s = torch.where(m > 0, s, torch.full_like(s, -127)).clamp(min=-127)
    return torch.where(fin, s + 127, torch.full_like(s, 255)).to(torch.int64)


def _amax(v: torch.Tensor) -> torch.Tensor:
    a = v.abs()
    return torch.where(torch.isnan(a).any(-1), torch.full(a.shape[:-1], float("nan"), dtype=a.dtype), a.amax(-1))


def store8(x: torch.Tensor):
    """Codes [D, 32 nb] and scale bytes [nb, D] of states ``x [D, B]``."""
    v = _blocks(x)
    byte = _scale_byte(_amax(v), 127.0)
    bad = (byte == 255)[..., None]
    c = torch.round(torch.where(bad, torch.zeros_like(v), v) / torch.exp2(byte.double() - 127)[..., None])
    c = torch.where(bad, torch.zeros_like(c), c)
    return c.reshape(x.shape[0], -1).to(torch.int8), byte.t().contiguous().to(torch.uint8)


def load8(codes: torch.Tensor, scales: torch.Tensor, B: int) -> torch.Tensor:
    D = codes.shape[0]
    p = torch.exp2(scales.double() - 127).t()
    p = torch.where(scales.t() == 255, torch.full_like(p, float("nan")), p)
    return (codes.double().reshape(D, -1, 32) * p[..., None]).reshape(D, -1)[:, :B]


def quant4(v: torch.Tensor):
    """Values [R, K] a 4-bit operand of ``v [R, K]`` stands for, its codes [R, Kp/2] and scale bytes."""
    R, K = v.shape
    kp = -(-K // 128) * 128
    w = _blocks(torch.nn.functional.pad(v.double(), (0, kp - K)))
    byte = _scale_byte(_amax(w), 6.0)
    bad = (byte == 255)[..., None]
    step = torch.exp2(byte.double() - 127)[..., None]
    u = torch.where(bad, torch.zeros_like(w), w).abs() / step
    d = (u[..., None] - GRID).abs()
    best = d.amin(-1, keepdim=True)
    even = torch.tensor([0, 2, 4, 6])
    tie = (d == best).sum(-1) == 2
    idx = d.argmin(-1)
    idx_even = even[(d[..., 0::2]).argmin(-1)]
    idx = torch.where(tie, idx_even, idx)
    val = torch.sign(w) * GRID[idx] * step
    val = torch.where(bad, torch.full_like(val, float("nan")), val)
    code = (idx + 8 * torch.signbit(w).to(idx.dtype)) * (~bad)
    code = code.reshape(R, kp // 2, 2).to(torch.uint8)
    rp = -(-R // 128) * 128
    full = torch.zeros(rp, kp // 32, dtype=torch.uint8)
    full[:R] = byte.to(torch.uint8)
    r = torch.arange(rp)[:, None]
    j = torch.arange(kp // 32)[None, :]
    scales = torch.zeros(rp // 128, kp // 128, 32, 4, 4, dtype=torch.uint8)
    scales[r // 128, j // 4, r % 32, r % 128 // 32, j % 4] = full
    return val.reshape(R, kp)[:, :K], code[..., 0] + 16 * code[..., 1], scales


def slope(act: str, x: torch.Tensor) -> torch.Tensor:
    return O.act_derivative(act, x)


def delta(e, xhat, act, alpha):
    return alpha * (e.double() @ O.act_forward(act, xhat.double()).t())


def backward(w, e, xhat, act):
    return slope(act, xhat.double()) * (w.double().t() @ e.double())
