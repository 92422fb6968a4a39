"""64-bit forms of the serving operators, for their tests, with the error bounds they are held to."""
from __future__ import annotations

import math

import torch

EPS32 = 2.0 ** -24  # half a step of a float32 value, relative
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: EPS32}
CODE_DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def code_grid(code: str) -> torch.Tensor:
    """Every value a code stands for, in order, zero in the middle; odd neighbours of even codes."""
    if code == "int8":
        return torch.arange(-127, 128, dtype=torch.float64)
    pos = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    pos = pos[:-1]  # the last pattern is NaN; 448 is the largest value
    return torch.tensor([-p for p in reversed(pos[1:])] + pos, dtype=torch.float64)


def quantise(x: torch.Tensor, code: str):
    """(values the codes stand for, exponent e) of 64-bit rows x (..., Dh): the
    exponent by trying them in turn, the code by looking for the nearest."""
    grid, c = code_grid(code), 448.0 if code == "e4m3" else 127.0
    x = x.double().cpu()
    a = x.abs().amax(-1)
    bad = ~torch.isfinite(a)
    a = torch.where(bad, 0.0, a)
    _, e = torch.frexp(a)
    e = torch.where(a == 0, -126, e - 12).clamp(min=-126)  # too small by a few ...
    for _ in range(8):                                      # ... so that the first that holds is the smallest
        e = torch.where(a > c * torch.exp2(e.double()), e + 1, e)
    v = torch.where(bad[..., None], 0.0, x) * torch.exp2(-e.double())[..., None]
    hi = torch.searchsorted(grid, v.contiguous()).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = v - grid[lo], grid[hi] - v
    even = (hi - grid.numel() // 2) % 2 == 0
    value = torch.where((above < below) | ((above == below) & even), grid[hi], grid[lo]) * torch.exp2(e.double())[..., None]
    return torch.where(bad[..., None], math.nan, value), torch.where(bad, 128, e)


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Interleaved pairs of x (n, heads, Dh) by cos / sin (n, Dh / 2), 64 bits."""
    z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], -1, 2).contiguous())
    return torch.view_as_real(z * torch.complex(cos.double(), sin.double())[:, None]).flatten(-2)


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, p_step: float = 0.0):
    """One row: q (H, Dh) over k / v (Hkv, len, Dh), all 64-bit values. Returns
    (out (H, Dh), bound): how far a float32 evaluation may be off before its
    output is rounded. A score's products and sums are off by at most
    (Dh + 4) half steps of the sum of its terms' magnitudes, so a probability by
    a factor within exp(2 d); its exponential and the sums over len terms add
    (len + 16) half steps; `p_step`: probabilities are rounded to that relative
    half step before they meet v."""
    H, Dh = q.shape
    Hkv, L, _ = k.shape
    if L == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    qh = q.view(Hkv, H // Hkv, Dh)
    s = torch.matmul(qh, k.transpose(1, 2)) * scale
    mag = torch.matmul(qh.abs(), k.abs().transpose(1, 2)) * abs(scale)
    p = torch.softmax(s, -1)
    out = torch.matmul(p, v)
    d = mag.amax(-1, keepdim=True) * (Dh + 4) * EPS32
    rel = torch.expm1(2 * d) + (L + 16) * 2 * EPS32 + p_step
    return out.reshape(H, Dh), (rel * torch.matmul(p, v.abs())).reshape(H, Dh)


def check_attention(got: torch.Tensor, ref: torch.Tensor, bound: torch.Tensor) -> None:
    """|got - ref| within the float32 bound and the half step of got's type (taken of the
    largest value the bound allows)."""
    half = HALF_STEP[got.dtype]
    err = (got.double().cpu() - ref).abs()
    tol = bound + half * (ref.abs() + bound) + 2.0 ** -126
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.3f} of its bound"
