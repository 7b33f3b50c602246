"""8-bit activations and the training operators on them, restated in 64 bits.

Test infrastructure only: plain CPU arithmetic, one definition per operator,
with no code shared with the product.  e4m3: 4 exponent bits (bias 7), 3
fraction bits, subnormal step 2^-9, largest value 448.
"""

from __future__ import annotations

import math

import torch

BLOCK = 128
E4M3_MAX = 448.0


def round_e4m3(q: torch.Tensor) -> torch.Tensor:
    """float64 values with |q| <= 448 to the nearest e4m3 value, ties to even."""
    _, k = torch.frexp(q)  # q = m * 2^k, 0.5 <= |m| < 1
    step = torch.ldexp(torch.ones_like(q), torch.clamp(k - 1, min=-6) - 3)
    return torch.round(q / step) * step


def block_exponent(amax: float) -> int:
    """Smallest e >= -127 with amax <= 448 * 2^e; 0 for amax 0."""
    if amax == 0.0:
        return 0
    e = -127
    while amax > math.ldexp(E4M3_MAX, e):
        e += 1
    return e


def _exponents(amax: torch.Tensor) -> torch.Tensor:
    return torch.tensor([block_exponent(float(a)) for a in amax.flatten()], dtype=torch.int64).reshape(amax.shape)


def _finite_abs(x):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))


def pack(x: torch.Tensor, mask=None):
    """x [rows, cols] -> (codes' values float64 [rows, cols], exponents [rows, blocks])."""
    x = x.double().cpu().clone()
    if mask is not None:
        x[~mask.cpu().reshape(-1)] = 0.0
    rows, cols = x.shape
    nb = -(-cols // BLOCK)
    codes = torch.empty_like(x)
    exps = torch.empty(rows, nb, dtype=torch.int64)
    for b in range(nb):
        blk = x[:, b * BLOCK:(b + 1) * BLOCK]
        e = _exponents(_finite_abs(blk).amax(1))
        q = round_e4m3(torch.ldexp(blk, -e[:, None]))
        q[~torch.isfinite(blk)] = math.nan
        codes[:, b * BLOCK:(b + 1) * BLOCK] = q
        exps[:, b] = e
    return codes, exps


def pack_weight(w: torch.Tensor):
    w = w.double().cpu()
    n, k = w.shape
    codes, exps = torch.empty_like(w), torch.empty(-(-n // BLOCK), -(-k // BLOCK), dtype=torch.int64)
    for i in range(exps.shape[0]):
        for j in range(exps.shape[1]):
            s = (slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK))
            e = block_exponent(float(_finite_abs(w[s]).max()))
            codes[s] = round_e4m3(torch.ldexp(w[s], torch.tensor(-e)))
            exps[i, j] = e
    return codes, exps


def value(codes: torch.Tensor, exps: torch.Tensor, rows_per_scale: int = 1) -> torch.Tensor:
    s = torch.ldexp(torch.ones(exps.shape, dtype=torch.float64), exps)
    s = s.repeat_interleave(rows_per_scale, 0)[: codes.shape[0]].repeat_interleave(BLOCK, 1)[:, : codes.shape[1]]
    return codes.double().cpu() * s


def gelu(h: torch.Tensor) -> torch.Tensor:
    return 0.5 * h * torch.special.erfc(-h / math.sqrt(2.0))


def gelu_slope(h: torch.Tensor) -> torch.Tensor:
    return 0.5 * torch.special.erfc(-h / math.sqrt(2.0)) + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)


def layernorm(x, weight, bias, eps, mask=None):
    """(y, mean, rstd) in float64, zeros for masked rows."""
    x = x.double().cpu()
    live = torch.ones(x.shape[0], dtype=torch.bool) if mask is None else mask.cpu().reshape(-1)
    x = torch.where(live[:, None], x, torch.zeros((), dtype=torch.float64))
    mean = x.mean(1)
    rstd = (x - mean[:, None]).square().mean(1).add(eps).rsqrt()
    y = (x - mean[:, None]) * rstd[:, None] * weight.double().cpu() + bias.double().cpu()
    zero = torch.zeros((), dtype=torch.float64)
    return torch.where(live[:, None], y, zero), torch.where(live, mean, zero), torch.where(live, rstd, zero)


def layernorm_backward(dy, x, weight, mean, rstd, mask=None, resid=None):
    """(dx, dweight, dbias, xhat) in float64 for given statistics."""
    dy, x, weight, mean, rstd = (t.double().cpu() for t in (dy, x, weight, mean, rstd))
    live = torch.ones(x.shape[0], dtype=torch.bool) if mask is None else mask.cpu().reshape(-1)
    zero = torch.zeros((), dtype=torch.float64)
    dy = torch.where(live[:, None], dy, zero)
    xhat = torch.where(live[:, None], (x - mean[:, None]) * rstd[:, None], zero)
    g = dy * weight
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if resid is not None:
        dx = dx + resid.double().cpu()
    return torch.where(live[:, None], dx, zero), (dy * xhat).sum(0), dy.sum(0), xhat
