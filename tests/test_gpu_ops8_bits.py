"""How many bits the 8-bit operators keep, against 64 bits and against the
same operator in plain 32-bit operations."""

import math

import pytest
import torch

from techjam_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rnd(shape, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV) * scale


def values(t, rows_per_scale=1):
    """The 64-bit values of an Act8 or Weight8 (cols a multiple of 128)."""
    s = torch.exp2(t.scales.view(torch.uint8).double() - 127)
    return t.codes.double() * s.repeat_interleave(rows_per_scale, 0)[: t.codes.shape[0]].repeat_interleave(128, 1)


def in_8_bits(v):
    """Values [rows, cols] as their 8-bit form holds them, in v's precision (cols a multiple of 128)."""
    b = v.unflatten(1, (-1, 128))
    m, k = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = torch.where(m <= 0.875, k - 9, k - 8)  # 448 = 0.875 * 2^9
    q = torch.ldexp(b, -e)
    _, k = torch.frexp(q)
    step = torch.ldexp(torch.ones_like(q), k.clamp_min(-5) - 4)
    return torch.ldexp(torch.round(q / step) * step, e).flatten(1)


def test_gelu_product_changes_no_more_codes_than_plain_32_bits():
    """A value whose 32-bit sum falls on the other side of a rounding boundary
    than the exact one gets the code next to it; the kernel may not do that
    more often than a plain 32-bit product, bias and GELU do.  Over 16 inputs
    of 33.5M values the plain form changes about 630 codes of g and 440 of h:
    counts whose ratio varies by 6-7% (one over the root of either, twice), so
    that 1.2 is three times that above an equal count."""
    m, n, k = 16384, 2048, 512
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    changed = {"g": [0, 0], "h": [0, 0]}
    try:
        for seed in range(16):
            a8, w8 = ops.checkpoint8(rnd((m, k), 3 * seed)), ops.pack_weight8(rnd((n, k), 3 * seed + 1, k ** -0.5))
            bias = rnd((n,), 3 * seed + 2, 0.1)
            a, w = values(a8), values(w8, 128)
            h = a @ w.t() + bias.double()
            want = {"h": in_8_bits(h), "g": in_8_bits(0.5 * h * torch.special.erfc(-h / math.sqrt(2.0)))}
            h = a.float() @ w.float().t() + bias
            plain = {"h": in_8_bits(h), "g": in_8_bits(0.5 * h * torch.special.erfc(h * -(0.5 ** 0.5)))}
            g8, h8 = ops.gemm8_gelu(a8, w8, bias)
            for key, own in (("g", values(g8)), ("h", values(h8))):
                changed[key][0] += int((own != want[key]).sum())
                changed[key][1] += int((plain[key].double() != want[key]).sum())
    finally:
        torch.backends.cuda.matmul.allow_tf32 = tf32
    assert ops.device_error() == 0
    for key, (own, plain) in changed.items():
        assert own <= 1.2 * plain, (key, own, plain)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_gelu_slope_keeps_its_tail(dt):
    """h in [-9, -1], relative to the slope itself: for a = |h| the exponent
    a^2 / 2 is rounded three times (constant, product, product: at most
    3 a^2 / 2 u), the exponential is 4 u off, and the rest (t with 4 u, nine
    terms whose magnitudes add up to 4 times their sum at most, two products
    and a difference of which the smaller term is at most 0.86) counts below
    60 u for a <= 1.5 and falls; then the product with dy and the output."""
    u = 2.0 ** -24
    h = -torch.linspace(1.0, 9.0, 100 * 1001, device=DEV).view(100, 1001)
    h = h.to(dt)
    dy = rnd(h.shape, 3).to(dt)
    x = h.double()
    slope = 0.5 * torch.special.erfc(-x / math.sqrt(2.0)) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    want = dy.double() * slope
    f = torch.finfo(dt)
    tol = ((1.5 * x * x + 66) * u + f.eps / 2) * want.abs() + f.smallest_normal * f.eps / 2
    got = ops.gelu_backward(dy, h).double()
    assert torch.all((got - want).abs() <= tol), float(((got - want).abs() / tol).max())


def test_gelu_slope_packed_tail():
    """A block of far negative values gets the scale and the codes of its own values."""
    h = -torch.linspace(6.0, 9.0, 64 * 128, device=DEV).view(64, 128)
    dy = torch.ones_like(h)
    dh, dh8 = ops.gelu_backward(dy, h, pack=True)
    x = h.double()
    want = 0.5 * torch.special.erfc(-x / math.sqrt(2.0)) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    assert torch.equal(values(dh8), in_8_bits(dh.double()))
    # half a step of a code with 3 fraction bits, or of the smallest under the row's scale (2^-10 of 2^-8 of its maximum)
    tol = (2.0 ** -4 + 1e-4) * want.abs() + 2.0 ** -17 * want.abs().amax(1, keepdim=True)
    assert torch.all((values(dh8) - want).abs() <= tol)
