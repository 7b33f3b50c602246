"""The tensor-core kernels of the 8-bit operators in their steady state: rings
and accumulators used over and over, several tiles a CTA, valid, masked and
empty tiles in turn.  Element by element against 64 bits; u is half a step of
fp32, and the tensor core's truncation counts 2^-22 of the magnitudes' sum for
each MMA that an accumulator takes (the alignment of the products and the sum)."""

import math

import pytest
import torch

from techjam_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
MMA = 2.0 ** -22


def rnd(shape, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV) * scale


def values(t, cols, rows_per_scale=1):
    s = torch.exp2(t.scales.view(torch.uint8).double() - 127)
    return t.codes.double() * s.repeat_interleave(rows_per_scale, 0)[: t.codes.shape[0]].repeat_interleave(128, 1)[:, :cols]


def close(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()}")


def stage_mask(rows, seed, run):
    """Runs of `run` rows that are whole, holed or empty, in a random order (the first whole, the second empty)."""
    g = torch.Generator().manual_seed(seed)
    m = torch.ones(rows, dtype=torch.bool)
    for i, kind in enumerate(torch.randint(0, 3, ((rows + run - 1) // run,), generator=g).tolist()):
        kind = {0: 0, 1: 2}.get(i, kind)
        part = m[i * run:(i + 1) * run]
        if kind == 1:
            part &= torch.rand(part.shape, generator=g) > 0.2
        elif kind == 2:
            part &= False
    return m.to(DEV)


# (stages of 64 tokens, 256 x 256 tiles): 66 on 72, 24 on 40, 11 on 112 for 74 pairs
# (some take two), 18 on 75
@pytest.mark.parametrize("rows,n,k", [(4200, 2048, 2304), (1500, 2048, 1280), (700, 4096, 1552), (1100, 1280, 3840)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
def test_wgrad_many_stages(rows, n, k, dt, masked):
    dy = rnd((rows, n), rows + n, 0.1).to(dt)
    x = rnd((rows, k), rows + k) * torch.exp2((torch.arange(k, device=DEV) // 128 * 3 % 5).float())
    x8 = ops.checkpoint8(x)
    xv, dv, m = values(x8, k), dy.double(), None
    if masked:
        m = stage_mask(rows, rows, 64)
        xv, dv = xv[m], dv[m]
        dy[~m] = math.nan
        x8.codes.view(torch.uint8)[~m] = 0x7f  # NaN
    dw, db = ops.linear_wgrad(dy, x8, m)
    again = ops.linear_wgrad(dy, x8, m)
    assert ops.device_error() == 0
    # 32 MMAs of 16 tokens per accumulator, one more for the start; then the accumulators' sum
    close(dw, dv.t() @ xv, (33 * MMA + (rows / 512 + 2) * U) * (dv.abs().t() @ xv.abs()) + 1e-30, "dweight")
    close(db, dv.sum(0), (rows + 64) * U * dv.abs().sum(0) + 1e-30, "dbias")
    assert torch.equal(dw, again[0]) and torch.equal(db, again[1])


# 160 tiles of 128 x 128 (40 of 256 x 256: single CTAs, some with two), and 250 of 256 x 256 for 74 pairs (four each);
# the last two with three and two accumulators a tile on either path
PRODUCTS = [(2000, 1280, 400), (6200, 2560, 144), (2000, 1280, 2080), (4000, 4096, 1168)]


def product_inputs(m, n, k, masked):
    a, w = rnd((m, k), m) * torch.exp(rnd((m, 1), 3)), rnd((n, k), n, k ** -0.5)
    a *= torch.exp2((torch.arange(k, device=DEV) // 128 * 5 % 7 - 3).float())
    w *= torch.exp2(-(torch.arange(k, device=DEV) // 128 * 3 % 5).float())
    a8, w8 = ops.checkpoint8(a), ops.pack_weight8(w)
    av, wv = values(a8, k), values(w8, k, 128)
    mask = stage_mask(m, k, 128) if masked else None
    if masked:
        a8.codes.view(torch.uint8)[~mask] = 0x7f
        av = torch.where(mask[:, None], av, 0.0)
    return a8, w8, av, wv, rnd((n,), 1, 0.5), mask


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
def test_product_many_tiles(m, n, k, out, masked):
    a8, w8, av, wv, bias, mask = product_inputs(m, n, k, masked)
    resid = rnd((m, n), 5) if out == torch.float32 else None
    live = torch.ones(m, 1, dtype=torch.bool, device=DEV) if mask is None else mask[:, None]
    base = av @ wv.t() + bias.double()
    want = torch.where(live, base + (0 if resid is None else resid.double()), 0.0)
    if masked and resid is not None:
        resid[~mask] = math.nan
    got = ops.gemm8(a8, w8, bias, mask, resid, out)
    again = ops.gemm8(a8, w8, bias, mask, resid, out)
    assert ops.device_error() == 0
    f = torch.finfo(out)
    steps = 33 if out == torch.float32 else k / 32 + 1
    tol = steps * MMA * (av.abs() @ wv.abs().t()) + (f.eps / 2 + 8 * U) * want.abs() + 8 * U * (base.abs() + bias.abs()) \
        + f.smallest_normal * f.eps / 2
    close(got, want, tol, "out")
    assert torch.all(got[~live.reshape(-1)] == 0) and torch.equal(got, again)


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("masked", [False, True])
def test_gelu_product_many_tiles(m, n, k, masked):
    """As test_product_many_tiles; a value may land on the code next to the
    exact one's, a scale beside the exact one only where the block's maximum
    lies within the error of the border between them."""
    a8, w8, av, wv, bias, mask = product_inputs(m, n, k, masked)
    live = torch.ones(m, 1, dtype=torch.bool, device=DEV) if mask is None else mask[:, None]
    got, again = ops.gemm8_gelu(a8, w8, bias, mask), ops.gemm8_gelu(a8, w8, bias, mask)
    assert ops.device_error() == 0
    h = av @ wv.t() + bias.double()
    err = 34 * MMA * (av.abs() @ wv.abs().t()) + 8 * U * (h.abs() + bias.abs())
    g = 0.5 * h * torch.special.erfc(-h / math.sqrt(2.0))
    for t, t2, want, e in ((got[0], again[0], g, 1.2 * err + 1e-6 * h.abs()), (got[1], again[1], h, err)):
        assert torch.equal(t.codes.view(torch.uint8), t2.codes.view(torch.uint8))
        assert torch.equal(t.scales.view(torch.uint8), t2.scales.view(torch.uint8))
        want, e = torch.where(live, want, 0.0), torch.where(live, e, 0.0)
        amax = want.unflatten(1, (-1, 128)).abs().amax(-1)
        frac, x = torch.frexp(amax)
        exps = torch.where(amax > 0, torch.where(frac <= 0.875, x - 9, x - 8), 0)
        have = t.scales.view(torch.uint8).int() - 127
        border = torch.ldexp(torch.full_like(amax, 448.0), torch.minimum(exps, have))
        beside = ((exps - have).abs() == 1) & ((amax - border).abs() <= e.unflatten(1, (-1, 128)).amax(-1))
        assert torch.all((exps == have) | beside)
        scale = torch.exp2(have.double()).repeat_interleave(128, 1)
        # half a step of 2^-3, relative to the value or to the smallest normal code's 2^-6
        close(values(t, n), want, 1.07 * e + 2.0 ** -4 * torch.maximum(want.abs(), 2.0 ** -6 * scale), "codes")
