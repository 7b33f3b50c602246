"""The training and 8-bit operators on the GPU against 64-bit restatements.

Tolerances are error bounds, element by element: u is half a step of fp32
(2^-24), `half(t)` half a relative step of the output's type; counts of
roundings stand where they are used.
"""

import math

import pytest
import torch

from oracle import act8
from techjam_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F = [torch.float32, torch.float16, torch.bfloat16]


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the smallest subnormal step: what a result near zero may lose."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def close(got, want, tol, what=""):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{((got - want).abs() / tol.clamp_min(1e-300))[bad].max().item():.3g} of the bound, first at "
                           f"{bad.nonzero()[0].tolist()}: {got[bad][0].item()} for {want[bad][0].item()}")


def rnd(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def padding(b, n, seed, hole=False):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(0, n + 1, (b,), generator=g)
    lengths[0] = n
    if b > 1:
        lengths[1] = 0
    m = torch.arange(n)[None, :] < lengths[:, None]
    if hole:
        m &= torch.rand(b, n, generator=g) > 0.3
    return m


def e8m0(exps):
    return (exps + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def act(values_codes, exps, dtype=torch.float32):
    return ops.Act8(values_codes.to(torch.float8_e4m3fn).to(DEV), e8m0(exps).to(DEV), dtype)


def check_pack(got, codes, exps, what=""):
    gs = got.scales.view(torch.uint8).cpu().long() - 127
    assert torch.equal(gs, exps), f"{what}: scales"
    gc = got.codes.float().cpu().double()
    assert torch.equal(torch.isnan(gc), torch.isnan(codes)), f"{what}: NaN places"
    assert torch.equal(torch.nan_to_num(gc), torch.nan_to_num(codes)), f"{what}: codes"


# ---------------------------------------------------------------- pack and restore
SPECIAL = [0.0, -0.0, 448.0, 448.00003, 1.75 * 2.0 ** 20, math.nextafter(1.75 * 2.0 ** 20, 2e9), 3.4028234e38, 2.0 ** -126,
           2.0 ** -140, 2.0 ** -149, 1e-30, math.inf, -math.inf, math.nan, 2.0 ** -9, 2.0 ** -10, 1.0625, 1.1875]


@pytest.mark.parametrize("dtype", F)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (5, 129), (33, 1000), (2, 4096), (257, 36), (7, 1001)])
def test_checkpoint_and_restore(rows, cols, dtype):
    x = rnd((rows, cols), rows + cols, scale=3.0)
    x *= torch.exp(3 * rnd((rows, 1), 5))
    x = x.to(dtype)
    got = ops.checkpoint8(x.to(DEV))
    codes, exps = act8.pack(x)
    check_pack(got, codes, exps)
    want = act8.value(codes, exps)
    assert torch.equal(ops.restore8(got, torch.float32).double().cpu(), want)
    # bf16 holds e4m3 times a power of two exactly, fp16 within its range
    assert torch.equal(ops.restore8(got, torch.bfloat16).double().cpu(), want)
    assert torch.equal(ops.restore8(got, torch.float16).cpu(), want.clamp(-65504, 65504).half())
    assert ops.restore8(got).dtype == dtype


def test_checkpoint_special_values():
    """Every special value alone in a block of ones, alone among zeros, and together."""
    rows = []
    for s in SPECIAL:
        for fill in (1.0, 0.0, s):
            r = torch.full((128,), fill)
            r[17] = s
            rows.append(r)
    x = torch.stack(rows)
    for d in F:
        xd = x.to(d)
        codes, exps = act8.pack(xd)
        got = ops.checkpoint8(xd.to(DEV))
        check_pack(got, codes, exps, str(d))
        want = act8.value(codes, exps)
        for t in F:  # beyond a type's range: its largest value
            back, lim = ops.restore8(got, t).cpu(), torch.finfo(t).max
            assert torch.equal(torch.isnan(back), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(back), torch.nan_to_num(want).clamp(-lim, lim).to(t))


def test_restore_every_code_and_scale():
    """All 256 codes under every one of the 256 scale bytes, 255 (NaN) included."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).view(torch.float8_e4m3fn)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 2).view(torch.float8_e8m0fnu)
    a = ops.Act8(codes.to(DEV), scales.to(DEV), torch.float32)
    want = codes.float().double() * torch.exp2(torch.arange(256).double() - 127)[:, None]
    want[255] = math.nan
    want = want.clamp(-torch.finfo(torch.float32).max, torch.finfo(torch.float32).max).float()  # exact within fp32's range
    got = ops.restore8(a).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_checkpoint_masked_rows_are_not_read():
    x = rnd((96, 200), 3)
    m = padding(3, 32, 1)
    x[~m.reshape(-1)] = math.nan
    got = ops.checkpoint8(x.to(DEV), m.to(DEV))
    check_pack(got, *act8.pack(x, m))


def test_checkpoint_unaligned_views():
    """Rows that start at odd addresses: contiguous views into a larger buffer."""
    for dtype in F:
        buf = rnd((1 + 64 * 132,), 11, dtype)
        x = buf.to(DEV)[1:].view(64, 132)
        assert x.is_contiguous()
        check_pack(ops.checkpoint8(x), *act8.pack(buf[1:].view(64, 132)))


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 257), (1000, 528), (64, 1024)])
@pytest.mark.parametrize("dtype", F)
def test_pack_weight(n, k, dtype, transpose):
    w = (rnd((n, k), n) * torch.exp(rnd((n, 1), 2))).to(dtype)
    got = ops.pack_weight8(w.to(DEV), transpose)
    codes, exps = act8.pack_weight(w)
    check_pack(got, *((codes.t(), exps.t()) if transpose else (codes, exps)))


# ---------------------------------------------------------------- layer norm
def norm_inputs(rows, d, xt, seed):
    x = (rnd((rows, d), seed) * (0.5 + torch.rand(d, generator=torch.Generator().manual_seed(seed))) +
         rnd((rows, 1), seed + 1)).to(xt)
    return x, 1 + rnd((d,), seed + 2, scale=0.3), rnd((d,), seed + 3, scale=0.3)


# a row's sum: 32 values per lane in a chain, 5 shuffles, up to 4 warps, the
# division: at most 42 roundings; 48 bounds them
SUM = 48 * U


def y_tolerance(x, y, w, b, mean, rstd, out):
    """xhat's error: the mean's (SUM of the mean magnitude, in units of the
    standard deviation), the variance's (half of 2 SUM: it is a sum of squares
    of deviations, each with the mean's error, whose first order cancels),
    rsqrt and three products; then two more roundings and the output's."""
    dev = (x.double() - mean[:, None]).abs() * rstd[:, None]
    mag = x.double().abs().mean(1, keepdim=True) * rstd[:, None]
    dx = SUM * mag + (SUM + 8 * U) * dev + (SUM * mag) ** 2 * dev
    return dx * w.double().abs() + 4 * U * (dev * w.double().abs() + b.double().abs()) + half(out) * y.abs() + tiny(out)


@pytest.mark.parametrize("rows,d", [(1, 1), (1, 256), (5, 64), (33, 1000), (130, 1001), (9, 2048), (6, 4096), (4, 2052),
                                    (3, 3999), (2000, 512)])
@pytest.mark.parametrize("xt", F)
def test_layernorm_forward(rows, d, xt):
    x, w, b = norm_inputs(rows, d, xt, rows + d)
    y, mean, rstd = act8.layernorm(x, w, b, 1e-5)
    for out in F:
        got = ops.layernorm_train(x.to(DEV), w.to(DEV), b.to(DEV), out_dtype=out)
        assert got.x8 is None and got.y.dtype == out
        close(got.y, y, y_tolerance(x, y, w, b, mean, rstd, out), f"y {out}")
        close(got.mean, mean, (SUM + U) * x.double().abs().mean(1) + 1e-30, "mean")
        mag = x.double().abs().mean(1) * rstd
        close(got.rstd, rstd, rstd * (SUM + 8 * U + (SUM * mag) ** 2), "rstd")


@pytest.mark.parametrize("rows,d", [(1, 256), (33, 1000), (70, 1001), (6, 4096), (9, 2048), (130, 100)])
def test_layernorm_forward_8bit(rows, d):
    """The 8-bit copy of x is that of checkpoint8, and the 8-bit y that of the
    32-bit y of the same call: the same values packed the same way."""
    x, w, b = norm_inputs(rows, d, torch.float32, 7)
    m = padding(1, rows, 3, hole=True).reshape(-1) if rows > 1 else None
    args = (x.to(DEV), w.to(DEV), b.to(DEV), None if m is None else m.to(DEV))
    f32 = ops.layernorm_train(*args, out_dtype=torch.float32, checkpoint=True)
    f8 = ops.layernorm_train(*args, out_dtype=torch.float8_e4m3fn, checkpoint=True)
    for f in (f32, f8):
        check_pack(f.x8, *act8.pack(x, m), "x8")
    check_pack(f8.y, *act8.pack(f32.y), "y8")
    assert torch.equal(f8.mean, f32.mean) and torch.equal(f8.rstd, f32.rstd)


@pytest.mark.parametrize("rows,d", [(1, 1), (1, 256), (5, 64), (33, 1000), (700, 1001), (9, 2048), (6, 4096), (40, 2052),
                                    (3000, 512), (2500, 1024)])
@pytest.mark.parametrize("xt,dt,kept,resid", [(torch.float32, torch.float16, False, True),
                                              (torch.float32, torch.bfloat16, True, True),
                                              (torch.bfloat16, torch.float32, False, False),
                                              (torch.float16, torch.float16, True, False),
                                              (torch.float16, torch.bfloat16, False, True),
                                              (torch.bfloat16, torch.bfloat16, True, True)])
def test_layernorm_backward(rows, d, xt, dt, kept, resid):
    x, w, _ = norm_inputs(rows, d, xt, rows + 3 * d)
    dy = rnd((rows, d), 17, dt, 0.1)
    r = rnd((rows, d), 19, xt, 0.1) if resid else None
    _, mean, rstd = act8.layernorm(x, w, w, 1e-5)
    mean, rstd = mean.float(), rstd.float()
    xd = ops.checkpoint8(x.to(DEV)) if kept else x.to(DEV)
    xv = act8.value(*act8.pack(x)) if kept else x
    dx, dw, db, xh = act8.layernorm_backward(dy, xv, w, mean, rstd, resid=r)
    got = ops.layernorm_backward(dy.to(DEV), xd, w.to(DEV), mean.to(DEV), rstd.to(DEV),
                                 resid_grad=None if r is None else r.to(DEV))
    assert got[0].dtype == xt
    g = dy.double() * w.double()
    xm = xv.double().abs() * rstd.double()[:, None] + mean.double().abs()[:, None] * rstd.double()[:, None]
    # xhat: the difference (rounded once against |x| + |mean|) and a product
    exh = 2 * U * (xh.abs() + xm)
    m0, m1 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    em1 = (g.abs() * exh).mean(1, keepdim=True) + (SUM + 4 * U) * m1
    tol = rstd.double()[:, None] * (4 * U * g.abs() + (SUM + 4 * U) * m0 + xh.abs() * (em1 + 4 * U * m1) + exh * m1)
    tol = tol + 3 * U * (dx.abs() + (r.double().abs() if resid else 0)) + half(xt) * dx.abs() + tiny(xt)
    close(got[0], dx, tol, "dx")
    # a column: rows in a chain per warp (3000 rows over 444 CTAs of 4), then
    # the CTA's warps and up to 444 partial rows in 32 chains: below 48
    close(got[1], dw, SUM * (dy.double() * xh).abs().sum(0) + (dy.double().abs() * exh).sum(0) + 1e-30, "dweight")
    close(got[2], db, SUM * dy.double().abs().sum(0) + 1e-30, "dbias")


@pytest.mark.parametrize("d", [100, 1024, 3000])
def test_layernorm_masked_rows(d):
    """Masked rows hold NaN in every input and leave zeros; a batch with no
    valid row at all leaves zero gradients."""
    b, n = 4, 37
    for m in (padding(b, n, 5), padding(b, n, 6, hole=True), torch.zeros(b, n, dtype=torch.bool)):
        flat = m.reshape(-1)
        x, w, bias = norm_inputs(b * n, d, torch.float32, d)
        dy, r = rnd((b * n, d), 1, scale=0.1), rnd((b * n, d), 2, scale=0.1)
        for t in (x, dy, r):
            t[~flat] = math.nan
        f = ops.layernorm_train(x.to(DEV), w.to(DEV), bias.to(DEV), m.to(DEV), out_dtype=torch.float32, checkpoint=True)
        y, mean, rstd = act8.layernorm(x, w, bias, 1e-5, m)
        assert torch.all(f.y.cpu()[~flat] == 0) and torch.all(f.mean.cpu()[~flat] == 0)
        assert torch.all(f.rstd.cpu()[~flat] == 0) and torch.all(f.x8.codes.float().cpu()[~flat] == 0)
        xs = torch.where(flat[:, None], x, torch.zeros(()))
        close(f.y, y, y_tolerance(xs, y, w, bias, mean, rstd, torch.float32) + 1e-30)
        for xin, xv in ((x.to(DEV), xs), (f.x8, act8.value(*act8.pack(x, m)))):
            dx, dw, db, _ = act8.layernorm_backward(torch.nan_to_num(dy), xv, w, f.mean, f.rstd, m, torch.nan_to_num(r))
            got = ops.layernorm_backward(dy.to(DEV), xin, w.to(DEV), f.mean, f.rstd, m.to(DEV), r.to(DEV))
            assert torch.all(got[0].cpu()[~flat] == 0)
            for a, e in zip(got, (dx, dw, db)):
                assert torch.isfinite(a).all()
                torch.testing.assert_close(a.double().cpu(), e, atol=2e-5, rtol=2e-5)
            if not flat.any():
                assert torch.all(got[1] == 0) and torch.all(got[2] == 0)


def test_layernorm_gradient_against_differences():
    """dx, dweight and dbias of the scalar sum(y * dy) against central
    differences of the forward kernel itself (fp32 in and out)."""
    rows, d = 3, 40
    x, w, b = norm_inputs(rows, d, torch.float32, 23)
    dy = rnd((rows, d), 24)
    f = ops.layernorm_train(x.to(DEV), w.to(DEV), b.to(DEV), out_dtype=torch.float32)
    dx, dw, db = ops.layernorm_backward(dy.to(DEV), x.to(DEV), w.to(DEV), f.mean, f.rstd)

    def loss(xx, ww, bb):
        return (act8.layernorm(xx, ww, bb, 1e-5)[0] * dy.double()).sum()

    for t, g, which in ((x, dx, 0), (w, dw, 1), (b, db, 2)):
        for idx in range(0, t.numel(), 7):
            v = [x.double(), w.double(), b.double()]
            e = torch.zeros(t.numel(), dtype=torch.float64)
            e[idx] = 1e-5
            lo, hi = list(v), list(v)
            lo[which], hi[which] = v[which] - e.view_as(v[which]), v[which] + e.view_as(v[which])
            # the difference's own error: 1e-10 of curvature, 1e-16 / 1e-5 of cancellation
            want = float((loss(*hi) - loss(*lo)) / 2e-5)
            assert abs(float(g.reshape(-1)[idx]) - want) <= 2e-5 * (1 + abs(want))


def test_layernorm_empty_and_in_place():
    w, b = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    f = ops.layernorm_train(torch.empty(0, 64, device=DEV), w, b)
    assert f.y.shape == (0, 64)
    dx, dw, db = ops.layernorm_backward(torch.empty(0, 64, device=DEV), torch.empty(0, 64, device=DEV), w, f.mean, f.rstd)
    assert dx.shape == (0, 64) and torch.all(dw == 0) and torch.all(db == 0)


# ---------------------------------------------------------------- GELU
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 129), (33, 1000), (17, 1001), (64, 2048)])
@pytest.mark.parametrize("dt", F)
def test_gelu_backward(rows, cols, dt):
    dy = rnd((rows, cols), 31, dt, 0.3)
    h = rnd((rows, cols), 32, scale=2.0).to(dt)
    h.view(-1)[:: 7] *= 10
    codes, exps = act8.pack(h)
    m = padding(1, rows, 1, hole=True) if rows > 1 else None
    md = None if m is None else m.to(DEV)
    for hin, hv in ((act(codes, exps), act8.value(codes, exps)), (h.to(DEV), h.double())):
        want = dy.double() * act8.gelu_slope(hv)
        # the series 0.75e-7, exponential and reciprocal a few u each on values below 1.2: 1e-6 bounds them
        tol = 1e-6 * dy.double().abs() + (half(dt) + 2 * U) * want.abs() + tiny(dt)
        if m is not None:
            want = want * m.reshape(-1, 1)
        dh = ops.gelu_backward(dy.to(DEV), hin, md)
        close(dh, want, tol, "dh")
        dh2, packed = ops.gelu_backward(dy.to(DEV), hin, md, pack=True)
        assert torch.equal(dh, dh2)
        check_pack(packed, *act8.pack(dh.cpu()), "packed")


def test_gelu_backward_extremes():
    h = torch.tensor([[0.0, -0.0, 40.0, -40.0, 1e20, -1e20, 3e38, math.inf, -math.inf, math.nan, 5.0, -5.0, -13.0, 1e-30]])
    dy = torch.ones_like(h)
    got = ops.gelu_backward(dy.to(DEV), h.to(DEV)).cpu()[0]
    want = torch.tensor([0.5, 0.5, 1, 0, 1, 0, 1, 1, 0, math.nan, 1.0000072, -7.2e-06, 0, 0.5])
    assert math.isnan(got[9])
    torch.testing.assert_close(torch.nan_to_num(got), torch.nan_to_num(want), atol=1e-6, rtol=0)


# ---------------------------------------------------------------- products
def product_inputs(m, n, k, seed):
    a = rnd((m, k), seed) * torch.exp(2 * rnd((m, 1), seed + 1))
    # blocks of K of very different scale, so that a scale applied to another block shows
    a *= torch.exp2((torch.arange(k) // 128 * 5 % 7 - 3).float())
    w = rnd((n, k), seed + 2, scale=k ** -0.5) * torch.exp2((torch.arange(n) // 128 % 3).float())[:, None]
    w *= torch.exp2(-(torch.arange(k) // 128 * 3 % 5).float())
    return a, w


def product_tolerance(av, wv, k, out, acc, steps):
    """Each MMA of 32 products adds with truncation to about 2^-23 of what it
    holds, which sum |a||w| bounds; twice that, for the alignment of the products."""
    return 2 * 2.0 ** -23 * steps * (av.abs() @ wv.abs().t()) + half(out) * acc.abs() + 4 * U * acc.abs() + tiny(out)


@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (1, 4096, 1024), (128, 128, 128), (129, 136, 144), (300, 264, 1040),
                                   (777, 1000, 528), (257, 2048, 640), (64, 64, 4112), (2000, 1024, 256),
                                   # enough 256 x 256 tiles for CTA pairs, ragged in each direction
                                   (2500, 2056, 272), (2304, 2304, 1168), (19000, 200, 32), (2304, 2056, 2064)])
@pytest.mark.parametrize("out", F)
def test_product(m, n, k, out):
    a, w = product_inputs(m, n, k, m + n + k)
    ac, ae = act8.pack(a)
    wc, we = act8.pack_weight(w)
    av, wv = act8.value(ac, ae), act8.value(wc, we, 128)
    w8 = ops.Weight8(wc.to(torch.float8_e4m3fn).to(DEV), e8m0(we).to(DEV))
    bias, resid = rnd((n,), 1), rnd((m, n), 2)
    acc = av @ wv.t()
    steps = 33 + k / 1024 if out == torch.float32 else k / 32 + 1
    got = ops.gemm8(act(ac, ae), w8, out_dtype=out)
    assert ops.device_error() == 0
    close(got, acc, product_tolerance(av, wv, k, out, acc, steps), "plain")
    full = acc + bias.double()
    tol = product_tolerance(av, wv, k, out, full, steps) + 2 * U * acc.abs()
    close(ops.gemm8(act(ac, ae), w8, bias.to(DEV), out_dtype=out), full, tol, "bias")
    if out == torch.float32:
        got = ops.gemm8(act(ac, ae), w8, bias.to(DEV), resid=resid.to(DEV), out_dtype=out)
        close(got, full + resid.double(), tol + 2 * U * (full.abs() + resid.double().abs()), "resid")
    assert ops.device_error() == 0


@pytest.mark.parametrize("n_tok,n,k", [(130, 256, 256), (1100, 1024, 256), (1100, 1024, 2064)])
@pytest.mark.parametrize("out", F)
def test_product_masked_rows(out, n_tok, n, k):
    b = 5
    m = padding(b, n_tok, 4, hole=True)
    m[2] = False  # whole tiles without a valid row
    m[3] = False
    flat = m.reshape(-1)
    a, w = product_inputs(b * n_tok, n, k, 5)
    ac, ae = act8.pack(a)
    ac[~flat] = math.nan
    wc, we = act8.pack_weight(w)
    resid = rnd((b * n_tok, n), 6)
    resid[~flat] = math.nan
    bias = rnd((n,), 7)
    got = ops.gemm8(act(ac, ae), ops.Weight8(wc.to(torch.float8_e4m3fn).to(DEV), e8m0(we).to(DEV)), bias.to(DEV),
                    m.to(DEV), resid.to(DEV) if out == torch.float32 else None, out)
    assert ops.device_error() == 0
    assert torch.all(got.cpu()[~flat] == 0)
    av, wv = act8.value(ac, ae)[flat], act8.value(wc, we, 128)
    want = av @ wv.t() + bias.double() + (resid.double()[flat] if out == torch.float32 else 0)
    close(got.cpu()[flat], want, product_tolerance(av, wv, k, out, want, k / 32 + 2) + 8 * U * (want.abs() + 4))


@pytest.mark.parametrize("m,n,k,scale", [(1, 16, 16, 1.0), (129, 144, 144, 1.0), (300, 2048, 512, 0.05),
                                         (1000, 512, 256, 4.0), (257, 1024, 1024, 1.0),
                                         (2500, 2064, 272, 1.0), (130, 256, 1168, 0.5), (2304, 2304, 1168, 0.2)])
def test_ffn_in(m, n, k, scale):
    """h and gelu(h) in 8 bits.  A value may land on the code next to the
    exact one's (the accumulator's error can carry it over a boundary), so the
    bound is half a code step (2^-4 of the value, or of e4m3's smallest normal
    2^-6 under the block's scale) plus the accumulator's; a scale may be off
    by one power of two only where the maximum sits on the boundary."""
    a, w = rnd((m, k), m), rnd((n, k), n, scale=k ** -0.5 * scale)
    ac, ae = act8.pack(a)
    wc, we = act8.pack_weight(w)
    av, wv = act8.value(ac, ae), act8.value(wc, we, 128)
    bias = rnd((n,), 1, scale=0.1 * scale)
    msk = padding(1, m, 2, hole=True).reshape(-1) if m > 1 else None
    g8, h8 = ops.gemm8_gelu(act(ac, ae), ops.Weight8(wc.to(torch.float8_e4m3fn).to(DEV), e8m0(we).to(DEV)), bias.to(DEV),
                            None if msk is None else msk.to(DEV))
    assert ops.device_error() == 0
    h = av @ wv.t() + bias.double()
    acc = product_tolerance(av, wv, k, torch.float32, h, k / 32 + 1) + 2 * U * (av.abs() @ wv.abs().t())
    for got, want, err in ((h8, h, acc), (g8, act8.gelu(h), 1.2 * acc + 1e-6 * h.abs())):
        if msk is not None:
            want, err = want * msk[:, None], err * msk[:, None]
        _, exps = act8.pack(want)
        gs = got.scales.view(torch.uint8).cpu().long() - 127
        off = gs != exps
        if off.any():
            amax = torch.stack([want[:, 128 * i:128 * i + 128].abs().amax(1) for i in range(exps.shape[1])], 1)
            edge = torch.ldexp(torch.tensor(448.0, dtype=torch.float64), torch.minimum(gs, exps))
            e128 = torch.stack([err[:, 128 * i:128 * i + 128].amax(1) for i in range(exps.shape[1])], 1)
            assert torch.all((gs - exps).abs()[off] == 1) and torch.all((amax - edge).abs()[off] <= e128[off])
        back = act8.value(got.codes.float(), gs)
        scale_of = torch.ldexp(torch.ones(gs.shape, dtype=torch.float64), gs).repeat_interleave(128, 1)[:, :n]
        close(back, want, 1.07 * err + 2.0 ** -4 * torch.maximum(want.abs(), 2.0 ** -6 * scale_of))


@pytest.mark.parametrize("m,n", [(40, 256), (2304, 2304)])
def test_nan_stays_in_its_column(m, n):
    """A NaN in one weight row is that column's alone, in the product and in both GELU outputs (CTA and pair kernels)."""
    a, w = rnd((m, 256), 1), rnd((n, 256), 2, scale=0.1)
    w[33, 7] = math.nan
    w[34, 200] = math.inf
    a8, w8 = ops.checkpoint8(a.to(DEV)), ops.pack_weight8(w.to(DEV))
    clean = w.clone()
    clean[33:35] = 0
    c8 = ops.pack_weight8(clean.to(DEV))
    bad = torch.zeros(n, dtype=torch.bool)
    bad[33:35] = True
    for out in F:
        got = ops.gemm8(a8, w8, out_dtype=out).cpu()
        assert torch.isnan(got[:, bad]).all() and not torch.isnan(got[:, ~bad]).any()
    for got, want in zip(ops.gemm8_gelu(a8, w8), ops.gemm8_gelu(a8, c8)):
        got, want = ops.restore8(got, torch.float32).cpu(), ops.restore8(want, torch.float32).cpu()
        assert torch.isnan(got[:, bad]).all() and not torch.isnan(got[:, ~bad]).any()
        assert torch.equal(got[:, 128:], want[:, 128:])
    assert ops.device_error() == 0


# ---------------------------------------------------------------- weight gradient
@pytest.mark.parametrize("rows,n,k", [(1, 8, 16), (64, 256, 256), (65, 264, 272), (633, 1000, 528), (1500, 256, 512),
                                      (5000, 512, 256), (130, 2048, 1024)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
def test_linear_wgrad(rows, n, k, dt, masked):
    dy = rnd((rows, n), rows + n, dt, 0.1)
    x = rnd((rows, k), rows + k) * torch.exp2((torch.arange(k) // 128 * 3 % 5).float())
    codes, exps = act8.pack(x)
    m = None
    if masked:
        m = padding(1, rows, 9, hole=True).reshape(-1)
        if rows > 400:
            m[100:300] = False  # a whole 64-token stage without a valid token
        dy[~m] = math.nan
        codes[~m] = math.nan
    x8 = act(codes, exps)
    dw, db = ops.linear_wgrad(dy.to(DEV), x8, None if m is None else m.to(DEV))
    assert ops.device_error() == 0
    live = slice(None) if m is None else m
    dv, xv = dy.double()[live], act8.value(codes, exps)[live]
    want = dv.t() @ xv
    # 32 MMAs of 16 products per accumulator (as product_tolerance), then one
    # rounding for each of at most rows / 512 accumulators
    mag = dv.abs().t() @ xv.abs()
    close(dw, want, (2 * 2.0 ** -23 * 33 + (rows / 512 + 2) * U) * mag + 1e-30, "dweight")
    # 32 tokens of a stage in a chain per thread, over the stages of a part
    close(db, dv.sum(0), (rows + 64) * U * dv.abs().sum(0) + 1e-30, "dbias")


def test_wgrad_no_valid_token():
    dy = torch.full((200, 64), math.nan, dtype=torch.bfloat16, device=DEV)
    x8 = ops.checkpoint8(torch.full((200, 128), math.nan, device=DEV))
    dw, db = ops.linear_wgrad(dy, x8, torch.zeros(200, dtype=torch.bool, device=DEV))
    assert torch.all(dw == 0) and torch.all(db == 0)
    dw, db = ops.linear_wgrad(dy[:0], ops.Act8(x8.codes[:0], x8.scales[:0], torch.float32))
    assert torch.all(dw == 0) and torch.all(db == 0)
    assert ops.device_error() == 0
