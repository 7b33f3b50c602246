"""Bounded waits of the 8-bit product on the GPU, without a fault: with a limit
of next to nothing a wait gives up after 64 tries (0.27 ms), which a sum over
262144 columns outlasts.  The kernel then records the site, leaves with nothing
in flight, and the same call with the default limit is right."""

import pytest
import torch

from techjam_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
K = 262144
SITES = range(401, 405)


def ones(rows, exponent):
    """Codes of 1.0 under the scale 2^exponent."""
    codes = torch.full((rows, K), 0x38, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    return codes, exponent + 127


def operands(m, n):
    a, ae = ones(m, -9)
    w, we = ones(n, -9)
    scale = lambda rows, byte: torch.full((rows, K // 128), byte, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    return ops.Act8(a, scale(m, ae), torch.float16), ops.Weight8(w, scale((n + 127) // 128, we))


# one tile of a single CTA; three tiles a CTA pair, so that loads, scales and MMAs wait for the epilogue that left
@pytest.mark.parametrize("m,n", [(128, 64), (3840, 3840)])
def test_expired_wait_leaves_in_order(m, n):
    a, w = operands(m, n)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.gemm8(a, w, out_dtype=torch.bfloat16, err=err)
    assert int(err) == 0
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    _lib.call("tj_set_wait_limit", 1)
    try:
        start.record()
        ops.gemm8(a, w, out_dtype=torch.bfloat16, err=err)
        end.record()
        torch.cuda.synchronize()
    finally:
        _lib.call("tj_set_wait_limit", 0)
    assert int(err) in SITES
    assert start.elapsed_time(end) < 1000
    err.zero_()
    # 262144 * 2^-18, exact in the accumulator
    assert torch.all(ops.gemm8(a, w, out_dtype=torch.bfloat16, err=err) == 1)
    assert int(err) == 0


def test_earlier_error_ends_no_later_call():
    """A word that holds an earlier call's site, the device's own or a caller's:
    the products and the weight gradient run to their end all the same, and the
    word keeps its site until it is read."""
    g = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    for m, n, k in ((300, 1024, 512), (3000, 2048, 640)):
        a, w, bias, resid = ops.checkpoint8(rnd(m, k)), ops.pack_weight8(rnd(n, k)), rnd(n), rnd(m, n)
        dy, x = rnd(m, n).bfloat16(), ops.checkpoint8(rnd(m, k))
        word = torch.zeros(1, dtype=torch.int32, device=DEV)

        def calls(err):
            out = [ops.gemm8(a, w, bias, out_dtype=t, err=err) for t in (torch.float16, torch.bfloat16)]
            out.append(ops.gemm8(a, w, bias, resid=resid, out_dtype=torch.float32, err=err))
            for t in ops.gemm8_gelu(a, w, bias, err=err):
                out += [t.codes.view(torch.uint8), t.scales.view(torch.uint8)]
            return out + list(ops.linear_wgrad(dy, x, err=err))

        want = calls(word)
        assert int(word) == 0
        word.fill_(403)
        for got, exp in zip(calls(word), want):
            assert torch.equal(got, exp)
        assert int(word) == 403
        own = ops._err_word(torch.cuda.current_device())
        own.fill_(502)
        for got, exp in zip(calls(None), want):
            assert torch.equal(got, exp)
        assert ops.device_error() == 502 and ops.device_error() == 0
