"""The training and 8-bit operators as a program uses them: one FFN sublayer
forward and backward, on other streams, captured into graphs, twice over, at
sizes past 32-bit offsets, and what the wrappers refuse."""

import math

import pytest
import torch

from oracle import act8
from techjam_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rnd(shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def ffn_inputs(b, n, d, f, seed=0):
    t = {"x": rnd((b * n, d), seed), "gamma": 1 + rnd((d,), seed + 1, 0.2), "beta": rnd((d,), seed + 2, 0.2),
         "w1": rnd((f, d), seed + 3, d ** -0.5), "b1": rnd((f,), seed + 4, 0.1),
         "w2": rnd((d, f), seed + 5, f ** -0.5), "b2": rnd((d,), seed + 6, 0.1),
         "dout": rnd((b * n, d), seed + 7, 0.1)}
    lengths = torch.randint(n // 2, n + 1, (b,), generator=torch.Generator().manual_seed(seed))
    lengths[-1] = 0
    t["mask"] = (torch.arange(n)[None, :] < lengths[:, None]).to(DEV)
    return t


def pack_weights(t):
    return {"w1": ops.pack_weight8(t["w1"]), "w2": ops.pack_weight8(t["w2"]),
            "w1t": ops.pack_weight8(t["w1"], transpose=True), "w2t": ops.pack_weight8(t["w2"], transpose=True)}


def ffn_step(t, w):
    """out = x + FFN(LayerNorm(x)) and every gradient for dout, activations kept in 8 bits."""
    m = t["mask"]
    ln = ops.layernorm_train(t["x"], t["gamma"], t["beta"], m, out_dtype=torch.float8_e4m3fn, checkpoint=True)
    g8, h8 = ops.gemm8_gelu(ln.y, w["w1"], t["b1"], m)
    out = ops.gemm8(g8, w["w2"], t["b2"], m, resid=t["x"], out_dtype=torch.float32)
    dout8 = ops.checkpoint8(t["dout"], m)
    dw2, db2 = ops.linear_wgrad(t["dout"].bfloat16(), g8, m)
    dg = ops.gemm8(dout8, w["w2t"], mask=m, out_dtype=torch.bfloat16)
    dh, dh8 = ops.gelu_backward(dg, h8, m, pack=True)
    dw1, db1 = ops.linear_wgrad(dh, ln.y, m)
    dy = ops.gemm8(dh8, w["w1t"], mask=m, out_dtype=torch.bfloat16)
    dx, dgamma, dbeta = ops.layernorm_backward(dy, ln.x8, t["gamma"], ln.mean, ln.rstd, m, t["dout"])
    return {"out": out, "dx": dx, "gamma": dgamma, "beta": dbeta, "w1": dw1, "b1": db1, "w2": dw2, "b2": db2}


@pytest.mark.parametrize("b,n,d,f", [(4, 100, 256, 1024), (3, 333, 512, 2048), (16, 512, 256, 1024)])
def test_ffn_sublayer_against_unpacked_gradients(b, n, d, f):
    """Against autograd of the same sublayer in 64 bits without any packing.  A
    packed factor is off by at most 2^-4 of each value, and sums of such
    products, whose errors are independent, by at most 2^-4 of their norm for
    each packed factor on the way: the counts below."""
    t = ffn_inputs(b, n, d, f)
    got = ffn_step(t, pack_weights(t))
    assert ops.device_error() == 0
    m = t["mask"].cpu().reshape(-1, 1)
    p = {k: v.double().cpu().requires_grad_() for k, v in t.items() if k not in ("mask", "dout")}
    x = torch.where(m, p["x"], 0.0)
    y = torch.nn.functional.layer_norm(x, (d,), p["gamma"], p["beta"], 1e-5)
    h = y @ p["w1"].t() + p["b1"]
    g = act8.gelu(h)
    out = torch.where(m, x + g @ p["w2"].t() + p["b2"], 0.0)
    out.backward(torch.where(m, t["dout"].double().cpu(), 0.0))
    want = {"out": out.detach(), "dx": p["x"].grad, "gamma": p["gamma"].grad, "beta": p["beta"].grad,
            "w1": p["w1"].grad, "b1": p["b1"].grad, "w2": p["w2"].grad, "b2": p["b2"].grad}
    # out: y, w1, g, w2 (on a branch smaller than x).  dw2: the three of g; db2:
    # dout in bf16.  dh: dout, w2, h and the three of h; dw1 adds y; dx adds
    # dh, w1 and x.
    packed = {"out": 4, "w2": 3, "b2": 2.0 ** -4, "b1": 6, "w1": 7, "beta": 8, "gamma": 9, "dx": 9}
    for k, v in want.items():
        err = float((got[k].double().cpu() - v).norm() / v.norm())
        assert err <= packed[k] * 2.0 ** -4, (k, err)
    flat = ~t["mask"].reshape(-1)
    assert torch.all(got["out"][flat] == 0) and torch.all(got["dx"][flat] == 0)


def test_ffn_sublayer_stages_fit_each_other():
    """Each stage of the step again from what the stage before it handed over."""
    t = ffn_inputs(4, 100, 256, 1024, seed=50)
    w = pack_weights(t)
    m = t["mask"]
    ln = ops.layernorm_train(t["x"], t["gamma"], t["beta"], m, out_dtype=torch.float8_e4m3fn, checkpoint=True)
    y = ops.restore8(ln.y, torch.float32)
    g8, h8 = ops.gemm8_gelu(ln.y, w["w1"], t["b1"], m)
    rows = m.reshape(-1)
    wv = act8.value(w["w1"].codes.float(), w["w1"].scales.view(torch.uint8).cpu().long() - 127, 128)
    h = (y.double().cpu() @ wv.t() + t["b1"].double().cpu()) * rows.cpu()[:, None]
    back = ops.restore8(h8, torch.float32).double().cpu()
    scale = torch.ldexp(torch.ones(h8.scales.shape, dtype=torch.float64), h8.scales.view(torch.uint8).cpu().long() - 127)
    step = 2.0 ** -4 * torch.maximum(h.abs(), 2.0 ** -6 * scale.repeat_interleave(128, 1))
    assert torch.all((back - h).abs() <= 1.001 * step + 1e-5)
    # the transposed weight is the transpose of the weight: same codes and scales
    assert torch.equal(w["w1t"].codes.view(torch.uint8), w["w1"].codes.view(torch.uint8).t())
    assert torch.equal(w["w1t"].scales.view(torch.uint8), w["w1"].scales.view(torch.uint8).t())


def test_same_call_same_bits():
    t = ffn_inputs(5, 300, 512, 1024, seed=3)
    w = pack_weights(t)
    a, b = ffn_step(t, w), ffn_step(t, w)
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_other_stream():
    """On a stream of its own, beside work on the default stream, with the
    inputs made on that stream."""
    t = ffn_inputs(4, 200, 256, 512, seed=9)
    w = pack_weights(t)
    want = ffn_step(t, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device=DEV)
    for _ in range(4):
        big = big @ big * 1e-3
    with torch.cuda.stream(side):
        t2 = {k: v.clone() for k, v in t.items()}
        w2 = pack_weights(t2)
        got = ffn_step(t2, w2)
    other = ffn_step(t, w)  # at the same time on the default stream
    side.synchronize()
    torch.cuda.synchronize()
    for k in want:
        assert torch.equal(got[k], want[k]) and torch.equal(other[k], want[k]), k
    assert ops.device_error() == 0


def test_captured_into_graphs():
    """Two graphs of the step, captured one after the other and replayed in
    turn with changed inputs, give the eager results; they share no workspace."""
    sets = [ffn_inputs(4, 150, 256, 512, seed=s) for s in (20, 30)]
    graphs, outs, statics, weights = [], [], [], []
    for t in sets:
        s = {k: v.clone() for k, v in t.items()}
        w = pack_weights(s)
        ffn_step(s, w)  # warm-up: kernel attributes, the error word
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ffn_step(s, w)
        graphs.append(g), outs.append(out), statics.append(s), weights.append(w)
    for turn in range(3):
        for t, s in zip(sets, statics):
            new = ffn_inputs(4, 150, 256, 512, seed=100 + turn)
            for k in ("x", "dout", "mask"):
                t[k] = new[k]
                s[k].copy_(new[k])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for t, w, out in zip(sets, weights, outs):
            want = ffn_step(t, w)
            for k in want:
                assert torch.equal(out[k], want[k]), (turn, k)
    assert ops.device_error() == 0
    del graphs


def test_offsets_past_32_bits():
    """2.15e9 elements: the last rows come out right."""
    rows, cols = 524291, 4100
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    x.fill_(1.0)
    tail = rnd((3, cols), 1, 2.0, torch.bfloat16)
    x[-3:] = tail
    a = ops.checkpoint8(x)
    codes, exps = act8.pack(tail.cpu())
    assert torch.equal(a.scales.view(torch.uint8)[-3:].cpu().long() - 127, exps)
    assert torch.equal(a.codes[-3:].float().cpu().double(), codes)
    dh = ops.gelu_backward(x, a)
    want = tail.double().cpu() * act8.gelu_slope(act8.value(codes, exps))
    assert torch.all((dh[-3:].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5)
    assert float(dh[0, 0]) == float(dh[-4, -1])
    del dh
    f = ops.layernorm_train(x[:, :4096].contiguous(), torch.ones(4096, device=DEV), torch.zeros(4096, device=DEV))
    y, _, _ = act8.layernorm(tail.cpu()[:, :4096], torch.ones(4096), torch.zeros(4096), 1e-5)
    assert torch.all((f.y[-3:].double().cpu() - y).abs() <= 2.0 ** -11 * y.abs() + 1e-4)


def test_c_entries_in_place():
    """resid may alias out (product) and resid_grad may alias dx (layer norm)."""
    a, w = ops.checkpoint8(rnd((300, 128), 1)), ops.pack_weight8(rnd((256, 128), 2, 0.1))
    resid = rnd((300, 256), 3)
    want = ops.gemm8(a, w, resid=resid, out_dtype=torch.float32)
    buf, err = resid.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    st = torch.cuda.current_stream().cuda_stream
    _lib.call("tj_gemm8", a.codes.data_ptr(), a.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), None, 300, 256,
              128, None, buf.data_ptr(), buf.data_ptr(), _lib.F32, err.data_ptr(), st)
    assert torch.equal(buf, want) and int(err) == 0
    x, dy, g = rnd((2000, 512), 4), rnd((2000, 512), 5), rnd((512,), 6)
    f = ops.layernorm_train(x, g, g)
    r = rnd((2000, 512), 7)
    want = ops.layernorm_backward(dy, x, g, f.mean, f.rstd, resid_grad=r)
    buf, dg, db = r.clone(), torch.empty(512, device=DEV), torch.empty(512, device=DEV)
    ws, wp, wn = ops._workspace("tj_layernorm_backward_workspace_bytes", x.device, 2000, 512)
    _lib.call("tj_layernorm_backward", dy.data_ptr(), _lib.F32, x.data_ptr(), None, g.data_ptr(), f.mean.data_ptr(),
              f.rstd.data_ptr(), 2000, 512, None, buf.data_ptr(), buf.data_ptr(), _lib.F32, dg.data_ptr(), db.data_ptr(),
              wp, wn, st)
    for got, exp in zip((buf, dg, db), want):
        assert torch.equal(got, exp)
    del ws


def test_wrappers_refuse():
    x, w = rnd((8, 64), 1), rnd((64,), 2)
    a = ops.checkpoint8(x)
    w8 = ops.pack_weight8(rnd((32, 64), 3))
    f = ops.layernorm_train(x, w, w)
    mask = torch.ones(8, dtype=torch.bool, device=DEV)
    bad = [
        lambda: ops.checkpoint8(x.t()), lambda: ops.checkpoint8(x.double()), lambda: ops.checkpoint8(x[0]),
        lambda: ops.checkpoint8(x, mask[:7]), lambda: ops.checkpoint8(x, mask.int()), lambda: ops.checkpoint8(x[:, :0]),
        lambda: ops.restore8(a, torch.float64), lambda: ops.restore8(ops.Act8(a.codes, a.scales[:4], x.dtype)),
        lambda: ops.restore8(x), lambda: ops.pack_weight8(x[:0]),
        lambda: ops.layernorm_train(x, w[:32], w), lambda: ops.layernorm_train(x, w.half(), w),
        lambda: ops.layernorm_train(x, w, w, out_dtype=torch.float64),
        lambda: ops.layernorm_backward(x, x[:4], w, f.mean, f.rstd),
        lambda: ops.layernorm_backward(x, x, w, f.mean[:4], f.rstd),
        lambda: ops.layernorm_backward(x, x, w, f.mean, f.rstd, resid_grad=x.half()),
        lambda: ops.layernorm_backward(x, ops.Act8(a.codes, a.scales, torch.int8), w, f.mean, f.rstd),
        lambda: ops.gelu_backward(x, x.half()), lambda: ops.gelu_backward(x[:4], a),
        lambda: ops.gemm8(a, ops.pack_weight8(rnd((32, 48), 3))), lambda: ops.gemm8(a, ops.pack_weight8(rnd((12, 64), 3))),
        lambda: ops.gemm8(a, w8, resid=rnd((8, 32), 1)), lambda: ops.gemm8(a, w8, w), lambda: ops.gemm8(a, a),
        lambda: ops.gemm8(a, w8, out_dtype=torch.int32), lambda: ops.gemm8(x, w8),
        lambda: ops.gemm8(a, ops.Weight8(w8.codes, w8.scales.repeat(2, 1))),
        lambda: ops.gemm8_gelu(a, ops.pack_weight8(rnd((24, 64), 3))),
        lambda: ops.linear_wgrad(x, a), lambda: ops.linear_wgrad(x.half()[:4], a),
        lambda: ops.linear_wgrad(rnd((8, 12), 1).half(), a),
        lambda: ops.linear_wgrad(x.half(), ops.checkpoint8(rnd((8, 24), 1))),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(_lib.TjError):
        ops.layernorm_train(rnd((2, 4100), 1), rnd((4100,), 1), rnd((4100,), 1))
    assert ops.device_error() == 0
