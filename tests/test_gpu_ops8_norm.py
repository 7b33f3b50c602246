"""Layer norm's gradients against differences of the forward kernel itself."""

import pytest
import torch

from oracle import act8
from techjam_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.mark.parametrize("rows,d", [(3, 40), (5, 1001), (2, 2052)])
def test_layernorm_gradient_against_its_own_forward(rows, d):
    """dx, dweight and dbias of sum(y * dy) against central differences of the
    kernel's fp32 output, step 2^-6.  Elements that a step does not touch come
    out the same bit for bit and cancel; of the others each y is off by at
    most 48 roundings in its sums and 16 more, relative to the magnitudes it
    is made of.  What the step itself leaves out (its square times the third
    derivative) is the difference of the 64-bit quotient and the 64-bit
    gradient."""
    g = torch.Generator().manual_seed(rows)
    x, dy = torch.randn(rows, d, generator=g), torch.randn(rows, d, generator=g)
    w, b = 1 + 0.3 * torch.randn(d, generator=g), torch.randn(d, generator=g)
    step = 2.0 ** -6
    f = ops.layernorm_train(x.to(DEV), w.to(DEV), b.to(DEV), out_dtype=torch.float32)
    grads = ops.layernorm_backward(dy.to(DEV), x.to(DEV), w.to(DEV), f.mean, f.rstd)
    y64, mean, rstd = act8.layernorm(x, w, b, 1e-5)
    exact = act8.layernorm_backward(dy, x, w, mean, rstd)[:3]
    xhat = ((x.double() - mean[:, None]) * rstd[:, None]).abs()
    off = 64 * U * ((xhat + (x.double().abs().mean(1) * rstd)[:, None]) * w.double().abs() + b.double().abs())
    weight = dy.double().abs() * off * 1.1  # of a stepped x, w or b in place of these

    def own(args):
        return (ops.layernorm_train(*(t.to(DEV) for t in args), out_dtype=torch.float32).y.double().cpu() * dy.double()).sum()

    def in_64(args):
        return (act8.layernorm(*args, 1e-5)[0] * dy.double()).sum()

    for which, t in enumerate((x, w, b)):
        for idx in range(0, t.numel(), max(1, t.numel() // 25)):
            sides = []
            for s in (step, -step):
                v = [x, w, b]
                v[which] = t.clone()
                v[which].view(-1)[idx] += s
                sides.append(v)
            wide = float(sides[0][which].view(-1)[idx].double() - sides[1][which].view(-1)[idx].double())
            quotient = float(own(sides[0]) - own(sides[1])) / wide
            in64 = float(in_64(sides[0]) - in_64(sides[1])) / wide
            touched = weight[idx // d] if which == 0 else weight[:, idx]
            want = float(exact[which].reshape(-1)[idx])
            tol = 2 * float(touched.sum()) / wide + abs(in64 - want) + 1e-5 * (1 + abs(want))
            assert abs(float(grads[which].reshape(-1)[idx]) - quotient) <= tol, (which, idx, quotient, want, tol)
            if d == 40 or which > 0:  # a narrow row, or a column: the bound tells a wrong gradient
                assert tol <= 0.1 * max(1.0, abs(want))
