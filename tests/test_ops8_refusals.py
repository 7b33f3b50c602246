"""What the training and 8-bit operators refuse, checked without a GPU: the C
entries answer before they touch a device, the Python wrappers before they
call them."""

import ctypes

import pytest
import torch

from techjam_b200 import _lib, build, ops

INVALID, UNSUPPORTED = 1, 2
P = 1 << 20  # a non-null, 16-byte aligned pointer that no refused call reads


@pytest.fixture(scope="module", autouse=True)
def built():
    build.build()


def status(name, *args):
    got = getattr(_lib.load(), name)(*args)
    if got != 0:
        assert _lib.load().tj_last_error(), name
    return got


@pytest.mark.parametrize("name,args,want", [
    # codes of an unknown type, no columns, negative rows, missing pointers
    ("tj_act8_pack", (P, 7, 4, 4, None, P, P, None), INVALID),
    ("tj_act8_pack", (P, _lib.E4M3, 4, 4, None, P, P, None), INVALID),
    ("tj_act8_pack", (P, 0, 4, 0, None, P, P, None), INVALID),
    ("tj_act8_pack", (P, 0, -1, 4, None, P, P, None), INVALID),
    ("tj_act8_pack", (P, 0, 4, 4, None, None, P, None), INVALID),
    ("tj_act8_pack", (P, 0, 1 << 40, 4096, None, P, P, None), UNSUPPORTED),
    ("tj_act8_unpack", (P, P, 4, 4, P, _lib.E4M3, None), INVALID),
    ("tj_act8_unpack", (None, P, 4, 4, P, 0, None), INVALID),
    ("tj_weight8_pack", (P, 0, 0, 4, 0, P, P, None), INVALID),
    ("tj_weight8_pack", (P, 9, 4, 4, 0, P, P, None), INVALID),
    ("tj_weight8_pack", (P, 0, 4, 4, 0, P, None, None), INVALID),
    ("tj_layernorm_train", (P, 0, P, P, 4, 4097, 1e-5, None, P, 1, None, P, P, None, None, None), UNSUPPORTED),
    ("tj_layernorm_train", (P, 0, P, P, 4, 0, 1e-5, None, P, 1, None, P, P, None, None, None), INVALID),
    ("tj_layernorm_train", (P, _lib.E4M3, P, P, 4, 64, 1e-5, None, P, 1, None, P, P, None, None, None), INVALID),
    ("tj_layernorm_train", (P, 0, P, None, 4, 64, 1e-5, None, P, 1, None, P, P, None, None, None), INVALID),
    # an 8-bit output without scales, scales without an 8-bit output, half of a copy
    ("tj_layernorm_train", (P, 0, P, P, 4, 64, 1e-5, None, P, _lib.E4M3, None, P, P, None, None, None), INVALID),
    ("tj_layernorm_train", (P, 0, P, P, 4, 64, 1e-5, None, P, 1, P, P, P, None, None, None), INVALID),
    ("tj_layernorm_train", (P, 0, P, P, 4, 64, 1e-5, None, P, 1, None, P, P, P, None, None), INVALID),
    ("tj_layernorm_backward", (P, 3, P, None, P, P, P, 4, 64, None, None, P, 0, P, P, P, 0, None), INVALID),
    ("tj_layernorm_backward", (P, 0, P, None, P, P, P, 4, 5000, None, None, P, 0, P, P, P, 0, None), UNSUPPORTED),
    ("tj_layernorm_backward", (P, 0, None, None, P, P, P, 4, 64, None, None, P, 0, P, P, P, 0, None), INVALID),
    ("tj_layernorm_backward_workspace_bytes", (4, 64, None), INVALID),
    ("tj_gelu_backward", (P, 3, P, None, 4, 64, None, P, None, None, None), INVALID),
    ("tj_gelu_backward", (P, 0, P, None, 4, 64, None, P, P, None, None), INVALID),
    ("tj_gelu_backward", (P, 0, P, None, 4, 64, None, None, None, None, None), INVALID),
    # widths off the vector and TMA steps, a residual without a 32-bit result, an unaligned bias
    ("tj_gemm8", (P, P, P, P, None, 4, 8, 24, None, None, P, 0, P, None), UNSUPPORTED),
    ("tj_gemm8", (P, P, P, P, None, 4, 12, 32, None, None, P, 0, P, None), UNSUPPORTED),
    ("tj_gemm8", (P, P, P, P, None, 4, 8, 32, None, P, P, 1, P, None), UNSUPPORTED),
    ("tj_gemm8", (P, P, P, P, P + 4, 4, 8, 32, None, None, P, 1, P, None), INVALID),
    ("tj_gemm8", (P, P, P, P, None, -1, 8, 32, None, None, P, 1, P, None), INVALID),
    ("tj_gemm8", (P, P, P, P, None, 4, 8, 32, None, None, P, 1, None, None), INVALID),
    ("tj_gemm8", (P, P, P, P, None, 4, 8, 32, None, None, P, 3, P, None), INVALID),
    ("tj_gemm8_gelu", (P, P, P, P, None, 4, 8, 32, None, P, P, P, P, P, None), UNSUPPORTED),
    ("tj_gemm8_gelu", (P, P, P, P, None, 4, 16, 32, None, P, None, P, P, P, None), INVALID),
    ("tj_wgrad8", (P, 0, P, P, 4, 8, 16, None, P, P, P, 1, P, None), UNSUPPORTED),
    ("tj_wgrad8_workspace_bytes", (4, 8, 16, None), INVALID),
])
def test_c_entries_refuse(name, args, want):
    assert status(name, *args) == want


@pytest.mark.parametrize("name,args", [
    ("tj_act8_pack", (None, 0, 0, 4, None, None, None, None)),
    ("tj_act8_unpack", (None, None, 0, 4, None, 0, None)),
    ("tj_layernorm_train", (None, 0, None, None, 0, 64, 1e-5, None, None, 1, None, None, None, None, None, None)),
    ("tj_gelu_backward", (None, 0, None, None, 0, 64, None, None, None, None, None)),
    ("tj_gemm8", (None, None, P, P, None, 0, 8, 32, None, None, None, 1, P, None)),
    ("tj_gemm8_gelu", (None, None, P, P, None, 0, 16, 32, None, None, None, None, None, P, None)),
])
def test_no_rows_is_no_work(name, args):
    assert status(name, *args) == 0


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(4, 64)
    w = torch.zeros(64)
    a = ops.Act8(torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu),
                 torch.float32)
    w8 = ops.Weight8(torch.zeros(64, 64).to(torch.float8_e4m3fn),
                     torch.zeros(1, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu))
    for call in (lambda: ops.checkpoint8(x), lambda: ops.restore8(a), lambda: ops.pack_weight8(x),
                 lambda: ops.layernorm_train(x, w, w), lambda: ops.layernorm_backward(x, x, w, w[:4], w[:4]),
                 lambda: ops.gelu_backward(x, x), lambda: ops.gemm8(a, w8), lambda: ops.gemm8_gelu(a, w8),
                 lambda: ops.linear_wgrad(x.half(), a)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
