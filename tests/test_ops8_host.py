"""Host-side bookkeeping of the training and 8-bit operators, without a GPU."""

import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from techjam_b200 import _lib, build, ops

INVALID, UNSUPPORTED = 1, 2
ROOT = Path(__file__).resolve().parent.parent

class Word:
    """A device's error word: counts as zeroed only once the device was waited for."""

    def __init__(self):
        self.value, self.order = 0, []

    def item(self):
        self.order.append("item")
        return self.value

    def zero_(self):
        self.order.append("zero")
        self.value = 0


def test_device_error_is_told_to_every_thread(monkeypatch):
    word = Word()
    monkeypatch.setattr(ops, "_err_word", lambda index: word)
    monkeypatch.setattr(ops, "_err_log", {})
    monkeypatch.setattr(ops, "_err_seen", threading.local())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: word.order.append("sync"))

    def elsewhere():
        got = []
        t = threading.Thread(target=lambda: got.append((ops.device_error("cuda:0"), ops.device_error("cuda:0"))))
        t.start()
        t.join()
        return got[0]

    assert ops.device_error("cuda:0") == 0
    word.value = 402
    word.order.clear()
    assert elsewhere() == (402, 0)
    # cleared, and waited for, before anybody is told
    assert word.order[:4] == ["sync", "item", "zero", "sync"]
    word.value = 503
    assert ops.device_error("cuda:0") == 402  # the other thread's reading took nothing from this one
    assert ops.device_error("cuda:0") == 0
    assert elsewhere() == (402, 0)  # a thread that has never asked: all since the start, the first of them
    assert ops.device_error("cuda:1") == 0


LEAN = """
import pytest
import torch
for owner, name in ((torch, "float8_e4m3fn"), (torch, "float8_e8m0fnu"), (torch._C, "_cuda_getCurrentRawStream"),
                    (torch._C, "_cuda_getDevice")):
    if hasattr(owner, name):
        delattr(owner, name)
from techjam_b200 import _lib, build, ops
assert callable(ops.layernorm) and callable(ops.gemm) and callable(ops.attention)
assert callable(ops._stream_of) and callable(ops._current_device)
a = ops.Act8(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), torch.float32)
w = torch.zeros(64, 64)
for call in (lambda: ops.restore8(a), lambda: ops.pack_weight8(w), lambda: ops._new_act(4, 64, "cpu", torch.float32),
             lambda: ops.gemm8(a, ops.Weight8(w, w))):
    try:
        call()
    except RuntimeError as e:
        assert "float8" in str(e)
    else:
        raise AssertionError("not refused")
print("fine")
"""


def test_a_torch_without_8_bit_types_keeps_the_other_operators():
    """The 8-bit operators say what they lack; the module and the operators of before do without."""
    got = subprocess.run([sys.executable, "-c", LEAN], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip().endswith("fine"), got.stderr


BIG = 0x7fffffff
P = 1 << 20  # a non-null, 16-byte aligned pointer that no refused call reads


@pytest.mark.parametrize("name,args,want", [
    # sizes that cannot be rounded up to a block or a tile in an int, or whose count of blocks passes 64 bits
    ("tj_act8_pack", (P, 0, 1, BIG, None, P, P, None), UNSUPPORTED),
    ("tj_act8_pack", (P, 0, 1 << 62, 4096, None, P, P, None), UNSUPPORTED),
    ("tj_act8_unpack", (P, P, 1, BIG, P, 0, None), UNSUPPORTED),
    ("tj_gelu_backward", (P, 0, P, None, 1, BIG, None, P, None, None, None), UNSUPPORTED),
    ("tj_weight8_pack", (P, 0, BIG, 4, 0, P, P, None), UNSUPPORTED),
    ("tj_weight8_pack", (P, 0, 4, BIG, 0, P, P, None), UNSUPPORTED),
    ("tj_weight8_pack", (P, 0, 65535 * 128 + 1, 4, 0, P, P, None), UNSUPPORTED),
    ("tj_gemm8", (P, P, P, P, None, 4, BIG - 7, 32, None, None, P, 0, P, None), UNSUPPORTED),
    # the workspace holds floats
    ("tj_layernorm_backward", (P, 0, P, None, P, P, P, 4, 64, None, None, P, 0, P, P, P + 2, 1 << 20, None), INVALID),
])
def test_c_entries_refuse_sizes_and_alignment(name, args, want):
    build.build()
    assert getattr(_lib.load(), name)(*args) == want
    assert _lib.load().tj_last_error()
