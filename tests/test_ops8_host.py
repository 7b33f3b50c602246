"""Host-side bookkeeping of the training and 8-bit operators, without a GPU."""

import threading

import torch

from techjam_b200 import ops


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
