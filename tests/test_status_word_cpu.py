"""CPU: the status word that kernels report into can be asked for first inside a graph
capture (a fake of the library's call stands in for the device)."""
import importlib

import torch

K = importlib.import_module("10_20_b200.kernels")
_lib = importlib.import_module("10_20_b200._lib")


def test_status_address_first_asked_for_inside_a_capture(monkeypatch):
    asked = []

    def call(name, *args, device=None):
        asked.append((name, device))
        args[0]._obj.value = 0x7000

    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for name in ("_status", "_status_address"):
        monkeypatch.setattr(K, name, {}, raising=False)
    dev = torch.device("cuda", 0)
    assert K.status_ptr(dev) == 0x7000
    assert K.status_ptr(dev) == 0x7000
    assert asked == [("v1x_status_word", dev)]      # asked for once


def test_status_word_refuses_no_place():
    assert _lib.lib().v1x_status_word(None) == _lib.V1X_ERR_INVALID
    assert b"status_word" in _lib.lib().v1x_last_error()
