"""GPU: a process whose first call of the library is captured.  The graph's kernels
report into the device's status word at every replay, as eager ones do."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]

PROGRAM = r"""
import importlib

import torch

K = importlib.import_module("10_20_b200.kernels")
L = importlib.import_module("10_20_b200.latent_attention")
lib = importlib.import_module("10_20_b200._lib")
dev = torch.device("cuda", 0)
g = torch.Generator(device=dev).manual_seed(1)
q = torch.randn((2, 8, 576), generator=g, device=dev).to(torch.bfloat16)
pool = torch.randn((300, 1, 576), generator=g, device=dev).to(torch.bfloat16)
ids = torch.arange(200, device=dev, dtype=torch.int32).repeat(2, 1)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, lse = L.attend_slots(q, pool, None, ids, 0.05)
    # a bounded wait that nothing ends, into the same word
    lib.call("v1x_selftest_wait_timeout", 1000000, K.status_ptr(dev), None, lib.stream_of(q), device=dev)
for _ in range(2):
    graph.replay()
    try:
        K.check_status(dev)
    except RuntimeError as e:
        assert f"status {lib.V1X_STATUS_TIMEOUT}" in str(e), e
    else:
        raise AssertionError("the wait was not reported")
    K.check_status(dev)                    # reset
want = L.attend_slots(q, pool, None, ids, 0.05)
assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
K.check_status(dev)
assert K.status_word(dev).data_ptr() == K.status_ptr(dev)
print("reported")
"""


def test_a_captured_first_call_reports(cuda_dev):
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "reported" in r.stdout, r.stdout + r.stderr
