"""The first call on a device inside a capture: refused, since it would allocate, and the process goes on to work."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

SCRIPT = """
import sys
sys.path.insert(0, %r)
import torch
import __graft_entry__ as entry
pkg = entry.load_package()
x = torch.randn((1, 2, 64, 64), device="cuda").half()
pages = torch.zeros((4, 2, 16, 64), device="cuda").half()
table, lengths = torch.arange(4, device="cuda").int()[None], torch.full((1,), 30, device="cuda").int()
lse = torch.zeros((1, 2, 64), device="cuda")
calls = [lambda: pkg.attention_backward(x, x, x, x, lse, x),
         lambda: pkg.cache_append(x[:, :, :1], x[:, :, :1], pages, pages, table, lengths),
         lambda: pkg.attention_decode(x[:, :, :1], pages, pages, table, lengths)]
side = torch.cuda.Stream()
for call in calls:
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            call()
    except pkg.FlashForwardError as e:
        assert e.code == pkg.FA_UNSUPPORTED and "capture" in str(e), e
    else:
        raise SystemExit("the capture was not refused")
for call in calls:
    call()
for call in calls:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    graph.replay()
pkg.check(torch.cuda.current_stream().cuda_stream)
print("fine")
"""


def test_first_call_in_a_capture_is_refused():
    r = subprocess.run([sys.executable, "-c", SCRIPT % ROOT], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": ROOT})
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
