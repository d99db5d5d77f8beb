"""flash_forward_check where a launch on the device timed out and another read an index that was out of range."""
import ctypes

import pytest
import torch

import paged_cache_oracle as oracle
from test_wait_runs_out import load_waittest

pytestmark = pytest.mark.gpu


def test_both_reports_are_given_one_after_the_other(pkg):
    """In the test build work item 0 of a backward pass never gets its last tile, and a page table names a page that is not
    there: the time-out is reported first, the index by the next check, and then nothing is left."""
    L = load_waittest()
    vp, i = ctypes.c_void_p, ctypes.c_int
    L.flash_backward_test_withhold.argtypes = [vp] * 9 + [i] * 4 + [vp, ctypes.c_size_t, vp]
    L.flash_decode.argtypes = pkg.lib().flash_decode.argtypes
    stream = torch.cuda.current_stream().cuda_stream
    g = torch.Generator().manual_seed(1)
    q, k, v, dout = (torch.randn((1, 2, 300, 64), generator=g).half().cuda() for _ in range(4))
    out, lse = pkg.attention_forward(q, k, v, return_lse=True)
    grads = [torch.zeros_like(q) for _ in range(3)]
    nbytes = pkg.lib().flash_backward_workspace_bytes(1, 2, 300)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    withheld = [x.data_ptr() for x in (q, k, v, out, dout, lse, *grads)] + [1, 2, 300, 64, ws.data_ptr(), nbytes, stream]

    b = oracle.Batch(2, [40], [1], 1, 2, 64, 16, "fp16")
    args, rows = b.cuda(), b.rows(4).cuda()
    args[2][0, 1] = b.k_pages.shape[0]
    cache, q_rows = pkg._cache_struct(torch, *args, None), pkg._rows_struct("q", rows, args[0], 4, 1, 1)
    dec = torch.zeros((1, 4, 1, 64), dtype=torch.half, device="cuda")
    dec_bytes = pkg.lib().flash_decode_workspace_bytes(1, 4, 2, 64)
    dec_ws = torch.empty(dec_bytes, dtype=torch.uint8, device="cuda")
    bad = (cache, q_rows, dec.data_ptr(), None, 1, 1, 4, 0.0, -1, None, dec_ws.data_ptr(), ctypes.c_size_t(dec_bytes), stream)

    pkg.check(stream)
    assert L.flash_forward_check(stream) == pkg.FA_OK
    for calls in ((0, 1), (1, 0)):
        for which in calls:
            assert (L.flash_decode(*bad) if which else L.flash_backward_test_withhold(*withheld)) == pkg.FA_OK
        assert L.flash_forward_check(stream) == pkg.FA_DEVICE_TIMEOUT
        assert b"ran out of time" in L.flash_forward_last_error()
        assert L.flash_forward_check(stream) == pkg.FA_BAD_INDEX
        assert b"out of range" in L.flash_forward_last_error()
        assert L.flash_forward_check(stream) == pkg.FA_OK
