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


def test_calls_that_wait_for_their_own_forward_leave_the_report_of_an_index(pkg):
    """The blocking forward calls check for a wait of theirs that ran out. A decode before them that met a page out of range is
    none of theirs: they return FA_OK, and the check that follows the decode still has its report."""
    L = pkg.lib()
    stream = torch.cuda.current_stream().cuda_stream
    b = oracle.Batch(3, [40], [1], 1, 2, 64, 16, "fp16")
    args, rows = b.cuda(), b.rows(4).cuda()
    args[2][0, 1] = -1
    g = torch.Generator().manual_seed(4)
    host = [torch.randn((1, 2, 200, 64), generator=g).half().contiguous() for _ in range(3)]
    q, k, v = (x.cuda() for x in host)
    want = pkg.attention_forward(q, k, v)
    out_host, out = torch.zeros_like(host[0]), torch.zeros_like(q)
    nbytes = L.flash_forward_host_workspace_bytes(200, 64, 2)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    one = ctypes.c_void_p * 1
    calls = [
        lambda: L.flash_forward_host(*(x.data_ptr() for x in host), out_host.data_ptr(), 1, 2, 200, 64, 0.0, 0, -1, -1,
                                     ws.data_ptr(), nbytes, 2),
        lambda: L.run_flash_attention_c(1, 2, 200, 64, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), None, None, 0, 0,
                                        0, 0, 0, None, 0.0, None),
        lambda: L.flash_forward_multi_gpu(1, (ctypes.c_int * 1)(torch.cuda.current_device()),
                                          *(one(x.data_ptr()) for x in (q, k, v, out)), (ctypes.c_int * 1)(2), 200, 64, 0.0, 0,
                                          -1, -1, None, 1),
    ]
    for call in calls:
        pkg.check(stream)
        out.zero_()
        pkg.attention_decode(rows, *args)
        torch.cuda.synchronize()
        assert call() == pkg.FA_OK
        assert torch.equal(out_host.cuda() if call is calls[0] else out, want)
        assert L.flash_forward_check(stream) == pkg.FA_BAD_INDEX
        assert L.flash_forward_check(stream) == pkg.FA_OK
