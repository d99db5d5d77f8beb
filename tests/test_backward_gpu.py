"""flash_backward on the GPU against the gradient's formula in 64 bits, and that formula's chain against differences.

Tolerances (Gradient in backward_oracle.py): P and dS are rounded to fp16 once each, half a step (2^-11) relative to the
element; errors of the fp32 scores move P by a factor within 2^-13 (scores of up to 2^6 with a relative error of 2^-20);
dO.V and delta are fp32 sums whose error 2^-18 of the terms' absolute sum covers; the outputs are rounded to fp16. Each is
multiplied out with the absolute values of the other operand."""
import ctypes
import math

import pytest
import torch

import backward_oracle as oracle
from test_wait_runs_out import load_waittest

pytestmark = pytest.mark.gpu


def tensors(seed, B, H, N, d, spread=1.0, grad=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, dout = (torch.randn((B, H, N, d), generator=g) for _ in range(4))
    return (q * spread).half(), k.half(), v.half(), (dout * grad).half()


def gpu_kwargs(kw):
    return {name: x.cuda() if isinstance(x, torch.Tensor) else x for name, x in kw.items()}


def check(pkg, q, k, v, dout, dlse=None, **kw):
    gq, gk, gv, gd = (x.cuda() for x in (q, k, v, dout))
    gkw = gpu_kwargs(kw)
    out, lse = pkg.attention_forward(gq, gk, gv, return_lse=True, **gkw)
    got = pkg.attention_backward(gq, gk, gv, out, lse, gd, dlse=None if dlse is None else dlse.cuda(), **gkw)
    pkg.check(torch.cuda.current_stream().cuda_stream)
    want = oracle.Gradient(q, k, v, out.cpu(), lse.cpu(), dout, dlse, **kw)
    for name, x in zip(("dq", "dk", "dv"), got):
        err, bound = (x.cpu().double() - getattr(want, name)).abs(), getattr(want, name + "_err")
        assert torch.isfinite(x).all(), name
        assert (err <= bound).all(), (name, float((err / bound).max()))
    return got


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("N", [1, 2, 17, 127, 128, 129, 255, 256, 300, 513, 1000])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(pkg, N, d, causal):
    check(pkg, *tensors(N + d, 2, 3, N, d), causal=causal)


@pytest.mark.parametrize("causal,wl,wr", [(True, 0, -1), (True, 1, -1), (True, 100, -1), (False, 0, 0), (False, 130, 5),
                                          (False, -1, 40), (False, 40, -1), (True, 127, 50), (True, 128, -1),
                                          (False, 2 ** 31 - 1, 2 ** 31 - 1), (False, 639, 639)])
@pytest.mark.parametrize("d", [64, 128])
def test_windows(pkg, causal, wl, wr, d):
    check(pkg, *tensors(wl % 1000 + d, 1, 2, 640, d), causal=causal, window_left=wl, window_right=wr)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal,wl", [(False, -1), (True, -1), (True, 150)])
def test_alibi(pkg, d, causal, wl):
    slopes = torch.tensor([0.5, 0.03, -0.004, 0.0])
    check(pkg, *tensors(7 + d, 2, 4, 391, d), causal=causal, window_left=wl, alibi_slopes=slopes)


@pytest.mark.parametrize("scale", [0.02, 0.5])
def test_scale(pkg, scale):
    check(pkg, *tensors(1, 1, 2, 300, 64), softmax_scale=scale, causal=True)


@pytest.mark.parametrize("grad", [2.0 ** -14, 2.0 ** -8, 64.0])
@pytest.mark.parametrize("spread", [0.25, 3.0])
def test_small_and_large_gradients_and_peaked_rows(pkg, grad, spread):
    """Without its scaling dS of a long, flat row would be lost in fp16 for the smallest of these gradients."""
    check(pkg, *tensors(3, 1, 2, 2000, 64, spread=spread, grad=grad))


def test_gradient_of_the_log_sum_exp(pkg):
    q, k, v, dout = tensors(4, 2, 2, 260, 128)
    dlse = torch.randn((2, 2, 260), generator=torch.Generator().manual_seed(5)) * 8
    check(pkg, q, k, v, dout, dlse=dlse, causal=True)
    check(pkg, q, k, v, torch.zeros_like(dout), dlse=dlse)


def test_zero_gradient(pkg):
    q, k, v, dout = tensors(6, 1, 2, 200, 64)
    for x in check(pkg, q, k, v, torch.zeros_like(dout)):
        assert not x.any()


def test_against_differences(pkg):
    """The kernel's gradients are the slope of the 64-bit forward: along random directions, central differences of
    sum(dO * O) + sum(dlse * lse) against the inner products, within what fp16 operands explain."""
    B, H, N, d = 1, 2, 150, 64
    q, k, v, dout = tensors(8, B, H, N, d)
    g = torch.Generator().manual_seed(9)
    dlse = torch.randn((B, H, N), generator=g)
    kw = dict(causal=True, window_left=60, alibi_slopes=torch.tensor([0.1, 0.02]))
    gq, gk, gv = q.cuda(), k.cuda(), v.cuda()
    out, lse = pkg.attention_forward(gq, gk, gv, return_lse=True, **gpu_kwargs(kw))
    got = [x.cpu().double() for x in pkg.attention_backward(gq, gk, gv, out, lse, dout.cuda(), dlse=dlse.cuda(),
                                                            **gpu_kwargs(kw))]
    bound = oracle.Gradient(q, k, v, out.cpu(), lse.cpu(), dout, dlse, **kw)
    x = [t.double() for t in (q, k, v)]

    def loss(args):
        o, l = oracle.forward(*args, **kw)
        return float((dout.double() * o).sum() + (dlse.double() * l).sum())
    for which, name in enumerate(("dq", "dk", "dv")):
        for _ in range(3):
            u = torch.randn(x[which].shape, generator=g, dtype=torch.float64)
            step = 2.0 ** -12
            ends = []
            for sign in (1, -1):
                moved = list(x)
                moved[which] = x[which] + sign * step * u
                ends.append(loss(moved))
            slope = (ends[0] - ends[1]) / (2 * step)
            # the errors of the elements are independent roundings: 6 sigma of their sum, each at most its bound; the output O
            # that delta is taken from is rounded too, which adds at most as much again
            room = 12 * float(((getattr(bound, name + "_err") * u) ** 2).sum().sqrt())
            assert abs(slope - float((got[which] * u).sum())) <= room + 1e-4 * abs(slope), name


def test_same_bits_every_time_and_strided_dout(pkg):
    q, k, v, dout = (x.cuda() for x in tensors(10, 2, 3, 700, 128))
    out, lse = pkg.attention_forward(q, k, v, causal=True, return_lse=True)
    first = pkg.attention_backward(q, k, v, out, lse, dout, causal=True)
    strided = dout.transpose(1, 2).contiguous().transpose(1, 2)
    given = [torch.full_like(q, math.nan) for _ in range(3)]
    second = pkg.attention_backward(q, k, v, out, lse, strided, causal=True, dq=given[0], dk=given[1], dv=given[2])
    for x, y, z in zip(first, second, given):
        assert y is z and torch.equal(x, y)


def test_many_heads_and_a_long_row(pkg):
    """More work items than CTAs that run at once, in several groups of heads: sampled heads against the formula."""
    B, H, N, d = 3, 40, 1100, 64
    q, k, v, dout = (x.cuda() for x in tensors(11, B, H, N, d))
    out, lse = pkg.attention_forward(q, k, v, causal=True, return_lse=True)
    got = pkg.attention_backward(q, k, v, out, lse, dout, causal=True)
    one = [pkg.attention_backward(*(x[b:b + 1, h:h + 1].contiguous() for x in (q, k, v, out, lse, dout)), causal=True)
           for b, h in ((0, 0), (1, 17), (2, 39))]
    for (b, h), single in zip(((0, 0), (1, 17), (2, 39)), one):
        for x, y in zip(got, single):
            assert torch.equal(x[b, h], y[0, 0])
    check(pkg, *tensors(12, 1, 1, 4500, 128), causal=True)


@pytest.mark.parametrize("d", [64, 128])
def test_many_items_again_and_again(pkg, d):
    """Calls that fill the GPU several times over give the same bits, call after call: no hand-over between the warps of a CTA
    may depend on how far one of them has got ahead."""
    q, k, v, dout = (x.cuda() for x in tensors(14, 2, 48, 1000, d))
    out, lse = pkg.attention_forward(q, k, v, causal=True, return_lse=True)
    first = pkg.attention_backward(q, k, v, out, lse, dout, causal=True)
    for _ in range(20):
        again = pkg.attention_backward(q, k, v, out, lse, dout, causal=True)
        assert all(torch.equal(x, y) for x, y in zip(first, again))
    pkg.check(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("kw", [dict(causal=True), dict(window_left=30, window_right=50), dict(causal=True, alibi=True)])
@pytest.mark.parametrize("N,d", [(1, 64), (128, 64), (200, 64), (256, 64), (257, 64), (3, 128), (100, 128), (128, 128), (129, 128)])
def test_short_heads_alone_and_among_many(pkg, N, d, kw):
    """A few short heads find their delta and norms in the kernel that uses them, many have a kernel for it: the same bits, and
    for the few the formula's gradient, with one of the log-sum-exp."""
    H = 5
    kw = dict(kw)
    if kw.pop("alibi", False):
        kw["alibi_slopes"] = torch.tensor([0.5, 0.1, 1.0, 0.02, 0.0])
    q, k, v, dout = tensors(40 + N + d, 31, H, N, d)
    dout[::2] *= 2.0 ** -10
    dlse = torch.randn((31, H, N), generator=torch.Generator().manual_seed(41))
    check(pkg, *(x[:2] for x in (q, k, v, dout)), dlse=dlse[:2], **kw)
    gq, gk, gv, gd, gl = (x.cuda() for x in (q, k, v, dout, dlse))
    gkw = gpu_kwargs(kw)
    out, lse = pkg.attention_forward(gq, gk, gv, return_lse=True, **gkw)
    many = pkg.attention_backward(gq, gk, gv, out, lse, gd, dlse=gl, **gkw)
    few = pkg.attention_backward(*(x[:2] for x in (gq, gk, gv, out, lse, gd)), dlse=gl[:2], **gkw)
    for x, y in zip(many, few):
        assert torch.equal(x[:2], y)


def test_two_streams_and_capture(pkg):
    q, k, v, dout = (x.cuda() for x in tensors(13, 1, 4, 600, 64))
    out, lse = pkg.attention_forward(q, k, v, return_lse=True)
    want = pkg.attention_backward(q, k, v, out, lse, dout)
    torch.cuda.synchronize()
    results = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(pkg.attention_backward(q, k, v, out, lse, dout))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = pkg.attention_backward(q, k, v, out, lse, dout)
    for _ in range(2):
        for x in captured:
            x.zero_()
        graph.replay()
        results.append([x.clone() for x in captured])
    pkg.check(torch.cuda.current_stream().cuda_stream)
    for r in results:
        assert all(torch.equal(x, y) for x, y in zip(r, want))


def test_training_step_of_one_layer(pkg):
    """Forward and backward as a training step makes them: the gradient of a projection's weights through the attention,
    against autograd of the same layer in 64 bits."""
    B, H, N, d, width = 2, 2, 200, 64, 96
    g = torch.Generator().manual_seed(20)
    x = (torch.randn((B, N, width), generator=g)).half()
    w = (torch.randn((3, width, H * d), generator=g) * width ** -0.5).half()
    dout = torch.randn((B, H, N, d), generator=g).half()

    def heads(t):
        return t.view(B, N, H, d).transpose(1, 2).contiguous()
    gx, gw = x.cuda(), w.cuda()
    q, k, v = (heads(gx @ gw[i]) for i in range(3))
    out, lse = pkg.attention_forward(q, k, v, causal=True, return_lse=True)
    grads = pkg.attention_backward(q, k, v, out, lse, dout.cuda(), causal=True)
    dw = [gx.flatten(0, 1).float().T @ t.transpose(1, 2).reshape(B * N, H * d).float() for t in grads]
    wd = w.double().requires_grad_()
    qkv = [(x.double() @ wd[i]).view(B, N, H, d).transpose(1, 2) for i in range(3)]
    o, _ = oracle.forward(*qkv, causal=True)
    (o * dout.double()).sum().backward()
    for i in range(3):
        # roundings of q, k, v, P, dS, O and the gradients, 2^-11 each and independent: relative to the whole 10 of them
        err = float((dw[i].cpu().double() - wd.grad[i]).norm() / wd.grad[i].norm())
        assert err <= 10 * 2.0 ** -11, (i, err)


def test_wait_gives_up_and_the_device_stays_usable(pkg):
    """Test build: work item 0 never gets its last tile. The launch returns, the check reports it, the next call is right."""
    L = load_waittest()
    vp, i = ctypes.c_void_p, ctypes.c_int
    L.flash_backward_test_withhold.argtypes = [vp] * 9 + [i] * 4 + [vp, ctypes.c_size_t, vp]
    L.flash_backward.argtypes = pkg.lib().flash_backward.argtypes
    for d, N in ((64, 900), (128, 600)):
        q, k, v, dout = (x.cuda() for x in tensors(30, 1, 2, N, d))
        out, lse = pkg.attention_forward(q, k, v, return_lse=True)
        want = pkg.attention_backward(q, k, v, out, lse, dout)
        stream = torch.cuda.current_stream().cuda_stream
        pkg.check(stream)
        grads = [torch.zeros_like(q) for _ in range(3)]
        nbytes = pkg.lib().flash_backward_workspace_bytes(1, 2, N)
        ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        ptrs = [x.data_ptr() for x in (q, k, v, out, dout, lse)]
        gptrs = [x.data_ptr() for x in grads]
        assert L.flash_backward_test_withhold(*ptrs, *gptrs, 1, 2, N, d, ws.data_ptr(), nbytes, stream) == pkg.FA_OK
        assert L.flash_forward_check(stream) == pkg.FA_DEVICE_TIMEOUT
        assert L.flash_forward_check(stream) == pkg.FA_OK
        assert L.flash_backward(*ptrs, None, *gptrs, 1, 2, N, d, 0.0, 0, -1, -1, None, ws.data_ptr(), nbytes,
                                stream) == pkg.FA_OK
        assert L.flash_forward_check(stream) == pkg.FA_OK
        for x, y in zip(grads, want):
            assert torch.equal(x, y)


def test_wait_gives_up_in_a_short_head(pkg):
    """The same where delta and the norms are found by the kernel itself."""
    L = load_waittest()
    vp, i = ctypes.c_void_p, ctypes.c_int
    L.flash_backward_test_withhold.argtypes = [vp] * 9 + [i] * 4 + [vp, ctypes.c_size_t, vp]
    for d, N in ((64, 200), (128, 70)):
        q, k, v, dout = (x.cuda() for x in tensors(31, 1, 2, N, d))
        out, lse = pkg.attention_forward(q, k, v, return_lse=True)
        want = pkg.attention_backward(q, k, v, out, lse, dout)
        stream = torch.cuda.current_stream().cuda_stream
        pkg.check(stream)
        grads = [torch.zeros_like(q) for _ in range(3)]
        nbytes = pkg.lib().flash_backward_workspace_bytes(1, 2, N)
        ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        ptrs = [x.data_ptr() for x in (q, k, v, out, dout, lse, *grads)]
        assert L.flash_backward_test_withhold(*ptrs, 1, 2, N, d, ws.data_ptr(), nbytes, stream) == pkg.FA_OK
        assert L.flash_forward_check(stream) == pkg.FA_DEVICE_TIMEOUT
        again = pkg.attention_backward(q, k, v, out, lse, dout)
        pkg.check(stream)
        assert all(torch.equal(x, y) for x, y in zip(again, want))
