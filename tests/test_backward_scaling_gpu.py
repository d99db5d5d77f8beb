"""flash_backward where one row of a head is infinite, or far larger than the others: the rows that it does not touch.

Tolerances: element by element those of test_backward_gpu.py; and for the whole, where errors that one large row would cause
are random and hide below a sum of absolute values, the 2-norm: every dS_ij is off by at most half a step of fp16 (2^-11) and
what the scores do to P (2^-13), every output by half a step, all of them independent of one another, so the squares add up;
2^-13 of the norm for what a row's elements share."""
import math

import pytest
import torch

import backward_oracle as oracle
from test_backward_gpu import gpu_kwargs, tensors

pytestmark = pytest.mark.gpu


def run(pkg, q, k, v, dout, dlse=None, **kw):
    gkw = gpu_kwargs(kw)
    out, lse = pkg.attention_forward(q.cuda(), k.cuda(), v.cuda(), return_lse=True, **gkw)
    got = pkg.attention_backward(q.cuda(), k.cuda(), v.cuda(), out, lse, dout.cuda(),
                                 dlse=None if dlse is None else dlse.cuda(), **gkw)
    pkg.check(torch.cuda.current_stream().cuda_stream)
    return out.cpu(), lse.cpu(), dict(zip(("dq", "dk", "dv"), (x.cpu() for x in got)))


def within(got, want, name, rows):
    """got[name] for these rows, element by element."""
    x, w, bound = got[name][:, :, rows].double(), getattr(want, name)[:, :, rows], getattr(want, name + "_err")[:, :, rows]
    assert torch.isfinite(x).all(), name
    assert ((x - w).abs() <= bound).all(), (name, float(((x - w).abs() / bound).max()))


@pytest.mark.parametrize("N,d,batch", [(640, 64, 1), (640, 128, 1), (200, 64, 1), (100, 128, 1), (200, 64, 40)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_other_rows_of_an_infinite_gradient(pkg, N, d, batch, value):
    """dO of one row holds an infinity or NaN. dQ of all other rows, and dK and dV of the tiles of 128 keys that the row does
    not see, are what they are without it. (Gradients and scores so large that P dS goes beyond fp16 if it is not scaled.)"""
    q, k, v, dout = tensors(N + d, batch, 2, N, d, spread=3.0, grad=64.0)
    row = N // 3
    dirty = dout.clone()
    dirty[0, 0, row, 5] = value
    dout[0, 0, row] = 0
    out, lse, got = run(pkg, q, k, v, dirty, causal=True)
    want = oracle.Gradient(q, k, v, out, lse, dout, causal=True)
    rest = [i for i in range(N) if i != row]
    within(got, want, "dq", rest)
    unseen = list(range((row // 128 + 1) * 128, N))
    for name in ("dk", "dv"):
        within(got, want, name, unseen)
    assert not torch.isfinite(got["dq"][0, 0, row]).all()


@pytest.mark.parametrize("d", [64, 128])
def test_other_rows_of_an_infinite_gradient_of_the_log_sum_exp(pkg, d):
    q, k, v, dout = tensors(50 + d, 1, 2, 500, d, spread=3.0, grad=64.0)
    dlse = torch.zeros((1, 2, 500))
    dlse[0, 1, 77] = math.inf
    out, lse, got = run(pkg, q, k, v, dout, dlse, causal=True)
    dlse[0, 1, 77] = 0
    want = oracle.Gradient(q, k, v, out, lse, dout, dlse, causal=True)
    within(got, want, "dq", [i for i in range(500) if i != 77])
    within(got, want, "dk", list(range(128, 500)))
    within(got, want, "dv", list(range(500)))  # P dO has no part of it


@pytest.mark.parametrize("d", [64, 128])
def test_rows_in_front_of_an_infinite_value(pkg, d):
    """V of a late key is infinite: rows of the tiles in front of it do not see it."""
    q, k, v, dout = tensors(60 + d, 1, 2, 640, d, spread=3.0, grad=64.0)
    v[0, 0, 500, 7] = math.inf
    out, lse, got = run(pkg, q, k, v, dout, causal=True)
    seen = [x[:, :, :384] for x in (q, k, v, out, lse, dout)]
    want = oracle.Gradient(*seen, causal=True)
    within({"dq": got["dq"][:, :, :384]}, want, "dq", list(range(384)))
    within({"dq": got["dq"][:, 1:]}, oracle.Gradient(*(x[:, 1:] for x in (q, k, v, out, lse, dout)), causal=True), "dq",
           list(range(640)))


def norm_within(got, q, k, v, out, lse, dout, dlse, rows_q, rows_k):
    """Errors in the 2-norm of dq over rows_q and of dk over rows_k against what independent roundings add up to."""
    want = oracle.Gradient(q, k, v, out, lse, dout, dlse, causal=True)
    x = [t.double() for t in (q, k, v, out, lse, dout)]
    scale = 1 / math.sqrt(q.shape[3])
    p = torch.exp(oracle.scores(x[0], x[1], causal=True) - x[4][..., None])
    delta = (x[5] * x[3]).sum(-1) - (0 if dlse is None else dlse.double())
    ds2 = (p * (x[5] @ x[2].transpose(2, 3) - delta[..., None])) ** 2
    h2, r = 2.0 ** -22, 2.0 ** -13
    var = {"dq": scale ** 2 * (h2 + r * r) * (ds2 @ x[1] ** 2) + h2 * want.dq ** 2,
           "dk": scale ** 2 * (h2 + r * r) * (ds2.transpose(2, 3) @ x[0] ** 2) + h2 * want.dk ** 2}
    for name, rows in (("dq", rows_q), ("dk", rows_k)):
        w = getattr(want, name)[:, :, rows]
        err = (got[name][:, :, rows].double() - w).norm()
        bound = var[name][:, :, rows].sum().sqrt() + r * w.norm()
        assert err <= bound, (name, float(err / bound))


@pytest.mark.parametrize("d", [64, 128])
def test_small_rows_beside_a_large_one(pkg, d):
    """One row of dO is 2^18 times the others, and one d_lse is 10^6 or near the end of fp32: no cost to the precision of other
    rows of dQ, nor of dK where the row is not seen."""
    N, row = 4096, 50
    q, k, v, dout = tensors(70 + d, 1, 1, N, d, grad=2.0 ** -6)
    large = dout.clone()
    large[0, 0, row] *= 2.0 ** 18
    rest, unseen = [i for i in range(N) if i != row], list(range(128, N))
    out, lse, got = run(pkg, q, k, v, large, causal=True)
    norm_within(got, q, k, v, out, lse, large, None, rest, unseen)
    for value in (1e6, 3e38):
        dlse = torch.zeros((1, 1, N))
        dlse[0, 0, row] = value
        out, lse, got = run(pkg, q, k, v, dout, dlse, causal=True)
        norm_within(got, q, k, v, out, lse, dout, dlse, rest, unseen)


def test_small_rows_beside_a_large_one_in_a_short_head(pkg):
    """The same bits where the kernel finds the norms itself and where another kernel has found them."""
    for N, d in ((200, 64), (100, 128), (256, 64), (128, 128)):
        q, k, v, dout = (x.cuda() for x in tensors(80 + N, 31, 5, N, d, grad=2.0 ** -6))
        dout[:, :, 3] *= 2.0 ** 18
        dout[1, 2, N - 2] = math.inf
        out, lse = pkg.attention_forward(q, k, v, causal=True, return_lse=True)
        many = pkg.attention_backward(q, k, v, out, lse, dout, causal=True)
        few = pkg.attention_backward(*(x[:2] for x in (q, k, v, out, lse, dout)), causal=True)
        for x, y in zip(many, few):
            assert torch.equal(x[:2].isnan(), y.isnan()) and torch.equal(x[:2].nan_to_num(7.0), y.nan_to_num(7.0))
