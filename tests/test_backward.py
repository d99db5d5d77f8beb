"""Refusals of flash_backward and its Python wrapper, its workspace, and its oracle against autograd. No GPU."""
import pytest
import torch

import backward_oracle as oracle
from test_paged_cache import Fake

P = 0x10000


def call(pkg, tensors=9 * [P], lse=P, d_lse=None, batch=1, heads=2, seqlen=128, head_dim=64, scale=0.0, slopes=None, ws=P,
         ws_bytes=1 << 40):
    q, k, v, o, d_o, dq, dk, dv = tensors[:8]
    return pkg.lib().flash_backward(q, k, v, o, d_o, lse, d_lse, dq, dk, dv, batch, heads, seqlen, head_dim, scale, 0, -1, -1,
                                    slopes, ws, ws_bytes, None)


def test_bad_arguments(pkg):
    bad = pkg.FA_INVALID_ARG
    for i in range(8):
        for value in (None, P + 8):
            t = 8 * [P]
            t[i] = value
            assert call(pkg, t) == bad
    for kw in (dict(lse=None), dict(lse=P + 2), dict(d_lse=P + 1), dict(slopes=P + 2), dict(batch=0), dict(heads=-1),
               dict(seqlen=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-35), dict(ws=None),
               dict(ws=P + 16), dict(ws_bytes=511), dict(batch=200, heads=300, seqlen=2 ** 31 - 1)):
        assert call(pkg, **kw) == bad, kw
        assert pkg.lib().flash_forward_last_error()
    assert call(pkg, head_dim=96) == pkg.FA_UNSUPPORTED
    assert call(pkg, batch=256, heads=256) == pkg.FA_UNSUPPORTED


def test_workspace_bytes(pkg):
    size = pkg.lib().flash_backward_workspace_bytes
    assert size(1, 1, 1) == 512 and size(2, 3, 100) == 2560 + 256
    assert size(2, 32, 8192) == 4 * 64 * 8192 + 12 * 64 * 64
    assert size(0, 1, 1) == size(1, -1, 1) == size(1, 1, 0) == 0


def test_no_gpu_is_an_error(pkg):
    if torch.cuda.is_available():
        pytest.skip("this check is for machines without a GPU")
    assert call(pkg) in (pkg.FA_CUDA_ERROR, pkg.FA_UNSUPPORTED)


class FakeTensor(Fake):
    def contiguous(self):
        return self


def test_wrapper_refuses_what_does_not_fit(pkg):
    half, shape = torch.float16, (2, 3, 50, 64)
    good = {x: FakeTensor(shape, half) for x in ("q", "k", "v", "out", "dout")}
    good["lse"] = FakeTensor(shape[:3], torch.float32)
    other = FakeTensor((2, 3, 51, 64), half)
    wrong = [{x: other} for x in ("q", "k", "v", "out", "dout", "dq", "dk", "dv")]
    wrong += [{x: FakeTensor(shape, torch.bfloat16)} for x in ("q", "dout", "dv")]
    wrong += [{x: FakeTensor(shape, half, device=1)} for x in ("k", "out", "dq")]
    wrong += [{x: FakeTensor(shape, half, stride=(9600, 64, 192, 1))} for x in ("q", "out", "dk")]
    wrong += [dict(lse=FakeTensor((2, 3, 49), torch.float32)), dict(lse=FakeTensor(shape[:3], half)),
              dict(dlse=FakeTensor((2, 3), torch.float32)), dict(alibi_slopes=FakeTensor((4,), torch.float32)),
              dict(out=None), dict(lse=None)]
    for change in wrong:
        with pytest.raises(AssertionError):
            pkg.attention_backward(**{**good, **change})


def test_oracle_is_the_gradient():
    """The formula of the oracle against torch's autograd of the 64-bit forward."""
    g = torch.Generator().manual_seed(1)
    q, k, v, dout = (torch.randn((1, 2, 40, 8), generator=g, dtype=torch.float64) for _ in range(4))
    dlse = torch.randn((1, 2, 40), generator=g, dtype=torch.float64)
    for kw in (dict(), dict(causal=True, window_left=7), dict(window_right=3, softmax_scale=0.7),
               dict(alibi_slopes=torch.tensor([0.3, -0.1]))):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out, lse = oracle.forward(*leaves, **kw)
        ((out * dout).sum() + (lse * dlse).sum()).backward()
        got = oracle.Gradient(q, k, v, out.detach(), lse.detach(), dout, dlse, **kw)
        for leaf, x in zip(leaves, (got.dq, got.dk, got.dv)):
            assert torch.allclose(leaf.grad, x, rtol=1e-10, atol=1e-12)
