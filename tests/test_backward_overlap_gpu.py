"""flash_backward refuses outputs that lie in the memory of its inputs or of one another."""
import pytest
import torch

from test_backward_gpu import tensors

pytestmark = pytest.mark.gpu


def test_overlapping_outputs_are_refused(pkg):
    B, H, N, d = 1, 2, 100, 64
    q, k, v, dout = (x.cuda() for x in tensors(90, B, H, N, d))
    out, lse = pkg.attention_forward(q, k, v, return_lse=True)
    want = pkg.attention_backward(q, k, v, out, lse, dout)
    ins = dict(q=q, k=k, v=v, out=out, lse=lse, dout=dout)
    kept = {name: x.clone() for name, x in ins.items()}
    n = q.numel()

    def refused(**kw):
        with pytest.raises(pkg.FlashForwardError) as e:
            pkg.attention_backward(**{**ins, **kw})
        assert e.value.code == pkg.FA_INVALID_ARG and "overlap" in str(e.value)
        torch.cuda.synchronize()
        assert all(torch.equal(x, kept[name]) for name, x in ins.items())

    for name in ("q", "k", "v", "out", "dout"):
        for grad in ("dq", "dk", "dv"):
            refused(**{grad: ins[name]})
    one = torch.empty_like(q)
    refused(dq=one, dk=one)
    refused(dk=one, dv=one)
    pool = torch.zeros(2 * n, device="cuda", dtype=torch.half)
    refused(dq=pool[:n].view_as(q), dv=pool[n - 8:2 * n - 8].view_as(q))
    mixed = pool[:n].copy_(q.flatten()).view_as(q)
    refused(q=mixed, dk=pool[n - 8:2 * n - 8].view_as(q))
    stats = torch.zeros(n, device="cuda", dtype=torch.half)  # lse in the middle of an output
    held = stats[64:64 + 2 * lse.numel()].view(torch.float32).view_as(lse).copy_(lse)
    refused(lse=held, dq=stats.view_as(q))
    refused(dlse=held, dv=stats.view_as(q))
    # side by side is not over one another
    pool = torch.full((3 * n,), 7.0, device="cuda", dtype=torch.half)
    grads = [pool[i * n:(i + 1) * n].view_as(q) for i in range(3)]
    got = pkg.attention_backward(**ins, dq=grads[0], dk=grads[1], dv=grads[2])
    for x, y in zip(got, want):
        assert torch.equal(x, y)
