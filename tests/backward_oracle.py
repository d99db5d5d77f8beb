"""The gradient of the attention in 64 bits, for the tests: the definition, differentiated by hand, and what its products'
operands add up to in absolute value (what roundings are relative to)."""
import math

import torch


def hidden(n, causal, wl, wr):
    i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
    m = torch.zeros(n, n, dtype=torch.bool)
    if causal:
        m |= j > i
    if wl >= 0:
        m |= j < i - wl
    if wr >= 0:
        m |= j > i + wr
    return m


def scores(q, k, causal=False, window_left=-1, window_right=-1, softmax_scale=0.0, alibi_slopes=None):
    """q, k: [B, H, N, d] in 64 bits; the scaled, biased scores, -infinity where hidden."""
    n, d = q.shape[2:]
    s = q @ k.transpose(2, 3) * (softmax_scale if softmax_scale > 0 else 1 / math.sqrt(d))
    if alibi_slopes is not None:
        gap = (torch.arange(n)[:, None] - torch.arange(n)[None, :]).abs().double()
        s = s - alibi_slopes.double()[None, :, None, None] * gap
    return s.masked_fill(hidden(n, causal, window_left, window_right), -math.inf)


def forward(q, k, v, **kw):
    s = scores(q, k, **kw)
    return torch.softmax(s, -1) @ v, torch.logsumexp(s, -1)


class Gradient:
    """dq, dk, dv of the formula with the given out and lse, and bounds on the kernel's errors (see the tests)."""

    def __init__(self, q, k, v, out, lse, dout, dlse=None, **kw):
        q, k, v, out, lse, dout = (x.double() for x in (q, k, v, out, lse, dout))
        d = q.shape[3]
        scale = kw.get("softmax_scale", 0.0)
        scale = scale if scale > 0 else 1 / math.sqrt(d)
        p = torch.exp(scores(q, k, **kw) - lse[..., None])
        delta = (dout * out).sum(-1) - (0 if dlse is None else dlse.double())
        ds = p * (dout @ v.transpose(2, 3) - delta[..., None])
        self.dq, self.dk, self.dv = scale * ds @ k, scale * ds.transpose(2, 3) @ q, p.transpose(2, 3) @ dout
        h, r = 2.0 ** -11, 2.0 ** -13  # half a step of fp16; what errors of the scores do to P
        # dO.V and delta in fp32: each a sum of d products
        size = p * (dout.abs() @ v.abs().transpose(2, 3) + (dout * out).abs().sum(-1)[..., None])
        ds_err = (h + r) * ds.abs() + 2.0 ** -18 * size
        tiny = 2.0 ** -24  # the smallest step of the fp16 outputs
        self.dq_err = scale * ds_err @ k.abs() + h * self.dq.abs() + tiny
        self.dk_err = scale * ds_err.transpose(2, 3) @ q.abs() + h * self.dk.abs() + tiny
        self.dv_err = (h + r) * p.transpose(2, 3) @ dout.abs() + h * self.dv.abs() + tiny
