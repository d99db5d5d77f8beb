"""Plain 64-bit implementation of the paged cache's operators, and batches to try them on, for the tests."""
import math

import torch

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


class Batch:
    """A pool of pages, a table, lengths and counts on the CPU. `fill` is what the pool holds where nothing was put."""

    def __init__(self, seed, lengths, counts, tokens, kv_heads, head_dim, page_size, dtype, fill=0.0, token_major=False,
                 spare=3):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.counts, self.tokens = list(lengths), list(counts), tokens
        self.kv_heads, self.head_dim, self.page_size, self.dtype = kv_heads, head_dim, page_size, DTYPES[dtype]
        need = [-(-n // page_size) for n in self.lengths]
        pool = sum(need) + spare
        order = torch.randperm(pool, generator=g).tolist()
        self.table = torch.full((len(self.lengths), max(max(need), 1) + 1), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        shape = (pool, page_size, kv_heads, head_dim) if token_major else (pool, kv_heads, page_size, head_dim)
        self.k_pages, self.v_pages = (torch.full(shape, fill, dtype=self.dtype) for _ in range(2))
        if token_major:
            self.k_pages, self.v_pages = self.k_pages.transpose(1, 2), self.v_pages.transpose(1, 2)
        self.k, self.v = [], []  # of every sequence, [kv_head][token][d]
        for b, n in enumerate(self.lengths):
            self.k.append(torch.randn((kv_heads, n, head_dim), generator=g).to(self.dtype))
            self.v.append(torch.randn((kv_heads, n, head_dim), generator=g).to(self.dtype))
            for j in range(n):
                page = self.table[b, j // page_size]
                self.k_pages[page, :, j % page_size] = self.k[b][:, j]
                self.v_pages[page, :, j % page_size] = self.v[b][:, j]
        self.gen = g

    def rows(self, heads, scale=1.0):
        """New rows, as a view of [batch][token][head]."""
        x = torch.randn((len(self.lengths), self.tokens, heads, self.head_dim), generator=self.gen) * scale
        return x.to(self.dtype).transpose(1, 2)

    def cuda(self):
        """k_pages, v_pages, page_table, lengths on the GPU, strides kept."""
        ints = torch.tensor(self.lengths, dtype=torch.int32).cuda()
        return [self.k_pages.cuda(), self.v_pages.cuda(), self.table.cuda(), ints]

    def cuda_counts(self):
        return torch.tensor(self.counts, dtype=torch.int32).cuda()


def decode(batch, q, softmax_scale=0.0, window_left=-1, alibi_slopes=None):
    """Returns O, log-sum-exp and sum_j P_j |V_j| (what roundings of P are relative to) in 64 bits."""
    n, heads, tokens, d = q.shape
    group = heads // batch.kv_heads
    scale = softmax_scale if softmax_scale > 0 else 1.0 / math.sqrt(d)
    out, size = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64)
    for b in range(n):
        for t in range(batch.counts[b] if batch.lengths[b] else 0):
            i = batch.lengths[b] - batch.counts[b] + t
            lo = 0 if window_left < 0 else max(0, i - window_left)
            for h in range(heads):
                k, v = (x[b][h // group, lo:i + 1].double() for x in (batch.k, batch.v))
                s = k @ q[b, h, t].double() * scale
                if alibi_slopes is not None:
                    s = s - float(alibi_slopes[h]) * torch.arange(i - lo, -1, -1, dtype=torch.float64)
                p = torch.softmax(s, 0)
                out[b, h, t], size[b, h, t] = p @ v, p @ v.abs()
                lse[b, h, t] = torch.logsumexp(s, 0)
    return out, lse, size


def rotate(x, angles, interleaved):
    """x: [..., d] in 64 bits, angles: [rotary_dim] cosines and sines."""
    half = len(angles) // 2
    c, s = angles[:half].double(), angles[half:].double()
    y = x.clone()
    first = torch.arange(half) * 2 if interleaved else torch.arange(half)
    second = first + 1 if interleaved else first + half
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    return y


def angles(positions, rotary_dim, base=10000.0):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (
        -2.0 * torch.arange(rotary_dim // 2, dtype=torch.float64) / rotary_dim)
    return torch.cat([a.cos(), a.sin()], 1).float()


def append(batch, k, v, q=None, rotary=None, interleaved=False):
    """The pools (64 bits) after the call, and the rotated queries."""
    k_pages, v_pages = batch.k_pages.double(), batch.v_pages.double()
    turned = torch.zeros(q.shape, dtype=torch.float64) if q is not None else None
    for b, (length, count) in enumerate(zip(batch.lengths, batch.counts)):
        for t in range(count):
            i = length - count + t
            page, slot = int(batch.table[b, i // batch.page_size]), i % batch.page_size
            row = k[b, :, t].double()
            k_pages[page, :, slot] = row if rotary is None else rotate(row, rotary[i], interleaved)
            v_pages[page, :, slot] = v[b, :, t].double()
            if q is not None:
                turned[b, :, t] = rotate(q[b, :, t].double(), rotary[i], interleaved)
    return k_pages, v_pages, turned
