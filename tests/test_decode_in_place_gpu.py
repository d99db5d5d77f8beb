"""flash_decode into the memory of its queries."""
import pytest
import torch

import paged_cache_oracle as oracle
from decode_plans import plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head_dim,q_heads,kv_heads,tokens,n,longest,kind", [
    (64, 8, 8, 1, 40, 3000, (0, 16, 0)),      # the line, cut items joined by a second launch
    (128, 8, 4, 2, 2, 1500, (0, 16, 8)),      # clusters
    (64, 4, 4, 1, 90, 900, (0, 16, 1)),       # a CTA an item
    (128, 200, 8, 4, 24, 1100, (1, 128, 0)),  # products of 128 rows, along the line
    (64, 96, 8, 9, 60, 900, (1, 128, 1)),     # and by a CTA an item
    (128, 14, 2, 40, 20, 800, (1, 128, 0)),   # several row tiles of a key head
])
def test_output_in_place_of_the_queries(pkg, head_dim, q_heads, kv_heads, tokens, n, longest, kind):
    lengths = [0, longest] + [(97 * i * i + 13 * i) % (longest + 1) for i in range(2, n)]
    counts = [min(m, 1 + i % tokens) for i, m in enumerate(lengths)]
    b = oracle.Batch(500 + n, lengths, counts, tokens, kv_heads, head_dim, 16, "fp16")
    d = plan(n, tokens, q_heads, kv_heads, b.table.shape[1] * 16, head_dim)
    assert (d.wide, d.part_rows, d.cluster) == kind
    args, counts = b.cuda(), b.cuda_counts()
    q = b.rows(q_heads).contiguous().cuda()
    want = pkg.attention_decode(q, *args, counts=counts)
    for _ in range(3):
        held = q.clone()
        assert pkg.attention_decode(held, *args, counts=counts, out=held) is held
        pkg.check(torch.cuda.current_stream().cuda_stream)
        assert torch.equal(held, want)
