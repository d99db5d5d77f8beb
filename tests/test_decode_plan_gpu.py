"""flash_decode on every way that a call is run, with windows that hide keys: against the plain implementation, with the
tolerances of test_paged_cache_gpu.py."""
import math

import pytest
import torch

import paged_cache_oracle as oracle
from decode_plans import plan
from test_paged_cache_gpu import check_decode, with_room

pytestmark = pytest.mark.gpu


def lengths_of(n, longest, step=97):
    """Lengths of every kind from 0 to `longest`, both among them."""
    return [0, longest] + [(step * i * i + 13 * i) % (longest + 1) for i in range(2, n)]


def windowed(seed, lengths, tokens, kv_heads, head_dim, page, dtype, window, fill):
    """A batch whose pages in front of the window are given back, and whose tokens in front of it are overwritten."""
    b = oracle.Batch(seed, lengths, [min(tokens, n) for n in lengths], tokens, kv_heads, head_dim, page, dtype, fill=fill)
    for i, n in enumerate(lengths):
        gone = max(0, n - b.counts[i] - window)
        for j in range(gone):
            b.k_pages[b.table[i, j // page], :, j % page] = fill
            b.v_pages[b.table[i, j // page], :, j % page] = fill
        b.table[i, :gone // page] = -1
    return b


def planned(b, q_heads, head_dim, window):
    return plan(len(b.lengths), b.tokens, q_heads, b.kv_heads, b.table.shape[1] * b.page_size, head_dim, window)


@pytest.mark.parametrize("dtype,fill,head_dim,q_heads,kv_heads,tokens,n,window,longest,page,part_rows", [
    ("fp16", math.nan, 128, 200, 8, 4, 12, 500, 1100, 16, 128),   # 100 rows
    ("bf16", math.inf, 64, 200, 8, 4, 12, 1020, 2000, 32, 128),
    ("bf16", math.nan, 128, 80, 8, 6, 21, 510, 900, 8, 64),       # 60 rows: two copies of them
    ("fp16", math.inf, 64, 80, 8, 6, 21, 1020, 1900, 16, 64),
    ("fp16", math.inf, 128, 96, 8, 2, 110, 500, 720, 24, 32),     # 24 rows: copies
    ("bf16", math.nan, 64, 96, 8, 2, 99, 1020, 1500, 16, 32),
    ("fp16", math.nan, 128, 14, 2, 40, 20, 333, 800, 40, 128),    # 280 rows: three row tiles
    ("bf16", math.inf, 64, 14, 2, 40, 20, 633, 1500, 40, 128),
])
def test_many_rows_behind_a_window(pkg, dtype, fill, head_dim, q_heads, kv_heads, tokens, n, window, longest, page,
                                   part_rows):
    """Products of 128 rows along the line and its join, keys hidden in front and behind."""
    b = windowed(200 + head_dim + tokens, lengths_of(n, longest), tokens, kv_heads, head_dim, page, dtype, window, fill)
    d = planned(b, q_heads, head_dim, window)
    assert d.wide and d.part_rows == part_rows and d.cluster == 0 and longest > window + tokens
    slopes = torch.linspace(-0.02, 0.4, q_heads) if dtype == "fp16" else None
    check_decode(pkg, b, b.rows(q_heads), counts=True, window_left=window, alibi_slopes=slopes)


@pytest.mark.parametrize("head_dim,longest,window", [(128, 460, -1), (128, 460, 130), (64, 900, -1), (64, 900, 300)])
def test_many_rows_by_a_cta_an_item(pkg, head_dim, longest, window):
    """Products of 128 rows where every item is a CTA's own: no line, no second launch, sequences without keys among them."""
    b = windowed(300 + head_dim, lengths_of(60, longest), 9, 8, head_dim, 16, "fp16", window if window >= 0 else 1 << 20, math.nan)
    d = planned(b, 96, head_dim, window)
    assert d.wide and d.part_rows == 128 and d.cluster == 1 and d.items > 148
    check_decode(pkg, b, b.rows(96), counts=True, window_left=window)


@pytest.mark.parametrize("head_dim,q_heads,kv_heads,tokens,n,longest,window,room,kind", [
    (64, 8, 8, 1, 12, 3000, 1500, False, (16, 0)),       # the line behind a window
    (128, 16, 8, 2, 12, 1500, 700, False, (16, 0)),
    (128, 20, 4, 4, 12, 1500, 700, False, (32, 0)),      # 20 rows
    (64, 40, 4, 4, 5, 2100, 1100, False, (64, 0)),       # 40 rows
    (64, 8, 4, 2, 2, 1500, 700, False, (16, 8)),         # clusters behind a window
    (128, 12, 2, 6, 2, 900, 300, False, (64, 8)),
    (128, 8, 1, 3, 3, 700, 150, False, (32, 4)),
    (64, 4, 4, 1, 90, 900, 600, False, (16, 1)),         # a CTA an item behind a window
    (128, 4, 2, 1, 30, 800, 30, True, (16, 1)),          # a window of one tile in a long sequence
])
def test_few_rows_behind_a_window(pkg, head_dim, q_heads, kv_heads, tokens, n, longest, window, room, kind):
    b = windowed(400 + head_dim + n, lengths_of(n, longest), tokens, kv_heads, head_dim, 16, "bf16", window, math.nan)
    if room:
        b = with_room(b)
    d = planned(b, q_heads, head_dim, window)
    assert not d.wide and (d.part_rows, d.cluster) == kind and longest > window + tokens
    check_decode(pkg, b, b.rows(q_heads), counts=True, window_left=window)
