"""flash_cache_append and flash_decode on the GPU against the plain 64-bit implementation.

Tolerances. Append: an element is a * cos - b * sin in fp32 (two roundings of products, one of the sum: 3 * 2^-24 of |a| +
|b| at most) rounded once to the cache's type: half a step of the value and that. Decode: P is rounded to the cache's type
(half a step each, relative: eps/2 of sum P|V|), the output once more (eps/2 of |O|); the scores are fp32 sums of d products
whose error moves P by a factor that 2^-13 of sum P|V| covers (scores of up to 2^6 with a relative error of 2^-20 give 2^-14
each, on a term and on the sum that it is divided by)."""
import math

import pytest
import torch

import paged_cache_oracle as oracle

pytestmark = pytest.mark.gpu
LSE_TOL = 5e-4  # as for flash_forward_lse: fp32 scores, ex2 and lg2


def check_decode(pkg, batch, q, dtype_eps=None, counts=False, **kw):
    slopes = kw.get("alibi_slopes")
    want, want_lse, size = oracle.decode(batch, q, **kw)
    gkw = dict(kw, alibi_slopes=None if slopes is None else slopes.cuda())
    out, lse = pkg.attention_decode(q.cuda(), *batch.cuda(), counts=batch.cuda_counts() if counts else None,
                                    return_lse=True, **gkw)
    pkg.check(torch.cuda.current_stream().cuda_stream)
    out, lse = out.cpu(), lse.cpu()
    assert out.is_contiguous() and torch.isfinite(out).all()
    eps = torch.finfo(batch.dtype).eps / 2
    bound = eps * (want.abs() + size) + 2.0 ** -13 * size + torch.finfo(batch.dtype).tiny
    err = (out.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    empty = torch.isinf(want_lse)
    assert (lse[empty] == -math.inf).all() and (out[empty] == 0).all()
    assert ((lse[~empty].double() - want_lse[~empty]).abs() <= LSE_TOL).all()
    return out, lse


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads,tokens,page,lengths", [
    (4, 4, 1, 16, [1]),                              # one key
    (8, 2, 1, 16, [1, 2, 15, 16, 17, 63, 64, 65]),   # around the ends of pages and tiles
    (8, 8, 1, 8, [129, 0, 77, 0]),                   # sequences without keys between others
    (6, 1, 1, 24, [0, 0, 300]),                      # pages that end inside a tile, first sequences empty
    (40, 2, 1, 128, [500, 41]),                      # 20 queries a key head: two groups of 16 rows
    (70, 1, 1, 64, [130]),                           # 70: more than a tile of 64 rows
    (7, 1, 3, 32, [3, 4, 200]),                      # several tokens, sequences that hold nothing else
    (16, 4, 8, 256, [600, 8]),
    (1, 1, 1, 16, [4100]),                           # cut among many CTAs
    (4, 4, 1, 16, [700, 0, 1, 130]),                 # clusters of CTAs with and without tiles
    (36, 4, 2, 64, [1000, 64]),                      # clusters, 18 rows
    (64, 2, 2, 64, [900]),                           # clusters, 64 rows
    (4, 2, 1, 16, [31 * i % 129 for i in range(90)]),  # a CTA for each of many short sequences
])
def test_decode(pkg, dtype, head_dim, q_heads, kv_heads, tokens, page, lengths):
    b = oracle.Batch(len(lengths) + head_dim, lengths, [min(tokens, n) for n in lengths], tokens, kv_heads, head_dim, page,
                     dtype)
    check_decode(pkg, b, b.rows(q_heads))


def with_room(batch, keys=1 << 19):
    """The same batch with a page table that has room for long sequences: how a call is computed depends on that room."""
    more = torch.full((len(batch.lengths), keys // batch.page_size), -7, dtype=torch.int32)
    more[:, :batch.table.shape[1]] = batch.table
    batch.table = more
    return batch


MANY_ROWS = [  # query heads, key heads, tokens, page, lengths
    (24, 1, 1, 16, [1]),                         # 24 rows, one key
    (8, 1, 3, 24, [3, 64, 65, 127, 128, 129]),   # around the ends of tiles
    (32, 1, 1, 8, [192, 0, 193, 0, 256, 257]),   # 32 rows; one, two and three tiles; sequences without keys between others
    (33, 1, 1, 64, [700, 41]),
    (16, 2, 8, 128, [500, 8, 1100]),             # 64 rows of either key head
    (65, 1, 1, 16, [330]),
    (20, 2, 10, 32, [10, 11, 640]),              # 100 rows
    (4, 1, 32, 16, [32, 150]),                   # 128 rows, a sequence that holds nothing else
    (43, 1, 3, 16, [260]),                       # 129 rows: two row tiles
    (4, 2, 150, 256, [150, 400]),                # 300 rows
    (20, 1, 1, 16, [3000]),                      # cut among many CTAs
    (40, 2, 1, 16, [37 * i * i % 300 for i in range(40)]),  # items that share CTAs
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads,tokens,page,lengths", MANY_ROWS)
def test_many_rows(pkg, dtype, head_dim, q_heads, kv_heads, tokens, page, lengths):
    b = oracle.Batch(70 + len(lengths) + head_dim, lengths, [min(tokens, n) for n in lengths], tokens, kv_heads, head_dim, page,
                     dtype)
    q = b.rows(q_heads)
    check_decode(pkg, b, q, counts=True)
    long = check_decode(pkg, with_room(b), q, counts=True)
    again = check_decode(pkg, b, q, counts=True)
    for x, y in zip(long, again):
        assert torch.equal(x, y)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("window,alibi", [(0, False), (1, True), (63, False), (64, True), (200, False), (100000, True)])
def test_many_rows_window_and_alibi(pkg, head_dim, window, alibi):
    b = with_room(oracle.Batch(71, [5, 64, 133, 700, 0], [5, 6, 6, 2, 0], 6, 2, head_dim, 16, "fp16"))
    slopes = torch.tensor([0.5, 0.01, -0.02, 0.0, 0.1, 0.2, 0.3, 0.003]) if alibi else None
    check_decode(pkg, b, b.rows(8), counts=True, window_left=window, alibi_slopes=slopes)


@pytest.mark.parametrize("head_dim,rows", [(64, 24), (64, 48), (64, 96), (128, 24), (128, 96)])
@pytest.mark.parametrize("fill", [math.nan, math.inf])
def test_many_rows_ignore_what_is_not_the_sequences(pkg, head_dim, rows, fill):
    b = oracle.Batch(72, [1, 40, 200, 317], [1, 2, 2, 1], 2, 1, head_dim, 32, "bf16", fill=fill)
    for window in (-1, 70):
        if window >= 0:
            for i, n in enumerate(b.lengths):
                gone = max(0, n - b.counts[i] - window)
                for j in range(gone):
                    b.k_pages[b.table[i, j // 32], :, j % 32] = fill
                    b.v_pages[b.table[i, j // 32], :, j % 32] = fill
                b.table[i, :gone // 32] = -1
        check_decode(pkg, with_room(b), b.rows(rows // 2), counts=True, window_left=window)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("rows", [24, 60, 120])
def test_many_rows_with_scores_that_grow(pkg, head_dim, rows):
    """The maximum of a row rises from tile to tile: scores with a deviation of 6, and keys that grow along the sequence."""
    b = oracle.Batch(73, [900, 400], [1, 1], 1, 1, head_dim, 16, "fp16")
    for i, n in enumerate(b.lengths):
        b.k[i] = (b.k[i] * torch.linspace(0.1, 1.5, n)[None, :, None]).half()
        for j in range(n):
            b.k_pages[b.table[i, j // 16], :, j % 16] = b.k[i][:, j]
    check_decode(pkg, with_room(b), b.rows(rows, scale=4.0))


def test_many_rows_bad_page_is_reported(pkg):
    b = with_room(oracle.Batch(74, [200, 90], [1, 1], 1, 1, 128, 16, "fp16"))
    q = b.rows(24)
    args = b.cuda()
    want = pkg.attention_decode(q.cuda(), *args)
    stream = torch.cuda.current_stream().cuda_stream
    pkg.check(stream)
    for bad in (-1, b.k_pages.shape[0], 2 ** 31 - 1):
        table = args[2].clone()
        table[0, 3] = bad
        out = pkg.attention_decode(q.cuda(), args[0], args[1], table, args[3])
        with pytest.raises(Exception):
            pkg.check(stream)
        assert torch.equal(out[1], want[1])
        pkg.check(stream)


def test_many_rows_on_two_streams_and_captured(pkg):
    b = with_room(oracle.Batch(75, [900, 130, 0, 77], [2, 2, 0, 1], 2, 2, 64, 16, "fp16"))
    q, args, counts = b.rows(40).cuda(), b.cuda(), b.cuda_counts()
    want = pkg.attention_decode(q, *args, counts=counts)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(pkg.attention_decode(q, *args, counts=counts))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = pkg.attention_decode(q, *args, counts=counts)
    args[3].copy_(torch.tensor([500, 1, 0, 77], dtype=torch.int32))
    counts.copy_(torch.tensor([2, 1, 0, 1], dtype=torch.int32))
    graph.replay()
    later = pkg.attention_decode(q, *args, counts=counts)
    pkg.check(torch.cuda.current_stream().cuda_stream)
    assert all(torch.equal(x, want) for x in outs) and torch.equal(captured, later)


@pytest.mark.parametrize("window", [0, 1, 63, 64, 200, 100000, 2 ** 31 - 1])
@pytest.mark.parametrize("alibi", [False, True])
def test_decode_window_and_alibi(pkg, window, alibi):
    b = oracle.Batch(5, [1, 64, 65, 333, 700], [1, 3, 3, 3, 3], 3, 2, 64, 16, "fp16")
    slopes = torch.tensor([0.5, 0.01, -0.02, 0.0]) if alibi else None
    check_decode(pkg, b, b.rows(4), counts=True, window_left=window, alibi_slopes=slopes)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_decode_many_sequences(pkg, dtype):
    """More sequences than lanes of a warp, lengths of every kind, some of them empty."""
    lengths = [(37 * i * i) % 400 for i in range(150)]
    b = oracle.Batch(3, lengths, [min(1, n) for n in lengths], 1, 2, 64, 16, dtype, token_major=True)
    check_decode(pkg, b, b.rows(4))


def test_decode_counts(pkg):
    """A padded batch: rows behind a sequence's count are 0 and -infinity, in tiles that no mask cuts too."""
    b = oracle.Batch(4, [500, 300, 4, 0, 129], [4, 1, 2, 0, 0], 4, 2, 128, 16, "fp16")
    check_decode(pkg, b, b.rows(6), counts=True)


@pytest.mark.parametrize("fill", [math.nan, math.inf])
@pytest.mark.parametrize("window", [-1, 70])
def test_decode_ignores_what_is_not_the_sequences(pkg, fill, window):
    """The rest of last pages, pages that no sequence names and pages in front of the window hold anything."""
    b = oracle.Batch(6, [1, 40, 200, 317], [1, 1, 1, 1], 1, 2, 128, 32, "fp16", fill=fill)
    if window >= 0:
        for i, n in enumerate(b.lengths):
            gone = max(0, n - 1 - window)
            for j in range(gone):  # tokens in front of the window: overwritten; whole pages: given back
                b.k_pages[b.table[i, j // 32], :, j % 32] = fill
                b.v_pages[b.table[i, j // 32], :, j % 32] = fill
            b.table[i, :gone // 32] = -1
    check_decode(pkg, b, b.rows(4), window_left=window)


def test_decode_large_scores_and_scale(pkg):
    b = oracle.Batch(8, [1000, 90], [1, 1], 1, 1, 64, 16, "fp16")
    check_decode(pkg, b, b.rows(2), softmax_scale=0.5)  # scores of +-15
    q = b.rows(2)
    out, _ = pkg.attention_decode(q.cuda() * 100, *b.cuda(), return_lse=True)  # scores of hundreds: one key takes all
    want, _, _ = oracle.decode(b, q * 100)
    assert torch.isfinite(out).all() and ((out.cpu().double() - want).abs() <= 2e-2).all()


def test_decode_nan_and_infinity_where_they_are_seen(pkg):
    b = oracle.Batch(9, [100, 100], [1, 1], 1, 1, 64, 16, "fp16")
    b.k_pages[b.table[1, 2], 0, 3, 5] = math.nan
    out, lse = pkg.attention_decode(b.rows(4).cuda(), *b.cuda(), return_lse=True)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()


def test_decode_is_the_same_every_time_and_on_views(pkg):
    b = oracle.Batch(10, [3000, 17, 900], [2, 2, 2], 2, 2, 128, 16, "bf16")
    args, q = b.cuda(), b.rows(8).cuda()
    first = pkg.attention_decode(q, *args, return_lse=True)
    # the same rows out of a fused projection, a table with longer rows, the pool in the middle of a larger one
    fused = torch.randn((3, 2, 12, 128), device="cuda").bfloat16()
    fused[:, :, 2:10] = q.transpose(1, 2)
    table = torch.full((3, args[2].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    table[:, :args[2].shape[1]] = args[2]
    pools = []
    for x in args[:2]:
        wide = torch.full((x.shape[0] + 2, x.shape[1] + 3, x.shape[2], x.shape[3]), math.nan, device="cuda", dtype=x.dtype)
        wide[1:-1, 2:4] = x
        pools.append(wide[1:-1, 2:4])
    second = pkg.attention_decode(fused.transpose(1, 2)[:, 2:10], *pools, table[:, :args[2].shape[1]], args[3],
                                  return_lse=True)
    for x, y in zip(first, second):
        assert torch.equal(x, y)


def test_decode_far_offsets(pkg):
    """A pool of more than 2^32 elements: the sequence's pages lie at its end."""
    pages, heads, page, d = 40000, 8, 128, 128  # 5.2e9 elements a tensor
    k = torch.zeros((pages, heads, page, d), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    b = oracle.Batch(11, [200], [1], 1, heads, d, page, "fp16", spare=0)
    k[-2:], v[-2:] = b.k_pages.cuda(), b.v_pages.cuda()
    table = b.table.clone()
    table[:, :2] += pages - 2
    q = b.rows(8)
    out, lse = pkg.attention_decode(q.cuda(), k, v, table.cuda(), b.cuda()[3], return_lse=True)
    near, near_lse = check_decode(pkg, b, q)
    assert torch.equal(out.cpu(), near) and torch.equal(lse.cpu(), near_lse)
    # and the append writes there
    new = b.rows(8)
    pkg.cache_append(new.cuda(), new.cuda(), k, v, table.cuda(), b.cuda()[3])
    pkg.check(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(k[table[0, 1], :, 199 - 128].cpu(), new[0, :, 0])
    assert int((k != 0).any(-1).sum()) <= 200 * heads


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head_dim,rotary_dim,token_major", [(64, 64, False), (64, 16, True), (128, 128, True),
                                                             (128, 96, False), (128, 32, False)])
def test_append(pkg, dtype, interleaved, head_dim, rotary_dim, token_major):
    lengths, counts = [1, 17, 5, 40, 0, 33], [1, 5, 5, 2, 0, 0]
    b = oracle.Batch(20 + rotary_dim, lengths, counts, 5, 2, head_dim, 16, dtype, token_major=token_major)
    k, v, q = b.rows(2), b.rows(2), b.rows(6)
    k[1, 0, 2, 3] = math.inf  # copied or turned like any other
    rotary = oracle.angles(64, rotary_dim)
    want = oracle.append(b, k, v, q, rotary, interleaved)
    k_pages, v_pages, table, lens = b.cuda()
    before = k_pages.clone()
    turned = pkg.cache_append(k.cuda(), v.cuda(), k_pages, v_pages, table, lens, counts=b.cuda_counts(), q=q.cuda(),
                              rotary=rotary.cuda(), interleaved=interleaved)
    pkg.check(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(v_pages.cpu().double(), want[1])
    eps = torch.finfo(b.dtype).eps / 2
    for got, w, src in ((k_pages.cpu(), want[0], 6.0), (turned.cpu(), want[2], 6.0)):
        same = torch.isinf(w) | torch.isnan(w)
        assert torch.equal(torch.isnan(got[same]), torch.isnan(w[same]))
        err = (got.double() - w).abs()[~same]
        # |a| + |b| of normal values is below 12
        assert (err <= eps * w[~same].abs() + 3 * 2.0 ** -24 * 2 * src + torch.finfo(b.dtype).tiny).all()
    touched = torch.zeros(k_pages.shape[0], 16, dtype=torch.bool)
    for i, (n, c) in enumerate(zip(lengths, counts)):
        for j in range(n - c, n):
            touched[b.table[i, j // 16], j % 16] = True
    untouched = ~touched[:, None, :, None].expand(k_pages.shape)
    assert torch.equal(k_pages.cpu()[untouched], before.cpu()[untouched])


def test_append_without_rotation_and_in_place(pkg):
    b = oracle.Batch(31, [9, 30], [3, 3], 3, 4, 64, 8, "fp16")
    k, v = b.rows(4), b.rows(4)
    want = oracle.append(b, k, v)
    args = b.cuda()
    assert pkg.cache_append(k.cuda(), v.cuda(), *args) is None
    assert torch.equal(args[0].cpu().double(), want[0]) and torch.equal(args[1].cpu().double(), want[1])
    rotary, q = oracle.angles(32, 64).cuda(), b.rows(4).cuda().contiguous()
    apart = pkg.cache_append(k.cuda(), v.cuda(), *args, q=q, rotary=rotary)
    same = pkg.cache_append(k.cuda(), v.cuda(), *args, q=q, rotary=rotary, q_out=q)
    assert same is q and torch.equal(q, apart)


def test_append_of_many_tokens_and_of_keys_alone(pkg):
    """More tokens than blocks that run at once (a block then has a whole token), and a rotation without queries."""
    lengths = [700, 333, 640]
    b = oracle.Batch(32, lengths, [640, 200, 640], 640, 2, 128, 16, "fp16")
    k, v, q = b.rows(2), b.rows(2), b.rows(6)
    rotary = oracle.angles(700, 64)
    want = oracle.append(b, k, v, q, rotary)
    args = b.cuda()
    turned = pkg.cache_append(k.cuda(), v.cuda(), *args, counts=b.cuda_counts(), q=q.cuda(), rotary=rotary.cuda())
    alone = b.cuda()
    assert pkg.cache_append(k.cuda(), v.cuda(), *alone, counts=b.cuda_counts(), rotary=rotary.cuda()) is None
    pkg.check(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(args[0], alone[0]) and torch.equal(args[1], alone[1])
    assert torch.equal(args[1].cpu().double(), want[1])
    # |a| + |b| of normal values is below 12
    for got, w in ((args[0].cpu(), want[0]), (turned.cpu(), want[2])):
        assert ((got.double() - w).abs() <= 2.0 ** -11 * w.abs() + 3 * 2.0 ** -24 * 12 + 2.0 ** -24).all()


def test_bad_indices_are_reported(pkg):
    """Pages, lengths, counts and positions outside their ranges become a status; the other sequences are unharmed."""
    stream = torch.cuda.current_stream().cuda_stream

    def reported():
        with pytest.raises(pkg.FlashForwardError) as e:
            pkg.check(stream)
        assert e.value.code == pkg.FA_BAD_INDEX
        pkg.check(stream)  # and forgotten

    b = oracle.Batch(40, [40, 200], [2, 2], 2, 2, 64, 16, "fp16")
    q, k = b.rows(4).cuda(), b.rows(2).cuda()
    good = pkg.attention_decode(q, *b.cuda())
    for page in (-1, b.k_pages.shape[0], 2 ** 30, -2 ** 31):
        args = b.cuda()
        args[2][0, 2] = page
        out = pkg.attention_decode(q, *args)
        reported()
        assert torch.equal(out[1], good[1])
        before = args[0].clone()
        pkg.cache_append(k[:1], k[:1], args[0], args[1], args[2][:1], args[3][:1])
        reported()
        assert torch.equal(args[0], before)
    for length in (-3, 10 ** 6, 2 ** 31 - 1):
        args = b.cuda()
        args[3][1] = length
        args[2][1] = args[2][0, 0]  # every page of the row can be read
        pkg.attention_decode(q, *args)
        reported()
        pkg.cache_append(k, k, *args)
        reported()
    for counts in ([3, 2], [-1, 2], [2, 2 ** 31 - 1]):
        pkg.attention_decode(q, *b.cuda(), counts=torch.tensor(counts, dtype=torch.int32).cuda())
        reported()
    args = b.cuda()
    before = args[0].clone()
    pkg.cache_append(k, k, *args, q=q, rotary=oracle.angles(150, 64).cuda())  # sequence 1 is at 198
    reported()
    assert torch.equal(args[0][args[2][1, 12].item()], before[args[2][1, 12].item()])


def test_generation_steps_captured_and_replayed(pkg):
    """Append and decode of a step as one graph, replayed with lengths that grow, against the same steps by call."""
    tokens, heads, kv_heads, d, page = 1, 8, 2, 64, 16
    b = oracle.Batch(50, [30, 5, 64], [1, 1, 1], tokens, kv_heads, d, page, "fp16", spare=8)
    spare = sorted(set(range(b.k_pages.shape[0])) - {int(x) for x in b.table.flatten() if x >= 0})
    for i, need in enumerate([2, 1, 4]):  # room to grow
        b.table[i, need] = spare[i]
    rotary = oracle.angles(128, d).cuda()
    steps = [(b.rows(kv_heads).cuda(), b.rows(kv_heads).cuda(), b.rows(heads).cuda()) for _ in range(4)]

    def step(k, v, q, k_pages, v_pages, table, lengths):
        turned = pkg.cache_append(k, v, k_pages, v_pages, table, lengths, q=q, rotary=rotary)
        return pkg.attention_decode(turned, k_pages, v_pages, table, lengths, return_lse=True)

    eager_args, want = b.cuda(), []
    for s in steps:
        want.append([x.clone() for x in step(*s, *eager_args)])
        eager_args[3] += 1
    args = b.cuda()
    held = [torch.empty_like(x) for x in steps[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held, *args)
    for s, w in zip(steps, want):
        for x, y in zip(held, s):
            x.copy_(y)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(got, w))
        args[3] += 1
    pkg.check(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(args[0], eager_args[0]) and torch.equal(args[1], eager_args[1])


def test_prompt_then_steps_is_the_forward(pkg):
    """A prompt through attention_forward, its keys into the cache, then one token at a time: the rows that attention_forward
    gives for the whole sequence."""
    B, H, N, d, prompt = 2, 4, 150, 128, 131
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((B, H, N, d), generator=g, device="cuda", dtype=torch.float16) for _ in range(3))
    whole, lse = pkg.attention_forward(q, k, v, causal=True, return_lse=True)
    k_pages, v_pages = (torch.full((20, H, 16, d), math.nan, device="cuda", dtype=torch.float16) for _ in range(2))
    table = torch.randperm(20, device="cuda").int().view(2, 10)
    lengths = torch.full((B,), prompt, dtype=torch.int32, device="cuda")
    pkg.cache_append(k[:, :, :prompt], v[:, :, :prompt], k_pages, v_pages, table, lengths)
    for i in range(prompt, N, 1):
        lengths += 1
        pkg.cache_append(k[:, :, i:i + 1], v[:, :, i:i + 1], k_pages, v_pages, table, lengths)
        out, out_lse = pkg.attention_decode(q[:, :, i:i + 1], k_pages, v_pages, table, lengths, return_lse=True)
        # both are within 2 eps/2 of sum P|V|, which is below 1.5 here, and of |O|
        assert ((out[:, :, 0] - whole[:, :, i]).abs().float() <= 4 * 2.0 ** -11 * 1.5).all()
        assert ((out_lse[:, :, 0] - lse[:, :, i]).abs() <= 2 * LSE_TOL).all()
    pkg.check(torch.cuda.current_stream().cuda_stream)


def test_on_two_streams(pkg):
    b = oracle.Batch(60, [2500, 700], [1, 1], 1, 4, 128, 16, "fp16")
    args, q = b.cuda(), b.rows(16).cuda()
    want = pkg.attention_decode(q, *args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(pkg.attention_decode(q, *args))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in outs)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("heads,room", [(8, False), (8, True), (40, False), (40, True), (100, True)])
def test_wait_gives_up_and_the_device_stays_usable(pkg, heads, room, head_dim):
    """Test build: a sequence never gets its last tile. The launch returns, the check reports it, the next call is right.
    With and without room for long sequences: clusters, or the line of tiles; and a row's warps, or products of 128 rows."""
    import ctypes

    from test_wait_runs_out import load_waittest

    L = load_waittest()
    L.flash_decode.argtypes = L.flash_decode_test_withhold.argtypes = pkg.lib().flash_decode.argtypes
    b = oracle.Batch(80, [900, 400], [1, 1], 1, 1, head_dim, 16, "fp16")
    if room:
        b = with_room(b)
    q, args = b.rows(heads).cuda(), b.cuda()
    want = pkg.attention_decode(q, *args)
    stream = torch.cuda.current_stream().cuda_stream
    pkg.check(stream)
    cache = pkg._cache_struct(torch, *args, None)
    rows = pkg._rows_struct("q", q, args[0], heads, 2, 1)
    out = torch.zeros((2, heads, 1, head_dim), device="cuda", dtype=q.dtype)
    nbytes = pkg.lib().flash_decode_workspace_bytes(1, heads, 1, head_dim)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    call = (cache, rows, out.data_ptr(), None, 2, 1, heads, 0.0, -1, None, ws.data_ptr(), ctypes.c_size_t(nbytes), stream)
    assert L.flash_decode_test_withhold(*call) == pkg.FA_OK
    assert L.flash_forward_check(stream) == pkg.FA_DEVICE_TIMEOUT
    assert L.flash_forward_check(stream) == pkg.FA_OK
    assert L.flash_decode(*call) == pkg.FA_OK
    assert L.flash_forward_check(stream) == pkg.FA_OK
    assert torch.equal(out, want)
