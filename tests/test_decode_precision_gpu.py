"""flash_decode on rows that one key dominates.

Tolerances: as in test_paged_cache_gpu.py; and where P is so small beside the row's maximum that fp16 holds it in steps,
half a step a key: P is kept as 2^14 P for up to 16 rows and as 2^7 P or more for more, so that is at most 2^-32 of the
maximum (2^-25 / 2^7), times |V|. The exact main term has no rounding of P, only that of the output."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def one_sequence_many_times(keys, values, copies, page=128):
    """A pool that holds one sequence [keys][d], and a table by which `copies` sequences share it."""
    n, d = keys.shape
    pages = n // page
    pools = [x.view(pages, 1, page, d).cuda() for x in (keys, values)]
    table = torch.arange(pages, dtype=torch.int32)[None].repeat(copies, 1).cuda()
    return pools + [table, torch.full((copies,), n, dtype=torch.int32).cuda()]


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("rows", [1, 24, 40, 128])
def test_a_long_tail_behind_a_dominating_key(pkg, rows, head_dim):
    """An early key 17.3 nats above 131071 others, whose values the output is made of: they have 4e-3 of the weight together,
    3e-8 each. Many sequences, so that a CTA has all of a sequence's keys."""
    n, copies = 131072, 320
    keys, values = torch.zeros((n, head_dim)), torch.ones((n, head_dim))
    keys[3, 0], values[3] = 17.3125, 0.0
    args = one_sequence_many_times(keys.half(), values.half(), copies)
    q = torch.zeros((copies, rows, 1, head_dim))
    q[..., 0] = 1.0
    out, lse = pkg.attention_decode(q.half().cuda(), *args, softmax_scale=1.0, return_lse=True)
    pkg.check(torch.cuda.current_stream().cuda_stream)
    total = math.exp(17.3125) + n - 1
    want = (n - 1) / total
    bound = 2.0 ** -11 * 2 * want + 2.0 ** -13 * want + n * 2.0 ** -32
    err = float((out.double() - want).abs().max())
    assert err <= bound, (err, bound)
    assert float((lse.double() - math.log(total)).abs().max()) <= 5e-4


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_a_dominating_key_whose_neighbour_row_moves(pkg, head_dim, dtype):
    """128 rows in products of 128: in a later tile the maximum of every second row grows by less than 2^8, that of the others
    by far more. The rows move along together, and the key that dominates a row has P = 1, without a rounding."""
    n, page = 1 << 16, 128
    eps = torch.finfo(dtype).eps / 2
    scale = math.log2(128.45) / 7.0 * math.log(2.0)  # a product of 7 is a P of 128.45: 128 in bf16
    g = torch.Generator().manual_seed(3)
    keys, values = torch.zeros((n, head_dim)), torch.randn((n, head_dim), generator=g).to(dtype)
    keys[:, 0] = keys[:, 1] = -40.0
    keys[1, 0] = keys[1, 1] = 0.0
    first_of_third_tile = 2 * (64 if head_dim == 128 else 128)
    keys[first_of_third_tile, 0], keys[first_of_third_tile, 1] = 7.0, 40.0
    args = one_sequence_many_times(keys.to(dtype), values, 4, page)
    q = torch.zeros((4, 128, 1, head_dim))
    q[:, ::2, :, 0] = 1.0
    q[:, 1::2, :, 1] = 1.0
    out = pkg.attention_decode(q.to(dtype).cuda(), *args, softmax_scale=scale).cpu().double()
    pkg.check(torch.cuda.current_stream().cuda_stream)
    for rows, dim in ((slice(0, None, 2), 0), (slice(1, None, 2), 1)):
        p = torch.softmax(keys[:, dim].double() * scale, 0)
        want = p @ values.double()
        size = p[:, None] * values.double().abs()
        minor = size.sum(0) - size[first_of_third_tile]
        bound = eps * (want.abs() + minor) + 2.0 ** -13 * size.sum(0)
        err = (out[:, rows, 0] - want).abs()
        assert (err <= bound).all(), (dim, float((err / bound).max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("rows", [1, 128, 300])
@pytest.mark.parametrize("power", [20, 24.9, 25.3, 26, 26.6, 27, 27.5, 28, 31])
def test_scores_so_large_that_steps_of_fp32_are(pkg, rows, head_dim, dtype, power):
    """Scores of 2^20 to 2^31 (log2 units), where fp32 has steps of up to 256: keys with the largest share the weight, evenly,
    in one tile and across tiles, also where the maximum has grown from a key one step below."""
    n = 1 << 14
    keys, values = torch.zeros((n, head_dim)), torch.randn((n, head_dim), generator=torch.Generator().manual_seed(5)).to(dtype)
    top = [5, 9, 4000, 4001, 9000, 16000]
    keys[:, 0] = -8.0
    keys[2, 0] = 8.0 - 2.0 ** -4 if dtype == torch.bfloat16 else 8.0 - 2.0 ** -7
    keys[top, 0] = 8.0
    q = torch.zeros((4, rows, 1, head_dim))
    q[..., 0] = 8.0
    args = one_sequence_many_times(keys.to(dtype), values, 4)
    scale = 2.0 ** power / 64 * math.log(2.0)
    out, lse = (x.cpu() for x in pkg.attention_decode(q.to(dtype).cuda(), *args, softmax_scale=scale, return_lse=True))
    pkg.check(torch.cuda.current_stream().cuda_stream)
    want = values[top].double().mean(0)
    # P of the six is 1, 2^7 or 2^14; the output is rounded, and the join divides in fp32
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -20 * values[top].double().abs().mean(0)
    assert ((out.double() - want).abs() <= bound).all()
    assert float((lse.double() / (2.0 ** power * math.log(2.0)) - 1).abs().max()) <= 2.0 ** -15
