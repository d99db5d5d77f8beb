"""attention_backward, cache_append and attention_decode answered natively (host/torch_binding.cpp) and by the Python code: the
same results, the same refusals."""
import math

import pytest
import torch

import paged_cache_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture
def python_code(pkg, monkeypatch):
    """Switches the native answers off."""
    def off():
        monkeypatch.setattr(pkg, "_native_operators", 3 * (lambda *a: NotImplemented,))
    return off


def calls(pkg):
    b = oracle.Batch(1, [40, 17], [2, 1], 2, 2, 64, 16, "bf16")
    q, k = b.rows(4).cuda(), b.rows(2).cuda()
    slopes, rotary = torch.tensor([0.1, 0.2, 0.3, 0.4]).cuda(), oracle.angles(64, 32).cuda()
    args, counts = b.cuda(), b.cuda_counts()
    x = [torch.randn((1, 4, 100, 64), device="cuda").half() for _ in range(4)]
    out, lse = pkg.attention_forward(*x[:3], causal=True, alibi_slopes=slopes, return_lse=True)
    return [
        lambda: pkg.cache_append(k, k, *args, counts=counts, q=q, rotary=rotary, interleaved=True),
        lambda: pkg.cache_append(k, k, *args, q=q, rotary=rotary, q_out=torch.zeros_like(q, memory_format=torch.contiguous_format)),
        lambda: (pkg.cache_append(k, k, *args), args[0].clone(), args[1].clone()),
        lambda: pkg.attention_decode(q, *args, counts=counts, softmax_scale=0.2, window_left=9, alibi_slopes=slopes,
                                     return_lse=True),
        lambda: pkg.attention_decode(q, *args, out=torch.zeros((2, 4, 2, 64), device="cuda").bfloat16()),
        lambda: pkg.attention_backward(*x[:3], out, lse, x[3], causal=True, alibi_slopes=slopes),
        lambda: pkg.attention_backward(*x[:3], out, lse, x[3], causal=True, window_left=5, softmax_scale=0.1,
                                       alibi_slopes=slopes, dlse=torch.ones_like(lse), dk=torch.zeros_like(x[0])),
    ]


def flat(r):
    return [r] if isinstance(r, torch.Tensor) else [x for x in r if x is not None]


def test_the_native_answer_is_the_python_codes(pkg, python_code):
    assert all(type(f).__name__ == "builtin_function_or_method" for f in pkg._native_operators), "the binding was not built"
    todo = calls(pkg)
    native = [flat(f()) for f in todo]
    python_code()
    for f, want in zip(todo, native):
        got = flat(f())
        assert len(got) == len(want)
        assert all(torch.equal(x, y) and x.dtype == y.dtype and x.stride() == y.stride() for x, y in zip(got, want))
    pkg.check(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("off", [False, True])
def test_refusals_are_the_same(pkg, python_code, off):
    if off:
        python_code()
    b = oracle.Batch(2, [40, 17], [1, 1], 1, 2, 64, 16, "fp16")
    q, k, (k_pages, v_pages, table, lengths) = b.rows(4).cuda(), b.rows(2).cuda(), b.cuda()
    for bad in ((q.float(), k_pages, v_pages, table, lengths), (q, k_pages, v_pages[:1], table, lengths),
                (q, k_pages, v_pages, table.long(), lengths), (q, k_pages, v_pages, table, lengths[:1]),
                (q, k_pages, v_pages, table, lengths.cpu()), (q[:1], k_pages, v_pages, table, lengths),
                (q, k_pages.float(), v_pages.float(), table, lengths)):
        with pytest.raises(AssertionError):
            pkg.attention_decode(*bad)
        with pytest.raises(AssertionError):
            pkg.cache_append(bad[0][:, :2], k, *bad[1:])
    with pytest.raises(pkg.FlashForwardError) as e:
        pkg.attention_decode(q[:, :3], k_pages, v_pages, table, lengths)
    assert e.value.code == pkg.FA_INVALID_ARG
    with pytest.raises(pkg.FlashForwardError):
        pkg.attention_decode(q, k_pages, v_pages, table, lengths, softmax_scale=math.nan)
    with pytest.raises(pkg.FlashForwardError):
        pkg.cache_append(k, k, k_pages, v_pages, table, lengths, rotary=torch.zeros((64, 24), device="cuda"))
    x = torch.zeros((1, 2, 64, 96), device="cuda").half()
    lse = torch.zeros((1, 2, 64), device="cuda")
    with pytest.raises(pkg.FlashForwardError) as e:
        pkg.attention_backward(x, x, x, x, lse, x)
    assert e.value.code == pkg.FA_UNSUPPORTED
    for args in ((x, x, x, x, lse[..., :1], x), (x, x, x, x.float(), lse, x), (x, x[:, :1], x, x, lse, x),
                 (x.cpu(), x, x, x, lse, x)):
        with pytest.raises(AssertionError):
            pkg.attention_backward(*args)
