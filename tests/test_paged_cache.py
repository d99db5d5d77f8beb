"""Refusals of flash_cache_append and flash_decode: status codes of the C ABI and the checks of the Python wrappers. No GPU."""
import ctypes

import pytest
import torch

P = 0x10000


def cache(pkg, **kw):
    fields = dict(k=P, v=P, page_stride=4 * 16 * 64, head_stride=16 * 64, token_stride=64, num_pages=10, page_size=16,
                  kv_heads=4, head_dim=64, dtype=pkg.FA_FP16, page_table=P, table_stride=5, max_pages=5, lengths=P,
                  counts=None)
    fields.update(kw)
    return pkg.PagedCacheStruct(**fields)


def rows(pkg, **kw):
    fields = dict(data=P, batch_stride=512, head_stride=64, token_stride=64)
    fields.update(kw)
    return pkg.RowsStruct(**fields)


def decode(pkg, c, q, batch=2, tokens=1, q_heads=8, o=P, lse=None, scale=0.0, slopes=None, ws=P, ws_bytes=1 << 40):
    return pkg.lib().flash_decode(c, q, o, lse, batch, tokens, q_heads, scale, -1, slopes, ws, ws_bytes, None)


def append(pkg, c, k, v, q=None, q_out=None, batch=2, tokens=1, q_heads=0, rotary=None, rotary_dim=0, positions=0):
    return pkg.lib().flash_cache_append(c, k, v, q, q_out, batch, tokens, q_heads, rotary, rotary_dim, positions, 0, None)


BAD_CACHES = [
    (dict(k=None), "INVALID"), (dict(v=None), "INVALID"), (dict(page_table=None), "INVALID"), (dict(lengths=None), "INVALID"),
    (dict(dtype=2), "UNSUPPORTED"), (dict(head_dim=96), "UNSUPPORTED"), (dict(kv_heads=0), "INVALID"),
    (dict(num_pages=0), "INVALID"), (dict(max_pages=0), "INVALID"), (dict(page_size=12), "UNSUPPORTED"),
    (dict(page_size=0), "UNSUPPORTED"), (dict(page_size=-8), "UNSUPPORTED"),
    (dict(max_pages=1 << 28, table_stride=1 << 28), "INVALID"), (dict(table_stride=4), "INVALID"),
    (dict(k=P + 8), "INVALID"), (dict(page_table=P + 2), "INVALID"), (dict(counts=P + 1), "INVALID"),
    (dict(page_stride=1020), "INVALID"), (dict(token_stride=32), "INVALID"), (dict(head_stride=-1024), "INVALID"),
    (dict(kv_heads=3), "INVALID"),
]


@pytest.mark.parametrize("change,status", BAD_CACHES, ids=[str(c) for c, _ in BAD_CACHES])
def test_bad_caches(pkg, change, status):
    want = {"INVALID": pkg.FA_INVALID_ARG, "UNSUPPORTED": pkg.FA_UNSUPPORTED}[status]
    c, r = cache(pkg, **change), rows(pkg)
    assert decode(pkg, c, r) == want
    assert pkg.lib().flash_forward_last_error()
    if "kv_heads" not in change or change["kv_heads"] == 0:
        assert append(pkg, c, r, r) == want


def test_bad_arguments(pkg):
    c, r, bad = cache(pkg), rows(pkg), pkg.FA_INVALID_ARG
    assert decode(pkg, None, r) == bad and append(pkg, None, r, r) == bad
    for q in (None, rows(pkg, data=None), rows(pkg, data=P + 4), rows(pkg, batch_stride=-8), rows(pkg, head_stride=60)):
        assert decode(pkg, c, q) == bad
        assert append(pkg, c, q, r) == bad and append(pkg, c, r, q) == bad
    for kw in (dict(batch=0), dict(tokens=0), dict(tokens=-1), dict(q_heads=0), dict(q_heads=7), dict(o=None), dict(o=P + 2),
               dict(lse=P + 2), dict(slopes=P + 1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-35),
               dict(ws=None), dict(ws_bytes=100), dict(ws=P + 4), dict(batch=2 ** 30, q_heads=8)):
        assert decode(pkg, c, r, **kw) == bad, kw
    for kw in (dict(q=r), dict(q=r, q_out=P), dict(q_out=P), dict(q_heads=8), dict(q=r, q_out=P, q_heads=8),
               dict(rotary=P, rotary_dim=64), dict(rotary=P + 4, rotary_dim=64, positions=9), dict(batch=0), dict(tokens=0),
               dict(q=r, q_out=P + 8, q_heads=8, rotary=P, rotary_dim=64, positions=9),
               dict(batch=2 ** 31 - 1, tokens=2 ** 31 - 1)):
        assert append(pkg, c, r, r, **kw) == bad, kw
    for dim in (8, 24, 80, -16):
        assert append(pkg, c, r, r, rotary=P, rotary_dim=dim, positions=9) == pkg.FA_UNSUPPORTED


def test_workspace_bytes(pkg):
    size = pkg.lib().flash_decode_workspace_bytes
    assert size(1, 32, 8, 128) == 296 * 2 * 16 * 130 * 4
    assert size(4, 32, 8, 64) == size(1, 16, 1, 64) == 296 * 2 * 16 * 66 * 4
    assert size(1, 17, 1, 64) == 148 * 2 * 32 * 66 * 4 and size(1, 33, 1, 64) == size(8, 8, 1, 64) == 148 * 2 * 64 * 66 * 4
    assert size(65, 1, 1, 64) == size(100, 8, 1, 64) == 148 * 2 * 128 * 66 * 4
    assert size(0, 8, 8, 64) == size(1, 8, 3, 64) == size(1, 8, 0, 64) == 0


def test_no_gpu_is_an_error(pkg):
    if torch.cuda.is_available():
        pytest.skip("this check is for machines without a GPU")
    c, r = cache(pkg), rows(pkg)
    assert decode(pkg, c, r) in (pkg.FA_CUDA_ERROR, pkg.FA_UNSUPPORTED)
    assert append(pkg, c, r, r) in (pkg.FA_CUDA_ERROR, pkg.FA_UNSUPPORTED)


class Fake:
    """Looks enough like a CUDA tensor for the wrappers' checks."""

    def __init__(self, shape, dtype, device=0, stride=None):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device("cpu")
        self.is_cuda, self._device = True, device
        self._stride = torch.empty(shape, device="meta").stride() if stride is None else stride

    def get_device(self):
        return self._device

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self, i=None):
        return self._stride if i is None else self._stride[i]

    def is_contiguous(self):
        return self._stride == torch.empty(self.shape, device="meta").stride()

    def data_ptr(self):
        return P


def test_wrappers_refuse_what_does_not_fit(pkg):
    half, i32 = torch.float16, torch.int32
    good = dict(k_pages=Fake((9, 2, 16, 64), half), v_pages=Fake((9, 2, 16, 64), half), page_table=Fake((3, 4), i32),
                lengths=Fake((3,), i32), counts=None)
    q, k = Fake((3, 4, 2, 64), half), Fake((3, 2, 2, 64), half)
    wrong = [
        dict(k_pages=Fake((9, 2, 16, 64), torch.float32)), dict(k_pages=torch.zeros((9, 2, 16, 64), dtype=half)),
        dict(v_pages=Fake((8, 2, 16, 64), half)), dict(v_pages=Fake((9, 2, 16, 64), half, device=1)),
        dict(v_pages=Fake((9, 2, 16, 64), half, stride=(2048, 64, 128, 1))),
        dict(page_table=Fake((2, 4), i32)), dict(page_table=Fake((3, 4), torch.int64)),
        dict(page_table=Fake((3, 4), i32, stride=(1, 3))), dict(page_table=Fake((12,), i32)),
        dict(lengths=Fake((4,), i32)), dict(lengths=Fake((3,), torch.int64)), dict(lengths=Fake((3,), i32, device=1)),
        dict(lengths=Fake((3,), i32, stride=(2,))), dict(counts=Fake((2,), i32)), dict(counts=Fake((3,), half)),
    ]
    for change in wrong:
        args = {**good, **change}
        with pytest.raises(AssertionError):
            pkg.attention_decode(q, **args)
        with pytest.raises(AssertionError):
            pkg.cache_append(k, k, **args)
    for bad_q in (Fake((3, 4, 2, 128), half), Fake((3, 4, 64), half), Fake((3, 4, 2, 64), torch.bfloat16),
                  Fake((3, 4, 2, 64), half, stride=(512, 128, 1, 2)), Fake((3, 4, 2, 64), half, device=1)):
        with pytest.raises(AssertionError):
            pkg.attention_decode(bad_q, **good)
        with pytest.raises(AssertionError):
            pkg.cache_append(k, k, q=bad_q, rotary=Fake((9, 64), torch.float32), **good)
    for bad_k in (Fake((3, 4, 2, 64), half), Fake((3, 2, 2, 64), torch.bfloat16), Fake((3, 2, 2, 128), half)):
        with pytest.raises(AssertionError):
            pkg.cache_append(bad_k, k, **good)
        with pytest.raises(AssertionError):
            pkg.cache_append(k, bad_k, **good)
    with pytest.raises(AssertionError):
        pkg.cache_append(k, k, rotary=Fake((9, 64), half), **good)
    with pytest.raises(AssertionError):
        pkg.cache_append(k, k, q_out=q, **good)
    with pytest.raises(AssertionError):
        pkg.cache_append(k, k, q=q, rotary=Fake((9, 64), torch.float32), q_out=Fake((3, 4, 1, 64), half), **good)
    with pytest.raises(AssertionError):
        pkg.attention_decode(q, out=Fake((3, 2, 4, 64), half), **good)
    with pytest.raises(AssertionError):
        pkg.attention_decode(q, alibi_slopes=Fake((3,), torch.float32), **good)
