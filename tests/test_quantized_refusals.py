"""What the entry points of pools in 8 and 4 bits and of shared pages refuse,
without a GPU (no kernel is launched on these paths)."""
import ctypes

import pytest
import torch

from test_paged_refusals import attention, batch


@pytest.fixture(scope="module")
def L():
    from adaptiveimi_amd import _lib

    return _lib.lib()


CODES = dict(format=1, key_exponents=256, value_exponents=256, exponent_page_stride=512, exponent_head_stride=64,
             exponent_row_stride=4)


def read(b=None, **over):
    from adaptiveimi_amd._lib import ReadPagesArgs

    a = ReadPagesArgs(batch=b or batch(), dtype=0, kv_heads=8, dim=128, key_pages=256, value_pages=256,
                      page_stride=16384, head_stride=2048, row_stride=128, rows=10, keys=256, values=256,
                      out_seq_stride=10240, out_head_stride=1280, out_row_stride=128)
    for k, v in over.items():
        setattr(a, k, v)
    return a


BAD_CODES = [
    (dict(format=4), 3, "format"),
    (dict(format=-1), 3, "format"),
    (dict(key_exponents=None), 1, "null exponents"),
    (dict(value_exponents=None), 1, "null exponents"),
    (dict(row_stride=120), 1, "16 bytes"),
    (dict(page_stride=16384 + 8), 1, "16 bytes"),
    (dict(exponent_row_stride=6), 1, "exponents must be multiples of 4"),
    (dict(exponent_head_stride=-4), 1, "exponents must be multiples of 4"),
    (dict(key_exponents=258), 1, "aligned to 4"),
    (dict(exponent_page_stride=1 << 33), 3, "2^32"),
    (dict(exponent_row_stride=1 << 30), 3, "2^32"),
]


@pytest.mark.parametrize("over,code,text", BAD_CODES)
def test_formats_refused(L, over, code, text):
    need = ctypes.c_size_t()
    a = attention(**{**CODES, **over})
    assert L.imi_paged_attention_workspace_size(ctypes.byref(a), ctypes.byref(need)) == code
    assert text in L.imi_last_error().decode()
    assert L.imi_paged_attention(ctypes.byref(a), None) == code
    assert L.imi_read_pages(ctypes.byref(read(**{**CODES, **over})), None) == code
    assert text in L.imi_last_error().decode()


def test_formats_refused_when_storing(L):
    from adaptiveimi_amd._lib import QkNormRopeArgs

    for over, code, text in BAD_CODES:
        a = QkNormRopeArgs(batch=batch(), dtype=0, query_heads=32, kv_heads=8, dim=128, query=256,
                           query_token_stride=4096, query_head_stride=128, key=256, key_token_stride=1024,
                           key_head_stride=128, value=256, value_token_stride=1024, value_head_stride=128, eps=1e-6,
                           query_out=256, query_out_token_stride=4096, query_out_head_stride=128, key_pages=256,
                           value_pages=256, page_stride=16384, head_stride=2048, row_stride=128)
        for k, v in {**CODES, **over}.items():
            setattr(a, k, v)
        assert L.imi_qk_norm_rope(ctypes.byref(a), None) == code, over
        assert text in L.imi_last_error().decode()


@pytest.mark.parametrize("over,b,code,text", [
    (dict(dtype=2), {}, 3, "dtype"),
    (dict(dim=96), {}, 3, "dim=96"),
    (dict(kv_heads=0), {}, 1, "heads"),
    (dict(rows=-1), {}, 1, "rows"),
    (dict(keys=None), {}, 1, "null"),
    (dict(values=264), {}, 1, "aligned"),
    (dict(out_row_stride=129), {}, 1, "strides"),
    (dict(rows=1 << 30), {}, 3, "too many rows"),
    ({}, dict(n_seqs=-1), 1, "negative"),
    ({}, dict(lens=None), 1, "null"),
    ({}, dict(page_size=24), 3, "power of two"),
    ({}, dict(n_pages=0), 1, "n_pages"),
    ({}, dict(page_table=None, n_pages=1), 1, "no page table"),
])
def test_read_pages_refuses(L, over, b, code, text):
    assert L.imi_read_pages(ctypes.byref(read(batch(**b), **over)), None) == code
    assert text in L.imi_last_error().decode()


def test_read_pages_of_nothing(L):
    assert L.imi_read_pages(ctypes.byref(read(batch(n_seqs=0), keys=None)), None) == 0
    assert L.imi_read_pages(ctypes.byref(read(rows=0, keys=None)), None) == 0
    # the new tokens are not looked at
    assert L.imi_read_pages(ctypes.byref(read(batch(n_tokens=0, max_query=0, query_start=None), rows=0)), None) == 0


def test_share_prefixes_refuses(L):
    need = ctypes.c_size_t()
    size = lambda b: L.imi_share_prefixes_workspace_size(ctypes.byref(b), ctypes.byref(need))
    share = lambda b, *a: L.imi_share_prefixes(ctypes.byref(b), None, *a, None)
    for over, code, text in ((dict(n_seqs=-1), 1, "negative"), (dict(page_table=None, n_pages=2), 1, "no"),
                             (dict(page_size=0), 1, "page_size"), (dict(page_size=24), 3, "power of two"),
                             (dict(table_stride=3), 1, "table_stride"), (dict(lens=None), 1, "null"),
                             (dict(query_start=None), 1, "null")):
        assert size(batch(**over)) == code, over
        assert share(batch(**over), 256, 256, 256, 256, 256, 8) == code
    assert size(batch(n_tokens=0, n_pages=0, max_query=0)) == 0 and need.value == 8
    for i in range(4):
        assert share(batch(), *[None if k == i else 256 for k in range(4)], 256, 8) == 1
    assert share(batch(), 256, 256, 256, 256, 256, 7) == 4 and share(batch(), 256, 256, 256, 256, None, 8) == 4
    assert share(batch(n_seqs=0), None, None, None, None, None, 0) == 0


def test_shared_goes_with_members(L):
    need = ctypes.c_size_t()
    size = lambda **b: L.imi_paged_attention_workspace_size(ctypes.byref(attention(batch(**b))), ctypes.byref(need))
    assert size(shared=256) == 1 and size(members=256) == 1 and size(shared=256, members=256, leaders=256) == 1
    assert size(shared=256, members=256, leaders=256, saved=256, share_bytes=-1) == 1
    assert size() == 0
    plain = need.value
    found = dict(shared=256, members=256, leaders=256, saved=256)
    assert size(**found, share_bytes=1) == 0 and need.value > plain
    # 100 pages cannot save what sharing costs
    assert size(**found) == 0 and need.value == plain
    assert size(**found, share_bytes=1 << 62) == 0 and need.value == plain
    # a window hides some of the common rows: nothing is attended together
    sizes = []
    for b in (batch(**found, share_bytes=1), batch()):
        a = attention(b, window=64)
        assert L.imi_paged_attention_workspace_size(ctypes.byref(a), ctypes.byref(need)) == 0
        sizes.append(need.value)
    assert sizes[0] == sizes[1]


def test_quantized_pages_refuses():
    from adaptiveimi_amd import ops

    codes, exps = torch.zeros((4, 2, 8, 64), dtype=torch.int8), torch.zeros((4, 2, 8, 2), dtype=torch.uint8)
    assert ops.QuantizedPages(codes, exps).format == 2
    assert ops.QuantizedPages(codes[..., :32].contiguous().view(torch.uint8), exps).format == 3
    assert ops.QuantizedPages.zeros(4, 2, 8, 64, "fp8", "cpu").codes.dtype is torch.float8_e4m3fn
    for bad in ((codes.float(), exps), (codes, exps.int()), (codes[0], exps[0])):
        with pytest.raises((TypeError, ValueError)):
            ops.QuantizedPages(*bad)
    for bad in ((codes, exps[:3]), (codes, exps[..., :1]), (codes.view(torch.uint8), exps),
                (torch.zeros((4, 2, 64, 8), dtype=torch.int8).transpose(2, 3), exps)):
        with pytest.raises(ValueError):
            ops.QuantizedPages(*bad)
    for kw in (dict(format="fp6"), dict(dim=48)):
        with pytest.raises(ValueError):
            ops.QuantizedPages.zeros(**{**dict(n_pages=4, kv_heads=2, page_size=8, dim=64, format="fp8",
                                               device="cpu"), **kw})
