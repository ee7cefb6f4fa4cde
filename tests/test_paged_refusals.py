"""What the paged cache's entry points refuse, without a GPU: the checks of
the C ABI (no kernel is launched on these paths) and of the Python layer."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def L():
    from adaptiveimi_amd import _lib

    return _lib.lib()


def batch(**over):
    from adaptiveimi_amd._lib import PagedBatchArgs

    b = PagedBatchArgs(page_table=256, table_stride=64, max_pages=64, n_pages=100, page_size=16, lens=256,
                       query_start=256, n_seqs=2, n_tokens=40, max_query=20)
    for k, v in over.items():
        setattr(b, k, v)
    return b


def attention(b=None, **over):
    from adaptiveimi_amd._lib import PagedAttentionArgs

    a = PagedAttentionArgs(batch=b or batch(), dtype=0, kv_heads=8, groups=4, dim=128, query=256,
                           query_token_stride=4096, query_head_stride=128, keys=256, values=256, page_stride=16384,
                           head_stride=2048, row_stride=128, scale=0.1, out=256, out_token_stride=4096,
                           out_head_stride=128)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,b,code,text", [
    (dict(dtype=2), {}, 3, "dtype"),
    (dict(dim=96), {}, 3, "dim=96"),
    (dict(kv_heads=0), {}, 1, "heads"),
    (dict(groups=0), {}, 1, "heads"),
    (dict(window=-1), {}, 1, "window"),
    (dict(sinks=-1), {}, 1, "sinks"),
    (dict(scale=0.0), {}, 1, "scale"),
    (dict(scale=-1.0), {}, 1, "scale"),
    (dict(scale=float("nan")), {}, 1, "scale"),
    (dict(scale=float("inf")), {}, 1, "scale"),
    (dict(query=None), {}, 1, "null"),
    (dict(keys=264), {}, 1, "aligned"),
    (dict(row_stride=129), {}, 1, "strides"),
    (dict(page_stride=-8), {}, 1, "strides"),
    ({}, dict(n_seqs=-1), 1, "negative"),
    ({}, dict(max_query=0), 1, "max_query"),
    ({}, dict(page_size=0), 1, "page_size"),
    ({}, dict(page_size=24), 3, "power of two"),
    ({}, dict(n_pages=0), 1, "n_pages"),
    ({}, dict(table_stride=63), 1, "table_stride"),
    ({}, dict(lens=None), 1, "null"),
    ({}, dict(page_table=None, n_pages=1), 1, "no page table"),
    ({}, dict(max_pages=1 << 27, table_stride=1 << 27), 3, "2^30"),
])
def test_attention_refuses(L, over, b, code, text):
    a = attention(batch(**b), **over)
    need = ctypes.c_size_t()
    assert L.imi_paged_attention_workspace_size(ctypes.byref(a), ctypes.byref(need)) == code
    assert text in L.imi_last_error().decode()
    assert L.imi_paged_attention(ctypes.byref(a), None) == code


def test_attention_workspace(L):
    need = ctypes.c_size_t()
    a = attention()
    assert L.imi_paged_attention_workspace_size(ctypes.byref(a), ctypes.byref(need)) == 0 and need.value > 0
    a.workspace, a.workspace_bytes = 256, need.value - 1
    assert L.imi_paged_attention(ctypes.byref(a), None) == 4
    # nothing to do: no workspace, no launch
    for b in (batch(n_seqs=0), batch(n_tokens=0)):
        a = attention(b, query=None)
        assert L.imi_paged_attention_workspace_size(ctypes.byref(a), ctypes.byref(need)) == 0 and need.value == 0
        assert L.imi_paged_attention(ctypes.byref(a), None) == 0


def norm(b=None, **over):
    from adaptiveimi_amd._lib import QkNormRopeArgs

    a = QkNormRopeArgs(batch=b or batch(), dtype=0, query_heads=8, kv_heads=2, dim=128, query=256,
                       query_token_stride=1536, query_head_stride=128, key=256, key_token_stride=1536,
                       key_head_stride=128, value=256, value_token_stride=1536, value_head_stride=128, inv_freq=256,
                       rotary=128, eps=1e-6, query_out=256, query_out_token_stride=1024, query_out_head_stride=128,
                       key_pages=256, value_pages=256, page_stride=4096, head_stride=2048, row_stride=128)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,b,code,text", [
    (dict(dtype=7), {}, 3, "dtype"),
    (dict(dim=80), {}, 3, "dim=80"),
    (dict(rotary=24), {}, 3, "rotary"),
    (dict(rotary=144), {}, 3, "rotary"),
    (dict(inv_freq=None), {}, 1, "inv_freq"),
    (dict(eps=-1.0), {}, 1, "eps"),
    (dict(eps=float("nan")), {}, 1, "eps"),
    (dict(query_heads=-1), {}, 1, "heads"),
    (dict(key_pages=None), {}, 1, "positions"),
    (dict(value=None), {}, 1, "null"),
    (dict(query_out=None), {}, 1, "null"),
    (dict(key=260), {}, 1, "aligned"),
    (dict(key_token_stride=1535), {}, 1, "strides"),
    ({}, dict(n_tokens=-1), 1, "n_tokens"),
    ({}, dict(page_size=12), 3, "power of two"),
])
def test_norm_refuses(L, over, b, code, text):
    a = norm(batch(**b), **over)
    assert L.imi_qk_norm_rope(ctypes.byref(a), None) == code
    assert text in L.imi_last_error().decode()


def table(**over):
    from adaptiveimi_amd._lib import PageTableArgs

    t = PageTableArgs(pages=256, stride=8, lens=512, refs=1024, n_seqs=4, max_pages=8, n_pages=32, page_size=16)
    for k, v in over.items():
        setattr(t, k, v)
    return t


def test_page_tables_refuse(L):
    from adaptiveimi_amd._lib import PagePool

    ref = ctypes.byref
    other = dict(pages=2256, lens=2512, refs=3024)
    for over, code, text in ((dict(page_size=0), 1, "page_size"), (dict(stride=7), 1, "stride"),
                             (dict(n_seqs=-1), 1, "negative"), (dict(refs=None), 1, "refs"),
                             (dict(lens=None), 1, "null"), (dict(max_pages=1 << 28, stride=1 << 28), 3, "2^31")):
        need = ctypes.c_size_t()
        for call in (lambda t: L.imi_extend_pages_workspace_size(ref(t), ref(need)),
                     lambda t: L.imi_compact_pages_workspace_size(ref(t), ref(need)),
                     lambda t: L.imi_fork_pages(ref(t), 256, ref(table(**other)), None),
                     lambda t: L.imi_extend_pages(ref(t), 256, 256, None, 0, 256, 1 << 20, None),
                     lambda t: L.imi_compact_pages(ref(t), 256, None, 0, 256, 1 << 20, None)):
            assert call(table(**over)) == code
            assert text in L.imi_last_error().decode()
    assert L.imi_fork_pages(ref(table()), 256, ref(table()), None) == 1
    assert "out must not be in" in L.imi_last_error().decode()
    assert L.imi_fork_pages(ref(table()), 256, ref(table(n_pages=31, **other)), None) == 1
    assert "differ" in L.imi_last_error().decode()
    assert L.imi_fork_pages(ref(table()), None, ref(table(**other)), None) == 1
    need = ctypes.c_size_t()
    assert L.imi_extend_pages_workspace_size(ref(table()), ref(need)) == 0
    assert L.imi_extend_pages(ref(table()), 256, 256, None, 0, 256, need.value - 1, None) == 4
    assert L.imi_compact_pages_workspace_size(ref(table()), ref(need)) == 0
    assert L.imi_compact_pages(ref(table()), 256, None, 0, 256, need.value - 1, None) == 4
    for pool in ((0, 64, 64), (264, 64, 64), (256, 48, 64), (256, 64, 8), (256, 72, 64), (256, 64, 0)):
        pools = (PagePool * 1)(PagePool(*pool))
        assert L.imi_extend_pages(ref(table()), 256, 256, pools, 1, 256, 1 << 20, None) == 1
        assert L.imi_compact_pages(ref(table()), 256, pools, 1, 256, 1 << 20, None) == 1
        assert "pool 0" in L.imi_last_error().decode()


def test_python_layer_refuses_host_tensors():
    import torch

    from adaptiveimi_amd import ops

    i32 = torch.zeros((2,), dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        ops.PagedBatch(None, i32, torch.zeros((3,), dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="HIP device"):
        ops.PageTable(torch.zeros((2, 4), dtype=torch.int32), i32, i32, 16)
    x = torch.zeros((2, 1, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="HIP device"):
        ops.qk_norm_rope(x, x, positions=i32)


def test_sizes_past_the_kernels_indexes(L):
    """Counts that 32-bit indexes of the kernels would not hold are refused."""
    ref = ctypes.byref
    need = ctypes.c_size_t()
    for over in (dict(n_seqs=(1 << 30) + 1), dict(n_tokens=(1 << 30) + 1)):
        a = attention(batch(**over))
        assert L.imi_paged_attention_workspace_size(ref(a), ref(need)) == 3
        assert "2^30" in L.imi_last_error().decode()
        assert L.imi_qk_norm_rope(ref(norm(batch(**over))), None) == 3
    long = dict(max_pages=1 << 27, table_stride=1 << 27)
    assert L.imi_qk_norm_rope(ref(norm(batch(**long))), None) == 3
    assert "2^30" in L.imi_last_error().decode()
    a = attention(batch(n_seqs=1 << 28, max_pages=1 << 20, table_stride=1 << 20), kv_heads=1024, groups=1)
    assert L.imi_paged_attention_workspace_size(ref(a), ref(need)) == 3
    assert "too much work" in L.imi_last_error().decode()
    for over in (dict(n_pages=(1 << 30) + 1), dict(n_seqs=(1 << 30) + 1), dict(max_pages=1, page_size=(1 << 31) - 1)):
        assert L.imi_compact_pages_workspace_size(ref(table(**over)), ref(need)) == 3


def test_attention_splits_more_heads_than_a_launch_has_workgroups(L):
    """Short sequences take a workgroup per (sequence, head) and no workspace,
    as long as a launch can hold them."""
    need = ctypes.c_size_t()
    short = dict(max_pages=2, table_stride=2, max_query=1)
    for n, shared in ((1 << 19, False), ((1 << 19) + 1, True)):
        a = attention(batch(n_seqs=n, n_tokens=n, **short))
        assert L.imi_paged_attention_workspace_size(ctypes.byref(a), ctypes.byref(need)) == 0
        assert (need.value > 0) == shared


def test_c_ints_are_not_taken_modulo():
    from adaptiveimi_amd import ops

    for x in (0, 1, -1, 2 ** 31 - 1, -2 ** 31):
        assert ctypes.c_int32(ops._c_int(x)).value == x
    for x in (2 ** 31, 2 ** 32 + 5, 2 ** 64):
        assert ctypes.c_int32(ops._c_int(x)).value == 2 ** 31 - 1
        assert ctypes.c_int32(ops._c_int(-x + 5 if x > 2 ** 31 else -x - 1)).value == -2 ** 31
