"""Shared batches at the sizes where sharing ends, without a GPU (no kernel is
launched on these paths)."""
import ctypes

import pytest

from test_paged_refusals import attention, batch


@pytest.fixture(scope="module")
def L():
    from adaptiveimi_amd import _lib

    return _lib.lib()


def workspace(L, a):
    need = ctypes.c_size_t()
    assert L.imi_paged_attention_workspace_size(ctypes.byref(a), ctypes.byref(need)) == 0, L.imi_last_error().decode()
    return need.value


@pytest.mark.parametrize("n_seqs,kv_heads,shares", [(1 << 19, 8, True), ((1 << 19) + 1, 8, False), (1 << 22, 1, True),
                                                    ((1 << 22) + 1, 1, False), (1 << 24, 8, False)])
def test_more_sequences_than_the_join_takes(L, n_seqs, kv_heads, shares):
    """Past 2^22 pairs of a sequence and a KV head nothing is attended together: the
    call is the one without, with its workspace, instead of one that is refused when
    some of its kernels have been launched."""
    found = dict(shared=256, members=256, leaders=256, saved=256, share_bytes=1)
    size = lambda **b: workspace(L, attention(batch(n_seqs=n_seqs, n_tokens=n_seqs, max_query=1, n_pages=1 << 24, **b),
                                              kv_heads=kv_heads, groups=1))
    assert (size(**found) > size()) == shares and (size(**found) == size()) != shares
