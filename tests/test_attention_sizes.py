"""Sizes of the attention calls without a GPU: scratch of very large blocks of queries and of problems beyond every limit."""
import ctypes as C

import pytest

from cuspamm_b200 import _lib

P = 1 << 20          # stands for a device address: 16-byte aligned, never read


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def problem(**change):
    a = _lib.SpammAttn()
    base = dict(dtype=0, batch=3, heads=8, kv_heads=2, dim=128, block=64, query_block=64, n_select=4, causal=1, max_q=100,
                tokens=250, scale=0.1, d_cu=P, d_lists=P, d_q=P, q_token=1024, q_head=128, d_k=P, k_token=256, k_head=128,
                d_v=P, v_token=256, v_head=128, d_o=P, o_token=1024, o_head=128, d_lse=P)
    for k, v in {**base, **change}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("max_q", [1, 2, 100, 8192])
def test_one_list_for_the_whole_sequence(lib, max_q):
    """A query block of 2^31 - 1 is one of max_q: the same scratch."""
    for n_select in (4, 40):
        sizes = []
        for query_block in (max_q, 2 ** 31 - 1):
            r = C.byref(problem(max_q=max_q, tokens=2 * max_q, query_block=query_block, n_select=n_select))
            sizes.append((lib.spamm_attn_select_scratch_bytes(r), lib.spamm_attn_forward_scratch_bytes(r),
                          lib.spamm_attn_backward_scratch_bytes(r)))
        assert sizes[0] == sizes[1]


@pytest.mark.parametrize("max_q", [2 ** 31 - 1, 2 ** 31 - 64])
def test_select_refuses_more_blocks_than_it_ranks_at_the_largest_bound(lib, max_q):
    r = C.byref(problem(max_q=max_q, query_block=2 ** 31 - 1))
    assert lib.spamm_attn_select_dev(r, None, 1, 0, P, P, 1 << 40, None) == 6
    assert b"16384" in lib.spamm_last_cuda_error()


@pytest.mark.parametrize("max_q,heads,kv_heads", [(1 << 26, 64, 1), (2 ** 31 - 1, 2, 1), (2 ** 31 - 1, 128, 1), (1 << 28, 16, 8)])
def test_backward_refuses_query_blocks_of_too_many_rows(lib, max_q, heads, kv_heads):
    """Query blocks of 2^28 rows and more (queries times heads of a key head), up to counts that pass 32 bits."""
    a = problem(max_q=max_q, query_block=2 ** 31 - 1, heads=heads, kv_heads=kv_heads, batch=1)
    r = C.byref(a)
    assert lib.spamm_attn_backward_scratch_bytes(r) == 0
    assert lib.spamm_attn_backward_dev(r, P, heads * 128, 128, P, P, P, P, 1 << 60, None) == 6
    assert lib.spamm_last_cuda_error().startswith(b"spamm_attn")
