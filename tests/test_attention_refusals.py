"""What the attention operators refuse, without a GPU: the C entry points check their arguments before they touch CUDA,
the Python calls check shapes, types and numbers before anything is queued."""
import ctypes as C

import pytest
import torch

from cuspamm_b200 import _lib

P = 1 << 20          # stands for a device address: 16-byte aligned, never read


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def problem(**change):
    a = _lib.SpammAttn()
    base = dict(dtype=0, batch=2, heads=8, kv_heads=2, dim=128, block=64, query_block=64, n_select=4, causal=1, max_q=100,
                tokens=150, scale=0.1, d_cu=P, d_lists=P, d_q=P, q_token=1024, q_head=128, d_k=P, k_token=256, k_head=128,
                d_v=P, v_token=256, v_head=128, d_o=P, o_token=1024, o_head=128, d_lse=P)
    for k, v in {**base, **change}.items():
        setattr(a, k, v)
    return a


PAGED = dict(n_pages=9, table_width=4, table_stride=4, d_table=P, d_lengths=P, d_status=P)
WRONG = [dict(dtype=2), dict(dim=96), dict(block=48), dict(block=0), dict(kv_heads=3), dict(kv_heads=0), dict(heads=258),
         dict(query_block=0), dict(n_select=-1), dict(n_select=1025), dict(batch=-1), dict(tokens=-1), dict(max_q=-1),
         dict(d_cu=None)]
WRONG_PAGED = [dict(d_table=None), dict(d_lengths=None), dict(d_status=None), dict(table_stride=3), dict(n_pages=-1),
               dict(table_width=-1), dict(table_width=1 << 30, table_stride=1 << 30)]


@pytest.mark.parametrize("change", WRONG + [{**PAGED, **w} for w in WRONG_PAGED])
def test_every_entry_point_refuses(lib, change):
    a = problem(**change)
    r = C.byref(a)
    assert lib.spamm_attn_forward_dev(r, P, 1 << 40, None) == 1
    assert lib.spamm_attn_select_dev(r, P, 0, 0, P, P, 1 << 40, None) == 1
    assert lib.spamm_attn_append_dev(r, P, P, P, None, 0, 0, None) == 1
    assert lib.spamm_attn_backward_dev(r, P, 1024, 128, P, P, P, P, 1 << 40, None) == 1
    assert lib.spamm_attn_forward_scratch_bytes(r) == 0
    assert lib.spamm_last_cuda_error().startswith(b"spamm_attn")


def test_null_problem(lib):
    assert lib.spamm_attn_forward_dev(None, None, 0, None) == 1
    assert lib.spamm_attn_select_dev(None, None, 0, 0, None, None, 0, None) == 1
    assert lib.spamm_attn_append_dev(None, None, None, None, None, 0, 0, None) == 1
    assert lib.spamm_attn_backward_dev(None, None, 0, 0, None, None, None, None, 0, None) == 1


@pytest.mark.parametrize("change", [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                                    dict(d_lists=None), dict(d_q=None), dict(d_q=P + 2), dict(q_token=1028), dict(k_head=4),
                                    dict(d_v=None), dict(d_o=P + 8), dict(o_head=129)])
def test_forward_and_backward_refuse_rows_and_scales(lib, change):
    r = C.byref(problem(**change))
    assert lib.spamm_attn_forward_dev(r, P, 1 << 40, None) == 1
    assert lib.spamm_attn_backward_dev(r, P, 1024, 128, P, P, P, P, 1 << 40, None) == 1


def test_backward_refuses(lib):
    r = C.byref(problem())
    ok = (r, P, 1024, 128, P, P, P, P)
    need = lib.spamm_attn_backward_scratch_bytes(r)
    assert need > 0
    assert lib.spamm_attn_backward_dev(*ok, need - 1, None) == 1                     # scratch too small
    assert lib.spamm_attn_backward_dev(r, P + 4, 1024, 128, P, P, P, P, need, None) == 1
    assert lib.spamm_attn_backward_dev(r, P, 1023, 128, P, P, P, P, need, None) == 1
    assert lib.spamm_attn_backward_dev(r, P, 1024, 128, P, None, P, P, need, None) == 1
    for wrong in (dict(n_select=0), PAGED, dict(d_lse=None)):
        assert lib.spamm_attn_backward_dev(C.byref(problem(**wrong)), P, 1024, 128, P, P, P, P, 1 << 40, None) == 1


def test_select_refuses(lib):
    r = C.byref(problem(n_select=8))
    need = lib.spamm_attn_select_scratch_bytes(r)
    assert need > 0
    for first, local in ((-1, 0), (0, -1), (9, 0), (1, 7), (7, 1)):                  # 1 + 7 + (64 + 64 - 2) // 64 > 8
        assert lib.spamm_attn_select_dev(r, None, first, local, P, P, need, None) == 1
    assert lib.spamm_attn_select_dev(r, None, 1, 1, None, P, need, None) == 1
    assert lib.spamm_attn_select_dev(r, None, 1, 1, P, P, need - 1, None) == 1
    assert lib.spamm_attn_select_dev(r, None, 1, 1, P, P + 4, need, None) == 1
    paged = problem(n_select=8, **PAGED)
    assert lib.spamm_attn_select_dev(C.byref(paged), None, 1, 1, P, None, 0, None) == 1   # no key sums
    long = problem(n_select=8, **{**PAGED, "table_width": 16385, "table_stride": 16385})
    assert lib.spamm_attn_select_dev(C.byref(long), P, 1, 1, P, None, 0, None) == 6
    assert b"16384" in lib.spamm_last_cuda_error()


def test_append_refuses(lib):
    a = problem(**PAGED)
    r = C.byref(a)
    for n in (-8, 4, 12, 72):
        assert lib.spamm_attn_append_dev(r, P, P, P, P, n, 0, None) == 1
    assert lib.spamm_attn_append_dev(r, None, P, P, None, 0, 0, None) == 1
    assert lib.spamm_attn_append_dev(r, P, P + 8, P, None, 0, 0, None) == 1
    assert lib.spamm_attn_append_dev(C.byref(problem()), P, P, P, None, 0, 0, None) == 1      # no pages


def test_empty_problems_need_nothing(lib):
    for change in (dict(tokens=0), dict(batch=0), dict(max_q=0)):
        a = problem(**change)
        assert lib.spamm_attn_forward_dev(C.byref(a), None, 0, None) == 0
        assert lib.spamm_attn_forward_scratch_bytes(C.byref(a)) == 0
    assert lib.spamm_attn_backward_dev(C.byref(problem(tokens=0)), None, 0, 0, None, None, None, None, 0, None) == 0


def test_python_calls_refuse():
    from cuspamm_b200 import PagedCache, block_sparse_attention, select_blocks

    q, k = torch.zeros(10, 4, 64, dtype=torch.bfloat16), torch.zeros(10, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 10], dtype=torch.int32)
    lists = torch.zeros(1, 1, 2, 4, dtype=torch.int32)

    def train(q=q, k=k, v=k, lists=lists, cu=cu, n=10, **kw):
        return block_sparse_attention(q, k, v, lists, cu, n, **kw)

    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q[:, :3]), dict(k=k[:5]), dict(v=k[:, :1]), dict(v=k.half()),
                dict(lists=lists[0]), dict(lists=lists.long()), dict(lists=lists[:, :, :1]), dict(cu=cu.long()), dict(n=65),
                dict(n=-1), dict(block=48), dict(query_block=0), dict(scale=0.0), dict(scale=float("nan")),
                dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)[..., ::2]),
                dict(lists=torch.zeros(1, 1, 2, 1025, dtype=torch.int32)), dict()):          # the last: not on a GPU
        with pytest.raises(ValueError):
            train(**bad)
    with pytest.raises(TypeError):
        train(n=torch.tensor(10))
    with pytest.raises(TypeError):
        train(q=q.numpy() if q.dtype == torch.float32 else [q])
    for bad in (dict(n_select=0), dict(n_select=2), dict(n_select=1025), dict(n_select=8, n_first=-1),
                dict(n_select=8, n_local=-1), dict(n_select=8)):
        with pytest.raises(ValueError):
            select_blocks(q, k, cu, 10, **bad)
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    for args in ((pages, pages[:2]), (pages.float(), pages.float()), (pages[:, :, :10], pages[:, :, :10]), (pages[0], pages[0]),
                 (pages, pages, torch.zeros(3, 2, 64, dtype=torch.float64)), (pages, pages)):
        with pytest.raises(ValueError):
            PagedCache(*args)
