"""What the batch operators take and refuse of their tensors' shapes and strides: no GPU is needed."""
import pytest
import torch

from genllm_b200 import _lib, batch

CPU = torch.device("cpu")


def test_an_empty_page_list_is_refused():
    """Its address is null, which would mean all pages."""
    lists = torch.zeros(2, 4, 3, dtype=torch.int32)
    assert batch._page_lists(lists, CPU, 2, 4) is lists
    for bad in (lists[..., :0], lists[..., :2], lists[:1], lists.float()):
        with pytest.raises(_lib.GkvError):
            batch._page_lists(bad, CPU, 2, 4)


def strided(shape, stride, dtype):
    n = sum((e - 1) * s for e, s in zip(shape, stride)) + 1
    return torch.as_strided(torch.zeros(n + 16, dtype=dtype), shape, stride)


@pytest.mark.parametrize("shape,stride", [((1, 8, 64), (1003, 64, 1)), ((3, 1, 64), (128, 5, 1)), ((1, 1, 64), (3, 7, 1))])
def test_strides_of_one_row_mean_nothing(shape, stride):
    t = strided(shape, stride, torch.bfloat16)
    assert batch._rows(t, "q", CPU, torch.bfloat16, (shape[0], None, 64)) is t


@pytest.mark.parametrize("shape,stride", [((2, 8, 64), (1003, 64, 1)), ((1, 2, 64), (128, 5, 1)), ((1, 1, 32), (64, 64, 2))])
def test_strides_of_several_rows_are_aligned(shape, stride):
    with pytest.raises(_lib.GkvError):
        batch._rows(strided(shape, stride, torch.bfloat16), "q", CPU, torch.bfloat16, (shape[0], None, shape[2]))


@pytest.mark.parametrize("shape,stride,fine", [((1, 5, 2), (7, 2, 1), True), ((3, 1, 2), (6, 9, 1), True), ((1, 1, 2), (5, 3, 1), True),
                                               ((2, 5, 2), (11, 2, 1), False), ((1, 5, 2), (20, 4, 1), False),
                                               ((2, 5, 2), (8, 2, 1), False)])
def test_strides_of_the_table(shape, stride, fine):
    table = strided(shape, stride, torch.int32)
    if fine:
        assert batch._table_stride(table) >= shape[1]
    else:
        with pytest.raises(_lib.GkvError):
            batch._table_stride(table)


def test_the_library_on_strides_of_one_row():
    """With one sequence, or one head, the refusal is the next one: the empty workspace."""
    import test_batch_refusals as r
    L = _lib.lib()
    status = L.gkv_batch_decode(r.C.byref(r.batch(batch=1)), r.C.byref(r.decode_args(
        q_stride_batch=1003, k_stride_batch=-5, v_stride_batch=77, workspace=None)), None)
    assert status == _lib.GKV_ERR_INVALID and b"workspace" in L.gkv_last_error()
    status = L.gkv_batch_decode(r.C.byref(r.batch(n_kv_heads=1)), r.C.byref(r.decode_args(
        n_q_heads=1, q_stride_head=3, k_stride_head=5, v_stride_head=7, workspace=None)), None)
    assert status == _lib.GKV_ERR_INVALID and b"workspace" in L.gkv_last_error()
    status = L.gkv_batch_select_pages(r.C.byref(r.batch(batch=1)), r.C.byref(r.select_args(q_stride_batch=1003, workspace=None)), None)
    assert status == _lib.GKV_ERR_INVALID and b"workspace" in L.gkv_last_error()
    # What lies behind one another is still told from what overlaps.
    args = r.decode_args(q=r.OUT + 16, q_stride_batch=-8, workspace=None)
    assert L.gkv_batch_decode(r.C.byref(r.batch(batch=1)), r.C.byref(args), None) == _lib.GKV_ERR_INVALID
    assert b"out overlaps" in L.gkv_last_error()
