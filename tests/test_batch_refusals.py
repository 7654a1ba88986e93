"""What the batch entry points refuse, before any CUDA call: no GPU is needed."""
import ctypes as C

import pytest

from genllm_b200 import _lib

INVALID, UNSUPPORTED = _lib.GKV_ERR_INVALID, _lib.GKV_ERR_UNSUPPORTED
ADDR = 1 << 20  # never read: every check comes first
OUT = 1 << 24


def batch(**changes):
    pool = _lib.PoolDesc(ADDR, ADDR, 10, 8, 128, _lib.GKV_BF16)
    b = _lib.Batch(pool, ADDR, ADDR, 16, 2, 16, 0)
    for k, v in changes.items():
        setattr(b.pool if hasattr(b.pool, k) else b, k, v)
    return b


def decode_args(**changes):
    a = _lib.BatchDecodeArgs(ADDR, 1024, 128, ADDR, ADDR, 1024, 128, 1024, 128, OUT, None, None, None, None, 0, 0, 16,
                             _lib.GKV_BF16, 0.1, 1.0, ADDR, 0)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


def select_args(**changes):
    a = _lib.BatchSelectArgs(ADDR, 1024, 128, ADDR, ADDR, 8, 1, 1, 1, 16, ADDR, 0)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


def evict_args(**changes):
    a = _lib.BatchEvictArgs(ADDR, ADDR, None, ADDR, ADDR, None, ADDR, 256, 64, 8, ADDR, 0)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


BAD_BATCH = [(dict(dtype=_lib.GKV_F32), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED),
             (dict(n_kv_heads=0), INVALID), (dict(n_kv_heads=257), INVALID), (dict(pool_pages=0), INVALID),
             (dict(k_base=None), INVALID), (dict(v_base=ADDR + 8), INVALID), (dict(batch=0), UNSUPPORTED),
             (dict(batch=4097), UNSUPPORTED), (dict(table_pages=0), INVALID), (dict(table_stride=15), INVALID),
             (dict(table_pages=1 << 28, table_stride=1 << 28), INVALID),
             (dict(batch=4096, table_pages=1 << 20, table_stride=1 << 20), UNSUPPORTED), (dict(table=None), INVALID),
             (dict(table=ADDR + 4), INVALID), (dict(lens=None), INVALID), (dict(device=-1), INVALID),
             (dict(device=64), INVALID)]


@pytest.mark.parametrize("changes,status", BAD_BATCH)
def test_batches(changes, status):
    L, b, n = _lib.lib(), batch(**changes), C.c_size_t()
    assert L.gkv_batch_decode(C.byref(b), C.byref(decode_args()), None) == status
    assert L.gkv_batch_decode_workspace(C.byref(b), 16, 0, C.byref(n)) == status
    assert L.gkv_batch_page_bounds(C.byref(b), None, 0, ADDR, None) == status
    assert L.gkv_batch_select_pages(C.byref(b), C.byref(select_args()), None) == status
    assert L.gkv_batch_select_workspace(C.byref(b), C.byref(n)) == status
    assert L.gkv_batch_evict(C.byref(b), C.byref(evict_args()), None) == status
    assert L.gkv_batch_evict_workspace(C.byref(b), C.byref(n)) == status


@pytest.mark.parametrize("changes,status", [
    (dict(q=None), INVALID), (dict(q=ADDR + 2), INVALID), (dict(q_stride_head=100), INVALID),
    (dict(q_stride_batch=1004), INVALID), (dict(k_new=None), INVALID), (dict(v_new=None), INVALID),
    (dict(k_stride_head=4), INVALID), (dict(v_stride_batch=2), INVALID), (dict(out=None), INVALID),
    (dict(out=ADDR + 4), INVALID), (dict(out_dtype=7), UNSUPPORTED), (dict(lse=ADDR + 1), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(n_q_heads=0), INVALID),
    (dict(n_q_heads=12), INVALID), (dict(n_q_heads=136), UNSUPPORTED), (dict(pages=ADDR, n_pages=0), INVALID),
    (dict(pages=ADDR, n_pages=4, weights_out=ADDR, weights_stride=256), UNSUPPORTED),
    (dict(weights_in=ADDR), INVALID), (dict(weights_out=ADDR, weights_stride=255), INVALID),
    (dict(weights_out=ADDR, weights_stride=256, decay=float("inf")), INVALID), (dict(workspace=None), INVALID),
    (dict(workspace=ADDR + 8), INVALID), (dict(out=ADDR), INVALID),
    (dict(q=OUT + 2 * 2 * 16 * 128 - 16), INVALID), (dict(q=OUT - 2 * (1024 + 16 * 128) + 16), INVALID),
    (dict(k_new=OUT + 16), INVALID), (dict(v_new=OUT - 16), INVALID),
    (dict(weights_in=ADDR, weights_out=ADDR + 4, weights_stride=256), INVALID)])
def test_decode(changes, status):
    assert _lib.lib().gkv_batch_decode(C.byref(batch()), C.byref(decode_args(**changes)), None) == status
    assert _lib.lib().gkv_last_error()


@pytest.mark.parametrize("changes,status", [
    (dict(q=None), INVALID), (dict(q_stride_head=4), INVALID), (dict(bounds=None), INVALID),
    (dict(bounds=ADDR + 8), INVALID), (dict(pages=None), INVALID), (dict(n_pages=0), INVALID),
    (dict(n_first=-1), INVALID), (dict(n_last=-1), INVALID), (dict(n_first=5, n_last=4), INVALID),
    (dict(n_first=2147483647, n_last=2147483647), INVALID), (dict(extra=-1), INVALID), (dict(extra=257), INVALID),
    (dict(n_q_heads=15), INVALID), (dict(n_q_heads=136), UNSUPPORTED), (dict(workspace=None), INVALID)])
def test_select(changes, status):
    assert _lib.lib().gkv_batch_select_pages(C.byref(batch()), C.byref(select_args(**changes)), None) == status


@pytest.mark.parametrize("changes,status", [
    (dict(weights=None), INVALID), (dict(weights_out=None), INVALID), (dict(positions_out=None), INVALID),
    (dict(seen=None), INVALID), (dict(lens_out=None), INVALID), (dict(tracked=ADDR), INVALID),
    (dict(weights=ADDR + 2), INVALID), (dict(stride=255), INVALID), (dict(n_keep=-1), INVALID),
    (dict(n_recent=-1), INVALID), (dict(n_recent=65), INVALID), (dict(workspace=None), INVALID),
    (dict(workspace=ADDR + 4), INVALID), (dict(weights_out=ADDR + 2 * 8 * 256 * 4 - 4), INVALID),
    (dict(positions=ADDR + 4), INVALID)])
def test_evict(changes, status):
    assert _lib.lib().gkv_batch_evict(C.byref(batch()), C.byref(evict_args(**changes)), None) == status


def message(call, args):
    """What the entry point says of arguments whose only fault is the empty workspace, or another one."""
    assert call(C.byref(batch()), C.byref(args), None) != _lib.GKV_OK
    return _lib.lib().gkv_last_error()


def test_outputs_on_inputs_are_named():
    L = _lib.lib()
    assert b"out overlaps" in message(L.gkv_batch_decode, decode_args(out=ADDR, workspace=None))
    assert b"workspace" in message(L.gkv_batch_decode, decode_args(workspace=None))
    span = 2 * (1024 + 16 * 128)  # bytes of q with these strides
    assert b"out overlaps" in message(L.gkv_batch_decode, decode_args(q=OUT - span + 16, workspace=None))
    assert b"workspace" in message(L.gkv_batch_decode, decode_args(q=OUT - span, workspace=None))
    assert b"workspace" in message(L.gkv_batch_decode, decode_args(
        weights_in=ADDR, weights_out=ADDR, weights_stride=256, workspace=None))
    end = ADDR + 2 * 8 * 256 * 4
    assert b"workspace" in message(L.gkv_batch_evict, evict_args(weights_out=end, workspace=None))
    assert b"successor" in message(L.gkv_batch_evict, evict_args(weights_out=end - 4, workspace=None))


def test_counts_that_32_bits_do_not_hold():
    from genllm_b200.batch import _count
    assert _count(7, "keep") == 7 and _count(2 ** 31 - 1, "keep") == 2 ** 31 - 1
    for bad in (2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1, 1.5, "3", None):
        with pytest.raises(_lib.GkvError):
            _count(bad, "keep")


def test_bounds_and_nulls():
    L, b, n = _lib.lib(), batch(), C.c_size_t()
    ref = C.byref
    assert L.gkv_batch_page_bounds(ref(b), None, 0, None, None) == INVALID
    assert L.gkv_batch_page_bounds(ref(b), None, 0, ADDR + 8, None) == INVALID
    assert L.gkv_batch_page_bounds(ref(b), ADDR + 2, 0, ADDR, None) == INVALID
    assert L.gkv_batch_page_bounds(ref(b), None, -1, ADDR, None) == INVALID
    assert L.gkv_batch_page_bounds(ref(b), None, 257, ADDR, None) == INVALID
    assert L.gkv_batch_decode(None, ref(decode_args()), None) == INVALID
    assert L.gkv_batch_decode(ref(b), None, None) == INVALID
    assert L.gkv_batch_select_pages(ref(b), None, None) == INVALID
    assert L.gkv_batch_evict(ref(b), None, None) == INVALID
    assert L.gkv_batch_decode_workspace(ref(b), 16, 0, None) == INVALID
    assert L.gkv_batch_decode_workspace(ref(b), 15, 0, ref(n)) == INVALID
    assert L.gkv_batch_select_workspace(ref(b), None) == INVALID
    assert L.gkv_batch_evict_workspace(ref(b), None) == INVALID
    assert L.gkv_batch_prepare(-1) == INVALID and L.gkv_batch_prepare(64) == INVALID
    assert L.gkv_batch_check_errors(-1, None) == INVALID
    many = batch(batch=4096, n_kv_heads=17)
    assert L.gkv_batch_evict(ref(many), ref(evict_args()), None) == UNSUPPORTED


def test_python_refusals_without_a_gpu():
    torch = pytest.importorskip("torch")
    from genllm_b200.batch import PagedBatch
    pool = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(_lib.GkvError):
        PagedBatch(pool, pool, torch.zeros(1, 2, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
