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
