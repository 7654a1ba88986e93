import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

# A reference tree that is there but empty counts as absent.
_REF = os.environ.get("GENLLM_REF") or os.path.join(os.path.dirname(ROOT), "reference")
if os.path.isdir(_REF) and not os.listdir(_REF):
    os.environ["GENLLM_REF"] = os.path.join(_REF, "absent")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200); run with -m gpu")


def _has_cuda():
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


def pytest_collection_modifyitems(config, items):
    if _has_cuda():
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)
