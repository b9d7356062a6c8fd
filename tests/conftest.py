import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "oracle")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a)")


# Tests that compare with the reference's own kernels.  Where its build is missing they
# fail, after all others, so that a run that stops at its first failure has run the rest.
NEED_REFERENCE = ("test_forward_tensorcore_vs_reference_kernels", "test_swtcf_vs_reference_converter",
                  "test_config2_vs_reference_kernel", "test_swtcf_spmm_vs_reference_kernel",
                  "test_swtcf_spmm_prepared_pull", "test_push_heavy_hub_window")


def pytest_collection_modifyitems(items):
    if not os.path.exists(os.path.join(ROOT, "oracle", "_ref", "libtcc_ref.so")):
        items.sort(key=lambda item: getattr(item, "originalname", item.name) in NEED_REFERENCE)  # stable


@pytest.fixture(scope="session")
def oracle():
    import oracle as O
    O.build()
    return O


def cuda_ok():
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


@pytest.fixture(scope="session")
def gpu():
    """The CUDA library on a GPU; a GPU test without a GPU is an error, not a skip."""
    import torch
    assert torch.cuda.is_available(), "gpu-marked test needs a CUDA device"
    from tcc_b200 import build
    build.build()
    from tcc_b200 import _lib
    _lib.lib()
    return torch.device("cuda:0")
