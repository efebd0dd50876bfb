import os
import sys

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
for p in (ROOT, os.path.join(ROOT, "oracle")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a)")


def pytest_collection_modifyitems(items):
    """The comparisons with the reference's own GPU library need it built from the
    reference's sources (make -C oracle ref).  Where neither is there, they are
    skipped and say so: as failures they would end a run with -x before every test
    behind them.  Where the sources are there, a missing library is a failure."""
    import oracle
    if os.path.exists(oracle.reference_gpu_lib_path()):
        return
    root = os.environ.get("MX_REFERENCE_ROOT") or os.path.join(os.path.dirname(ROOT), "reference")
    if os.path.isfile(os.path.join(root, "moonxi-net-gpu", "cuda", "cuda_kernels.cu")):
        return
    skip = pytest.mark.skip(reason="neither the reference's GPU library nor its sources are here")
    for item in items:
        if getattr(item, "originalname", "") == "test_vs_reference_cuda_matmul":
            item.add_marker(skip)


@pytest.fixture(scope="session")
def cuda_device():
    """The CUDA device for GPU tests.  GPU tests fail (never skip) when no
    device is usable: a silent skip would hide a missing native path."""
    import torch
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    torch.cuda.set_device(0)
    return torch.device("cuda", 0)
