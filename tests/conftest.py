"""pytest configuration: markers and import path."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run with -m gpu on a B200 box)")
    config.addinivalue_line("markers", "multigpu: needs at least two CUDA devices")
    config.addinivalue_line("markers", "slow: long-running soak test")


def pytest_collection_modifyitems(config, items):
    """Skips GPU tests on machines without the hardware they need."""
    try:
        import torch
        ngpu = torch.cuda.device_count() if torch.cuda.is_available() else 0
    except Exception:
        ngpu = 0
    for item in items:
        if "gpu" in item.keywords and ngpu < 1:
            item.add_marker(pytest.mark.skip(reason="no CUDA device"))
        if "multigpu" in item.keywords and ngpu < 2:
            item.add_marker(pytest.mark.skip(reason="needs >= 2 CUDA devices"))


#: modules whose kernels give up a wait that runs out with an error word and incomplete results
_STATUS = ("test_gpu_paged_attention", "test_gpu_paged_cache", "test_gpu_w4", "test_gpu_generate", "test_gpu_serving", "test_gpu_attention_weights",
           "test_gpu_packed_attention", "test_gpu_packed_edges", "test_gpu_packed_gradients", "test_gpu_rotary", "test_gpu_sample", "test_gpu_sample_weights", "test_gpu_prompts")


@pytest.fixture(autouse=True)
def kernels_report_no_error(request):
    """No wait ran out in the kernels of a test that answers token by token."""
    yield
    if request.module.__name__.rpartition(".")[2] in _STATUS:
        from mccl_b200 import _C
        assert _C.gemm_error_flag() == 0
