import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run with -m gpu on a B200)")


@pytest.fixture(scope="session")
def cuda_device():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def kv8_waits_hold(request):
    """After each test of the 8-bit cache: no bounded wait of its attention kernels has expired in it."""
    yield
    if request.module.__name__.startswith("test_kv8"):
        import torch

        if torch.cuda.is_available():
            from prime_kernels_b200 import kv8

            kv8.check_status()
