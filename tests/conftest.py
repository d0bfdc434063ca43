import importlib
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP kernels)")


@pytest.fixture(scope="session")
def mga():
    """The product package (its directory name is not a Python identifier)."""
    return importlib.import_module("mtp-glora_amd")


@pytest.fixture(scope="session")
def dev():
    import torch
    if not torch.cuda.is_available():
        raise RuntimeError("GPU tests need a visible GPU")
    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def seeded():
    """Every test begins with the same generators, so that a failure repeats."""
    import torch
    torch.manual_seed(20240)
