import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X GPU")


def gpu_available() -> bool:
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


@pytest.fixture(scope="session")
def golden():
    import numpy as np
    return dict(np.load(ROOT / "tests" / "golden" / "ref_vectors.npz"))


@pytest.fixture(autouse=True)
def _no_default_device_left():
    """A default device that a test sets ends with it (torch.set_default_device("cpu") sets one, too)."""
    yield
    torch = sys.modules.get("torch")
    if torch is not None and getattr(torch, "_GLOBAL_DEVICE_CONTEXT", None) is not None and \
            getattr(torch._GLOBAL_DEVICE_CONTEXT, "device_context", None) is not None:
        torch.set_default_device(None)
