"""No test runs under a default device that an earlier one has set."""
import torch


def _set():
    return getattr(torch._GLOBAL_DEVICE_CONTEXT, "device_context", None) is not None


def test_sets_one():
    torch.set_default_device("meta")
    assert _set() and torch.empty(1).device.type == "meta"


def test_starts_without():
    assert not _set() and torch.empty(1).device.type == "cpu"
