"""Caches with a scale for each block of tokens and head: refusals, on the CPU."""
import pytest
import torch

from nano_qwen_amd import kernels
from tests.test_gpu_append import refusals


@pytest.fixture
def host(monkeypatch):
    """The shim's and the library's checks, with tensors on the host: what passes them all fails at its launch (status -3)."""
    if torch.cuda.is_available():
        pytest.skip("would launch on host memory")
    monkeypatch.setattr(kernels, "_check_one_device", lambda *a: 0)
    monkeypatch.setattr(kernels, "_current_device", lambda: 0)
    monkeypatch.setattr(kernels, "raw_stream", lambda i: 0)


def test_append_refusals(host):
    good, bad = refusals("cpu")
    with pytest.raises(RuntimeError, match="status -3"):
        kernels.append_kvcache(**good)
    for kw in bad:
        with pytest.raises(RuntimeError) as e:
            kernels.append_kvcache(**(good | kw))
        assert "status -3" not in str(e.value), (list(kw), str(e.value))


def test_append_refuses_tensors_on_the_host():
    good, _ = refusals("cpu")
    with pytest.raises(RuntimeError, match="HIP device"):
        kernels.append_kvcache(**good)
