"""Caches with a scale for each block of tokens and head: refusals, on the CPU."""
import pytest
import torch

from nano_qwen_amd import kernels
from tests import test_gpu_blocks
from tests.test_gpu_append import refusals


def buffer(n):
    """``n`` bytes, aligned as a device's are."""
    t = torch.empty(n + 256, dtype=torch.uint8)
    return t[-t.data_ptr() % 256:][:n]


@pytest.fixture
def host(monkeypatch):
    """The shim's and the library's checks, with tensors on the host: what passes them all fails at its launch (status -3)."""
    if torch.cuda.is_available():
        pytest.skip("would launch on host memory")
    monkeypatch.setattr(kernels, "_check_one_device", lambda *a: 0)
    monkeypatch.setattr(kernels, "_current_device", lambda: 0)
    monkeypatch.setattr(kernels, "raw_stream", lambda i: 0)
    monkeypatch.setattr(kernels, "_decode_counters_and_workspace", lambda *a: (None, buffer(1 << 26)))
    monkeypatch.setattr(kernels, "prefill_workspace", lambda d: torch.zeros(64, dtype=torch.int32))
    monkeypatch.setitem(kernels._prefill_parts, (0, 0), buffer(1 << 27))
    monkeypatch.setitem(kernels._span_parts, (0, 0), buffer(1 << 27))


def test_append_refusals(host):
    good, bad = refusals("cpu")
    with pytest.raises(RuntimeError, match="status -3"):
        kernels.append_kvcache(**good)
    for kw in bad:
        with pytest.raises(RuntimeError) as e:
            kernels.append_kvcache(**(good | kw))
        assert "status -3" not in str(e.value), (list(kw), str(e.value))


def test_append_refuses_a_table_without_rows(host):
    """Rows of positions outside the table are NaN, but are read from its first row all the same."""
    good, _ = refusals("cpu")
    rot = 64
    pos = torch.zeros(good["key"].shape[0], dtype=torch.int64)
    for rows in (0, 1):
        kw = good | dict(positions=pos, rotary_dim=rot, cos_sin_cache=torch.zeros(4, rot)[:rows], query=None)
        with pytest.raises(RuntimeError) as e:
            kernels.append_kvcache(**kw)
        assert ("status -3" in str(e.value)) == (rows == 1), str(e.value)


def test_append_refuses_tensors_on_the_host():
    good, _ = refusals("cpu")
    with pytest.raises(RuntimeError, match="HIP device"):
        kernels.append_kvcache(**good)


def test_attention_refusals(host):
    for call, c, args, kw in test_gpu_blocks.refusals("cpu"):
        with pytest.raises(RuntimeError) as e:
            getattr(c, call)(*args, **kw)
        assert "status -3" not in str(e.value), (call, args, list(kw), str(e.value))
    for new in ([2, 3], [1, 1]):
        c = test_gpu_blocks.Case(new, [40, 5], 8, 2, 128, torch.bfloat16, 64, 32).to("cpu")
        for call in (c.prefill, c.decode)[:1 if new[0] > 1 else 2]:
            for args in ((), (40, 1)):
                with pytest.raises(RuntimeError, match="status -3"):
                    call(*args)
