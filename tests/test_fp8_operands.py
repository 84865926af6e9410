"""What the Python entry points of the FP8 operators refuse by looking at their operands, without a GPU:
nothing here reaches the library."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from hmoe import block, fp8  # noqa: E402


@pytest.fixture
def on_host(monkeypatch):
    """The entry points' checks on host tensors."""
    monkeypatch.setattr(fp8, "_torch", lambda: torch)
    monkeypatch.setattr(block, "_torch", lambda: torch)
    monkeypatch.setattr(block, "check_on_device", lambda *t: t[0].device)


# one byte a value, but not OCP e4m3
OTHERS = [torch.float8_e5m2, torch.float8_e4m3fnuz, torch.float8_e5m2fnuz, torch.int8, torch.bool]


@pytest.mark.parametrize("dtype", OTHERS)
def test_matrix_of_other_bytes(on_host, dtype):
    """Bytes of another 8-bit type are not read as e4m3."""
    q, scale = torch.zeros((2, 128), dtype=torch.uint8), torch.ones((2, 1))
    with pytest.raises(ValueError, match="e4m3"):
        fp8.Matrix(q.view(dtype), scale, 128, 1)
    for good in (torch.uint8, torch.float8_e4m3fn):
        assert fp8.Matrix(q.view(good), scale, 128, 1).rows == 2


@pytest.mark.parametrize("dtype", OTHERS)
@pytest.mark.parametrize("which", range(3))
def test_checkpoint_of_other_bytes(on_host, dtype, which):
    """A checkpoint in e5m2 or a format with another bias is refused, not decoded as e4m3."""
    w = [torch.zeros((2, 128, 128), dtype=torch.uint8) for _ in range(3)]
    s = [torch.ones((2, 1, 1)) for _ in range(3)]
    with pytest.raises(ValueError, match="e4m3"):
        block.DeviceExpertLayer.from_fp8(*[t.view(dtype) if i == which else t for i, t in enumerate(w)], *s)
    for good in (torch.uint8, torch.float8_e4m3fn):
        layer = block.DeviceExpertLayer.from_fp8(*[t.view(good) for t in w], *s)
        assert (layer.experts, layer.hidden, layer.inter) == (2, 128, 128)
