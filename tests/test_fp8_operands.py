"""What the Python entry points of the FP8 operators refuse by looking at their operands, without a GPU:
nothing here reaches the library."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from hmoe import block, fp8, stack  # noqa: E402


@pytest.fixture
def on_host(monkeypatch):
    """The entry points' checks on host tensors."""
    monkeypatch.setattr(fp8, "_torch", lambda: torch)
    monkeypatch.setattr(block, "_torch", lambda: torch)
    monkeypatch.setattr(stack, "_torch", lambda: torch)
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


@pytest.fixture
def calls(on_host, monkeypatch):
    """The library's calls, recorded instead of made; tensors pass as on a GPU."""
    import contextlib
    made = []
    monkeypatch.setattr(fp8, "check_on_device", lambda *t: t[0].device)
    monkeypatch.setattr(fp8.capi, "call", lambda *a: made.append(a))
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *d: type("S", (), {"cuda_stream": 0}))
    return made


def _views():
    x = torch.randn(8, 12)
    yield "a row of a strided block", x[::2, ::2][:1, :1]
    yield "a column of one, any stride", x.as_strided((4, 1), (1, 7))
    yield "a row, broadcast", torch.randn(12).as_strided((1, 12), (0, 1))
    yield "a row, negative-free stride of a slice", x[:1, ::2]
    yield "a row of a transposed view", x.t()[:1]
    yield "a column", x[:, 3:4]
    yield "a column of every third row", x[::3, 3:4]
    yield "a whole matrix", x
    yield "a transposed view", x.t()
    yield "a block of a matrix", x[2:5, 4:9]
    yield "every second column", x[:, ::2]
    yield "one row repeated", torch.randn(12).expand(5, 12)
    yield "one value repeated", torch.randn(1, 1).expand(5, 12)


@pytest.mark.parametrize("what,x", list(_views()), ids=lambda v: v if isinstance(v, str) else "")
def test_quantize_views(calls, what, x):
    """Whatever the view, the library gets strides that it takes and that name the view's elements: the
    stride of a dimension of one is any number, also one that the library would refuse."""
    m = fp8.quantize(x)
    (name, pointer, _, rows, width, row_stride, col_stride, *_), = calls
    assert name == "hm_fp8_quantize" and (rows, width) == tuple(x.shape) == (m.rows, m.width)
    assert row_stride > 0 and col_stride > 0 and 1 in (row_stride, col_stride)
    at = torch.arange(rows)[:, None] * row_stride + torch.arange(width) * col_stride
    if pointer == x.data_ptr():      # else a copy, whose strides are its shape's
        own = x.as_strided((int(at.max()) + 1,), (1,))
        assert torch.equal(own[at], x)
    else:
        assert (row_stride, col_stride) == (width, 1)


def _one_device(*tensors):
    """check_on_device with the host in the place of a GPU."""
    devices = {t.device for t in tensors if t is not None}
    if len(devices) != 1:
        raise ValueError(f"the operands must share one GPU, got {devices}")
    return devices.pop()


@pytest.mark.parametrize("part", ["packed", "scale"])
def test_experts_of_a_layer_elsewhere(calls, monkeypatch, part):
    """Both of a layer's arrays have to be where the rows are."""
    monkeypatch.setattr(fp8, "check_on_device", _one_device)
    monkeypatch.setattr(fp8, "workspace_bytes", lambda *a: 16)
    w = [torch.zeros((2, 128, 128), dtype=torch.uint8) for _ in range(3)]
    layer = block.DeviceExpertLayer.from_fp8(*w, *[torch.ones((2, 1, 1)) for _ in range(3)])
    args = torch.ones((4, 128)), torch.tensor([0, 4, 4], dtype=torch.int32), torch.arange(4, dtype=torch.int32)
    fp8.experts(layer, *args)
    assert len(calls) == 1
    setattr(layer, part, getattr(layer, part).to("meta"))
    with pytest.raises(ValueError, match="share one GPU"):
        fp8.experts(layer, *args)
    assert len(calls) == 1


@pytest.mark.parametrize("entry", ["block", "stack"])
def test_layer_on_another_device(on_host, monkeypatch, entry):
    """A block and a stack refuse an FP8 layer that is not on the current device, whose memory their
    buffers and their stream belong to."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    w = [torch.zeros((2, 128, 128), dtype=torch.uint8) for _ in range(3)]
    layer = block.DeviceExpertLayer.from_fp8(*w, *[torch.ones((2, 1, 1)) for _ in range(3)])
    layer.packed = type("Elsewhere", (), {"device": torch.device("cuda", 1)})()
    with pytest.raises(ValueError, match="cuda:1"):
        if entry == "block":
            block.MoEBlock(layer, 1)._buffers(4)
        else:
            stack.MoEStack([layer], [torch.zeros((128, 2))], 1)
