"""moe_decode and lora_linear of tensors on another device than the current one: every question to the library is asked with theirs current, since it
answers for the current device's number of SMs. With stand-ins for the tensors and the library: no GPU."""
import torch
import pytest

from dqmoe_b200 import _lib, ops


class Stub:
    """A tensor on cuda:1, as far as the front end looks."""
    def __init__(self, *shape, dtype=torch.bfloat16):
        self.shape, self.dtype, self.device, self.is_cuda = torch.Size(shape), dtype, torch.device("cuda", 1), True

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 256

    def numel(self):
        return self.shape.numel()

    def element_size(self):
        return self.dtype.itemsize

    def new_empty(self, shape, dtype=None):
        return Stub(*([shape] if isinstance(shape, int) else shape), dtype=dtype or self.dtype)


@pytest.mark.parametrize("current", [0, 1])
def test_asked_on_the_tensors_device(monkeypatch, current):
    at, asked = [current], []

    class Device:
        def __init__(self, index):
            self.index = index if isinstance(index, int) else index.index

        def __enter__(self):
            at.append(self.index)

        def __exit__(self, *_):
            at.pop()

    class Library:
        def __getattr__(self, name):
            def fn(*args):
                asked.append((name, at[-1]))
                return 4096 if name.endswith("_bytes") else 0
            return fn

    monkeypatch.setattr(_lib, "load", lambda: Library())
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: at[-1], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)

    T, H, I, E = 4, 256, 128, 8
    x = Stub(T, H)
    ops.moe_decode(x, Stub(E, H), Stub(E, 2 * I, H), None, Stub(E, H, I), None, 2, quant_mode=0, out=Stub(T, H))
    a = (x, Stub(64, H), Stub(3, 16, H), Stub(3, 64, 16), Stub(T, dtype=torch.int32))
    ops.lora_linear(*a)
    assert [name for name, _ in asked] == ["dqmoe_moe_decode_workspace_bytes", "dqmoe_moe_decode", "dqmoe_lora_linear_workspace_bytes", "dqmoe_lora_linear"]
    assert [device for _, device in asked] == [1] * 4
    assert at == [current]
