"""Refusals of the projection with adapters, and its workspace arithmetic: neither needs a GPU."""
import ctypes

import pytest
import torch

from dqmoe_b200 import _lib, ops


def call(**kw):
    """dqmoe_lora_linear with host addresses that are never read: every case below is refused before the first CUDA call."""
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    a = dict(x=at, ldx=64, w=at, lora_a=at, lora_b=at, ids=at, scale=at, bias=at, y=at, ldy=128, workspace=at, workspace_bytes=256, T=4, N=128, K=64,
             L=2, R=16, type=7, stream=None)
    a.update(kw)
    lib = _lib.load()
    rc = lib.dqmoe_lora_linear(*a.values())
    return rc, lib.dqmoe_last_error().decode() if rc else ""


@pytest.mark.parametrize("bad,word", [
    (dict(R=12), "R=12"), (dict(R=136), "R=136"), (dict(R=0), "R > 0"), (dict(L=0), "L > 0"), (dict(K=60), "K=60"), (dict(T=-1), "T >= 0"),
    (dict(N=0), "N > 0"), (dict(type=6), "type=6"), (dict(type=0), "type=0"), (dict(ldx=56), "ldx=56"), (dict(ldx=68), "ldx=68"),
    (dict(ldy=127), "ldy=127"), (dict(x=None), "x != nullptr"), (dict(ids=None), "ids != nullptr"), (dict(workspace=None), "is not aligned"),
    (dict(N=(1 << 24) + 8), "too large"), (dict(L=1 << 27), "too large"), (dict(workspace_bytes=128), "the projection needs"),
])
def test_refusals(bad, word):
    rc, message = call(**bad)
    assert rc in (1, 3) and message.startswith("[ASSERT FAILED] lora.cu") and word in message, message


def test_misaligned_operands():
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    for name, by in (("x", 8), ("w", 8), ("lora_a", 8), ("lora_b", 8), ("y", 1), ("ids", 2), ("scale", 2), ("bias", 2), ("workspace", 16)):
        assert call(**{name: at + by})[0] == 1, name
    assert call(T=0, x=None)[0] == 0


def test_workspace_is_host_arithmetic():
    for N in (128, 4096, 6144):
        sizes = [ops.lora_linear_workspace_bytes(T, N, 4096, 8, 16) for T in [*range(0, 600), *range(600, 20000, 37)]]
        assert all(0 < a <= b for a, b in zip(sizes, sizes[1:])) and all(s % 256 == 0 for s in sizes)  # the longest batch's serves all
    assert ops.lora_linear_workspace_bytes(4, 128, 64, 2, 20) == 0


def test_checks_of_the_front_end():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.lora_linear(x, x, x[None], x[None], torch.zeros(2, dtype=torch.int32))
