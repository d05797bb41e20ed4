"""Refusals of the MoE layer for a few tokens, and its workspace arithmetic: neither needs a GPU."""
import ctypes

import pytest
import torch

from dqmoe_b200 import _lib, ops


def call(**kw):
    """dqmoe_moe_decode with host addresses that are never read: every case below is refused before the first CUDA call."""
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    a = dict(x=at, w_router=at, router_type=7, b=at, b_scale=at, b1=at, b1_scale=at, out=at, workspace=at, workspace_bytes=256, T=4, H=256,
             I=128, E=8, k=2, n_shared=0, scoring=0, quant_mode=1024, stream=None)
    a.update(kw)
    lib = _lib.load()
    rc = lib.dqmoe_moe_decode(*a.values())
    return rc, lib.dqmoe_last_error().decode() if rc else ""


@pytest.mark.parametrize("bad,word", [
    (dict(T=33), "at most 32 tokens"), (dict(T=-1), "at most 32 tokens"), (dict(k=9), "k <= E"), (dict(k=0), "k > 0"),
    (dict(E=64, k=33), "kMaxTopk"), (dict(E=1020, n_shared=5), "at most 1024 experts"), (dict(n_shared=-1), "n_shared >= 0"),
    (dict(H=264), "multiples of 16"), (dict(I=120), "multiples of 16"), (dict(quant_mode=2048), "quant_mode=2048"),
    (dict(quant_mode=3), "quant_mode=3"), (dict(scoring=2), "scoring"), (dict(router_type=1), "router_type=1"), (dict(x=None), "x_bf16"),
    (dict(b_scale=None), "b_scale"), (dict(workspace=None), "is not aligned"), (dict(H=1 << 18), "too large"),
    (dict(H=131072, I=131072, E=1000), "too large"), (dict(workspace_bytes=256), "the layer needs"),
])
def test_refusals(bad, word):
    rc, message = call(**bad)
    assert rc in (1, 3) and message.startswith("[ASSERT FAILED] moe_decode.cu") and word in message, message


def test_misaligned_operands():
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    for name in ("x", "w_router", "b", "b1"):
        assert call(**{name: at + 8})[0] == 1
    assert call(workspace=at + 16)[0] == 1
    assert call(T=0, x=None)[0] == 0


@pytest.mark.parametrize("mode", [0, 256, 512, 1024])
def test_workspace_for_the_most_tokens_serves_fewer(mode):
    for H, I, E, k, shared in ((4096, 14336, 8, 2, 0), (7168, 2048, 256, 8, 1), (2048, 768, 128, 8, 0)):
        sizes = [ops.moe_decode_workspace_bytes(T, H, I, E, k, shared, mode) for T in range(1, 33)]
        assert all(0 < a <= b for a, b in zip(sizes, sizes[1:])) and all(s % 256 == 0 for s in sizes)
        assert ops.moe_decode_workspace_bytes(33, H, I, E, k, shared, mode) == 0


def test_no_cpu_path():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.moe_decode(x, x, x, None, x, None, 1)


def test_wait_limit_is_checked():
    lib = _lib.load()
    assert lib.dqmoe_set_wait_limit(-1) == 1 and "cycles >= 0" in lib.dqmoe_last_error().decode()
    assert lib.dqmoe_set_wait_limit(5) == 0 and lib.dqmoe_set_wait_limit(0) == 0
