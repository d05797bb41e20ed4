"""Waits of moe_decode and lora_linear that run out: the call ends, says so in the status word, and leaves the next one unharmed.

With a limit of one clock cycle an ordinary call gives up at its first wait that looks at the clock in each turn: for an expert's fc1, which takes
microseconds, and for the slots of the mixed rows' B. All other waits end because the block's flag is up, or by the same limit."""
import pytest
import torch

import test_gpu_lora as lora
import test_gpu_moe_decode as moe
from dqmoe_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def run_out(call, codes):
    """`call` with the usual limit, with that of a cycle, and with the usual one again."""
    want = call()
    assert ops.device_status() == 0
    lib = _lib.load()
    _lib.check(lib.dqmoe_set_wait_limit(1))
    try:
        call()
        assert ops.device_status() in codes
    finally:
        _lib.check(lib.dqmoe_set_wait_limit(0))
    assert ops.device_status() == 0  # cleared
    assert torch.equal(call(), want) and ops.device_status() == 0


@pytest.mark.parametrize("mode", ["bf16", "block"])
@pytest.mark.parametrize("T", [1, 16, 32])
def test_moe_decode(mode, T):
    a = moe.make(91, mode, T, 2048, 2048, 1, 1)  # one expert: whoever begins fc2 has its fc1 to wait for
    run_out(lambda: ops.moe_decode(**a), (301, 302))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K,L,R", [(40, 2048, 1024, 16, 16), (200, 640, 1032, 8, 72), (2661, 1720, 2048, 40, 128)])
def test_lora_linear(dtype, T, N, K, L, R):
    """Parts of a tile, a tile per block, and pairs of blocks."""
    a = lora.make(93, T, N, K, L, R, dtype, "random")
    run_out(lambda: ops.lora_linear(**a), (311, 312))


def test_several_calls_at_once():
    """Calls of other streams beside one that gives up, and calls behind it on its stream."""
    a, b = moe.make(95, "tensor", 8, 2048, 2048, 1, 1), lora.make(97, 64, 2048, 2048, 16, 16)
    want = ops.moe_decode(**a), ops.lora_linear(**b)
    lib = _lib.load()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        before = ops.lora_linear(**b)
    _lib.check(lib.dqmoe_set_wait_limit(1))
    try:
        ops.moe_decode(**a)
    finally:
        _lib.check(lib.dqmoe_set_wait_limit(0))
    after = ops.moe_decode(**a), ops.lora_linear(**b)
    assert ops.device_status() in (301, 302)
    torch.cuda.synchronize()
    assert torch.equal(before, want[1]) and torch.equal(after[0], want[0]) and torch.equal(after[1], want[1])
    assert ops.device_status() == 0
