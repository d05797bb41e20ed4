"""Sigmoid scores of logits far below zero: the chosen experts' weights are ratios of scores, which fp32 has also where a score by itself is none of
its numbers any more.

Tolerance of a weight: expf and the division are off by some 2^-22 of the value, the difference of two logits by 2^-24 of at most 40, the sum of k <= 8
scores by k 2^-24: 64 2^-24 of the value in all; and a score that is not above 2^-24 of the largest may count as 0.
"""
import pytest
import torch

import test_gpu_moe_decode as moe
from dqmoe_b200 import ops

pytestmark = pytest.mark.gpu


def weights_in_64_bits(logits, k):
    order = torch.argsort(logits.double(), dim=1, descending=True, stable=True)[:, :k]
    score = torch.sigmoid(logits.double().gather(1, order))
    return order, score / score.sum(1, keepdim=True)


def logits_around(T, E, seed):
    """Rows whose largest logits lie between 30 and -600, on both sides of where a score or its reciprocal leaves fp32."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    top = torch.tensor([30.0, 0.0, -17.0, -60.0, -71.9, -72.0, -72.1, -80.0, -87.0, -88.7, -88.8, -89.0, -100.0, -104.0, -200.0, -600.0], device="cuda")
    spread = torch.tensor([0.5, 8.0, 20.0], device="cuda")
    row = torch.arange(T, device="cuda")
    logits = -torch.rand(T, E, generator=g, device="cuda") * spread[row % 3, None]
    logits[row, torch.randint(0, E, (T,), generator=g, device="cuda")] = 0
    return logits + top[row % 16, None]


@pytest.mark.parametrize("E,k", [(8, 2), (64, 6), (128, 8), (256, 8), (1000, 6), (3, 3)])
def test_weights_of_the_router(E, k):
    logits = logits_around(96, E, E)
    ids, weights = ops.route_topk(logits, k, "sigmoid")
    order, want = weights_in_64_bits(logits, k)
    assert torch.equal(ids.long(), order)
    off = (weights.double() - want).abs()
    assert (off <= 64 * 2.0 ** -24 * want + 2.0 ** -24).all(), float(off.max())


def test_tokens_without_a_number_stay_what_they_were():
    logits = torch.full((3, 8), -float("inf"), device="cuda")
    logits[1, 3] = -300.0
    logits[2] = float("nan")
    ids, weights = ops.route_topk(logits, 2, "sigmoid")
    assert weights[0].isnan().all() and weights[2].isnan().all()
    assert ids[1].tolist() == [3, 0] and weights[1].tolist() == [1.0, 0.0]


@pytest.mark.parametrize("mode", list(moe.MODES))
@pytest.mark.parametrize("T", [5, 20])
def test_the_layer_for_a_few_tokens(mode, T):
    """Every logit of the even tokens near -100: their rows are what the formula says, not NaN."""
    a = moe.make(81, mode, T, 512, 256, 12, 3, shared=1)
    a["w_router"][:, 0] = -12.5
    a["x"][:, 0] = 0
    a["x"][::2, 0] = 8
    out = ops.moe_decode(**a, scoring="sigmoid")
    ref, size = moe.reference(a, "sigmoid")
    moe.check(out, ref, size)


@pytest.mark.parametrize("T", [5, 200])
def test_the_block(T):
    """moe_block on logits near -100 is moe_block on the logits whose softmax over the chosen is the same: scores this small are exponentials."""
    g = torch.Generator(device="cuda").manual_seed(83)
    H, I, E, k = 256, 384, 12, 3
    x, b, b1 = ((torch.randn(*n, generator=g, device="cuda") * s).bfloat16() for n, s in (((T, H), 1), ((E, 2 * I, H), 0.05), ((E, H, I), 0.05)))
    logits = torch.randint(-64, 64, (T, E), generator=g, device="cuda") / 32.0 + torch.arange(E, device="cuda") / 512.0
    low = ops.moe_block(x, logits - 128, b, None, b1, None, k, "sigmoid", quant_mode=0)
    want = ops.moe_block(x, logits, b, None, b1, None, k, "softmax", quant_mode=0)
    assert torch.equal(low, want) and low.isfinite().all() and ops.device_status() == 0
