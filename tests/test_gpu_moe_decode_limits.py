"""moe_decode where an expert's intermediate leaves fp32's range: what dqmoe.h says of the tokens that chose it, and nothing for the others."""
import pytest
import torch

import test_gpu_moe_decode as moe
from dqmoe_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [7, 30])
@pytest.mark.parametrize("mode", list(moe.MODES))
def test_an_intermediate_beyond_fp32(mode, T):
    a = moe.make(101, mode, T, 512, 384, 6, 2)
    clean = ops.moe_decode(**a)
    victim = int(torch.topk(a["x"][0].double() @ a["w_router"].double().T, 2).indices[0])
    if mode == "bf16":
        a["b"][victim] *= 2.0 ** 100  # gate and value of some 2^98: their product is infinite
    else:
        a["b_scale"].view(6, -1)[victim] *= 2.0 ** 100
    out = ops.moe_decode(**a)
    chosen = torch.topk(a["x"].double() @ a["w_router"].double().T, 2, dim=1).indices
    hit = (chosen == victim).any(1)
    assert ops.device_status() == 0 and hit.any() and (~hit).any()
    assert torch.equal(out[~hit], clean[~hit])
    if mode == "bf16":
        assert not out[hit].isfinite().any()
    else:
        assert out[hit].isnan().all()
