"""The projection with adapters (ops.lora_linear) where scale * (x A^T) lies near the ends of fp16's range, against the formula in 64 bits.

Tolerance, h = half a step of the type (fp16 2^-11, bf16 2^-8), z = scale * (x A^T), D = sum |z| |B| per result:
  - the result is rounded once, off by h of its value, or, where it is not a normal number of fp16, by 2^-25;
  - each z is rounded once, off by h of its value, or, where what is stored is not normal, by 2^-25. A row is stored as it is only if its largest |z|
    is R 2^-14 or more: R such errors then come to R 2^-25 <= h max |z|. A row with a power of two has its largest at 2^14 or more: less still.
    All |B| of an adapter here lie within [b, 2 b], so these errors end as 2 h max |z| b <= 2 h D at most;
  - fp32 sums of K products, 16 or more of which are added at once (by the tensor core, or by 32 lanes each for itself), are off by (K / 16 + 8)
    2^-24 of the sum of their magnitudes at most; of the R products alike.
"""
import pytest
import torch

from dqmoe_b200 import ops
from test_gpu_lora import make

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def check(out, a):
    """w is zero in all of these: the adapters' part alone."""
    assert ops.device_status() == 0
    x, R, K = a["x"].double(), a["lora_a"].shape[1], a["lora_a"].shape[2]
    h = HALF_STEP[out.dtype]
    y, D, inner = (torch.zeros(out.shape, dtype=torch.float64, device="cuda") for _ in range(3))
    for i in range(a["lora_a"].shape[0]):
        rows = torch.nonzero(a["ids"] == i).view(-1)
        if rows.numel():
            A, B, s = a["lora_a"][i].double(), a["lora_b"][i].double(), float(a["scale"][i])
            z = s * (x[rows] @ A.T)
            y[rows], D[rows], inner[rows] = z @ B.T, z.abs() @ B.abs().T, s * (x[rows].abs() @ A.abs().T) @ B.abs().T
    off = (out.double() - y).abs()
    bound = h * (y.abs() + 3 * D) + (K / 16 + 8) * 2.0 ** -24 * inner + (R / 16 + 8) * 2.0 ** -24 * D + (2.0 ** -25 if out.dtype == torch.float16 else 0)
    assert (off <= bound).all(), (float((off - bound).max()), float(off.norm() / y.norm()))


def small_inner(seed, T, N, K, L, R, run, exponent, dtype="fp16"):
    """z of some 2^exponent in each row with an adapter, B so large that the adapters' part is of order one; no projection beside it."""
    a = make(seed, T, N, K, L, R, dtype, run)
    a["w"].zero_()
    magnitude = 2.0 ** min(-exponent, 12)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    sign = torch.randint(0, 2, (L, N, R), generator=g, device="cuda") * 2 - 1
    a["lora_b"] = ((1 + torch.rand(L, N, R, generator=g, device="cuda")) * sign * magnitude).to(a["x"].dtype)
    a["scale"] = torch.full((L,), 2.0 ** exponent, device="cuda")
    return a


# both forms of shrink (a block per row up to 32 MiB of A read, tiles beyond), both forms of the products (runs of whole chunks, rows in any order)
FORMS = [(48, 264, 512, 5, 16), (200, 256, 640, 4, 128), (600, 384, 512, 3, 8), (1221, 3280, 1280, 2, 8), (40, 256, 8192, 6, 64)]


@pytest.mark.parametrize("run", [512, 3])
@pytest.mark.parametrize("exponent", [-6, -12, -16, -20, -24, -40])
@pytest.mark.parametrize("T,N,K,L,R", FORMS)
def test_inner_values_below_fp16(T, N, K, L, R, exponent, run):
    a = small_inner(71, T, N, K, L, R, run, exponent)
    out = ops.lora_linear(**a)
    check(out, a)
    if exponent >= -20:  # what the output can represent is there
        assert (out[a["ids"] >= 0] != 0).float().mean() > 0.9


@pytest.mark.parametrize("run", [512, 3])
@pytest.mark.parametrize("T,N,K,L,R", [(48, 264, 512, 5, 16), (600, 384, 512, 6, 32)])
def test_rows_of_all_magnitudes_side_by_side(T, N, K, L, R, run):
    """Adapters whose z are small, ordinary and beyond the range, and one that is zero, in one batch."""
    a = small_inner(73, T, N, K, L, R, run, 0)
    for i, exponent in enumerate([-20, 0, 20, -30, -11, 3][:L]):
        a["scale"][i] = 2.0 ** exponent
        a["lora_b"][i] *= 2.0 ** -exponent if exponent > 0 else 2.0 ** min(-exponent, 11)
    a["lora_a"][1] = 0
    out = ops.lora_linear(**a)
    check(out, a)
    assert (out[a["ids"] == 1] == 0).all()


@pytest.mark.parametrize("run", [512, 3])
def test_small_values_of_bf16(run):
    """bf16 has fp32's range: nothing is lost there."""
    a = small_inner(75, 300, 256, 512, 4, 16, run, -40, "bf16")
    a["scale"].fill_(2.0 ** -100)
    a["lora_b"] *= 2.0 ** 88
    check(ops.lora_linear(**a), a)
