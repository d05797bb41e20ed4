"""The projection with adapters (ops.lora_linear) on both sides of 32 MiB of A that the rows of a batch read, where up to 256 rows go from a block
per row and 16 ranks to tiles of 64 rows on the tensor core: tiles that are not full, the smallest ones, one to four of them, with a cluster for
each slice of K and several clusters that share a tile's adapters.

Tolerance, h = half a step of the type, z = scale * (x A^T): the result and each z are rounded once; fp32 sums of K products, of which 16 or more are
added at once, are off by (K / 16 + 8) 2^-24 of the sum of their magnitudes at most.
"""
import pytest
import torch

from dqmoe_b200 import ops
from test_gpu_lora import TYPES, make

pytestmark = pytest.mark.gpu

LIMIT = 32 << 20
SHAPES = [  # T, N, K, L, R; tiles of 64 rows unless marked
    (20, 256, 8192, 20, 128), (40, 136, 6080, 6, 128), (65, 384, 4096, 40, 128), (64, 256, 8192, 64, 40), (63, 128, 8200, 3, 72), (129, 264, 8184, 5, 24),
    (256, 256, 4096, 64, 16),  # a block per row: 32 MiB
    (256, 256, 4104, 64, 16), (255, 128, 8264, 17, 8),
    (255, 128, 8224, 17, 8),   # a block per row: 32.0 MiB
    (2, 64, 65544, 2, 128), (1, 64, 131072, 2, 128),  # the last one a block per row: 32 MiB
    (1, 64, 131080, 2, 128),
]


def test_the_shapes_lie_on_both_sides():
    rows = [T * R * K * 2 <= LIMIT for T, N, K, L, R in SHAPES]
    assert [i for i, r in enumerate(rows) if r] == [6, 9, 11]


@pytest.mark.parametrize("ids", ["random", 1, 30, "none"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,N,K,L,R", SHAPES)
def test_against_64_bits(T, N, K, L, R, dtype, ids):
    a = make(T + K, T, N, K, L, R, dtype, ids, bias=T % 2 == 0, scale=T % 3 != 0)
    ws = torch.full((ops.lora_linear_workspace_bytes(T, N, K, L, R),), 0xff, dtype=torch.uint8, device="cuda")  # NaN, as floats
    out = torch.full((T + 1, N), -7.0, dtype=TYPES[dtype][0], device="cuda")
    ops.lora_linear(**a, out=out[:T], workspace=ws)
    assert ops.device_status() == 0 and (out[T] == -7).all()
    x, w, h = a["x"].double(), a["w"].double(), TYPES[dtype][1]
    y, size, D = x @ w.T, x.abs() @ w.abs().T, torch.zeros(T, N, dtype=torch.float64, device="cuda")
    if a["bias"] is not None:
        y += a["bias"].double()
        size += a["bias"].double().abs()
    for i in range(L):
        rows = torch.nonzero(a["ids"] == i).view(-1)
        if rows.numel():
            s, A, B = 1.0 if a["scale"] is None else float(a["scale"][i]), a["lora_a"][i].double(), a["lora_b"][i].double()
            z = s * (x[rows] @ A.T)
            y[rows] += z @ B.T
            D[rows] += z.abs() @ B.abs().T
            size[rows] += s * (x[rows].abs() @ A.abs().T) @ B.abs().T
    off = (out[:T].double() - y).abs()
    assert (off <= h * (y.abs() + D) + (K / 16 + 8) * 2.0 ** -24 * (size + D)).all(), float(off.norm() / y.norm())
    assert float(off.norm() / y.norm()) <= h
    assert torch.equal(ops.lora_linear(**a), out[:T])
