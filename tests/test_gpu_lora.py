"""The shared projection with adapters (ops.lora_linear) against the same formula in 64 bits.

Tolerances, h = half a step of the type (bf16 2^-8, fp16 2^-11): the result is rounded once (h of the value), x A^T may be rounded once (h
of each of the products that make up the adapter's part, D = the sum of their magnitudes), and a sum of up to 8192 products in 32 bits
is off by less than 2^-14 of the sum of their magnitudes. As a 2-norm over many values these are independent: below h in all as long as the adapter's
part is not larger than the projection's.
"""
import pytest
import torch

from dqmoe_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = {"bf16": (torch.bfloat16, 2.0 ** -8), "fp16": (torch.float16, 2.0 ** -11)}


def make(seed, T, N, K, L, R, dtype="bf16", ids="random", bias=False, scale=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    t = TYPES[dtype][0]
    if ids == "random":
        i = torch.randint(-1, L + 1, (T,), generator=g, device="cuda")  # L itself is outside, too
    elif ids == "none":
        i = torch.full((T,), -1, device="cuda")
    else:  # runs of that many rows
        run = torch.randint(0, L, (T // ids + 1,), generator=g, device="cuda")
        i = run.repeat_interleave(ids)[:T]
    return dict(x=rand(T, K).to(t), w=(rand(N, K) * 0.02).to(t), lora_a=(rand(L, R, K) * K ** -0.5).to(t),
                lora_b=(rand(L, N, R) * 0.05 * R ** -0.5).to(t), ids=i.to(torch.int32),
                scale=0.5 + torch.rand(L, generator=g, device="cuda") if scale else None, bias=rand(N) if bias else None)


def reference(a):
    """(result, magnitudes of the projection's sum, of the adapters') in 64 bits."""
    x, w = a["x"].double(), a["w"].double()
    y, size, mine = x @ w.T, x.abs() @ w.abs().T, torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    if a["bias"] is not None:
        y += a["bias"].double()
        size += a["bias"].double().abs()
    for i in range(a["lora_a"].shape[0]):
        rows = torch.nonzero(a["ids"] == i).view(-1)
        if rows.numel():
            s = 1.0 if a["scale"] is None else float(a["scale"][i])
            z = s * (x[rows] @ a["lora_a"][i].double().T)
            b = a["lora_b"][i].double()
            y[rows] += z @ b.T
            mine[rows] += z.abs() @ b.abs().T
    return y, size, mine


def check(out, a, dtype="bf16"):
    assert ops.device_status() == 0
    y, size, mine = reference(a)
    h = TYPES[dtype][1]
    off = (out.double() - y).abs()
    assert (off <= h * (y.abs() + mine) + 2.0 ** -14 * (size + mine)).all(), float((off - h * y.abs()).max())
    rel = float(off.norm() / y.norm())
    assert rel <= h, rel


SHAPES = [  # T, N, K, L, R, ids
    (1, 128, 64, 1, 8, "random"), (1, 4096, 4096, 8, 16, 1), (3, 136, 72, 4, 8, "random"), (16, 1000, 328, 5, 24, 1), (17, 513, 520, 64, 16, "random"),
    (33, 2048, 1024, 3, 64, "random"), (64, 6144, 4096, 64, 16, 1), (65, 200, 2880, 9, 40, 7), (100, 8, 8, 2, 8, "random"),
    (128, 1536, 512, 40, 128, 1), (129, 1536, 512, 40, 128, 1), (200, 640, 1032, 4, 72, 200), (256, 384, 256, 2, 16, 256), (257, 1, 256, 2, 16, 256),
    (333, 2880, 2880, 32, 64, 9), (512, 256, 4096, 7, 32, 100), (1000, 512, 512, 3, 8, "none"), (1023, 896, 640, 6, 96, 300), (2048, 4096, 512, 5, 16, 700),
    (4099, 1152, 192, 33, 48, 1000), (700, 3000, 64, 64, 8, "random"), (224, 384, 256, 2, 16, 100), (225, 384, 200, 5, 128, 3),
    (481, 256, 128, 8, 72, 16), (960, 128, 64, 3, 64, 17),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,N,K,L,R,ids", SHAPES)
def test_against_64_bits(dtype, T, N, K, L, R, ids):
    a = make(T + N + K, T, N, K, L, R, dtype, ids, bias=T % 2 == 0, scale=T % 3 != 0)
    need = ops.lora_linear_workspace_bytes(T, N, K, L, R)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")  # NaN, as floats
    out = torch.full((T + 1, N), -7.0, dtype=TYPES[dtype][0], device="cuda")
    ops.lora_linear(**a, out=out[:T], workspace=ws)
    check(out[:T], a, dtype)
    assert (out[T] == -7).all()
    assert torch.equal(ops.lora_linear(**a), out[:T])  # whichever block finishes a tile


PAIRS = [  # large enough for pairs of blocks: whole tiles in one round and in two, split ones, a last tile of one block, ragged rows
    (1214, 3096, 1280, 5, 16, 400), (2089, 3336, 1024, 9, 32, 37), (2413, 2312, 2048, 6, 64, 300), (2661, 1720, 2048, 40, 128, "random"),
    (2989, 2480, 1024, 64, 8, 1), (1221, 3280, 1280, 3, 24, "none"),
    (1282, 3384, 2400, 6, 16, 300), (3899, 1200, 2048, 20, 64, 61), (2916, 656, 4096, 8, 40, "random"),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,N,K,L,R,ids", PAIRS)
def test_large_batches_against_64_bits(dtype, T, N, K, L, R, ids):
    test_against_64_bits(dtype, T, N, K, L, R, ids)


@pytest.mark.parametrize("T", [5, 90, 400])
def test_rows_that_lie_apart(T):
    """x as a slice of a wider matrix, y into one: what stands beside it stays."""
    a = make(5, T, 264, 320, 6, 16)
    wide = torch.randn(T, 1000, device="cuda").bfloat16()
    wide[:, 8:328] = a["x"]
    out = torch.full((T, 777), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.lora_linear(**{**a, "x": wide[:, 8:328]}, out=out[:, 101:365])
    check(out[:, 101:365], a)
    assert (out[:, :101] == 3).all() and (out[:, 365:] == 3).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,run", [(40, 1), (300, 5), (600, 300)])
def test_rows_do_not_see_other_adapters(T, run, dtype):
    """An adapter full of infinities and NaN changes the rows that have it, and no others."""
    a = make(7, T, 384, 512, 8, 16, dtype, run)
    a["ids"][::11] = -1
    clean = ops.lora_linear(**a)
    bad = int(a["ids"][1])
    a["lora_a"][bad] = float("nan")
    a["lora_b"][bad, :, 3] = float("inf")
    out = ops.lora_linear(**a)
    hit = a["ids"] == bad
    assert torch.equal(out[~hit], clean[~hit]) and out[hit].isnan().all() and ops.device_status() == 0
    a["x"][2] = float("inf")  # one row of x
    again = ops.lora_linear(**a)
    rest = ~hit
    rest[2] = False
    assert torch.equal(again[rest], clean[rest]) and not again[2].isfinite().any()


@pytest.mark.parametrize("run", [512, 3])
def test_inner_values_beyond_fp16(run):
    """x A^T may pass fp16's range where the result does not."""
    a = make(9, 512, 256, 512, 2, 8, "fp16", run)
    a["lora_a"].mul_(3e4)
    a["lora_b"].mul_(1e-4)
    a["scale"].fill_(4.0)
    assert float((a["x"].double() @ a["lora_a"][int(a["ids"][0])].double().T).abs().max()) * 4 > 65504
    check(ops.lora_linear(**a), a, "fp16")


@pytest.mark.parametrize("run", [512, 3])
def test_inner_values_beyond_fp16_in_large_batches(run):
    a = make(31, 1221, 3280, 1280, 2, 8, "fp16", run)
    a["lora_a"].mul_(3e4)
    a["lora_b"].mul_(1e-4)
    a["scale"].fill_(4.0)
    a["lora_a"][1].mul_(1e-4)  # one adapter stays in range: chunks with and without powers of two
    check(ops.lora_linear(**a), a, "fp16")


def test_large_batches_do_not_see_other_adapters():
    a = make(33, 1214, 3096, 1280, 8, 16, "bf16", 150)
    a["ids"][::97] = -1
    clean = ops.lora_linear(**a)
    bad = int(a["ids"][1])
    a["lora_b"][bad, :, 3] = float("inf")
    a["lora_a"][bad] = float("nan")
    out = ops.lora_linear(**a)
    hit = a["ids"] == bad
    assert torch.equal(out[~hit], clean[~hit]) and out[hit].isnan().all() and ops.device_status() == 0


def test_one_workspace_for_all_batches():
    """A workspace for the longest batch serves all, one call after the other without waiting."""
    T, N, K, L, R = 1300, 1536, 512, 12, 32
    ws = torch.full((ops.lora_linear_workspace_bytes(T, N, K, L, R),), 0xff, dtype=torch.uint8, device="cuda")
    a = make(35, T, N, K, L, R, ids=5)
    got = []
    for t in (1300, 1, 17, 640, 64, 255, 257, 1300, 31, 900):
        part = {**a, "x": a["x"][:t], "ids": a["ids"][:t]}
        got.append((part, ops.lora_linear(**part, workspace=ws)))
    for part, out in got:
        check(out, part)


@pytest.mark.parametrize("T,N,K,L,R,ids", [(1, 4096, 4096, 8, 16, 1), (48, 2048, 1024, 16, 128, 1), (333, 2880, 512, 32, 64, 9), (1214, 3096, 1280, 5, 16, 400)])
def test_the_workspace_is_all_that_it_needs(T, N, K, L, R, ids):
    need = ops.lora_linear_workspace_bytes(T, N, K, L, R)
    ws = torch.full((need + (1 << 20),), 0xa5, dtype=torch.uint8, device="cuda")
    a = make(51, T, N, K, L, R, ids=ids)
    check(ops.lora_linear(**a, workspace=ws[:need]), a)
    assert (ws[need:] == 0xa5).all()


def test_adapters_far_apart():
    """Adapters whose B begins behind 2^31 elements."""
    T, N, K, L, R = 40, 28672, 64, 600, 128
    assert (L - 1) * N * R > 1 << 31
    b = torch.empty(L, N, R, dtype=torch.bfloat16, device="cuda")
    a = make(53, T, N, K, 3, R, ids=13)  # as three adapters ...
    b[0], b[1], b[L - 1] = a["lora_b"][0], a["lora_b"][1], a["lora_b"][2]
    far_a = torch.zeros(L, R, K, dtype=torch.bfloat16, device="cuda")
    far_a[0], far_a[1], far_a[L - 1] = a["lora_a"][0], a["lora_a"][1], a["lora_a"][2]
    far_scale = torch.ones(L, device="cuda")
    far_scale[[0, 1, L - 1]] = a["scale"]
    for ids in (a["ids"], torch.arange(T, dtype=torch.int32, device="cuda") % 3):  # direct products and mixed ones
        near = {**a, "ids": ids}
        far = {**near, "ids": torch.where(ids == 2, L - 1, ids).int(), "lora_a": far_a, "lora_b": b, "scale": far_scale}
        out = ops.lora_linear(**far)
        check(out, near)
        assert torch.equal(out, ops.lora_linear(**near))


def test_captured_and_replayed():
    a = make(11, 48, 1024, 768, 16, 16)
    ws = torch.empty(ops.lora_linear_workspace_bytes(48, 1024, 768, 16, 16), dtype=torch.uint8, device="cuda")
    out = torch.empty(48, 1024, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.lora_linear(**a, out=out, workspace=ws)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for _ in range(3):
            ops.lora_linear(**a, out=out, workspace=ws)
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(200 + seed)
        a["x"].copy_(torch.randn(48, 768, generator=g, device="cuda").bfloat16())
        a["ids"].copy_(torch.randint(-1, 16, (48,), generator=g, device="cuda"))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        check(out, a)


def test_streams_at_once():
    calls = [make(13 + i, *s) for i, s in enumerate([(64, 2048, 2048, 16, 16), (300, 1024, 1024, 4, 32), (1, 4096, 2048, 4, 8), (1500, 512, 512, 8, 64)])]
    want = [ops.lora_linear(**a) for a in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(5):
        for i, (a, s) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.lora_linear(**a))
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


def test_large_batches_at_once():
    """Pairs of blocks of two calls and a decode batch between them compete for the SMs."""
    calls = [make(41 + i, *s) for i, s in enumerate([(1214, 3096, 1280, 5, 16), (40, 2048, 1024, 16, 16), (2413, 2312, 2048, 6, 64)])]
    want = [ops.lora_linear(**a) for a in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(6):
        for i, (a, s) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.lora_linear(**a))
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


@pytest.mark.parametrize("mode", ["bf16", "block"])
def test_a_serving_step(mode):
    """A decode batch of ten tenants: the output projection with each one's adapter, a residual, then the MoE layer with its residual,
    twice in a row without waiting and through one workspace."""
    import test_gpu_moe_decode as moe
    T, H, K, L, R = 10, 512, 640, 6, 16
    p = make(21, T, H, K, L, R)
    m = moe.make(22, mode, T, H, 384, 12, 3, shared=1)
    size = max(ops.lora_linear_workspace_bytes(T, H, K, L, R), ops.moe_decode_workspace_bytes(T, H, 384, 12, 3, 1, moe.MODES[mode]))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    h, steps = m["x"], []
    for _ in range(2):
        y = ops.lora_linear(**p, workspace=ws)
        x = h + y
        o = ops.moe_decode(**{**m, "x": x}, workspace=ws)
        steps.append((y, x, o))
        h = x + o
    for y, x, o in steps:
        check(y, p)
        moe.check(o, *moe.reference({**m, "x": x}))


def test_empty_batch():
    a = make(23, 2, 64, 64, 2, 8)
    assert ops.lora_linear(**{**a, "x": a["x"][:0], "ids": a["ids"][:0]}).shape == (0, 64)
