"""The MoE layer for a few tokens (ops.moe_decode) against the same formulas in 64 bits.

Tolerances. The result is rounded to bf16: half a step, 2^-8 of the value. The intermediate is held to 2^-9 of each value (two e4m3 parts)
or better, so a result is off by at most 2^-9 of A = the sum of the magnitudes that it is added up from, if all of those errors
had one sign; fp32 sums and the split of x are below 2^-12 of A at these lengths. As a 2-norm over many values: errors of the rounding
are spread over +-2^-8, 2^-8 / sqrt 3 of it, and so are those of the split over +-2^-9 of independent terms: below 2^-8 in all.
"""
import pytest
import torch

from dqmoe_b200 import ops

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
MODES = {"bf16": 0, "tensor": 256, "channel": 512, "block": 1024}


def quantise(w, mode):
    if mode == "bf16":
        return w, None
    e, rows, cols = w.shape
    if mode == "block":
        p = torch.nn.functional.pad(w, (0, -cols % 128, 0, -rows % 128)).float()
        p = p.view(e, p.shape[1] // 128, 128, p.shape[2] // 128, 128)
        s = p.abs().amax(dim=(2, 4), keepdim=True).clamp(min=1e-4) / 448
        q = (p / s).to(FP8).view(e, p.shape[1] * 128, p.shape[3] * 128)[:, :rows, :cols].contiguous()
        return q, s.view(e, p.shape[1], p.shape[3])
    f = w.float()
    s = f.abs().amax(dim=(1, 2) if mode == "tensor" else 2, keepdim=True).clamp(min=1e-4) / 448
    return (f / s).to(FP8), s.reshape(e) if mode == "tensor" else s.reshape(e, rows)


def dequantise(w, s, mode):
    w = w.double()
    if mode == "bf16":
        return w
    if mode == "block":
        r = torch.arange(w.shape[1], device=w.device) // 128
        c = torch.arange(w.shape[2], device=w.device) // 128
        return w * s.double()[:, r][:, :, c]
    return w * s.double().reshape(w.shape[0], -1, 1)


def make(seed, mode, T, H, I, E, k, shared=0, router=torch.bfloat16, w_std=0.02):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    b, b_scale = quantise((rand(E + shared, 2 * I, H) * w_std).bfloat16(), mode)
    b1, b1_scale = quantise((rand(E + shared, H, I) * w_std).bfloat16(), mode)
    return dict(x=rand(T, H).bfloat16(), w_router=(rand(E, H) * H ** -0.5).to(router), b=b, b_scale=b_scale, b1=b1, b1_scale=b1_scale, k=k,
                quant_mode=MODES[mode], n_shared=shared)


def reference(a, scoring="softmax"):
    """(result, sum of the magnitudes it is added up from), both in 64 bits."""
    mode = {v: n for n, v in MODES.items()}[a["quant_mode"]]
    x = a["x"].double()
    E, k = a["w_router"].shape[0], a["k"]
    logits = x @ a["w_router"].double().T
    order = torch.argsort(logits, dim=1, descending=True, stable=True)
    if k < E:
        gap = logits.gather(1, order[:, k - 1:k + 1])
        assert (gap[:, 0] - gap[:, 1]).min() > 1e-5  # nothing here hangs on the last bits of a logit
    chosen = order[:, :k]
    score = torch.softmax(logits, 1).gather(1, chosen) if scoring == "softmax" else torch.sigmoid(logits.gather(1, chosen))
    weight = torch.zeros(x.shape[0], E + a["n_shared"], dtype=torch.float64, device=x.device)
    weight[:, E:] = 1
    weight.scatter_(1, chosen, score / score.sum(1, keepdim=True))
    out, size = torch.zeros_like(x), torch.zeros_like(x)
    for e in range(E + a["n_shared"]):
        rows = torch.nonzero(weight[:, e]).view(-1)
        if not rows.numel():
            continue
        w = dequantise(a["b"][e:e + 1], None if a["b_scale"] is None else a["b_scale"][e:e + 1], mode)[0]
        w1 = dequantise(a["b1"][e:e + 1], None if a["b1_scale"] is None else a["b1_scale"][e:e + 1], mode)[0]
        h = x[rows] @ w.T
        I = w1.shape[1]
        act = torch.nn.functional.silu(h[:, :I]) * h[:, I:] * weight[rows, e, None]
        out[rows] += act @ w1.T
        size[rows] += act.abs() @ w1.abs().T
    return out, size


def check(out, ref, size):
    assert ops.device_status() == 0
    off = (out.double() - ref).abs()
    assert (off <= 2.0 ** -8 * ref.abs() + (2.0 ** -9 + 2.0 ** -12) * size).all(), float((off / size).max())
    rel = float(off.norm() / ref.norm())
    assert rel <= 2.0 ** -8, rel


SHAPES = [  # T, H, I, E, k, shared, scoring
    (1, 256, 128, 4, 2, 0, "softmax"), (5, 1024, 2048, 8, 2, 0, "softmax"), (8, 272, 208, 5, 5, 0, "sigmoid"),
    (9, 640, 336, 3, 1, 1, "softmax"), (16, 1040, 64, 20, 3, 2, "sigmoid"), (17, 16, 16, 1, 1, 0, "softmax"),
    (32, 2048, 768, 128, 8, 0, "softmax"), (31, 144, 1040, 300, 8, 1, "sigmoid"), (2, 2880, 2880, 6, 3, 0, "softmax"),
    (32, 512, 256, 40, 32, 0, "softmax"), (1, 7168, 2048, 16, 8, 1, "sigmoid"), (24, 4096, 1008, 8, 2, 0, "softmax"),
]


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("T,H,I,E,k,shared,scoring", SHAPES)
def test_against_64_bits(mode, T, H, I, E, k, shared, scoring):
    a = make(7 * T + H + I, mode, T, H, I, E, k, shared)
    ref, size = reference(a, scoring)
    need = ops.moe_decode_workspace_bytes(T, H, I, E, k, shared, MODES[mode])
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")  # what stands in a workspace is of no consequence: NaN, for one
    out = torch.full((T + 1, H), -7.0, dtype=torch.bfloat16, device="cuda")
    ops.moe_decode(**a, scoring=scoring, workspace=ws, out=out[:T])
    check(out[:T], ref, size)
    assert (out[T] == -7).all()
    again = ops.moe_decode(**a, scoring=scoring, workspace=ws)
    assert torch.equal(again, out[:T])  # whichever block finishes a tile


@pytest.mark.parametrize("mode", ["bf16", "block"])
def test_fp32_router(mode):
    a = make(3, mode, 6, 384, 256, 12, 4, router=torch.float32)
    check(ops.moe_decode(**a), *reference(a))


def test_agrees_with_the_block_on_its_own_logits():
    """bf16 weights: the same layer as moe_block on the same logits, which rounds each product and the intermediate to bf16."""
    a = make(5, "bf16", 12, 1024, 512, 8, 2)
    logits = a["x"].float() @ a["w_router"].float().T
    block = ops.moe_block(a["x"], logits, a["b"], None, a["b1"], None, 2, quant_mode=0)
    out = ops.moe_decode(**a)
    assert float((out.double() - block.double()).norm() / out.double().norm()) < 4 * 2.0 ** -8


@pytest.mark.parametrize("mode", list(MODES))
def test_tokens_do_not_touch_each_other(mode):
    """A NaN in one token, and an expert full of NaN that another token does not choose, leave the others bit for bit."""
    a = make(11, mode, 7, 512, 384, 6, 2, shared=1)
    clean = ops.moe_decode(**a)
    logits = a["x"].double() @ a["w_router"].double().T
    chosen = torch.topk(logits, 2, dim=1).indices
    a["x"][3, 5] = float("nan")
    out = ops.moe_decode(**a)
    keep = torch.tensor([t for t in range(7) if t != 3], device="cuda")
    assert torch.equal(out[keep], clean[keep]) and out[3].isnan().all()
    a["x"][3, 5] = 0
    victim = int(chosen[0, 0])
    if mode == "bf16":
        a["b"][victim] = float("nan")
        a["b1"][victim] = float("inf")
    else:
        a["b"].view(torch.uint8)[victim] = 0x7f
        a["b1"].view(torch.uint8)[victim] = 0x7f
    out = ops.moe_decode(**a)
    now = torch.topk(a["x"].double() @ a["w_router"].double().T, 2, dim=1).indices
    spared = torch.tensor([t for t in range(7) if t != 3 and not (now[t] == victim).any()], device="cuda")
    assert spared.numel() and torch.equal(out[spared], clean[spared])
    assert out[0].isnan().all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("mode", ["bf16", "channel"])
def test_masked_logits(mode):
    """Tokens whose logits are all NaN have no expert: NaN for them alone; tokens of zeros (all logits 0) take the lowest ids."""
    a = make(13, mode, 4, 256, 128, 5, 2)
    a["x"][1] = 0
    out = ops.moe_decode(**a)
    assert (out[1] == 0).all()
    a["x"][0] = float("nan")
    a["x"][2] = float("nan")
    a["x"][3] = float("nan")
    a["x"][1] = float("nan")
    out = ops.moe_decode(**a)  # no expert is hit at all
    assert out.isnan().all() and ops.device_status() == 0


@pytest.mark.parametrize("mode", ["tensor", "block"])
def test_small_and_large_values_of_a_group(mode):
    """Values 2^-13 below their group's largest are still exact, smaller ones are off by 2^-21 of it."""
    a = make(17, mode, 8, 512, 256, 4, 2)
    a["x"][:, ::2] *= 2.0 ** -12
    a["x"][:, 1::4] *= 2.0 ** 20
    a["x"][2] *= 2.0 ** -60
    a["x"][4] *= 2.0 ** -120
    keep = torch.tensor([0, 1, 3, 5, 6, 7], device="cuda")
    a["x"] = a["x"].contiguous()
    a["w_router"] = (a["w_router"].float() * 2.0 ** -14).bfloat16()
    ref, size = reference({**a, "x": a["x"][keep]})
    out = ops.moe_decode(**a)
    check(out[keep], ref, size)
    assert out.isfinite().all()


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("T,H,I,E,k,shared", [(1, 1024, 2048, 8, 2, 0), (5, 528, 272, 6, 3, 1), (16, 2048, 768, 24, 4, 0), (32, 1024, 512, 40, 8, 2)])
def test_the_workspace_is_all_that_it_needs(mode, T, H, I, E, k, shared):
    need = ops.moe_decode_workspace_bytes(T, H, I, E, k, shared, MODES[mode])
    ws = torch.full((need + (1 << 20),), 0xa5, dtype=torch.uint8, device="cuda")
    ws[:need] = 0xff  # NaN, as floats
    a = make(61 + T, mode, T, H, I, E, k, shared)
    out = ops.moe_decode(**a, workspace=ws[:need])
    check(out, *reference(a))
    assert (ws[need:] == 0xa5).all()


def test_captured_and_replayed_on_another_stream():
    a = make(19, "block", 8, 1024, 512, 16, 4, shared=1)
    ws = torch.empty(ops.moe_decode_workspace_bytes(8, 1024, 512, 16, 4, 1, 1024), dtype=torch.uint8, device="cuda")
    out = torch.empty(8, 1024, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.moe_decode(**a, workspace=ws, out=out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for _ in range(3):  # layers back to back on one workspace
            ops.moe_decode(**a, workspace=ws, out=out)
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(100 + seed)
        a["x"].copy_(torch.randn(8, 1024, generator=g, device="cuda").bfloat16())
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        check(out, *reference(a))


def test_two_streams_at_once():
    """Calls that overlap on the GPU, each with a workspace of its own."""
    calls = [make(23 + i, m, 16, 2048, 768, 32, 8) for i, m in enumerate(["bf16", "block", "channel", "tensor"])]
    want = [ops.moe_decode(**a) for a in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(5):
        for i, (a, s) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.moe_decode(**a))
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


def test_a_step_after_a_step():
    """Layers with a residual that read one another's output without waiting, through one workspace, with calls of other sizes between."""
    a = make(29, "channel", 4, 512, 256, 8, 2, w_std=0.1)
    other = make(30, "channel", 32, 512, 512, 24, 4)
    size = max(ops.moe_decode_workspace_bytes(4, 512, 256, 8, 2, 0, 512), ops.moe_decode_workspace_bytes(32, 512, 512, 24, 4, 0, 512))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    x = a["x"]
    seen = []
    for _ in range(6):
        y = ops.moe_decode(**{**a, "x": x}, workspace=ws)
        ops.moe_decode(**other, workspace=ws)
        seen.append((x, y))
        x = a["x"] + y / (1 + y.abs().amax(dim=1, keepdim=True))  # the layer alone is quadratic in x and would leave the type's range
    for x, y in seen:
        check(y, *reference({**a, "x": x}))


@pytest.mark.parametrize("T", [1, 8, 16, 32])
@pytest.mark.parametrize("mode", list(MODES))
def test_many_calls_without_waiting(mode, T):
    """The next call's blocks take over an SM as soon as this one's leave it."""
    a = make(37, mode, T, 2048, 768, 128, 8)
    want = ops.moe_decode(**a)
    torch.cuda.synchronize()
    outs = [ops.moe_decode(**a) for _ in range(40)]
    assert ops.device_status() == 0
    assert all(torch.equal(o, want) for o in outs)


def test_empty_batch():
    a = make(31, "block", 3, 256, 128, 4, 2)
    out = ops.moe_decode(**{**a, "x": a["x"][:0]})
    assert out.shape == (0, 256)
