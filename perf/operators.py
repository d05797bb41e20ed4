"""The operators of a serving step: the MoE layer for a few tokens, and a projection with the adapters of many requests.

  moe    ops.moe_decode: from the activations x [T, H] of at most 32 tokens, the router's weights and the experts' weights to
         the layer's output [T, H]: logits = x Wr^T, the k largest, weights (softmax or sigmoid of the chosen, divided by their
         sum), out = sum over the chosen of weight * W2 (silu(G x) * (V x)), shared experts with weight 1. The experts' weights
         are bf16 or e4m3 with scales per tensor, per channel or per 128x128 block; the activations are not quantised.
  lora   ops.lora_linear: y = x W^T + bias + scale_a (x A_a^T) B_a^T, with the adapter a of each row's request; rows whose id is
         outside [0, L) have none.

Shapes: Mixtral-8x7B (H 4096, I 14336, 8 experts, top 2; its projections of queries, keys and values together 6144 rows),
one of eight ranks' share of DeepSeek-V3's experts (H 7168, I 2048, 32 experts, top 8, one shared), Qwen-MoE (H 2048, I 768,
128 experts, top 8), the wide bf16 shape of the reference's driver (2880 x 2880, 64 experts, top 3) and small odd models.
"""
import math

import torch

own = False

FP8 = torch.float8_e4m3fn
MIXTRAL = dict(H=4096, I=14336, E=8, k=2)
DEEPSEEK_RANK = dict(H=7168, I=2048, E=32, k=8)
QWEN = dict(H=2048, I=768, E=128, k=8)
WIDE = dict(H=2880, I=2880, E=64, k=3)
SMALL = dict(H=1024, I=2048, E=8, k=2)
QUANT = {"bf16": 0, "tensor": 256, "channel": 512, "block": 1024}


def _moe(quant, T, shape, *, scoring="softmax", shared=0):
    return dict(op="moe", quant=quant, T=T, scoring=scoring, shared=shared, **shape)


def _lora(T, N, K, L, R, requests, *, dtype="bf16", bias=False):
    return dict(op="lora", T=T, N=N, K=K, L=L, R=R, requests=requests, dtype=dtype, bias=bias)


def listed():
    return [
        # a few users of a small model on one card: latency of the whole layer
        dict(name="moe_small_block_5", **_moe("block", 5, SMALL)),
        # one user's next token, unquantised model
        dict(name="moe_bf16_1", **_moe("bf16", 1, MIXTRAL)),
        # the same model per-tensor FP8, a decode batch that hits every expert
        dict(name="moe_tensor_16", **_moe("tensor", 16, MIXTRAL)),
        # one rank's experts of a 256-expert model with its shared expert, a speculative batch
        dict(name="moe_block_8", **_moe("block", 8, DEEPSEEK_RANK, scoring="sigmoid", shared=1)),
        # many small experts, the largest batch of this path
        dict(name="moe_channel_32", **_moe("channel", 32, QWEN)),
        # odd row lengths, unquantised
        dict(name="moe_wide_bf16_3", **_moe("bf16", 3, WIDE)),
        # one user's next token through the output projection with that user's adapter
        dict(name="lora_1", **_lora(1, 4096, 4096, 8, 16, 1)),
        # a decode batch of as many tenants: queries, keys and values
        dict(name="lora_decode_64", **_lora(64, 6144, 4096, 64, 16, 64)),
        # a chunk of prefill beside decoding requests, fp16, high rank, with a bias
        dict(name="lora_chunk_333", **_lora(333, 2880, 2880, 32, 64, 40, dtype="fp16", bias=True)),
        # prefill of a few requests
        dict(name="lora_prefill_4096", **_lora(4096, 4096, 4096, 16, 32, 6)),
        # prefill of many requests through a shared expert's first projection, odd length
        dict(name="lora_prefill_8191", **_lora(8191, 4096, 7168, 64, 16, 24)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        quant = rng.choice(["bf16", "tensor", "channel", "block"])
        scoring = rng.choice(["softmax", "sigmoid"])
        T = _log_int(rng, 1, 32)
        if rng.random() < 0.5:
            shape = rng.choice([MIXTRAL, DEEPSEEK_RANK, QWEN, WIDE])
        else:  # odd models
            E = _log_int(rng, 3, 256)
            shape = dict(H=16 * _log_int(rng, 20, 250), I=16 * _log_int(rng, 12, 80), E=E, k=rng.randint(1, min(8, E)))
        return _moe(quant, T, shape, scoring=scoring, shared=rng.choice([0, 0, 1, 2]))
    T = _log_int(rng, 1, 8192)
    requests = T if rng.random() < 0.4 and T <= 512 else rng.randint(1, min(T, 48))
    return _lora(T, 8 * _log_int(rng, 40, 760), 8 * _log_int(rng, 40, 760), rng.randint(1, 64), rng.choice([8, 16, 24, 32, 64, 128]),
                 requests, dtype=rng.choice(["bf16", "bf16", "fp16"]), bias=rng.random() < 0.3)


# ---------------------------------------------------------------------------------------------------- inputs

def _quantise(w, quant):
    """(weights, scales) of bf16 weights [e, rows, cols]: e4m3 with amax / 448 of each expert, row or 128x128 block."""
    if quant == "bf16":
        return w, None
    e, rows, cols = w.shape
    if quant == "block":
        p = torch.nn.functional.pad(w, (0, -cols % 128, 0, -rows % 128)).float()
        p = p.view(e, p.shape[1] // 128, 128, p.shape[2] // 128, 128)
        s = p.abs().amax(dim=(2, 4), keepdim=True).clamp(min=1e-4) / 448
        q = (p / s).to(FP8).view(e, p.shape[1] * 128, p.shape[3] * 128)[:, :rows, :cols].contiguous()
        return q, s.view(e, p.shape[1], p.shape[3])
    f = w.float()
    s = f.abs().amax(dim=(1, 2) if quant == "tensor" else 2, keepdim=True).clamp(min=1e-4) / 448
    return (f / s).to(FP8), s.view(e) if quant == "tensor" else s.view(e, rows)


def _weights(g, E, rows, cols, quant):
    step = max(1, (1 << 27) // (rows * cols))
    parts = [_quantise(torch.randn(min(step, E - e), rows, cols, generator=g, device="cuda", dtype=torch.bfloat16).mul_(0.02), quant)
             for e in range(0, E, step)]
    if quant == "bf16":
        return torch.cat([q for q, _ in parts]), None
    return torch.cat([q.view(torch.uint8) for q, _ in parts]).view(FP8), torch.cat([s for _, s in parts])


def _request_ids(g, case):
    """Each row's adapter: the rows of a request stand together, the requests take the adapters in a random order, and every
    eighth request has none."""
    T, L, requests = case["T"], case["L"], case["requests"]
    cuts = torch.randperm(T - 1, generator=g, device="cuda")[:requests - 1] + 1
    request = torch.zeros(T, dtype=torch.int64, device="cuda")
    request[cuts] = 1
    request = request.cumsum(0)
    ids = torch.randperm(L, generator=g, device="cuda")[request % L]
    return torch.where(request % 8 == 7, -1, ids).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape, dtype=torch.bfloat16: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    if case["op"] == "moe":
        T, H, I, E = case["T"], case["H"], case["I"], case["E"]
        b, b_scale = _weights(g, E + case["shared"], 2 * I, H, case["quant"])
        b1, b1_scale = _weights(g, E + case["shared"], H, I, case["quant"])
        return dict(case=case, x=rand(T, H), w_router=rand(E, H).mul_(H ** -0.5), b=b, b_scale=b_scale, b1=b1, b1_scale=b1_scale)
    T, N, K, L, R = case["T"], case["N"], case["K"], case["L"], case["R"]
    dtype = torch.float16 if case["dtype"] == "fp16" else torch.bfloat16
    return dict(case=case, x=rand(T, K, dtype=dtype), w=rand(N, K, dtype=dtype).mul_(0.02),
                lora_a=rand(L, R, K, dtype=dtype).mul_(K ** -0.5), lora_b=rand(L, N, R, dtype=dtype).mul_(0.02),
                ids=_request_ids(g, case), scale=0.5 + 1.5 * torch.rand(L, generator=g, device="cuda"),
                bias=rand(N, dtype=torch.float32) if case["bias"] else None)


# ---------------------------------------------------------------------------------------------------- one pass

def _dequantised(w, scale, quant):
    w = w.float()
    if quant == "tensor":
        return w.mul_(scale[:, None, None])
    if quant == "channel":
        return w.mul_(scale[:, :, None])
    if quant == "block":
        rows, cols = torch.arange(w.shape[1], device=w.device) // 128, torch.arange(w.shape[2], device=w.device) // 128
        return w.mul_(scale[:, rows][:, :, cols])
    return w


def _moe_plain(st):
    """Every expert on every token, then the sum over the chosen: a token's weight of an expert that it did not choose masks the
    product out."""
    case, x = st["case"], st["x"].float()
    T, H, I, E, k, shared = (case[n] for n in ("T", "H", "I", "E", "k", "shared"))
    logits = x.double() @ st["w_router"].double().T  # chosen by value: 64 bits next to a border
    top, chosen = torch.sort(logits, dim=1, descending=True, stable=True)
    top, chosen = top[:, :k].float(), chosen[:, :k]
    score = torch.exp(top - top[:, :1]) if case["scoring"] == "softmax" else 1 / (1 + torch.exp(-top))
    weight = torch.zeros(T, E + shared, device=x.device)
    weight[:, E:] = 1
    weight.scatter_(1, chosen, score / score.sum(1, keepdim=True))
    h = (x @ _dequantised(st["b"], st["b_scale"], case["quant"]).view(-1, H).T).view(T, E + shared, 2, I)
    gate, value = h[:, :, 0], h[:, :, 1]
    act = torch.where(weight[:, :, None] > 0, weight[:, :, None] * gate / (1 + torch.exp(-gate)) * value, 0)
    y = torch.bmm(act.transpose(0, 1), _dequantised(st["b1"], st["b1_scale"], case["quant"]).transpose(1, 2))
    return y.sum(0).to(torch.bfloat16)


def _lora_plain(st):
    """The inner products of every adapter, of which each row keeps its own, then the same for the outer ones."""
    x, ids, L = st["x"].float(), st["ids"], st["lora_a"].shape[0]
    T, R = x.shape[0], st["lora_a"].shape[1]
    mine = (torch.arange(L, device=ids.device) == ids[:, None]) * st["scale"]  # [T, L]
    z = (x @ st["lora_a"].float().view(L * R, -1).T).view(T, L, R) * mine[:, :, None]
    y = x @ st["w"].float().T + z.view(T, L * R) @ st["lora_b"].float().permute(0, 2, 1).reshape(L * R, -1)
    if st["bias"] is not None:
        y += st["bias"]
    return y.to(st["x"].dtype)


def run(st):
    case = st["case"]
    if own:
        from dqmoe_b200 import ops
        if case["op"] == "moe":
            return ops.moe_decode(st["x"], st["w_router"], st["b"], st["b_scale"], st["b1"], st["b1_scale"], case["k"],
                                  scoring=case["scoring"], quant_mode=QUANT[case["quant"]], n_shared=case["shared"])
        return ops.lora_linear(st["x"], st["w"], st["lora_a"], st["lora_b"], st["ids"], scale=st["scale"], bias=st["bias"])
    return _moe_plain(st) if case["op"] == "moe" else _lora_plain(st)


# ---------------------------------------------------------------------------------------------------- what it takes

def work(case):
    if case["op"] == "moe":
        T, H, I, E, k, shared, quant = (case[n] for n in ("T", "H", "I", "E", "k", "shared", "quant"))
        hit = E * (1 - (1 - k / E) ** T) + shared  # experts that some token chooses, in the mean
        scales = {"bf16": 0, "tensor": 8, "channel": 4 * (2 * I + H), "block": 4 * (-(-2 * I // 128) * -(-H // 128) + -(-H // 128) * -(-I // 128))}
        expert = 3 * H * I * (2 if quant == "bf16" else 1) + scales[quant]
        return {"bytes": int(hit * expert + 2 * E * H + 4 * T * H), "flops": 6 * T * (k + shared) * H * I + 2 * T * E * H}
    T, N, K, L, R, requests = (case[n] for n in ("T", "N", "K", "L", "R", "requests"))
    used = len({i % L for i in range(requests) if i % 8 != 7})
    rows = T * sum(i % 8 != 7 for i in range(requests)) // requests
    return {"bytes": 2 * (T * K + N * K + used * R * (K + N) + T * N) + 4 * (T + L + (N if case["bias"] else 0)),
            "flops": 2 * T * N * K + 2 * rows * R * (K + N)}


# ---------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"].double()
    if case["op"] == "lora":
        y = x @ st["w"].double().T
        if st["bias"] is not None:
            y += st["bias"].double()
        for a in range(case["L"]):
            rows = torch.nonzero(st["ids"] == a).view(-1)
            if rows.numel():
                y[rows] += st["scale"][a].double() * (x[rows] @ st["lora_a"][a].double().T @ st["lora_b"][a].double().T)
        return y
    H, I, E, k = case["H"], case["I"], case["E"], case["k"]

    def expert(w, s, e):
        w = w[e].double()
        if s is None:
            return w
        if s.dim() < 3:
            return w * s[e].double().reshape(-1, 1)
        full = s[e].double().repeat_interleave(128, 0).repeat_interleave(128, 1)
        return w * full[:w.shape[0], :w.shape[1]]

    logits = x @ st["w_router"].double().T
    order = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :k]
    chosen = torch.zeros_like(logits, dtype=torch.bool).scatter_(1, order, True)
    score = torch.softmax(logits, 1) if case["scoring"] == "softmax" else torch.sigmoid(logits)
    score = torch.where(chosen, score, 0)
    score = score / score.sum(1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(E + case["shared"]):
        rows = torch.nonzero(chosen[:, e]).view(-1) if e < E else torch.arange(x.shape[0], device=x.device)
        if rows.numel():
            h = x[rows] @ expert(st["b"], st["b_scale"], e).T
            y = (torch.nn.functional.silu(h[:, :I]) * h[:, I:]) @ expert(st["b1"], st["b1_scale"], e).T
            out[rows] += y * (score[rows, e, None] if e < E else 1)
    return out
