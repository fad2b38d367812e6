"""The operators between and around the adapter linears of a transformer block, and their plain forms.

  rotate_axes      rotary positions with several axes (time, row, column)
  qk_norm_rotate   RMS norm of each head of q and k, with that rotation in the same pass
  int8_linear      8-bit integer linear, one scale per token and one per output channel, with the
                   adapters' rank-16 expand added to it

``own`` false: elementary torch operations in 32 bits (the angles in 64), rounded once at the
end.  ``own`` true: the calls a user makes of ``lithe_b200.kernels``.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
RANK = 16
#: Widths, heads and batch of the transformer that this repository serves (lithe_b200/flux_model.py, bench.py).
HIDDEN, HEADS, HEAD_DIM, BATCH, TEXT, IMAGE = 3072, 24, 128, 14, 512, 4096


def _rotate(name, **kw):
    return {"name": name, "op": "rotate", "batch": 1, "tokens": 1, "heads": HEADS, "dim": HEAD_DIM,
            "axes": "16,56,56", "theta": 10000.0, "pairing": "interleaved", "type": "bf16", "fused": False,
            "far": 64, "grid": 0, **kw}


def _norm(name, **kw):
    return {"name": name, "op": "norm_rotate", "batch": 1, "tokens": 1, "heads": HEADS, "kv_heads": HEADS,
            "dim": HEAD_DIM, "axes": "16,56,56", "theta": 10000.0, "pairing": "interleaved", "type": "bf16",
            "far": 64, "per_sample": False, "before": 0, **kw}


def _linear(name, **kw):
    return {"name": name, "op": "linear", "samples": 1, "rows": 1, "k": HIDDEN, "n": HIDDEN, "type": "bf16",
            "bias": True, "lora": False, **kw}


def listed():
    return [
        # one new token's queries: the smallest call, all latency
        _rotate("rotate_token"),
        # the queries of a video latent of 21 frames of 30 x 52 patches, contiguous
        _rotate("rotate_video", tokens=21 * 30 * 52, grid=52, far=21),
        # a vision encoder's 37 x 37 patches and one more token, read out of a fused q/k/v projection, in fp32,
        # with the pairs half a head apart and the last dimensions left as they are
        _rotate("rotate_patches", batch=3, tokens=37 * 37 + 1, heads=16, dim=80, axes="16,24,24", pairing="halves",
                type="fp32", fused=True),
        # q and k of one token
        _norm("norm_rotate_token"),
        # q and k of the image stream of a 1024 x 1024 batch, written behind the text tokens of the joint buffer
        _norm("norm_rotate_image", batch=BATCH, tokens=IMAGE, before=TEXT),
        # grouped heads with positions of each sample's own, fractional (stretched grids), an odd length
        _norm("norm_rotate_grouped", batch=5, tokens=1021, heads=32, kv_heads=8, dim=64, axes="16,24,24",
              pairing="halves", type="fp16", per_sample=True, far=3000),
        # the time embedding of one sample: one row, the weights' latency
        _linear("linear_row"),
        # the modulation of every sample of a batch: few rows, many weights
        _linear("linear_modulation", samples=BATCH, n=6 * HIDDEN),
        # the text stream's projections with an adapter for each sample
        _linear("linear_text", samples=BATCH, rows=TEXT, lora=True),
        # the image stream's feed-forward, in and out: the largest
        _linear("linear_image_in", samples=BATCH, rows=IMAGE, n=4 * HIDDEN, lora=True),
        _linear("linear_image_out", samples=BATCH, rows=1024, k=4 * HIDDEN),
        # odd sizes: rows, channels and lengths that no tile divides
        _linear("linear_odd", rows=1237, k=1898, n=1091, type="fp16", bias=False),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "norm_rotate", "linear", "linear"])
    if op == "linear":
        lora = rng.random() < 0.4
        samples = rng.randint(1, 16)
        rows = _between(rng, 1, 3000)
        k, n = _between(rng, 64, 13000), _between(rng, 64, 13000)
        while samples * rows * k * n > BATCH * IMAGE * HIDDEN * 4 * HIDDEN:
            rows = max(1, rows // 2)
        if rng.random() < 0.6:
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        return {"op": op, "samples": samples, "rows": rows, "k": k, "n": n,
                "type": "bf16" if lora else rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.7, "lora": lora}
    dim = rng.choice([32, 40, 64, 72, 80, 96, 128, 128, 160, 192, 256])
    parts = rng.randint(1, 4)
    cut = [2 * rng.randint(1, dim // (2 * parts)) for _ in range(parts)]
    case = {"op": op, "batch": rng.randint(1, 8), "tokens": _between(rng, 1, 6000), "heads": rng.randint(1, 32), "dim": dim,
            "axes": ",".join(map(str, cut)), "theta": rng.choice([256.0, 10000.0, 1e6]),
            "pairing": rng.choice(["interleaved", "halves"]), "type": rng.choice(["bf16", "fp16", "fp32"]),
            "far": _between(rng, 8, 100000)}
    if op == "rotate":
        return {**case, "fused": rng.random() < 0.5, "grid": 0}
    group = rng.choice([1, 1, 2, 4])
    case["kv_heads"] = max(1, case["heads"] // group)
    case["heads"] = case["kv_heads"] * group
    return {**case, "per_sample": rng.random() < 0.5, "before": rng.choice([0, 0, 77, 512])}


def _positions(case, gen):
    axes = len(case["axes"].split(","))
    s = case["tokens"]
    if case.get("grid"):    # frame, row and column of each patch, as whole numbers
        i = torch.arange(s, device=DEVICE)
        w, h = case["grid"], s // (case["grid"] * case["far"])
        return torch.stack([i // (w * h), i // w % h, i % w], dim=-1).to(torch.int32)
    shape = (case["batch"], s, axes) if case.get("per_sample") else (s, axes)
    p = torch.rand(shape, device=DEVICE, generator=gen) * case["far"]
    return p if case.get("per_sample") else p.floor().to(torch.int64)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    t = TYPES[case["type"]]

    def normal(*shape, std=1.0, to=t):
        return (torch.randn(*shape, device=DEVICE, generator=gen) * std).to(to)

    state = dict(case)
    if case["op"] == "linear":
        m, k, n = case["samples"] * case["rows"], case["k"], case["n"]
        x = normal(m, k)
        x *= (1 + 9 * (torch.rand(k, device=DEVICE, generator=gen) < 0.01)).to(t)     # activations have loud channels
        pitch = -(-k // 16) * 16                                    # weight rows start on 16-byte boundaries
        weight = torch.zeros(n, pitch, dtype=torch.int8, device=DEVICE)[:, :k]
        full = torch.randn(n, k, device=DEVICE, generator=gen) * 0.02
        scale = full.abs().amax(1) * (1.0 / 127)
        weight.copy_((full / scale[:, None]).round().clamp(-127, 127).to(torch.int8))
        state.update(x=x.view(case["samples"], case["rows"], k), weight=weight, scale=scale,
                     bias=normal(n, std=0.1) if case["bias"] else None,
                     h=normal(m, RANK, std=0.5) if case["lora"] else None,
                     b_dec=normal(case["samples"], n, RANK, std=0.1) if case["lora"] else None)
        return state
    b, s, heads, dim = case["batch"], case["tokens"], case["heads"], case["dim"]
    state["positions"] = _positions(case, gen)
    state["axes"] = tuple(int(v) for v in case["axes"].split(","))
    if case["op"] == "rotate":
        if case["fused"]:
            state["x"] = normal(b, s, 3, heads, dim)[:, :, 0]
        else:
            state["x"] = normal(b, s, heads, dim)
        return state
    kv = case["kv_heads"]
    state.update(q=normal(b, s, heads, dim, std=2.0), k=normal(b, s, kv, dim, std=0.5),
                 weight_q=1 + normal(dim, std=0.1), weight_k=1 + normal(dim, std=0.1),
                 joint_q=torch.zeros(b, case["before"] + s, heads, dim, dtype=t, device=DEVICE),
                 joint_k=torch.zeros(b, case["before"] + s, kv, dim, dtype=t, device=DEVICE))
    return state


def _angles(positions, axes, theta):
    """cos and sin of every pair's angle, (..., pairs) in 32 bits; the angles themselves in 64."""
    freq = torch.cat([theta ** (-torch.arange(0, d, 2, dtype=torch.float64, device=positions.device) / d) for d in axes])
    which = torch.cat([torch.full((d // 2,), i, device=positions.device) for i, d in enumerate(axes)])
    a = positions.double()[..., which] * freq
    return a.cos().float(), a.sin().float()


def _turn(x, cos, sin, pairing):
    """x (b, s, heads, dim) in 32 bits, turned by its tokens' angles; what lies behind the pairs stays."""
    r = 2 * cos.shape[-1]
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    if pairing == "interleaved":
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., r:]], dim=-1) if r < x.shape[-1] else y


def _normed(x, weight):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()


def _plain_linear(state):
    x = state["x"].flatten(0, 1).float()
    most = x.abs().amax(1, keepdim=True)
    q = (x * 127 / most).round()
    y = q @ state["weight"].float().t()
    y = y * (most * (1.0 / 127)) * state["scale"]
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if state["h"] is not None:
        h, b = state["h"].float(), state["b_dec"].float()
        y = y + torch.bmm(h.view(b.shape[0], -1, RANK), b.transpose(1, 2)).flatten(0, 1)
    return y.to(state["x"].dtype).view(*state["x"].shape[:2], -1)


def run(state):
    if own:
        from lithe_b200 import kernels
        if state["op"] == "linear":
            return kernels.int8_linear(state["x"], state["weight"], state["scale"], state["bias"], h=state["h"],
                                       b_dec=state["b_dec"])
        how = dict(theta=state["theta"], pairing=state["pairing"])
        if state["op"] == "rotate":
            return kernels.rotate_axes(state["x"], state["positions"], state["axes"], **how)
        at = state["before"]
        kernels.qk_norm_rotate(state["q"], state["k"], state["weight_q"], state["weight_k"], state["positions"],
                               state["axes"], out_q=state["joint_q"][:, at:], out_k=state["joint_k"][:, at:], **how)
        return state["joint_q"], state["joint_k"]
    if state["op"] == "linear":
        return _plain_linear(state)
    cos, sin = _angles(state["positions"], state["axes"], state["theta"])
    if state["op"] == "rotate":
        return _turn(state["x"].float(), cos, sin, state["pairing"]).to(state["x"].dtype)
    at = state["before"]
    state["joint_q"][:, at:] = _turn(_normed(state["q"], state["weight_q"]), cos, sin, state["pairing"])
    state["joint_k"][:, at:] = _turn(_normed(state["k"], state["weight_k"]), cos, sin, state["pairing"])
    return state["joint_q"], state["joint_k"]


def work(case):
    size = SIZES[case["type"]]
    if case["op"] == "linear":
        m, k, n = case["samples"] * case["rows"], case["k"], case["n"]
        lora = (m * RANK + case["samples"] * n * RANK) * 2 if case["lora"] else 0
        return {"bytes": m * k * size + n * k + n * 4 + (n * size if case["bias"] else 0) + m * n * size + lora,
                "flops": 2 * m * n * (k + (RANK if case["lora"] else 0))}
    tokens, parts = case["batch"] * case["tokens"], len(case["axes"].split(","))
    heads = case["heads"] + case.get("kv_heads", 0)
    rows = tokens if case.get("per_sample") else case["tokens"]
    each = 4 if case.get("per_sample") or case.get("grid") else 8
    values = tokens * heads * case["dim"]
    # a rotation is 3 operations a value; the norm adds its square and sum, the scale and the weight
    return {"bytes": 2 * values * size + rows * parts * each, "flops": values * (3 if case["op"] == "rotate" else 7)}


def _exact_turn(x, positions, axes, theta, pairing):
    """The rotation as a product of complex numbers, pair by pair."""
    angle = []
    for i, d in enumerate(axes):
        step = torch.exp(torch.arange(0, d, 2, dtype=torch.float64, device=x.device) * (-math.log(theta) / d))
        angle.append(positions[..., i, None].double() * step)
    angle = torch.cat(angle, -1)
    r = 2 * angle.shape[-1]
    turn = torch.polar(torch.ones_like(angle), angle)[..., None, :]
    head, rest = x[..., :r], x[..., r:]
    if pairing == "interleaved":
        z = torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * turn
        y = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(*(p.contiguous() for p in head.chunk(2, -1))) * turn
        y = torch.cat([z.real, z.imag], -1)
    return torch.cat([y, rest], -1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "linear":
        x = state["x"].double()
        unit = x.abs().amax(-1, keepdim=True) / 127
        steps = torch.round(x * 127 / x.abs().amax(-1, keepdim=True))
        y = torch.einsum("brk,nk->brn", steps, state["weight"].double() * state["scale"].double()[:, None]) * unit
        if state["bias"] is not None:
            y += state["bias"].double()
        if state["h"] is not None:
            y += torch.einsum("brj,bnj->brn", state["h"].double().view(case["samples"], case["rows"], RANK),
                              state["b_dec"].double())
        return y
    how = (state["positions"], state["axes"], state["theta"], state["pairing"])
    if case["op"] == "rotate":
        return _exact_turn(state["x"].double(), *how)
    outs = []
    for x, weight, joint in ((state["q"], state["weight_q"], state["joint_q"]), (state["k"], state["weight_k"], state["joint_k"])):
        x = x.double()
        x = x / (x.square().sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt() * weight.double()
        y = joint.double()
        y[:, case["before"]:] = _exact_turn(x, *how)
        outs.append(y)
    return tuple(outs)
