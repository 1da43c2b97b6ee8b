"""Performance cases of the feed-forward block's operators in 8-bit floating point: products with a scale for each block of 128,
a mixture-of-experts layer for a few tokens, and the norms before and after a block fused with its gate and residual scale.

Every case is one pass as a model server makes it, on tensors that are on the GPU already.  Numbers in 8-bit floating point are
e4m3 (largest value 448).  Activations have a scale per row and 128 of k, chosen at the call: the least power of two with which the
block's largest magnitude is at most 448.  Weights have one per block of 128 x 128, kept with them.  Results are bf16.
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # one token through an up-projection of a 7B layer: the weights are read once, latency counts
        {"name": "linear_fp8_1", "kind": "linear", "M": 1, "K": 4096, "N": 11008, "bias": False, "scales": "pow2"},
        # a decode batch through the down-projection: a long K, few columns
        {"name": "linear_fp8_24_down", "kind": "linear", "M": 24, "K": 11008, "N": 4096, "bias": False, "scales": "f32"},
        # a classifier-like head on a ragged batch: no size is a multiple of a block or tile
        {"name": "linear_fp8_ragged", "kind": "linear", "M": 391, "K": 1000, "N": 3001, "bias": True, "scales": "f32"},
        # a prompt of 2048 tokens through an up-projection
        {"name": "linear_fp8_2048", "kind": "linear", "M": 2048, "K": 4096, "N": 11008, "bias": True, "scales": "f32"},
        # a feed-forward block of a 7B layer between two others: the residual is updated, normed and quantised, and the MLP runs on it
        {"name": "ffn_fp8_16", "kind": "ffn", "M": 16, "K": 4096, "N": 11008},
        {"name": "ffn_fp8_1024", "kind": "ffn", "M": 1024, "K": 4096, "N": 11008},
        # one token through a layer of small experts, bf16 weights
        {"name": "moe_1", "kind": "moe", "T": 1, "E": 64, "k": 8, "H": 2048, "I": 1024, "type": "bf16", "scoring": "softmax"},
        # a small decode batch through a large layer, weights in 8 bits as a block-scaled checkpoint holds them
        {"name": "moe_8_fp8", "kind": "moe", "T": 8, "E": 128, "k": 8, "H": 4096, "I": 1536, "type": "fp8", "scoring": "sigmoid"},
        # two experts a token, a width that is no multiple of a block, several tokens at each expert
        {"name": "moe_32_ragged", "kind": "moe", "T": 32, "E": 16, "k": 2, "H": 1000, "I": 1376, "type": "bf16", "scoring": "softmax"},
        # the seam between two blocks for one token
        {"name": "norm_1", "kind": "norm", "M": 1, "H": 4096, "post": True, "gate": "row", "residual": "bf16"},
        # a ragged batch, a gate for every row, the residual stream in 32 bits
        {"name": "norm_ragged", "kind": "norm", "M": 391, "H": 1000, "post": True, "gate": "rows", "residual": "f32"},
        # a long prompt
        {"name": "norm_8192", "kind": "norm", "M": 8192, "H": 4096, "post": True, "gate": "row", "residual": "bf16"},
    ]


def _size(rng, lo, hi, step=1):
    """A size from [lo, hi], even over the logarithm, a multiple of step."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "ffn", "moe", "moe", "norm", "norm"])
    if kind == "linear":
        step = rng.choice([128, 128, 16, 1])  # most layers are whole blocks, some are not
        return {"kind": kind, "M": _size(rng, 1, 32) if rng.random() < 0.4 else _size(rng, 33, 2048), "K": _size(rng, 256, 8192, step),
                "N": _size(rng, 256, 11008, step), "bias": rng.random() < 0.5, "scales": rng.choice(["pow2", "f32"])}
    if kind == "ffn":
        return {"kind": kind, "M": _size(rng, 1, 32) if rng.random() < 0.5 else _size(rng, 33, 1024), "K": _size(rng, 512, 4096, 64),
                "N": _size(rng, 1024, 11008, 64)}
    if kind == "moe":
        E = rng.choice([8, 16, 24, 64, 96, 128])
        return {"kind": kind, "T": _size(rng, 1, 32), "E": E, "k": rng.randint(1, 8), "H": _size(rng, 512, 4096, rng.choice([128, 128, 8])),
                "I": _size(rng, 256, 1536, 32), "type": rng.choice(["bf16", "fp8"]) if E < 96 else "fp8", "scoring": rng.choice(["softmax", "sigmoid"])}
    return {"kind": kind, "M": _size(rng, 1, 8192), "H": _size(rng, 64, 4096, rng.choice([128, 8, 1])), "post": rng.random() < 0.7,
            "gate": rng.choice(["none", "row", "rows"]), "residual": rng.choice(["bf16", "f32"])}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _blocks(n):
    return -(-n // 128)


def _rand(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(shape, std=1.0, dtype=torch.bfloat16):
        return torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16 if dtype == torch.float8_e4m3fn else torch.float32).mul_(std).clamp_(-448, 448).to(dtype)

    def uniform(shape, lo, hi):
        return torch.rand(shape, device=DEV, generator=g) * (hi - lo) + lo

    def weight8(shape, std, scales):
        """e4m3 weights [..., N, K] of that deviation and the scales [..., N / 128, K / 128] of their blocks, as a checkpoint holds them."""
        s = uniform(shape[:-2] + (_blocks(shape[-2]), _blocks(shape[-1])), 0.7, 1.4).mul_(std / 100)
        if scales == "pow2":
            s = torch.exp2(torch.round(torch.log2(s)))
        return normal(shape, 100.0, torch.float8_e4m3fn), s

    return normal, uniform, weight8


_TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def prepare(case, seed):
    kind = case["kind"]
    normal, uniform, weight8 = _rand(seed)
    s = {"kind": kind}
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["w"], s["ws"] = weight8((N, K), 0.02, case["scales"])
        s["x"] = normal((M, K))
        s["bias"] = normal((N,), 0.1, torch.float32) if case["bias"] else None
        s["y"] = torch.empty((M, N), device=DEV, dtype=torch.bfloat16)
        if own:
            import mm_amx_amd as mx
            s["op"] = mx.LinearFp8()
            s["op"].set_weight(s["w"], s["ws"])
    elif kind == "ffn":
        M, K, N = case["M"], case["K"], case["N"]
        for name, shape in (("gate", (N, K)), ("up", (N, K)), ("down", (K, N))):
            s["w_" + name], s["s_" + name] = weight8(shape, 0.02, "f32")
        s["f"], s["residual"] = normal((M, K)), normal((M, K))
        s["pre"] = uniform((K,), 0.5, 1.5).to(torch.bfloat16)
        if own:
            import mm_amx_amd as mx
            s["op"] = mx.MLP()
            s["op"].setup(s["w_gate"], s["w_up"], s["w_down"], scales=(s["s_gate"], s["s_up"], s["s_down"]))
    elif kind == "moe":
        T, E, H, I = case["T"], case["E"], case["H"], case["I"]
        s["k"], s["scoring"] = case["k"], case["scoring"]
        s["x"], s["router"] = normal((T, H)), normal((E, H), 1 / math.sqrt(H))
        s["bias"] = normal((E,), 0.05, torch.float32) if case["scoring"] == "sigmoid" else None  # (moves the choice, not the weights)
        s["scales"] = None
        if case["type"] == "fp8":
            (g, sg), (u, su), (d, sd) = (weight8(shape, 0.02, "f32") for shape in ((E, I, H), (E, I, H), (E, H, I)))
            s["w_gate"], s["w_up"], s["w_down"], s["scales"] = g, u, d, (sg, su, sd)
        else:
            s["w_gate"], s["w_up"], s["w_down"] = normal((E, I, H), 0.02), normal((E, I, H), 0.02), normal((E, H, I), 0.02)
        if own:
            import mm_amx_amd as mx
            s["op"] = mx.MoE(top_k=case["k"], scoring=case["scoring"], renormalize=True, scale=1.5)
            s["op"].setup(s["router"], s["w_gate"], s["w_up"], s["w_down"], scales=s["scales"], bias=s["bias"])
    else:
        M, H = case["M"], case["H"]
        s["f"], s["residual"] = normal((M, H), 2.0), normal((M, H), 1.0, _TYPE[case["residual"]])
        s["post"] = uniform((H,), 0.5, 1.5).to(torch.bfloat16) if case["post"] else None
        s["pre"] = uniform((H,), 0.5, 1.5).to(torch.bfloat16)
        s["gate"] = None if case["gate"] == "none" else normal((H,) if case["gate"] == "row" else (M, H), 0.5)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _spread(scales, N, K):
    """Scales of blocks as a factor for every element of [..., N, K]."""
    return scales.repeat_interleave(128, -1)[..., :K].repeat_interleave(128, -2)[..., :N, :]


def _through_fp8(x):
    """What x [M, K] is after quantisation: e4m3 values times the power of two of their 128 of k."""
    M, K = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -K % 128)).view(M, -1, 128)
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # m in [0.5, 1): 448 is 0.875 * 2^9
    scale = torch.ldexp(torch.ones_like(m), (e - torch.where(m <= 0.875, 9, 8)).clamp_min(-126))
    return ((x / scale).to(torch.float8_e4m3fn).float() * scale).view(M, -1)[:, :K]


def _rms(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _silu(x):
    return x / (1 + torch.exp(-x))


def _linear(x, w, scales):
    return x @ (w.float() * _spread(scales, *w.shape)).T


def _seam(f, residual, post, gate, scale, pre):
    u = f.float() if post is None else _rms(f.float(), post)
    r = residual.float() + scale * (u if gate is None else gate.float() * u)
    return r, _rms(r, pre)


def _moe(s):
    x, (E, I, H), k = s["x"].float(), s["w_gate"].shape, s["k"]
    logits = x.double() @ s["router"].double().T  # (64 bits: a choice next to a border)
    p = torch.softmax(logits, -1) if s["scoring"] == "softmax" else torch.sigmoid(logits)
    rank = p if s["bias"] is None else p + s["bias"].double()
    ids = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :k]
    chosen = p.gather(1, ids)
    w = torch.zeros_like(p).scatter(1, ids, 1.5 * chosen / chosen.sum(-1, keepdim=True)).float()
    wide = lambda name, n: s["w_" + name].float() if s["scales"] is None else s["w_" + name].float() * _spread(s["scales"][n], *s["w_" + name].shape[1:])  # noqa: E731
    h = _silu(x @ wide("gate", 0).view(E * I, H).T) * (x @ wide("up", 1).view(E * I, H).T)  # [T, E I]
    h = (h.view(-1, E, I) * w[:, :, None]).transpose(0, 1).contiguous()
    return torch.bmm(h, wide("down", 2).transpose(1, 2).contiguous()).sum(0).to(torch.bfloat16)


def run(s):
    kind = s["kind"]
    if own:
        import mm_amx_amd as mx
        if kind == "linear":
            s["op"].forward(s["x"], s["y"], bias=s["bias"])
            return s["y"]
        if kind == "ffn":
            r, z = mx.block_norm(s["f"], s["residual"], scale=0.7, pre_weight=s["pre"], eps=EPS, quantize=True)
            return r, s["op"].run(z)
        if kind == "moe":
            return s["op"].run(s["x"])
        return mx.block_norm(s["f"], s["residual"], post=s["post"] is not None, post_weight=s["post"], gate=s["gate"], scale=0.7,
                             pre_weight=s["pre"], eps=EPS)
    if kind == "linear":
        y = _linear(_through_fp8(s["x"]), s["w"], s["ws"])
        s["y"].copy_(y if s["bias"] is None else y + s["bias"])
        return s["y"]
    if kind == "ffn":
        r, z = _seam(s["f"], s["residual"], None, None, 0.7, s["pre"])
        z = _through_fp8(z)
        h = _silu(_linear(z, s["w_gate"], s["s_gate"])) * _linear(z, s["w_up"], s["s_up"])
        return r.to(torch.bfloat16), _linear(_through_fp8(h), s["w_down"], s["s_down"]).to(torch.bfloat16)
    if kind == "moe":
        return _moe(s)
    r, z = _seam(s["f"], s["residual"], s["post"], s["gate"], 0.7, s["pre"])
    return r.to(s["residual"].dtype), z.to(torch.bfloat16)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": 2 * M * K + N * K + 4 * _blocks(N) * _blocks(K) + (4 * N if case["bias"] else 0) + 2 * M * N,
                "flops": 2 * M * K * N}
    if kind == "ffn":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": 3 * (N * K + 4 * _blocks(N) * _blocks(K)) + 2 * K + 8 * M * K, "flops": 6 * M * K * N}
    if kind == "moe":
        T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
        touched = E * (1 - (1 - k / E) ** T)  # experts that some token chose: what is expected of even choices
        each = 2 * H * I * 3 if case["type"] == "bf16" else 3 * (H * I + 4 * _blocks(H) * _blocks(I))
        return {"bytes": touched * each + 2 * E * H + 4 * T * H, "flops": T * k * 6 * H * I + 2 * T * E * H}
    M, H = case["M"], case["H"]
    stream = 2 if case["residual"] == "bf16" else 4
    return {"bytes": M * H * (4 + 2 * stream + (2 if case["gate"] == "rows" else 0)) + 2 * H * (1 + case["post"] + (case["gate"] == "row")), "flops": 10 * M * H}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _exact_fp8(x):
    """x [M, K] after quantisation, from the grid of e4m3: 3 bits behind the leading one, exponents from -6."""
    out = torch.zeros_like(x)
    for k0 in range(0, x.shape[1], 128):
        b = x[:, k0:k0 + 128]
        m, e = torch.frexp(b.abs().amax(1, keepdim=True) / 448)  # 2^(e-1) <= amax / 448 < 2^e
        s = torch.exp2(torch.where(m > 0.5, e, e - 1).clamp_min(-126).double())
        v = b / s
        step = torch.exp2((torch.frexp(v).exponent - 1).clamp_min(-6).double() - 3)
        out[:, k0:k0 + 128] = torch.round(v / step) * step * s  # (to the even one of two that are as near)
    return out


def _exact_weight(w, scales):
    w = w.double()
    for n in range(scales.shape[0]):
        for k in range(scales.shape[1]):
            w[128 * n:128 * n + 128, 128 * k:128 * k + 128] *= scales[n, k].double()
    return w


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "linear":
        y = _exact_fp8(s["x"].double()) @ _exact_weight(s["w"], s["ws"]).T
        return y if s["bias"] is None else y + s["bias"].double()
    if kind == "ffn":
        r = s["residual"].double() + 0.7 * s["f"].double()
        z = _exact_fp8(r / (r.square().mean(1, keepdim=True) + EPS).sqrt() * s["pre"].double())
        g, u = (z @ _exact_weight(s["w_" + n], s["s_" + n]).T for n in ("gate", "up"))
        return r, _exact_fp8(g * torch.sigmoid(g) * u) @ _exact_weight(s["w_down"], s["s_down"]).T
    if kind == "moe":
        x, k = s["x"].double(), s["k"]
        logits = x @ s["router"].double().T
        p = torch.softmax(logits, 1) if s["scoring"] == "softmax" else 1 / (1 + torch.exp(-logits))
        key = p if s["bias"] is None else p + s["bias"].double()
        taken = torch.zeros_like(p, dtype=torch.bool)
        for _ in range(k):  # the largest that is left, the lowest index of equal ones
            best = torch.where(taken, -math.inf, key).argmax(1, keepdim=True)
            taken.scatter_(1, best, True)
        w = p * taken
        w = 1.5 * w / w.sum(1, keepdim=True)
        y = torch.zeros_like(x)
        for e in range(case["E"]):
            at = taken[:, e].nonzero().flatten()
            if len(at):
                g, u, d = (s["w_" + n][e].double() if s["scales"] is None else _exact_weight(s["w_" + n][e], s["scales"][i][e])
                           for i, n in enumerate(("gate", "up", "down")))
                h = x[at] @ g.T
                y[at] += w[at, e, None] * ((h * torch.sigmoid(h) * (x[at] @ u.T)) @ d.T)
        return y
    f, r = s["f"].double(), s["residual"].double()
    if case["post"]:
        f = f / (f.square().mean(1, keepdim=True) + EPS).sqrt() * s["post"].double()
    r = r + 0.7 * f * (1.0 if s["gate"] is None else s["gate"].double())
    return r, r / (r.square().mean(1, keepdim=True) + EPS).sqrt() * s["pre"].double()
