"""Performance cases of the operators in microscaled 4-bit floating point - quantisation of rows and back, products, a feed-forward block - and of
the drawing of tokens from logits.

Every case is one pass as a model server makes it, on tensors that are on the GPU already.  Numbers in 4 bits are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives) with a scale, a power of two in 8 bits, for each row and 32 of k.  Where a program quantises, the scale is the least power of two with which the
block's largest magnitude is below 7, so that it rounds to 6 at most; ties go to the even one.  Results of products are bf16.

A token is drawn from weights e^((l - max l) / temperature): the top_k largest stay, of those the shortest run, in descending order, that holds top_p of their
weight, of those what has min_p of the largest weight at least; among equal logits the lowest index comes first.  The token is the first in the order of the vocabulary up to which
the weights that stay come to more than u of their sum.  Temperature 0 takes the largest.
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # one token's activations in front of several products
        {"name": "quantize_1", "kind": "quantize", "M": 1, "K": 4096, "x": "bf16"},
        # a prompt's, which another operator left in 32 bits
        {"name": "quantize_2048", "kind": "quantize", "M": 2048, "K": 11008, "x": "f32"},
        # one token through an up-projection of a 7B layer: the weights are read once, latency counts
        {"name": "linear_1", "kind": "linear", "M": 1, "K": 4096, "N": 11008, "x": "bf16", "bias": False, "weights": "mxfp4"},
        # a decode batch through the down-projection: a long K, few columns
        {"name": "linear_24_down", "kind": "linear", "M": 24, "K": 11008, "N": 4096, "x": "bf16", "bias": True, "weights": "mxfp4"},
        # a classifier-like head on a ragged batch, weights that the program quantises itself: no size is a multiple of a block or tile
        {"name": "linear_ragged", "kind": "linear", "M": 391, "K": 1001, "N": 3001, "x": "f32", "bias": True, "weights": "bf16"},
        # a prompt of 2048 tokens through an up-projection
        {"name": "linear_2048", "kind": "linear", "M": 2048, "K": 4096, "N": 11008, "x": "bf16", "bias": True, "weights": "mxfp4"},
        # a feed-forward block of a 7B layer between two others: the residual is updated, normed and quantised, and the MLP runs on it
        {"name": "ffn_16", "kind": "ffn", "M": 16, "K": 4096, "N": 11008},
        {"name": "ffn_1024", "kind": "ffn", "M": 1024, "K": 4096, "N": 11008},
        # the next token of one sequence, the usual filters
        {"name": "sample_1", "kind": "sample", "B": 1, "V": 32000, "type": "f32", "k": "50", "p": "0.9", "min_p": "0", "T": "0.8"},
        # a ragged batch over a large vocabulary, no top_k: the shortest run that holds 95 % of everything
        {"name": "sample_33_top_p", "kind": "sample", "B": 33, "V": 100003, "type": "f32", "k": "0", "p": "0.95", "min_p": "0", "T": "1"},
        # a server's batch in which every request has filters of its own, some none, some take the largest
        {"name": "sample_64_mixed", "kind": "sample", "B": 64, "V": 131072, "type": "bf16", "k": "rows", "p": "rows", "min_p": "rows", "T": "rows"},
        # many sequences, drawn from everything
        {"name": "sample_256_plain", "kind": "sample", "B": 256, "V": 131072, "type": "f32", "k": "0", "p": "1", "min_p": "0", "T": "1"},
    ]


def _size(rng, lo, hi, step=1):
    """A size from [lo, hi], even over the logarithm, a multiple of step."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "ffn", "sample", "sample", "sample"])
    if kind == "quantize":
        return {"kind": kind, "M": _size(rng, 1, 2048), "K": _size(rng, 32, 11008, rng.choice([32, 8, 1])), "x": rng.choice(["bf16", "f32"])}
    if kind == "linear":
        step = rng.choice([128, 128, 32, 2])  # most layers are whole blocks, some are not; two values share a byte
        weights = rng.choice(["mxfp4", "mxfp4", "bf16"])
        return {"kind": kind, "M": _size(rng, 1, 32) if rng.random() < 0.4 else _size(rng, 33, 2048), "K": _size(rng, 256, 8192, step if weights == "mxfp4" else 1),
                "N": _size(rng, 256, 11008, rng.choice([64, 16, 1])), "x": rng.choice(["bf16", "bf16", "f32"]), "bias": rng.random() < 0.5, "weights": weights}
    if kind == "ffn":
        return {"kind": kind, "M": _size(rng, 1, 32) if rng.random() < 0.5 else _size(rng, 33, 1024), "K": _size(rng, 512, 4096, 32), "N": _size(rng, 1024, 11008, 32)}
    # (the number of candidates is any, the others come in hundredths; as texts, since "rows" stands for values of each row's own)
    k = rng.choice(["0", "0", "1", str(_size(rng, 2, 200)), str(_size(rng, 200, 5000)), "rows"])
    return {"kind": kind, "B": _size(rng, 1, 256), "V": _size(rng, 1000, 131072, rng.choice([64, 1])), "type": rng.choice(["bf16", "f32"]), "k": k,
            "p": rng.choice(["1", "0.%02d" % rng.randint(10, 99), "0.%02d" % rng.randint(80, 99), "rows"]), "min_p": rng.choice(["0", "0", "0.%02d" % rng.randint(1, 30), "rows"]),
            "T": rng.choice(["1", "0.%02d" % rng.randint(20, 99), "1.%02d" % rng.randint(1, 99), "rows"])}


# ---- inputs -----------------------------------------------------------------------------------------------------------
_TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def _rand(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(shape, std=1.0, dtype=torch.bfloat16):
        return torch.randn(shape, device=DEV, generator=g).mul_(std).to(dtype)

    def uniform(shape, lo, hi):
        return torch.rand(shape, device=DEV, generator=g) * (hi - lo) + lo

    def weight4(N, K):
        """Weights [N, K] as a checkpoint holds them: two codes a byte, the first in its low half, and the biased exponents of their scales [N, K / 32]; a deviation of some 0.02."""
        v = torch.randn((N, K), device=DEV, generator=g).mul_(2.2)
        code = torch.bucketize(v.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)) + 8 * (v < 0)
        code = code.to(torch.uint8)
        return code[:, 0::2] | code[:, 1::2] << 4, torch.randint(119, 122, (N, -(-K // 32)), device=DEV, generator=g, dtype=torch.uint8)

    return normal, uniform, weight4


def prepare(case, seed):
    kind = case["kind"]
    normal, uniform, weight4 = _rand(seed)
    s = {"kind": kind}
    if kind == "quantize":
        s["x"] = normal((case["M"], case["K"]), 1.0, _TYPE[case["x"]])
    elif kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["w"], s["ws"] = weight4(N, K) if case["weights"] == "mxfp4" else (normal((N, K), 0.02), None)
        s["x"] = normal((M, K), 1.0, _TYPE[case["x"]])
        s["bias"] = normal((N,), 0.1, torch.float32) if case["bias"] else None
        s["y"] = torch.empty((M, N), device=DEV, dtype=torch.bfloat16)
        if own:
            import mm_amx_amd as mx
            s["op"] = mx.LinearMxfp4()
            s["op"].set_weight(s["w"], s["ws"])
    elif kind == "ffn":
        M, K, N = case["M"], case["K"], case["N"]
        for name, shape in (("gate", (N, K)), ("up", (N, K)), ("down", (K, N))):
            s["w_" + name], s["s_" + name] = weight4(*shape)
        s["f"], s["residual"] = normal((M, K)), normal((M, K))
        s["pre"] = uniform((K,), 0.5, 1.5).to(torch.bfloat16)
        if own:
            import mm_amx_amd as mx
            s["op"] = mx.MLP()
            s["op"].setup(s["w_gate"], s["w_up"], s["w_down"], scales=(s["s_gate"], s["s_up"], s["s_down"]))
    else:
        B, V = case["B"], case["V"]
        l = normal((B, V), 2.0, torch.float32)
        l += 10 * (uniform((B, V), 0, 1) < 12 / V) * uniform((B, V), 0.3, 1)  # the few tokens that the context makes likely
        l[:, V - V // 500:] = -math.inf  # a vocabulary padded to a size that suits its product
        s["logits"] = l.to(_TYPE[case["type"]])
        s["u"] = uniform((B,), 0, 1)
        number = lambda name, rows, of: rows if case[name] == "rows" else of(case[name])  # noqa: E731
        off = uniform((B,), 0, 1) < 0.3
        s["k"] = number("k", torch.where(off, 0, uniform((B,), 1, 200).to(torch.int32)).to(torch.int32), int)
        s["p"] = number("p", torch.where(uniform((B,), 0, 1) < 0.3, 1.0, uniform((B,), 0.5, 0.99)), float)
        s["min_p"] = number("min_p", torch.where(uniform((B,), 0, 1) < 0.5, 0.0, uniform((B,), 0.01, 0.2)), float)
        s["T"] = number("T", torch.where(uniform((B,), 0, 1) < 0.2, 0.0, uniform((B,), 0.3, 1.5)), float)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _power(biased):
    """2^(biased - 127) of whole numbers from 1 to 254."""
    return (biased.to(torch.int32) << 23).view(torch.float32)


def _through_fp4(x):
    """What x [M, K] is after quantisation: e2m1 values times the power of two of their 32 of k."""
    M, K = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -K % 32)).view(M, -1, 32)
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # m in [0.5, 1): 7 is 0.875 * 2^3
    scale = _power((e - torch.where(m < 0.875, 3, 2) + 127).clamp(1, 254))
    v = x / scale
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.round(v / step) * step * scale).view(M, -1)[:, :K]


def _wide(w, scales):
    """Weights [N, K] in 32 bits: quantised here, or from their codes."""
    if scales is None:
        return _through_fp4(w)
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=w.device)
    code = torch.stack((w & 15, w >> 4), -1).flatten(1).long()
    return torch.where(code >= 8, -1.0, 1.0) * table[code & 7] * _power(scales).repeat_interleave(32, 1)[:, :code.shape[1]]


def _silu(x):
    return x / (1 + torch.exp(-x))


def _sample(s):
    l = s["logits"].double()  # (64 bits: sums over a vocabulary, a token next to the border)
    B, V = l.shape
    column = lambda v: v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((B, 1), float(v), device=l.device, dtype=torch.float64)  # noqa: E731
    T, k, p, min_p = (column(s[n]) for n in ("T", "k", "p", "min_p"))
    k = torch.where(T == 0, 1.0, torch.where(k == 0, float(V), k))
    T = torch.where(T == 0, 1.0, T)
    l, at = torch.sort(l, dim=1, descending=True, stable=True)
    w = torch.exp((l - l[:, :1]) / T)
    w = torch.where(torch.arange(V, device=l.device) < k, w, 0)
    before = torch.cumsum(w, 1) - w
    w = torch.where(((before < p * w.sum(1, keepdim=True)) | (p >= 1)) & (w >= min_p), w, 0)
    run = torch.cumsum(torch.zeros_like(w).scatter(1, at, w), 1)
    return (run <= s["u"].double()[:, None] * run[:, -1:]).sum(1).to(torch.int32)


def run(s):
    kind = s["kind"]
    if own:
        import mm_amx_amd as mx
        if kind == "quantize":
            return mx.dequantize_mxfp4(mx.quantize_mxfp4(s["x"]))
        if kind == "linear":
            s["op"].forward(s["x"], s["y"], bias=s["bias"])
            return s["y"]
        if kind == "ffn":
            r, z = mx.block_norm(s["f"], s["residual"], scale=0.7, pre_weight=s["pre"], eps=EPS, quantize="mxfp4")
            return r, s["op"].run(z)
        return mx.sample(s["logits"], s["u"], temperature=s["T"], top_k=s["k"], top_p=s["p"], min_p=s["min_p"])
    if kind == "quantize":
        return _through_fp4(s["x"]).to(torch.bfloat16)
    if kind == "linear":
        y = _through_fp4(s["x"]) @ _wide(s["w"], s["ws"]).T
        s["y"].copy_(y if s["bias"] is None else y + s["bias"])
        return s["y"]
    if kind == "ffn":
        r = s["residual"].float() + 0.7 * s["f"].float()
        z = _through_fp4(r * torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS) * s["pre"].float())
        h = _silu(z @ _wide(s["w_gate"], s["s_gate"]).T) * (z @ _wide(s["w_up"], s["s_up"]).T)
        return r.to(torch.bfloat16), (_through_fp4(h) @ _wide(s["w_down"], s["s_down"]).T).to(torch.bfloat16)
    return _sample(s)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "quantize":  # the rows and the values that they become; what is held in between, half a byte each, need not leave the chip's caches
        return {"bytes": case["M"] * case["K"] * ((2 if case["x"] == "bf16" else 4) + 2), "flops": 4 * case["M"] * case["K"]}
    if kind == "sample":
        B, V = case["B"], case["V"]
        return {"bytes": B * V * (2 if case["type"] == "bf16" else 4) + 8 * B, "flops": 4 * B * V}
    M, K, N = case["M"], case["K"], case["N"]
    held = lambda N, K: N * -(-K // 2) + N * -(-K // 32)  # noqa: E731
    if kind == "linear":
        return {"bytes": (2 if case["x"] == "bf16" else 4) * M * K + held(N, K) + (4 * N if case["bias"] else 0) + 2 * M * N, "flops": 2 * M * K * N}
    return {"bytes": 2 * held(N, K) + held(K, N) + 2 * K + 8 * M * K, "flops": 6 * M * K * N}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _exact_fp4(x):
    """x [M, K] after quantisation, by the nearest of the eight magnitudes: what lies past the middle of two goes up, on the middle to the even one."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=x.device, dtype=torch.float64)
    middle = (grid[1:] + grid[:-1]) / 2
    out = torch.zeros_like(x)
    for k0 in range(0, x.shape[1], 32):
        b = x[:, k0:k0 + 32]
        m, e = torch.frexp(b.abs().amax(1, keepdim=True) / 7)  # 2^(e-1) <= amax / 7 < 2^e
        s = torch.exp2(torch.where(m == 0, -126, e).clamp_min(-126).double())
        a = (b / s).abs()
        low, high = torch.bucketize(a, middle), torch.bucketize(a, middle, right=True)  # (they differ on a middle)
        out[:, k0:k0 + 32] = torch.sign(b) * grid[torch.where(low % 2 == 0, low, high)] * s
    return out


def _exact_weight(w, scales):
    if scales is None:
        return _exact_fp4(w.double())
    out = torch.empty((w.shape[0], 2 * w.shape[1]), device=w.device, dtype=torch.float64)
    for half in range(2):
        c = (w >> 4 * half) & 15
        e, m = (c >> 1 & 3).double(), (c & 1).double()
        out[:, half::2] = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e - 1)) * (1 - 2 * (c >> 3).double())
    for b in range(scales.shape[1]):
        out[:, 32 * b:32 * b + 32] *= torch.exp2(scales[:, b:b + 1].double() - 127)
    return out


def _exact_token(l, u, T, k, p, min_p):
    """The token of one row of logits."""
    order = torch.argsort(-l, stable=True)
    if T == 0:
        return int(order[0])
    if k:
        order = order[:k]
    share = torch.softmax(l[order] / T, 0)
    if p < 1:
        order = order[:int((torch.cumsum(share, 0) < p).sum()) + 1]
    share = share[:len(order)]
    order = order[share >= min_p * share[0]].sort().values
    run = torch.cumsum(torch.exp((l[order] - l.max()) / T), 0)
    return int(order[torch.searchsorted(run, u * run[-1], right=True)])


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "quantize":
        return _exact_fp4(s["x"].double())
    if kind == "linear":
        y = _exact_fp4(s["x"].double()) @ _exact_weight(s["w"], s["ws"]).T
        return y if s["bias"] is None else y + s["bias"].double()
    if kind == "ffn":
        r = s["residual"].double() + 0.7 * s["f"].double()
        z = _exact_fp4(r / (r.square().mean(1, keepdim=True) + EPS).sqrt() * s["pre"].double())
        g, u = (z @ _exact_weight(s["w_" + n], s["s_" + n]).T for n in ("gate", "up"))
        return r, _exact_fp4(g * torch.sigmoid(g) * u) @ _exact_weight(s["w_down"], s["s_down"]).T
    l, B = s["logits"].double(), case["B"]
    T, k, p, min_p = ((v.tolist() if isinstance(v, torch.Tensor) else [v] * B) for v in (s["T"], s["k"], s["p"], s["min_p"]))
    return torch.tensor([_exact_token(l[b], s["u"][b].double(), T[b], k[b], p[b], min_p[b]) for b in range(B)], dtype=torch.int32, device=l.device)
