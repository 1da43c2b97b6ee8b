"""The mixture-of-experts layer for a few tokens against its definition in 64 bits."""
import numpy as np
import pytest
import torch

import ffn_util as u

pytestmark = pytest.mark.gpu

import mm_amx_amd as mx  # noqa: E402

E4 = torch.float8_e4m3fn


def normal(shape, seed, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def experts(E, H, I, f8, seed=1):
    """(w_gate, w_up, w_down, scales or None, the three in 64 bits)."""
    shapes = ((E, I, H), (E, I, H), (E, H, I))
    if not f8:
        w = [normal(s, seed + i, 0.05) for i, s in enumerate(shapes)]
        return (*w, None, [u.f64(t) for t in w])
    g = torch.Generator().manual_seed(seed)
    w = [(torch.randn(s, generator=g) * 100).clamp(-448, 448).to(E4).cuda() for s in shapes]
    sc = [(torch.rand((E, u.blocks(s[1]), u.blocks(s[2])), generator=g) * 5e-4 + 2e-4).cuda() for s in shapes]
    return (*w, tuple(sc), [u.f64(t) * u.spread(u.f64(s), *t.shape[1:]) for t, s in zip(w, sc)])


def layer(E, H, I, f8, k=2, seed=1, **kw):
    wg, wu, wd, sc, full = experts(E, H, I, f8, seed)
    moe = mx.MoE(k, **kw)
    moe.setup(normal((E, H), seed + 9, 1 / np.sqrt(H)), wg, wu, wd, scales=sc)
    return moe, full


def definition(x, ids, weights, full):
    """y and its bound for given choices."""
    wg, wu, wd = full
    E, I, H = wg.shape
    y, bound = np.zeros_like(x), np.zeros_like(x)
    total = np.zeros_like(x)
    n_h, n_i = H + 16, I + 16
    for t in range(x.shape[0]):
        for e, w in zip(ids[t], weights[t]):
            if not 0 <= e < E:
                continue
            g, v = wg[e] @ x[t], wu[e] @ x[t]
            h, eh = u.gated(g, n_h * u.U * (np.abs(wg[e]) @ np.abs(x[t])), v, n_h * u.U * (np.abs(wu[e]) @ np.abs(x[t])))
            eh = eh + np.abs(h) * (2.0 ** -16 + 4 * u.U)  # the two bf16 that hold it, and the weight's product
            y[t] += w * (wd[e] @ h)
            bound[t] += abs(w) * (np.abs(wd[e]) @ eh)
            total[t] += abs(w) * (np.abs(wd[e]) @ np.abs(h))
    return y, bound + (2 * n_i + 2 * ids.shape[1] * u.blocks(I)) * u.U * total


def routing(x, router, k, scoring, renormalize, scale, bias):
    logits = x @ router.T
    with np.errstate(over="ignore"):
        p = 1 / (1 + np.exp(-logits)) if scoring == "sigmoid" else np.exp(logits - logits.max(1, keepdims=True))
    if scoring == "softmax":
        p = p / p.sum(1, keepdims=True)
    key = p + (0 if bias is None else bias)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(p, ids, 1)
    return ids, scale * (w / w.sum(1, keepdims=True) if renormalize else w), key


# ---- routing -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,H,E,k", [(1, 8, 1, 1), (1, 1000, 64, 8), (2, 7, 5, 5), (7, 513, 65, 3), (9, 256, 128, 16), (33, 100, 200, 4), (5, 2048, 1024, 6), (200, 64, 16, 2)])
@pytest.mark.parametrize("scoring,renormalize,biased", [("softmax", True, False), ("softmax", False, True), ("sigmoid", True, True), ("sigmoid", False, False)])
def test_route(T, H, E, k, scoring, renormalize, biased):
    x, r = normal((T, H), 1), normal((E, H), 2, 1.5 / np.sqrt(H))
    b = normal((E,), 3, 0.1, torch.float32) if biased else None
    ids, w = mx.moe_route(x, r, k, scoring, renormalize, 2.5, b)
    want_ids, want_w, key = routing(u.f64(x), u.f64(r), k, scoring, renormalize, 2.5, None if b is None else u.f64(b))
    got = ids.cpu().numpy()
    # the order goes by the 64-bit keys but for what 32-bit partial sums of 8 products are off: 8 u sum |x r|, and key's slope is 1 at most
    slack = 2 * 8 * u.U * (np.abs(u.f64(x)) @ np.abs(u.f64(r)).T).max()
    assert (got >= 0).all() and (got < E).all() and all(len(set(row)) == k for row in got)
    mine, best = np.take_along_axis(key, got, 1), np.take_along_axis(key, want_ids, 1)
    assert (np.abs(mine - best) <= slack).all()
    same = (got == want_ids).all(1)
    assert same.mean() > 0.9  # (near ties within the slack are rare)
    assert (np.abs(w.cpu().numpy() - want_w) <= 1e-5 * want_w + slack * 2.5)[same].all()


def test_route_ties_go_to_the_lowest_index():
    x, r = torch.ones((3, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((130, 64), dtype=torch.bfloat16, device="cuda")
    ids, w = mx.moe_route(x, r, 4)
    assert ids.cpu().tolist() == [[0, 1, 2, 3]] * 3 and torch.equal(w.cpu(), torch.full((3, 4), 0.25))
    r[70] = 1
    r[129] = 1
    assert mx.moe_route(x, r, 4)[0].cpu().tolist() == [[70, 129, 0, 1]] * 3
    b = torch.zeros(130, device="cuda")
    b[5] = 2.0
    assert mx.moe_route(x, r, 4, scoring="sigmoid", bias=b)[0].cpu().tolist() == [[5, 70, 129, 0]] * 3


def test_shares_of_small_sigmoids():
    x, r = torch.ones((2, 64), dtype=torch.bfloat16, device="cuda"), torch.full((5, 64), -4.0, dtype=torch.bfloat16, device="cuda")
    r[3, 0] = -3.0  # logits -256, and -255 for expert 3: p is e^-256 and e^-255
    for bias in (None, torch.zeros(5, device="cuda")):
        ids, w = mx.moe_route(x, r, 2, scoring="sigmoid", bias=bias)
        assert ids.cpu().tolist() == [[3, 0]] * 2
        want = torch.tensor([1 / (1 + np.exp(-1.0)), 1 / (1 + np.exp(1.0))]).float()
        assert ((w.cpu() - want).abs() <= 2.0 ** -23 * want).all()


@pytest.mark.parametrize("logits,masked", [((0.0, -110.0, -112.0), 0), ((0.0, -102.0, -102.5), 0), ((3.0, -88.0, -90.0, -87.0), 0), ((0.0, -800.0, -801.0), 0),
                                           ((300.0, -500.0, -501.0, -499.0), 0), ((0.0, -1.0, -2.0), 0), ((0.0, -30000.0, -30000.0), 0), ((-50.0, -50.0, 0.0), 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("mask", [-float("inf"), -2.0])
def test_shares_of_choices_far_below_the_largest(logits, masked, scoring, mask):
    """A bias keeps the expert of the largest logit out: the shares of the others are what they are among themselves, however small their p.  e^x in 64 bits and
    a sum of a few terms are off by less than 2^-45, so what counts is the rounding of a weight to 32 bits, half a step of 2^-24."""
    E, k = len(logits), len(logits) - 1
    x = torch.zeros((2, 64), dtype=torch.bfloat16, device="cuda")
    x[:, 0] = x[:, 1] = 1
    r = torch.zeros((E, 64), dtype=torch.bfloat16, device="cuda")
    for e, l in enumerate(logits):  # (two summands of at most 8 bits each)
        r[e, 0] = l
        r[e, 1] = l - float(r[e, 0])
    assert [float(v) for v in r.double().sum(1)] == list(logits)
    bias = torch.zeros(E, device="cuda")
    bias[masked] = mask
    ids, w = mx.moe_route(x, r, k, scoring, True, 2.5, bias)
    l = np.array(logits)
    chosen = [e for e in range(E) if e != masked]
    # log p but for what all experts of a token have in common
    log_p = l if scoring == "softmax" else np.where(l < 0, l - np.log1p(np.exp(-np.abs(l))), -np.log1p(np.exp(-np.abs(l))))
    share = np.zeros(E)
    share[chosen] = np.exp(log_p[chosen] - log_p[chosen].max())
    share *= 2.5 / share.sum()
    for t in range(2):
        assert sorted(ids[t].tolist()) == chosen
        assert (np.abs(u.f64(w)[t] - share[ids[t].tolist()]) <= 2.0 ** -23 * share[ids[t].tolist()] + 2.0 ** -149).all(), (w[t], share[ids[t].tolist()])


def test_shares_of_sigmoids_that_64_bits_cannot_hold():
    x = torch.ones((2, 64), dtype=torch.bfloat16, device="cuda")
    r = torch.zeros((5, 64), dtype=torch.bfloat16, device="cuda")
    r[:, 0] = -2048.0
    r[3, 1] = 1.0  # logits -2048, and -2047 for expert 3: e^-l is past the largest double
    ids, w = mx.moe_route(x, r, 2, scoring="sigmoid")
    want = torch.tensor([1 / (1 + np.exp(-1.0)), 1 / (1 + np.exp(1.0))]).float()
    assert ids.cpu().tolist() == [[3, 0]] * 2 and ((w.cpu() - want).abs() <= 2.0 ** -23 * want).all()


def test_route_with_nan_stays_in_range():
    x, r = normal((4, 64), 1), normal((40, 64), 2, 0.2)
    want = mx.moe_route(x, r, 3)[0]
    x[2, 5] = float("nan")
    r[7, 3] = float("nan")
    ids, w = mx.moe_route(x, r, 3)
    got = ids.cpu()
    assert ((got >= 0) & (got < 40)).all() and (got[2] == torch.tensor([0, 1, 2])).all()
    assert not (got[[0, 1, 3]] == 7).any()
    keep = [t for t in (0, 1, 3) if 7 not in want[t].tolist()]
    assert keep and torch.equal(ids[keep], want[keep])


# ---- experts -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,H,I,E,k", [(1, 64, 32, 1, 1), (1, 1000, 96, 8, 3), (3, 129, 32, 5, 2), (8, 512, 160, 16, 4), (16, 256, 64, 3, 2), (17, 300, 288, 4, 4), (32, 130, 96, 2, 1),
                                      (33, 264, 128, 8, 2), (70, 100, 64, 6, 3), (5, 33, 416, 40, 16), (2, 2064, 64, 4, 2), (20, 1200, 96, 5, 2)])
@pytest.mark.parametrize("f8", [False, True])
def test_experts(T, H, I, E, k, f8):
    moe, full = layer(E, H, I, f8, min(k, E))
    x = normal((T, H), 5)
    g = torch.Generator().manual_seed(6)
    ids = torch.stack([torch.randperm(max(E, k), generator=g)[:k] for _ in range(T)]).to(torch.int32).cuda()
    w = torch.rand((T, k), generator=g).cuda()
    want, bound = definition(u.f64(x), ids.cpu().numpy(), u.f64(w), full)
    y = mx.moe_experts(x, ids, w, moe.gate_up, moe.down, E, I)
    u.close(y, want, bound, torch.bfloat16)
    wide = torch.full((T + 2, H + 3), 7.0, device="cuda")
    mx.moe_experts(x, ids, w, moe.gate_up, moe.down, E, I, y=wide[:T, :H])
    u.close(wide[:T, :H], want, bound, torch.float32)
    assert (wide[:, H:] == 7).all() and (wide[T:] == 7).all()


@pytest.mark.parametrize("f8", [False, True])
def test_choices_of_no_expert_the_same_twice_and_all_of_one(f8):
    T, H, I, E = 40, 200, 96, 6
    moe, full = layer(E, H, I, f8)
    x = normal((T, H), 5)
    ids = torch.full((T, 3), -1, dtype=torch.int32)
    ids[0] = torch.tensor([2, 2, 2])
    ids[1] = torch.tensor([5, -1, 5])
    ids[2] = torch.tensor([E, 1 << 30, 3])
    ids[5:] = 4
    w = torch.rand((T, 3), generator=torch.Generator().manual_seed(1)).cuda()
    y = mx.moe_experts(x, ids.cuda(), w, moe.gate_up, moe.down, E, I)
    want, bound = definition(u.f64(x), ids.numpy(), u.f64(w), full)
    u.close(y, want, bound * 2, torch.bfloat16)
    assert (y[3] == 0).all() and (y[4] == 0).all()
    none = mx.moe_experts(x, torch.full((T, 3), -1, dtype=torch.int32, device="cuda"), w, moe.gate_up, moe.down, E, I)
    assert (none == 0).all()


def in_scratch_of(fill, moe, x, ids, w, E, H, I):
    """moe_experts in scratch memory that holds these bytes, with a guard behind it."""
    from mm_amx_amd import _lib as L
    T, k = ids.shape
    f8 = isinstance(moe.gate_up, tuple)
    need = L.lib().mmx_moe_experts_scratch_bytes(T, H, I, k)
    scratch = torch.full((need + 64,), fill, dtype=torch.uint8, device="cuda")
    y = torch.empty((T, H), device="cuda")
    gu, gs, d, ds = (*moe.gate_up, *moe.down) if f8 else (moe.gate_up, None, moe.down, None)
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    assert L.lib().mmx_moe_experts(L.F8 if f8 else L.BF16, x.data_ptr(), H * 2, ids.data_ptr(), w.data_ptr(), T, H, I, E, k, at(gu), at(gs), at(d), at(ds), L.F32, y.data_ptr(),
                                   H * 4, scratch.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
    assert (scratch[need:] == fill).all()
    return y


@pytest.mark.parametrize("T,E,choices", [
    (1, 2, [-1, -1, 0, 1]), (1, 2, [0, 0, 1]), (1, 1, [-1, 5, 0]), (1, 1, [0, 0, 0]), (1, 3, [7, 1, 1, -1, 2, 0, 0, 1 << 30, 2]), (1, 6, [-1, 5, 5, 2]), (1, 6, [-1, -1]), (1, 16, [3] * 16),
    (33, 2, [-1, -1, 0, 1]), (33, 2, [1, 1, 0]), (33, 3, [-1, -1, -1, 2, 2, 1]), (33, 8, [-1, 7, 7]), (2, 2, [-1, 1, 1, 0]), (65, 1, [-1, 0])])
@pytest.mark.parametrize("f8", [False, True])
def test_no_expert_and_the_same_twice_for_a_token_alone_in_its_group(T, E, choices, f8):
    """Also where a token names more experts than there are, as a shard of a few of a layer's experts is asked: what one of them is not chosen for, the scratch's
    old contents are not taken for."""
    H, I, k = 72, 64, len(choices)
    moe, full = layer(E, H, I, f8, 1)
    x = normal((T, H), 5)
    g = torch.Generator().manual_seed(6)
    ids = torch.randint(-1, E + 1, (T, k), generator=g, dtype=torch.int32)
    ids[0] = ids[T - 1] = torch.tensor(choices, dtype=torch.int32)
    ids, w = ids.cuda(), torch.rand((T, k), generator=g).cuda()
    want, bound = definition(u.f64(x), ids.cpu().numpy(), u.f64(w), full)
    for fill in (0xff, 0x7f, 0):  # (0xffff is a NaN in bf16, 0x7f7f a large value)
        u.close(in_scratch_of(fill, moe, x, ids, w, E, H, I), want, bound * 2, torch.float32, f"scratch {fill:#x}")


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("T", [1, 5, 40])
def test_layer(T, f8):
    E, H, I, k = 16, 256, 96, 4
    moe, full = layer(E, H, I, f8, k, scoring="sigmoid", scale=1.5)
    x = normal((T, H), 3)
    ids, w = mx.moe_route(x, moe.router, k, "sigmoid", True, 1.5)
    want, bound = definition(u.f64(x), ids.cpu().numpy(), u.f64(w), full)
    u.close(moe.run(x), want, bound, torch.bfloat16)
    y = torch.empty((T, H), device="cuda")
    assert moe.run(x, y) is y
    u.close(y, want, bound, torch.float32)
    # rows of a wider tensor, not 16-byte aligned
    wide = torch.zeros((T, H + 5), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:H + 3] = x
    assert torch.equal(moe.run(wide[:, 3:H + 3]), moe.run(x))


def test_a_bad_token_is_its_own():
    E, H, I, k = 8, 128, 64, 2
    moe, _ = layer(E, H, I, False, k)
    x = normal((20, H), 3)
    clean = moe.run(x)
    x[4, 9] = float("inf")
    x[11, 0] = float("nan")
    y = moe.run(x)
    others = [t for t in range(20) if t not in (4, 11)]
    assert torch.equal(y[others], clean[others]) and torch.isnan(y[11]).all()


@pytest.mark.parametrize("f8", [False, True])
def test_values_past_the_largest_are_infinite(f8):
    E, H, I = 2, 128, 64
    big = torch.full((E, I, H), 256.0, device="cuda")
    wd = torch.ones((E, H, I), device="cuda")
    wd[:, 1::2] = -1
    moe = mx.MoE(1)
    moe.setup(torch.zeros((E, H), dtype=torch.bfloat16, device="cuda"), *(w.to(torch.bfloat16) for w in (big, big, wd)), compress="fp8" if f8 else None)
    x = torch.zeros((3, H), dtype=torch.bfloat16, device="cuda")
    x[0, 0], x[1, 0] = 2.0 ** 60, 1  # gate = up = 2^68: their product is past 2^128; and 2^16 of 64 of them
    y = moe.run(x).cpu().float()
    assert (y[0, ::2] == float("inf")).all() and (y[0, 1::2] == -float("inf")).all()
    assert (y[1, ::2] == 2.0 ** 22).all() and (y[1, 1::2] == -2.0 ** 22).all() and (y[2] == 0).all()


@pytest.mark.parametrize("T,H", [(1, 200), (5, 1100), (40, 200), (33, 1100)])
def test_scratch_of_any_contents_and_the_same_bits_each_time(T, H):
    """Workgroups that share columns count in the scratch who is there: whatever it held, and in whichever order they come, the sums are the same."""
    from mm_amx_amd import _lib as L
    I, E, k = 96, 6, 3
    moe, _ = layer(E, H, I, False, k)
    x = normal((T, H), 5)
    ids, w = mx.moe_route(x, moe.router, k)
    want = mx.moe_experts(x, ids, w, moe.gate_up, moe.down, E, I)
    need = L.lib().mmx_moe_experts_scratch_bytes(T, H, I, k)
    y = torch.empty_like(x)
    scratch = torch.empty(need + 64, dtype=torch.uint8, device="cuda")
    for fill in (0, 1, 3, 0x7f, 0xff):
        for _ in range(4):
            scratch.fill_(fill)
            y.fill_(7)
            assert L.lib().mmx_moe_experts(L.BF16, x.data_ptr(), H * 2, ids.data_ptr(), w.data_ptr(), T, H, I, E, k, moe.gate_up.data_ptr(), None, moe.down.data_ptr(), None,
                                           L.BF16, y.data_ptr(), H * 2, scratch.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
            assert torch.equal(y, want) and (scratch[need:] == fill).all()


def test_more_tokens_than_a_grid_has_rows():
    """Launches are made for 262140 tokens (routing) and 2097120 (experts) at a time: the tokens on both sides of those borders, and the last ones."""
    T, H, E, I = 2097120 + 33, 8, 4, 32
    moe, full = layer(E, H, I, False, 1)
    x = torch.randn((T, H), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    ids, w = mx.moe_route(x, moe.router, 1, renormalize=False)
    y = mx.moe_experts(x, ids, w, moe.gate_up, moe.down, E, I)
    at = torch.tensor([t for b in (4, 262140, 524280, 2097120, T) for t in range(b - 4, min(b + 4, T))])
    xs, got = u.f64(x[at]), ids[at].cpu().numpy()
    _, want_w, key = routing(xs, u.f64(moe.router), 1, "softmax", False, 1.0, None)
    slack = 2 * 8 * u.U * (np.abs(xs) @ np.abs(u.f64(moe.router)).T).max()
    assert (np.abs(np.take_along_axis(key, got, 1) - key.max(1, keepdims=True)) <= slack).all()
    assert (np.abs(u.f64(w[at]) - want_w) <= 1e-5 * want_w + slack).all()
    want, bound = definition(xs, got, u.f64(w[at]), full)
    u.close(y[at], want, bound, torch.bfloat16)


@pytest.mark.parametrize("T", [1, 3, 33])
def test_a_shard_of_a_layers_experts(T):
    """Experts 4 to 6 of 12, packed by a layer of their own, whose tokens have eight choices each: ids less 4, and what is not theirs out of range."""
    E, H, I, k = 12, 136, 64, 8
    wg, wu, wd, _, full = experts(E, H, I, False)
    router, x = normal((E, H), 9, 0.1), normal((T, H), 5)
    shard = mx.MoE(k)
    shard.setup(router[4:7], wg[4:7], wu[4:7], wd[4:7])
    ids, w = mx.moe_route(x, router, k)
    y = mx.moe_experts(x, ids - 4, w, shard.gate_up, shard.down, 3, I)
    want, bound = definition(u.f64(x), ids.cpu().numpy() - 4, u.f64(w), [f[4:7] for f in full])
    u.close(y, want, bound, torch.bfloat16)


def test_compressed_from_bf16_weights():
    E, H, I = 4, 256, 128
    wg, wu, wd, _, _ = experts(E, H, I, False)
    router, x = normal((E, H), 10, 0.1), normal((6, H), 3)
    a, b = mx.MoE(2), mx.MoE(2)
    a.setup(router, wg, wu, wd)
    b.setup(router, wg, wu, wd, compress="fp8")
    d = (a.run(x).float() - b.run(x).float()).norm() / a.run(x).float().norm()
    assert d < 3 * 2.0 ** -4  # (three matrices quantised to 4 significant bits)


def test_graph_and_streams():
    E, H, I, k = 16, 256, 96, 4
    for f8 in (False, True):
        moe, _ = layer(E, H, I, f8, k)
        xs = [normal((T, H), T) for T in (1, 9, 40)]
        want = [moe.run(x) for x in xs]
        side = torch.cuda.Stream()
        graphs = []
        for x in xs:
            with torch.cuda.stream(side):
                moe.run(x)
                side.synchronize()
                gr = torch.cuda.CUDAGraph()
                with torch.cuda.graph(gr, stream=side):
                    y = moe.run(x)
                graphs.append((gr, y))
        torch.cuda.synchronize()
        for _ in range(4):
            for (gr, y), x, w in zip(graphs, xs, want):
                y.zero_()
                torch.cuda.synchronize()
                with torch.cuda.stream(side):
                    gr.replay()
                eager = moe.run(x)
                torch.cuda.synchronize()
                assert torch.equal(y, w) and torch.equal(eager, w)


def test_setup_refuses_a_bias_that_run_could_not_take():
    E, H, I = 4, 128, 64
    wg, wu, wd, _, _ = experts(E, H, I, False)
    router, b = normal((E, H), 1), torch.zeros(E, device="cuda")
    for bias in (b.double(), b.half(), b[:3], b[None], b.cpu(), [0.0] * E):
        with pytest.raises(mx.MmxError, match="bias"):
            mx.MoE(2).setup(router, wg, wu, wd, bias=bias)
    mx.MoE(2).setup(router, wg, wu, wd, bias=b)


def test_refusals_on_the_gpu():
    E, H, I = 4, 128, 64
    moe, _ = layer(E, H, I, False)
    x = normal((3, H), 1)
    assert moe.run(x[:0]).shape == (0, H)
    ids, w = mx.moe_route(x, moe.router, 2)
    for bad in (dict(ids=ids.long()), dict(ids=ids[:2]), dict(weights=w.double()), dict(ids=ids.t().contiguous().t()), dict(E=0), dict(E=2000), dict(E=5), dict(I=63),
                dict(I=96), dict(x=x.float()), dict(gate_up=moe.gate_up[:-1]), dict(down=(moe.down, None)), dict(y=torch.empty((2, H), device="cuda")),
                dict(y=torch.empty((3, H), dtype=torch.float16, device="cuda"))):
        with pytest.raises(mx.MmxError):
            mx.moe_experts(**{**dict(x=x, ids=ids, weights=w, gate_up=moe.gate_up, down=moe.down, E=E, I=I), **bad})
    for bad in (dict(top_k=0), dict(top_k=5), dict(scoring="none"), dict(bias=torch.zeros(3, device="cuda")), dict(router=moe.router[:, :64]), dict(x=x.cpu())):
        with pytest.raises(mx.MmxError):
            mx.moe_route(**{**dict(x=x, router=moe.router, top_k=2), **bad})
    with pytest.raises(mx.MmxError):
        mx.MoE(2).run(x)
    with pytest.raises(mx.MmxError):
        mx.MoE(2).setup(moe.router, *(normal(s, 1) for s in ((E, 40, H), (E, 40, H), (E, H, 40))))
