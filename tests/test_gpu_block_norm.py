"""The norms around a block, its gate and the residual stream, against their definition in 64 bits; and the block's operators together."""
import numpy as np
import pytest
import torch

import ffn_util as u

pytestmark = pytest.mark.gpu

import mm_amx_amd as mx  # noqa: E402


def normal(shape, seed, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def definition(f, residual, post, post_weight, gate, scale, pre, pre_weight, eps, offset):
    """(r, bound of r, z, bound of z before rounding to their types).  A sum of n squares is off by n u relative, its root by half of that; every factor is one
    rounding, 2^-23 each with room."""
    n = f.shape[1]
    v, ev = f, np.zeros_like(f)
    if post:
        inv = 1 / np.sqrt((f * f).mean(1, keepdims=True) + eps)
        v = f * inv * (1 if post_weight is None else offset + post_weight)
        ev = np.abs(v) * (n / 2 + 8) * u.U
        if post_weight is not None:  # (offset + weight may cancel)
            ev = ev + np.abs(f * inv) * u.U * (abs(offset) + np.abs(post_weight))
    s = scale * (1 if gate is None else gate)
    r = (0 if residual is None else residual) + s * v
    er = np.abs(s) * ev + 3 * u.U * (np.abs(s * v) + (0 if residual is None else np.abs(residual)))
    z, ez = r, er
    if pre:
        mean = (r * r).mean(1, keepdims=True) + eps
        inv = 1 / np.sqrt(mean)
        # what r's own errors do to the mean of its squares
        em = (2 * np.abs(r) * er + er * er).mean(1, keepdims=True) / mean
        w = 1 if pre_weight is None else offset + pre_weight
        z = r * inv * w
        ez = er * inv * np.abs(w) + np.abs(z) * ((n / 2 + 8) * u.U + em)
        if pre_weight is not None:
            ez = ez + np.abs(r * inv) * u.U * (abs(offset) + np.abs(pre_weight))
    return r, er, z, ez


SIZES = [(1, 1), (1, 4096), (3, 7), (5, 128), (4, 512), (7, 513), (9, 1000), (2, 1025), (391, 1000), (6, 2048), (3, 2049), (2, 4100), (3, 8192), (2, 8200), (2, 16384), (1, 20000), (2, 32768)]


@pytest.mark.parametrize("M,H", SIZES)
@pytest.mark.parametrize("kind", ["pre", "residual", "full", "full32", "rows", "post_only", "plain"])
def test_seam(M, H, kind):
    f = normal((M, H), 1, 2.0)
    dt = torch.float32 if kind in ("full32", "rows") else torch.bfloat16
    res = None if kind in ("pre", "plain") else normal((M, H), 2, 1.0, dt)
    post = kind in ("full", "full32", "rows", "post_only")
    pw = normal((H,), 3, 0.3) if kind in ("full", "full32") else None
    gate = normal((H,), 4, 0.5) if kind == "full" else normal((M, H), 4, 0.5) if kind == "rows" else None
    pre = kind not in ("post_only", "plain")
    nw = normal((H,), 5, 0.3) if kind in ("pre", "residual", "full", "full32") else None
    kw = dict(post=post, post_weight=pw, gate=gate, scale=0.7, pre=pre, pre_weight=nw, eps=1e-5, weight_offset=1.0)
    r, z = mx.block_norm(f, res, **kw)
    g = lambda t: None if t is None else u.f64(t)  # noqa: E731
    want_r, er, want_z, ez = definition(u.f64(f), g(res), post, g(pw), g(gate), 0.7, pre, g(nw), 1e-5, 1.0)
    assert r.dtype == dt and z.dtype == torch.bfloat16
    u.close(r, want_r, er, dt, "r")
    u.close(z, want_z, ez, torch.bfloat16, "z")
    # quantised: z is off by ez, so e4m3 and scale are those of some value within it
    r2, zq = mx.block_norm(f, res, quantize=True, **kw)
    assert torch.equal(r, r2)
    q, s = zq
    codes, scales = q.cpu().view(torch.uint8).numpy(), u.f64(s)
    got = u.value_rows(codes, scales)
    spread = np.repeat(scales, 128, 0)[:H].T
    assert (np.abs(got - want_z) <= ez + np.maximum(2.0 ** -4 * (np.abs(want_z) + ez), 2.0 ** -10 * spread)).all()
    pad = np.zeros((M, u.blocks(H) * 128))
    pad[:, :H] = np.abs(want_z)
    epad = np.zeros_like(pad)
    epad[:, :H] = ez
    top = pad.reshape(M, -1, 128)
    lo, hi = (top - epad.reshape(M, -1, 128)).max(-1), (top + epad.reshape(M, -1, 128)).max(-1)
    assert (scales.T >= u.scale_of(np.maximum(lo, 0))).all() and (scales.T <= u.scale_of(hi)).all()
    assert not zq.padded.cpu().view(torch.uint8).numpy()[:, H:].any()


def test_in_place_strides_and_rows_behind():
    M, H = 6, 300
    wide = lambda seed, dt=torch.bfloat16: normal((M + 2, H + 7), seed, 1.0, dt)  # noqa: E731
    for dt in (torch.bfloat16, torch.float32):
        f, res, gate, z = wide(1), wide(2, dt), wide(3), wide(4)
        w = normal((H,), 5)
        at = (slice(0, M), slice(3, H + 3))
        want = mx.block_norm(f[at].contiguous(), res[at].contiguous(), post=True, gate=gate[at].contiguous(), pre_weight=w, scale=-1.25)
        before, zb = res.clone(), z.clone()
        r, zz = mx.block_norm(f[at], res[at], post=True, gate=gate[at], pre_weight=w, scale=-1.25, r=res[at], z=z[at])
        assert torch.equal(res[at], want[0]) and torch.equal(z[at], want[1])
        for got, old in ((res, before), (z, zb)):
            mask = torch.ones_like(old, dtype=torch.bool)
            mask[at] = False
            assert torch.equal(got[mask], old[mask])
    # r not wanted
    for q in (False, True):
        a, b = mx.block_norm(f[at], None, pre_weight=w, quantize=q), mx.block_norm(f[at], None, pre_weight=w, quantize=q, r=False)
        c = mx.block_norm(f[at], None, pre_weight=w, quantize=q, r=False, z=a[1])  # (a z of its own: the Python form)
        bits = lambda v: (v.q if q else v).contiguous().view(torch.uint8)  # noqa: E731
        assert b[0] is None and c[0] is None and torch.equal(bits(a[1]), bits(b[1])) and torch.equal(bits(a[1]), bits(c[1]))
    # one row of gate for all, as a view too
    f, res, gate = normal((M, H), 1), normal((M, H), 2), normal((H,), 3)
    a = mx.block_norm(f, res, gate=gate)
    for g in (gate[None], gate[None].expand(M, H)):
        b = mx.block_norm(f, res, gate=g)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("H", [128, 1000, 4096, 20000])
def test_rows_do_not_touch_each_other(H):
    f, res = normal((9, H), 1), normal((9, H), 2)
    clean = mx.block_norm(f, res, post=True)
    f[3, H // 2] = float("nan")
    f[5, 0] = float("inf")
    f[7] = 0
    res[7] = 0
    r, z = mx.block_norm(f, res, post=True)
    others = [0, 1, 2, 4, 6, 8]
    assert torch.equal(r[others], clean[0][others]) and torch.equal(z[others], clean[1][others])
    assert torch.isnan(z[3]).all() and torch.isnan(z[5]).all() and (z[7] == 0).all() and (r[7] == 0).all()


@pytest.mark.parametrize("H", [128, 1000, 4096, 20000])
def test_rows_whose_squares_32_bits_cannot_hold(H):
    f, res = normal((6, H), 1), normal((6, H), 2, 1.0, torch.float32)
    clean = mx.block_norm(f, res, post=True)
    f[1] = 2.0 ** 64  # a square of 2^128 alone
    f[4] = 0
    f[4, H // 2] = -(2.0 ** 63)  # 2^126: not yet
    r, z = mx.block_norm(f, res, post=True)
    others = [0, 2, 3, 5]
    assert torch.equal(r[others], clean[0][others]) and torch.equal(z[others], clean[1][others])
    assert torch.equal(r[1], res[1])  # (what the norm made zeros of, added)
    want = definition(u.f64(f), u.f64(res), True, None, None, 1.0, True, None, 1e-6, 0.0)
    u.close(r[4:5], want[0][4:5], want[1][4:5], torch.float32)
    u.close(z[4:5], want[2][4:5], want[3][4:5], torch.bfloat16)


def test_a_block_as_it_is_used():
    """Norm and quantise, MLP on the quantised rows, the seam to a mixture of experts, and the last seam: each step against the step's own
    definition on what the step before it gave."""
    M, K, N, E, I = 20, 256, 384, 8, 96
    x = normal((M, K), 1)
    w = [normal(s, 2 + i, 0.05) for i, s in enumerate(((N, K), (N, K), (K, N)))]
    mlp, moe = mx.MLP(), mx.MoE(2)
    mlp.setup(*w, compress="fp8")
    moe.setup(normal((E, K), 20, 0.1), normal((E, I, K), 21, 0.05), normal((E, I, K), 22, 0.05), normal((E, K, I), 23, 0.05))
    nw = [normal((K,), 30 + i, 0.1) for i in range(4)]

    def block():
        r, zq = mx.block_norm(x, pre_weight=nw[0], weight_offset=1.0, quantize=True)
        f = mlp.run(zq)
        r2, z = mx.block_norm(f, r, post=True, post_weight=nw[1], pre_weight=nw[2], weight_offset=1.0)
        g = moe.run(z)
        r3, _ = mx.block_norm(g, r2, post=True, post_weight=nw[3], weight_offset=1.0, pre=False)
        return r, zq.q, f, r2, z, g, r3

    r, q, f, r2, z, g, r3 = block()
    assert torch.equal(r, x)
    want = definition(u.f64(f), u.f64(r), True, u.f64(nw[1]), None, 1.0, True, u.f64(nw[2]), 1e-6, 1.0)
    u.close(r2, want[0], want[1], torch.bfloat16)
    u.close(z, want[2], want[3], torch.bfloat16)
    want = definition(u.f64(g), u.f64(r2), True, u.f64(nw[3]), None, 1.0, False, None, 1e-6, 1.0)
    u.close(r3, want[0], want[1], torch.bfloat16)
    assert torch.equal(mlp.run(mx.quantize_fp8(z)), mlp.run(z)) and torch.equal(moe.run(z), g)
    # the whole of it as one graph, replayed beside eager passes
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        block()
        side.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            out = block()
    torch.cuda.synchronize()
    keep = x.clone()
    for i in range(4):
        x.copy_(keep if i % 2 == 0 else keep * 0.5)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            gr.replay()
        eager = block()
        torch.cuda.synchronize()
        assert all(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in zip(out, eager))


def test_refusals_on_the_gpu():
    f, res, w = normal((3, 64), 1), normal((3, 64), 2), normal((64,), 3)
    r, z = mx.block_norm(f[:0], res[:0], post=True, quantize=True)
    assert r.shape == (0, 64) and z.shape == (0, 64)
    for bad in (dict(f=f.float()), dict(f=f[0]), dict(residual=res[:2]), dict(residual=res.half()), dict(post_weight=w), dict(pre=False, pre_weight=w),
                dict(pre_weight=w[:63]), dict(pre_weight=w.float()), dict(gate=w[:63]), dict(gate=res[:2]), dict(gate=w.float()), dict(r=res.float()), dict(z=res.float()),
                dict(quantize=True, z=res), dict(f=f.t()), dict(residual=res.cpu()), dict(f=f.expand(3, 64)[:1].expand(3, 64))):
        with pytest.raises(mx.MmxError):
            mx.block_norm(**{**dict(f=f, residual=res), **bad})
    with pytest.raises(mx.MmxError):
        mx.block_norm(normal((1, 40000), 1))


def test_the_stack_of_the_demo():
    """Three layers of the MLP demo over e4m3 weights beside torch's: x, the weights and the intermediate are each quantised to 4 significant bits (2^-4 at most)."""
    from mm_amx_amd import mlp_llama
    out = mlp_llama.perf_llama7b_MLP(M=5, num_layers=2, rounds=1, hidden_size=256, intermediate_size=704, verbose=False, fp8=True)
    assert out["fp8"]["per_layer_us"] > 0 and out["rel_err_fp8_one_layer"] < 4 * 2.0 ** -4
