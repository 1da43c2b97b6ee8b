"""Microscaled 4-bit floating point: quantisers, packing, products and the MLP over them, against their definitions in 64 bits."""
import copy

import numpy as np
import pytest
import torch

import ffn_util as u
import mxfp4_util as m4

pytestmark = pytest.mark.gpu

import mm_amx_amd as mx  # noqa: E402


def bits(t):
    return t.detach().cpu().contiguous().view(torch.uint8).numpy()


def normal(shape, seed, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def weight(N, K, seed, lo=117, hi=122):
    """Codes uint8 [N, K / 2] and scales uint8 [N, K / 32] as a checkpoint holds them, and the values."""
    g = np.random.default_rng(seed)
    codes, b = g.integers(0, 16, (N, K), dtype=np.uint8), g.integers(lo, hi, (N, m4.blocks(K)), dtype=np.uint8)
    return torch.from_numpy(m4.pairs(codes)).cuda(), torch.from_numpy(b).cuda(), m4.values(codes, b)


def in_wide(t, extra, fill):
    """The same values in rows `extra` elements longer than they are, and the whole buffer."""
    wide = torch.full((t.shape[0], t.shape[1] + extra), fill, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]], wide


def same_codes(got, want):
    """Equal but for the sign of zero, which does not matter to any product."""
    assert np.array_equal(np.where(got == 8, 0, got), np.where(want == 8, 0, want))


def check_rows(rows, x):
    want, b = m4.quantize(u.f64(x))
    codes, s, rest, rest_s = m4.unpack(bits(rows.packed), *x.shape)
    assert np.array_equal(s, b)
    live = np.repeat(b != 255, 32, 1)[:, :x.shape[1]]
    same_codes(codes[live], want[live])
    assert not (rest & 7).any() and not (rest_s == 255).any()
    return codes, s


# ---- quantisers --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,K", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 7), (33, 1000), (130, 256), (2, 11008), (64, 257), (31, 511)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_bits_and_back(M, K, dtype):
    x = normal((M, K), M * K, 3.0, dtype)
    rows = mx.quantize_mxfp4(x)
    codes, s = check_rows(rows, x)
    q, scales = rows
    assert np.array_equal(m4.single(bits(q), K), codes) and np.array_equal(bits(scales), s) and rows.shape == (M, K)
    if K % 2:
        assert not (bits(q)[:, -1] >> 4).any()
    for t in (torch.bfloat16, torch.float32):
        y = mx.dequantize_mxfp4(rows, t)
        assert y.dtype == t and np.array_equal(u.f64(y), m4.values(codes, s))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_special_values(dtype):
    x = torch.zeros((16, 96), dtype=dtype)
    x[1, 3] = 6.0                          # scale 1
    x[2, 3] = 6.96875                      # still rounds to 6
    x[3, 3] = 7.0                          # would round to 8: scale 2
    x[4, :96] = torch.arange(96) * 0.125 - 6
    x[5, 5], x[5, 6], x[5, 40] = float("inf"), 1.0, 2.0  # the block is NaN, the next one is not
    x[6, 0], x[6, 1] = float("nan"), 1.0
    x[7, 0] = 2.0 ** -133                  # subnormal: to zero
    x[8, 0], x[8, 1] = 2.0 ** -126, 2.0 ** -128
    x[9, 0] = 3.0e38
    x[10, 0], x[10, 1:32] = 6.0, 0.25      # half of the smallest: to zero
    x[11, 0], x[11, 1:32] = -6.0, 0.75     # between 0.5 and 1: the even one
    x[12, 0], x[12, 1:32] = 6.0, -5.0      # between 4 and 6
    x[13, 0], x[13, 1:32] = 6.0, 3.5       # between 3 and 4
    x[14, 0], x[14, 1:32] = -6.0, -2.5
    x[15, 0] = -0.0
    rows = mx.quantize_mxfp4(x.cuda())
    codes, s = check_rows(rows, x)
    assert list(s[1:4, 0]) == [127, 127, 128] and s[5, 0] == s[6, 0] == 255 and s[5, 1] == 126
    back = mx.dequantize_mxfp4(rows, torch.float32)
    # (3.0e38 is 3.53 * 2^126, which rounds to 4 * 2^126 = 2^128: infinite in 32 bits)
    with np.errstate(over="ignore"):
        assert np.array_equal(u.f64(back), m4.values(codes, s).astype(np.float32).astype(np.float64), equal_nan=True) and torch.isinf(back[9, 0])
    assert torch.isnan(back[5, :32]).all() and not torch.isnan(back[5, 32:]).any()


def test_quantize_reads_rows_of_any_stride():
    base = normal((9, 333), 5)
    for x in (base[:, 1:302], base[::2, 3:300], base[2:3, 5:6], normal((40, 70), 6, 1.0, torch.float32)[3:, 1:]):
        check_rows(mx.quantize_mxfp4(x), x)


@pytest.mark.parametrize("M,K", [(1, 2), (5, 31), (33, 100), (64, 512), (70, 1001)])
def test_rows_from_elsewhere_and_back(M, K):
    g = np.random.default_rng(M)
    codes, b = g.integers(0, 16, (M, K), dtype=np.uint8), g.integers(0, 256, (M, m4.blocks(K)), dtype=np.uint8)
    q, s = torch.from_numpy(m4.pairs(codes)).cuda(), torch.from_numpy(b).cuda()
    if K % 2:
        q[:, -1] |= 0x30  # (what an odd row's last byte has in its other half is left out)
    wide_q, wide_s = in_wide(q, 3, 255)[0], in_wide(s, 5, 7)[0]
    for a, c in ((q, s), (wide_q, wide_s)):
        rows = mx.Mxfp4Rows.of(a, c, K)
        got, gs, rest, rest_s = m4.unpack(bits(rows.packed), M, K)
        assert np.array_equal(got, codes) and np.array_equal(gs, b) and not rest.any() and not (rest_s == 255).any()
        assert np.array_equal(bits(rows.q), m4.pairs(codes)) and np.array_equal(bits(rows.scales), b)
    y = mx.dequantize_mxfp4(rows, torch.float32)
    want = m4.values(codes, b)
    with np.errstate(over="ignore"):
        assert np.array_equal(u.f64(y), want.astype(np.float32).astype(np.float64), equal_nan=True)  # (past 2^128 infinite)


def test_types_of_torch_for_codes_and_scales():
    if not hasattr(torch, "float4_e2m1fn_x2"):
        pytest.skip("this torch has no 4-bit floating point")
    q, s, v = weight(64, 128, 1)
    rows = mx.Mxfp4Rows.of(q.view(torch.float4_e2m1fn_x2), s.view(torch.float8_e8m0fnu))
    assert np.array_equal(u.f64(mx.dequantize_mxfp4(rows, torch.float32)), v)


@pytest.mark.parametrize("N,K", [(32, 128), (96, 200), (160, 1000)])
def test_gate_up_pairs_alternate(N, K):
    (g, gs, gv), (v, vs, vv) = weight(N, K, 1), weight(N, K, 2)
    packed = mx.pack_gate_up_mxfp4(g, v, (gs, vs))
    codes, b, _, _ = m4.unpack(bits(packed), 2 * N, K)
    both = m4.values(codes, b).reshape(N // 32, 2, 32, K)
    assert np.array_equal(both[:, 0].reshape(N, K), gv) and np.array_equal(both[:, 1].reshape(N, K), vv)
    gb, ub = normal((N, K), 3, 0.02), normal((N, K), 4, 0.5)
    codes, b, _, _ = m4.unpack(bits(mx.pack_gate_up_mxfp4(gb, ub)), 2 * N, K)
    both, bs = codes.reshape(N // 32, 2, 32, K), b.reshape(N // 32, 2, 32, -1)
    for i, w in enumerate((gb, ub)):
        want, wb = m4.quantize(u.f64(w))
        same_codes(both[:, i].reshape(N, K), want)
        assert np.array_equal(bs[:, i].reshape(N, -1), wb)


# ---- products ----------------------------------------------------------------------------------------------------------
SIZES = [(1, 2, 1), (1, 128, 16), (1, 4096, 96), (2, 126, 33), (8, 2048, 100), (9, 2048, 64), (15, 130, 31), (16, 640, 160), (17, 1000, 200), (31, 2048, 129), (33, 300, 500), (48, 4100, 64),
         (64, 1152, 130), (65, 128, 257), (100, 516, 70), (127, 2304, 40), (129, 1000, 300), (200, 130, 513), (256, 1024, 256), (257, 384, 258),
         (300, 4096, 65), (391, 1000, 3001), (513, 700, 1030), (1000, 260, 90), (1030, 2050, 520), (2049, 130, 290)]


@pytest.mark.parametrize("M,K,N", SIZES)
def test_product(M, K, N):
    x = normal((M, K), 1)
    q, s, w = weight(N, K, 2)
    packed = mx.pack_mxfp4(q, s)
    rows = mx.quantize_mxfp4(x)
    want, bound = m4.product(m4.values(*m4.quantize(u.f64(x))), w)
    y = torch.full((M, N), 7.0, device="cuda")
    mx.gemm_mxfp4(rows, packed, N, mx.Epilogue(y, mx.PP_NONE))
    u.close(y, want, bound, torch.float32, mx.last_kernel())
    # from bf16 and from fp32: the same rows, quantised on the way
    for t in (x, x.float()):
        y2 = torch.empty_like(y)
        mx.gemm_mxfp4(t, packed, N, mx.Epilogue(y2, mx.PP_NONE))
        u.close(y2, want, bound, torch.float32, mx.last_kernel())
    # bias, into bf16 rows with a gap that stays as it was
    b = normal((N,), 3, 0.3, torch.float32)
    y3, wide = in_wide(torch.empty((M, N), dtype=torch.bfloat16, device="cuda"), 5, 9.0)
    mx.gemm_mxfp4(rows, packed, N, mx.Epilogue(y3, mx.PP_BIAS, bias=b))
    u.close(y3, want + u.f64(b), bound + u.U * np.abs(u.f64(b)) + u.U * np.abs(want), torch.bfloat16, mx.last_kernel())
    assert (wide[:, N:] == 9.0).all()


@pytest.mark.parametrize("M", [1, 12, 16, 20, 40, 100, 300])
def test_small_whole_numbers_are_exact(M):
    """Values and scales whose sums 24 bits hold: every result is exact, and with it every index of the layout."""
    K, N = 1056, 200
    g = np.random.default_rng(M)
    codes, wc = g.choice([0, 1, 2, 4, 9, 10, 12], (M, K)).astype(np.uint8), g.choice([0, 1, 2, 4, 9, 10, 12], (N, K)).astype(np.uint8)
    b, wb = g.integers(126, 129, (M, m4.blocks(K)), dtype=np.uint8), g.integers(126, 129, (N, m4.blocks(K)), dtype=np.uint8)
    t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    y = torch.empty((M, N), device="cuda")
    mx.gemm_mxfp4(mx.Mxfp4Rows.of(t(m4.pairs(codes)), t(b)), mx.pack_mxfp4(t(m4.pairs(wc)), t(wb)), N, mx.Epilogue(y, mx.PP_NONE))
    assert np.array_equal(u.f64(y), m4.values(codes, b) @ m4.values(wc, wb).T)


@pytest.mark.parametrize("M", [1, 16, 20, 40, 100, 130, 300])
def test_gelu_is_the_polynomial_of_the_other_products(M, po):
    K, N = 256, 96
    x, (q, s, _) = normal((M, K), 1), weight(N, K, 2)
    packed = mx.pack_mxfp4(q, s)
    plain, y = torch.empty((M, N), device="cuda"), torch.empty((M, N), device="cuda")
    b = normal((N,), 3, 0.3, torch.float32)
    mx.gemm_mxfp4(x, packed, N, mx.Epilogue(plain, mx.PP_NONE))
    mx.gemm_mxfp4(x, packed, N, mx.Epilogue(y, mx.PP_BIAS | mx.PP_GELU, bias=b))
    want = po.pp(plain.cpu().numpy(), po.PP_BIAS | po.PP_GELU, po.F32, bias=b.cpu().numpy())
    assert np.array_equal(y.cpu().numpy(), want)


@pytest.mark.parametrize("M,K,N", [(1, 128, 32), (3, 1000, 96), (9, 5000, 32), (16, 256, 160), (17, 700, 64), (40, 1152, 288), (64, 130, 32), (129, 512, 128), (257, 1000, 416), (600, 260, 96)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gate_up(M, K, N, dtype):
    x = normal((M, K), 1)
    (g, gs, gv), (v, vs, vv) = weight(N, K, 2), weight(N, K, 3)
    packed = mx.pack_gate_up_mxfp4(g, v, (gs, vs))
    a = m4.values(*m4.quantize(u.f64(x)))
    want, bound = u.gated(*m4.product(a, gv), *m4.product(a, vv))
    for t in (mx.quantize_mxfp4(x), x):
        y, wide = in_wide(torch.empty((M, N), dtype=dtype, device="cuda"), 3, 9.0)
        mx.gemm_mxfp4(t, packed, 2 * N, mx.Epilogue(y, mx.PP_SILU_GATE))
        u.close(y, want, bound, dtype, mx.last_kernel())
        assert (wide[:, N:] == 9.0).all()


@pytest.mark.parametrize("M", [1, 16, 33, 100, 300])
def test_rows_do_not_touch_each_other(M):
    """A row of infinities and NaN, and blocks of zeros, leave the other rows' bits as they are; the rows behind the last are not written."""
    K, N = 512, 160
    x, (q, s, _) = normal((M, K), 1), weight(N, K, 2)
    packed = mx.pack_mxfp4(q, s)
    out = torch.full((M + 3, N), 5.0, device="cuda")
    mx.gemm_mxfp4(x, packed, N, mx.Epilogue(out[:M], mx.PP_NONE))
    clean = out.clone()
    x[M // 2, 7], x[M // 2, 300] = float("inf"), float("nan")
    mx.gemm_mxfp4(x, packed, N, mx.Epilogue(out[:M], mx.PP_NONE))
    assert torch.isnan(out[M // 2]).all()
    others = [m for m in range(M + 3) if m != M // 2]
    assert torch.equal(out[others], clean[others]) and (out[M:] == 5.0).all()
    x[M // 2] = 0
    mx.gemm_mxfp4(x, packed, N, mx.Epilogue(out[:M], mx.PP_NONE))
    assert (out[M // 2] == 0).all()


@pytest.mark.parametrize("M", [1, 20, 40, 300])
def test_what_memory_behind_the_last_row_holds_does_not_matter(M):
    """Rows from M up of the last panel are never written: whatever is there, scales of 255 among it."""
    K, N = 300, 70
    x, (q, s, _) = normal((M, K), 1), weight(N, K, 2)
    packed = mx.pack_mxfp4(q, s)
    y = [torch.empty((M, N), device="cuda") for _ in range(2)]
    for fill, out in zip((0, 255), y):
        rows = mx.Mxfp4Rows.empty(M, K, x.device)
        rows.packed.fill_(fill)
        made = mx.quantize_mxfp4(x)
        codes, b, _, _ = m4.unpack(bits(made.packed), M, K)
        t = torch.from_numpy(m4.pairs(codes)).cuda(), torch.from_numpy(b).cuda()
        from mm_amx_amd import mxfp4
        mxfp4._repack(*t, M, K, 0, rows.packed)
        w = packed.clone()
        mx.gemm_mxfp4(rows, w, N, mx.Epilogue(out, mx.PP_NONE))
    assert torch.equal(*y)


@pytest.mark.parametrize("M", [1, 16, 40, 300])
def test_scales_at_the_ends(M):
    """Scales from 2^-127 to 2^127 whose products come to something that 32 bits hold, exactly; 255 makes a NaN of its row or column."""
    K, N = 32, 96
    codes = np.full((M, K), 2, np.uint8)
    wc = np.full((N, K), 3, np.uint8)
    b, wb = np.array([254, 0, 127])[np.arange(M) % 3][:, None].astype(np.uint8), np.array([0, 254, 127])[np.arange(N) % 3][:, None].astype(np.uint8)
    wb[5] = 255
    t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    y = torch.empty((M, N), device="cuda")
    mx.gemm_mxfp4(mx.Mxfp4Rows.of(t(m4.pairs(codes)), t(b)), mx.pack_mxfp4(t(m4.pairs(wc)), t(wb)), N, mx.Epilogue(y, mx.PP_NONE))
    want = 48.0 * m4.power(b) * m4.power(wb).T
    with np.errstate(over="ignore"):
        want = want.astype(np.float32).astype(np.float64)
    got = u.f64(y)
    assert np.isnan(got[:, 5]).all()
    keep = np.arange(N) != 5
    normal_range = keep & ((np.abs(want) >= 2.0 ** -126) | (want == 0)).all(0)
    assert np.array_equal(got[:, normal_range], want[:, normal_range])
    assert (np.abs(got[:, keep] - want[:, keep])[np.isfinite(want[:, keep])] <= 2.0 ** -126).all()  # (below it a result may be zero)


# ---- layers ------------------------------------------------------------------------------------------------------------
def test_linear_layer_takes_both_kinds_of_weights():
    M, K, N = 20, 301, 200
    x, wb = normal((M, K), 1), normal((N, K), 2, 0.02)
    lin = mx.LinearMxfp4()
    lin.set_weight(wb)
    y = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    lin.forward(x, y)
    a, codes = m4.values(*m4.quantize(u.f64(x))), m4.quantize(u.f64(wb))
    u.close(y, *m4.product(a, m4.values(*codes)), torch.bfloat16)
    other = copy.deepcopy(lin)
    y2 = torch.empty_like(y)
    other.forward(mx.quantize_mxfp4(x), y2)
    assert torch.equal(y, y2)
    K = 300
    q, s, w = weight(N, K, 3)
    lin.set_weight(q, s)
    b = normal((N,), 4, 1.0, torch.float32)
    lin.forward(x[:, :K], y, bias=b)
    a = m4.values(*m4.quantize(u.f64(x[:, :K])))
    want, bound = m4.product(a, w, 2)
    u.close(y, want + u.f64(b), bound + 2 * u.U * np.abs(u.f64(b)), torch.bfloat16)


@pytest.mark.parametrize("M,K,N", [(1, 256, 96), (7, 300, 352), (16, 1024, 512), (30, 640, 256), (33, 640, 288), (100, 512, 384), (200, 260, 160), (513, 384, 1056)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mlp_is_its_two_products_with_the_intermediate_quantised_from_32_bits(M, K, N, dtype):
    """Step by step through the public calls, bit for bit."""
    x = normal((M, K), 1)
    (g, gs, _), (v, vs, _), (d, ds, dv) = weight(N, K, 5), weight(N, K, 6), weight(K, N, 7)
    mlp = mx.MLP()
    mlp.setup(g, v, d, scales=(gs, vs, ds))
    y, wide = in_wide(torch.empty((M, K), dtype=dtype, device="cuda"), 3, 9.0)
    rows = mx.quantize_mxfp4(x)
    mlp.run(rows, y)
    assert (wide[:, K:] == 9.0).all()
    h = torch.empty((M, N), device="cuda")
    mx.gemm_mxfp4(rows, mx.pack_gate_up_mxfp4(g, v, (gs, vs)), 2 * N, mx.Epilogue(h, mx.PP_SILU_GATE))
    hq, want = mx.quantize_mxfp4(h), torch.empty((M, K), dtype=dtype, device="cuda")
    mx.gemm_mxfp4(hq, mx.pack_mxfp4(d, ds), K, mx.Epilogue(want, mx.PP_NONE))
    assert torch.equal(y, want)
    value, bound = m4.product(m4.values(*m4.quantize(u.f64(h))), dv)
    u.close(y, value, bound, dtype)
    if dtype == torch.bfloat16:
        assert torch.equal(copy.deepcopy(mlp).run(rows), want)


@pytest.mark.parametrize("M", [1, 5, 24, 70])
def test_mlp_from_bf16_rows_and_weights(M):
    K, N = 256, 192
    x, w = normal((M, K), 1), [normal(s, 2 + i, 0.05) for i, s in enumerate(((N, K), (N, K), (K, N)))]
    mlp = mx.MLP()
    mlp.setup(*w, compress="mxfp4")
    rows = mx.quantize_mxfp4(x)
    # (M = 1 and 5 quantise x in the product, whose sums are added in the same order)
    assert torch.equal(mlp.run(x), mlp.run(rows)) and torch.equal(mlp.run(x.float()), mlp.run(rows))
    codes = [m4.values(*m4.quantize(u.f64(t))) for t in w]
    a = m4.values(*m4.quantize(u.f64(x)))
    h, bound = u.gated(*m4.product(a, codes[0]), *m4.product(a, codes[1]))
    # A value of h that is off by `bound` may go to a neighbouring one of e2m1: by its block's largest step, 2 of its scale, where it lies next to a border
    hv, hb = m4.quantize(h)
    p = np.repeat(m4.power(hb), 32, 1)[:, :N]
    border = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5])
    near = (np.abs(np.abs(h / p)[..., None] - border) <= (bound / p)[..., None]).any(-1)
    # (where the block's largest is next to a border of its scale, all of the block; by its whole value then)
    top = np.abs(h.reshape(M, -1, 32)).max(-1)
    edge = np.repeat(np.abs(top / 7 / m4.power(hb) - 1) * 7 <= 1e-4, 32, 1) | np.repeat(np.abs(top / 3.5 / m4.power(hb) - 1) <= 1e-4, 32, 1)
    step = np.where(edge, np.abs(h) + 2 * p, np.where(near, 2 * p, 0))
    want, sums = m4.product(m4.values(hv, hb), codes[2])
    u.close(mlp.run(x), want, sums + step @ np.abs(codes[2]).T, torch.bfloat16)


@pytest.mark.parametrize("M,H", [(1, 64), (3, 300), (5, 512), (40, 1000), (300, 2048), (2, 4096), (260, 4095), (33, 8192), (2, 16384), (1, 20000)])
@pytest.mark.parametrize("residual", [torch.bfloat16, torch.float32])
def test_block_norm_quantises(M, H, residual):
    """r as without quantising; z quantised from 32 bits: against z in fp32 from the definition, a value next to a border may go to either side."""
    f, r0 = normal((M, H), 1), normal((M, H), 2, 1.0, residual)
    w = normal((H,), 3)
    r, z = mx.block_norm(f, r0, scale=0.7, pre_weight=w, quantize="mxfp4")
    plain_r, plain_z = mx.block_norm(f, r0, scale=0.7, pre_weight=w)
    assert torch.equal(r, plain_r) and z.shape == (M, H)
    codes, b, rest, rest_s = m4.unpack(bits(z.packed), M, H)
    assert not (rest & 7).any() and not (rest_s == 255).any()
    rr = u.f64(r0) + np.float64(np.float32(0.7)) * u.f64(f)
    exact = rr / np.sqrt((rr ** 2).mean(1, keepdims=True) + 1e-6) * u.f64(w)
    got = m4.values(codes, b)
    # relative error of z: r one rounding, sum of squares H + 8 roundings / 2, rsqrt 2, products 3
    err = np.abs(exact) * (H / 64 + 16) * u.U
    p = np.repeat(m4.power(b), 32, 1)[:, :H]
    a = np.abs(exact) / p
    half = np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1.0))
    top = np.abs(np.pad(exact, ((0, 0), (0, -H % 32)))).reshape(M, -1, 32).max(-1) / m4.power(b)
    tol = (H / 64 + 16) * u.U * 8
    assert (top < 7 + tol).all() and ((top >= 3.5 - tol) | (b == 1)).all()
    assert (np.abs(got - exact) <= half * p + err).all()
    # without norm and weights: the quantiser's bits of a sum that is exact
    one = mx.block_norm(f, None, pre=False, quantize="mxfp4", r=False)[1]
    check_rows(one, f)
    out = mx.Mxfp4Rows.empty(M, H, f.device)
    assert mx.block_norm(f, r0, scale=0.7, pre_weight=w, quantize="mxfp4", z=out)[1] is out
    again = m4.unpack(bits(out.packed), M, H)
    assert np.array_equal(again[0], codes) and np.array_equal(again[1], b)


def test_graph_and_streams():
    """Replays of a captured layer beside eager calls of it on another stream: the scratch of each is its own."""
    K, N = 512, 256
    mlp = mx.MLP()
    mlp.setup(normal((N, K), 1, 0.05), normal((N, K), 2, 0.05), normal((K, N), 3, 0.05), compress="mxfp4")
    xs = [normal((M, K), 10 + M) for M in (1, 20, 200)]
    want = [mlp.run(x) for x in xs]
    side = torch.cuda.Stream()
    graphs = []
    for x in xs:
        with torch.cuda.stream(side):
            mlp.run(x)
            side.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                y = mlp.run(x)
            graphs.append((gr, y))
    torch.cuda.synchronize()
    for _ in range(4):
        for (gr, y), x, w in zip(graphs, xs, want):
            y.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                gr.replay()
            eager = mlp.run(x)
            torch.cuda.synchronize()
            assert torch.equal(y, w) and torch.equal(eager, w)


def test_nothing_to_do():
    q, s, _ = weight(64, 128, 1)
    packed = mx.pack_mxfp4(q, s)
    x = torch.empty((0, 128), dtype=torch.bfloat16, device="cuda")
    rows = mx.quantize_mxfp4(x)
    assert rows.shape == (0, 128) and rows.q.shape == (0, 64) and mx.dequantize_mxfp4(rows).shape == (0, 128)
    for a in (x, rows):
        mx.gemm_mxfp4(a, packed, 64, mx.Epilogue(torch.empty((0, 64), device="cuda"), mx.PP_NONE))
    assert mx.block_norm(x, quantize="mxfp4")[1].shape == (0, 128)


def test_refusals_on_the_gpu():
    q, s, _ = weight(96, 256, 1)
    packed = mx.pack_mxfp4(q, s)
    x = normal((4, 256), 1)
    y = torch.empty((4, 96), device="cuda")
    ok = lambda **k: mx.gemm_mxfp4(**{**dict(A=x, Bpacked=packed, N=96, ep=mx.Epilogue(y, mx.PP_NONE)), **k})  # noqa: E731
    ok()
    for bad in (dict(A=x.half()), dict(A=x[:, :0]), dict(A=x.t()), dict(A=q), dict(Bpacked=packed[:-1]), dict(Bpacked=packed.view(2, -1)), dict(Bpacked=packed[8:]),
                dict(N=97), dict(N=0), dict(N=96.0), dict(ep=mx.Epilogue(y[:, :95], mx.PP_NONE)), dict(A=mx.Mxfp4Rows(mx.quantize_mxfp4(x).packed, 40, 256)),
                dict(A=mx.Mxfp4Rows(mx.quantize_mxfp4(x).packed, 4, 0)), dict(A=mx.quantize_mxfp4(normal((4, 520), 1))),
                dict(ep=mx.Epilogue(y.half(), mx.PP_NONE)), dict(ep=mx.Epilogue(y, mx.PP_DEQUANT)), dict(ep=mx.Epilogue(y, mx.PP_QUANT)),
                dict(ep=mx.Epilogue(y, mx.PP_BIAS)), dict(ep=mx.Epilogue(y, mx.PP_BIAS, bias=torch.zeros(95, device="cuda"))),
                dict(ep=mx.Epilogue(y, mx.PP_SILU_GATE)), dict(ep=mx.Epilogue(y[:3], mx.PP_NONE)), dict(A=x.cpu()), dict(ep=None)):
        with pytest.raises(mx.MmxError):
            ok(**bad)
    for call in (lambda: mx.quantize_mxfp4(x.half()), lambda: mx.quantize_mxfp4(x[0]), lambda: mx.quantize_mxfp4(x[:, :0]), lambda: mx.pack_mxfp4(q), lambda: mx.pack_mxfp4(q, s[:, :1]),
                 lambda: mx.pack_mxfp4(q, s.float()), lambda: mx.pack_gate_up_mxfp4(q[:40], q[:40], (s[:40], s[:40])), lambda: mx.pack_gate_up_mxfp4(q, q, (s,)),
                 lambda: mx.pack_mxfp4(q, s, out=packed[:-1]), lambda: mx.Mxfp4Rows.of(q, s, 300), lambda: mx.dequantize_mxfp4(x), lambda: mx.dequantize_mxfp4(mx.quantize_mxfp4(x), torch.half),
                 lambda: mx.block_norm(x, quantize="fp4"), lambda: mx.block_norm(x, quantize="mxfp4", z=mx.quantize_fp8(x)), lambda: mx.block_norm(x, quantize=True, z=mx.quantize_mxfp4(x)),
                 lambda: mx.MLP().setup(q, q, q, scales=(s, s, s)), lambda: mx.MLP().setup(x, x, x.t(), compress="mxfp8")):
        with pytest.raises(mx.MmxError):
            call()


@pytest.mark.parametrize("M,K,N,pair,kernel", [
    (4096, 300, 4090, False, "256x256"), (582, 110, 19008, True, "256x256"), (2048, 4096, 5900, False, "256x192"), (700, 520, 21952, True, "128x128"), (1030, 10900, 4090, False, "128x256"),
    (264, 4159, 14528, True, "128x256"), (223, 103, 17257, False, "128x128"), (900, 400, 8192, True, "128x128"), (700, 1000, 4001, False, "128x128_k_by_2"),
    (513, 1000, 4032, True, "128x128_k_by_2"), (68, 5225, 15139, False, "64x128_k_by_2"), (73, 127, 9216, True, "64x128_k_by_2"), (300, 2950, 5056, True, "64x128_k_by_2"),
    (391, 1001, 3001, False, "64x64"), (300, 260, 3008, True, "64x64_k_by_2_pair"), (65, 3100, 705, False, "32x32_k_by_8"), (33, 2950, 130, False, "32x32_k_by_8"), (35, 349, 13318, False, "64x64_k_by_2"),
    (33, 3100, 704, True, "64x64_k_by_2_pair"), (70, 2950, 128, True, "64x64_k_by_2_pair"), (33, 100, 70, False, "32x32_k_by_8"), (65, 1300, 2050, False, "32x32_k_by_8"), (65, 128, 1537, False, "32x64_k_by_4"), (100, 2600, 4001, False, "32x64_k_by_4"), (20, 300, 9000, False, "rows_32"), (31, 515, 70, False, "rows_32"),
    (17, 300, 640, True, "rows_32_pair"), (16, 1000, 65, False, "rows_16"), (9, 5000, 192, True, "rows_16_pair"), (3, 1000, 190, False, "rows_16"), (3, 1000, 192, True, "rows_16_pair")])
def test_every_kernel_that_products_choose(M, K, N, pair, kernel):
    """Sizes with rows, k and columns left over, an even and an odd number of chunks of k, one band of eight rows of tiles and more.  N: packed columns."""
    rows = mx.quantize_mxfp4(normal((M, K), 1))
    a = torch.from_numpy(m4.values(*m4.unpack(bits(rows.packed), M, K)[:2])).cuda()
    wb = normal((N, K), 2, 0.05)
    codes = [mx.quantize_mxfp4(w) for w in ((wb[:N // 2], wb[N // 2:]) if pair else (wb,))]
    w = [mx.dequantize_mxfp4(c, torch.float32).double() for c in codes]
    packed = mx.pack_gate_up_mxfp4(wb[:N // 2].contiguous(), wb[N // 2:].contiguous()) if pair else mx.pack_mxfp4(wb)
    product = lambda b: (a @ b.T, (m4.blocks(K) + 4) * u.U * (a.abs() @ b.abs().T))  # noqa: E731 (m4.product, on the GPU in 64 bits)
    n = N // 2 if pair else N
    for dtype in (torch.float32, torch.bfloat16):
        y, wide = in_wide(torch.empty((M, n), dtype=dtype, device="cuda"), 3, 9.0)
        mx.gemm_mxfp4(rows, packed, N, mx.Epilogue(y, mx.PP_SILU_GATE if pair else mx.PP_NONE))
        assert mx.last_kernel() == f"mxfp4_{kernel}"
        if pair:
            (g, eg), (v, ev) = product(w[0]), product(w[1])
            want, bound = u.gated(*(t.cpu().numpy() for t in (g, eg, v, ev)))
        else:
            want, bound = (t.cpu().numpy() for t in product(w[0]))
        u.close(y, want, bound, dtype, kernel)
        assert (wide[:, n:] == 9.0).all()
        if dtype == torch.float32 and not pair:  # (one addition more)
            b = normal((N,), 5, 1.0, torch.float32)
            biased = torch.empty((M, N), device="cuda")
            mx.gemm_mxfp4(rows, packed, N, mx.Epilogue(biased, mx.PP_BIAS, bias=b))
            assert torch.equal(biased, y + b)


@pytest.mark.parametrize("M,K,N", [(40, 640, 288), (300, 512, 1056), (700, 520, 10976), (1030, 5000, 4000), (900, 400, 4096), (264, 4159, 7264), (700, 1000, 2016), (130, 1000, 4096)])
def test_the_intermediate_of_every_tile_is_quantised_as_by_the_quantiser(M, K, N):
    """The MLP's own quantisation in the tiles that a pair can have, against its two products through the public calls, bit for bit."""
    x = mx.quantize_mxfp4(normal((M, K), 1))
    g, v, d = normal((N, K), 2, 0.05), normal((N, K), 3, 0.05), normal((K, N), 4, 0.05)
    mlp = mx.MLP()
    mlp.setup(g, v, d, compress="mxfp4")
    h, want = torch.empty((M, N), device="cuda"), torch.empty((M, K), device="cuda")
    mx.gemm_mxfp4(x, mx.pack_gate_up_mxfp4(g, v), 2 * N, mx.Epilogue(h, mx.PP_SILU_GATE))
    mx.gemm_mxfp4(mx.quantize_mxfp4(h), mx.pack_mxfp4(d), K, mx.Epilogue(want, mx.PP_NONE))
    assert torch.equal(mlp.run(x, torch.empty((M, K), device="cuda")), want)


def test_weights_of_more_than_4_gib():
    """Panels past 2^32 bytes: columns at the far end of [600000, 14336] weights, of which the others are zero."""
    N, K, M = 600000, 14336, 3
    packed = torch.zeros(-(-N // 32) * -(-K // 256) * 4352, dtype=torch.uint8, device="cuda")
    assert packed.numel() > 2 ** 32
    w = normal((64, K), 2, 0.05)
    part = mx.pack_mxfp4(w)
    packed[packed.numel() - part.numel():] = part
    x = normal((40, K), 1)
    a, b = m4.values(*m4.quantize(u.f64(x))), m4.values(*m4.quantize(u.f64(w)))
    want, bound = m4.product(a, b)
    for M in (3, 40):
        y = torch.full((M, N), 5.0, dtype=torch.bfloat16, device="cuda")
        mx.gemm_mxfp4(x[:M], packed, N, mx.Epilogue(y, mx.PP_NONE))
        u.close(y[:, N - 64:], want[:M], bound[:M], torch.bfloat16, mx.last_kernel())
        assert (y[:, :N - 64] == 0).all()
        del y


def test_native_and_python_calls_agree(monkeypatch):
    from mm_amx_amd import _lib as L
    K, N = 300, 96
    x, w = normal((20, K), 1), normal((N, K), 2, 0.05)
    d = normal((K, N), 3, 0.05)
    packed, bias = mx.pack_mxfp4(w), normal((N,), 4, 1.0, torch.float32)
    gu, down = mx.pack_gate_up_mxfp4(w, w), mx.pack_mxfp4(d)

    def calls():
        y = torch.empty((20, N), device="cuda")
        mx.gemm_mxfp4(x, packed, N, mx.Epilogue(y, mx.PP_BIAS, bias=bias))
        rows = mx.quantize_mxfp4(x)
        r, z = mx.block_norm(x, x, quantize="mxfp4")
        return [y, mx.dequantize_mxfp4(rows), mx.dequantize_mxfp4(rows, torch.float32), mx.mlp_mxfp4(rows, gu, down, N), mx.mlp_mxfp4(x, gu, down, N, y=torch.empty((20, K), device="cuda")), r,
                mx.dequantize_mxfp4(z)]

    native = calls()
    assert L._native is not None
    monkeypatch.setattr(L, "_native", None)
    for a, b in zip(native, calls()):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_packed_weights_on_disk(tmp_path):
    from mm_amx_amd import packed_io
    N, K = 160, 300
    packed = mx.pack_mxfp4(normal((N, K), 1))
    path = str(tmp_path / "w.safetensors")
    packed_io.save_packed(path, packed, "mxfp4", K, N)
    w = packed_io.load_packed(path)
    assert torch.equal(w["packed"], packed) and w["scales"] is None and (w["dtype"], w["K"], w["N"]) == ("mxfp4", K, N)
    for bad in (dict(packed=packed[:-1]), dict(scales=torch.ones(N)), dict(K=2 * K)):
        with pytest.raises(mx.MmxError):
            packed_io.save_packed(path, **{**dict(packed=packed, dtype="mxfp4", K=K, N=N), **bad})


def test_the_stack_over_4_bit_weights_with_a_head_and_tokens():
    from mm_amx_amd import mlp_llama
    out = mlp_llama.perf_llama7b_MLP(M=5, num_layers=2, rounds=1, hidden_size=256, intermediate_size=704, verbose=False, vocab=1000)
    assert out["tokens"].shape == (5,) and bool(((out["tokens"] >= 0) & (out["tokens"] < 1000)).all())
    # three quantisations to 3 significant bits, 2^-2 of a value at most, against none
    assert out["rel_err_mxfp4_one_layer"] < 3 * 2.0 ** -2


def test_any_true_value_of_quantize_is_e4m3(monkeypatch):
    from mm_amx_amd import _lib as L
    x = normal((20, 300), 1)
    r, want = mx.block_norm(x, x, quantize=True)
    for native in (L._native, None):
        monkeypatch.setattr(L, "_native", native)
        for quantize in (1, 2, 3):
            r1, z = mx.block_norm(x, x, quantize=quantize)
            assert type(z) is mx.Fp8Rows and torch.equal(r1, r) and torch.equal(z.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(z.scales, want.scales)


def test_a_refused_setup_leaves_the_mlp_running():
    N, K = 96, 256
    w, d = normal((N, K), 1, 0.05), normal((K, N), 2, 0.05)
    x = normal((5, K), 3)
    mlp = mx.MLP()
    mlp.setup(w, w, d, compress="mxfp4")
    want = mlp.run(x)
    for bad in (dict(w_up=w[:32], compress="fp8"), dict(w_up=w[:32]), dict(w_gate=w.cpu()), dict(w_down=d.float(), compress="fp8"), dict(w_down=d.float()), dict(w_down=d.half(), compress="mxfp4")):
        with pytest.raises(mx.MmxError):
            mlp.setup(**{**dict(w_gate=w, w_up=w, w_down=d), **bad})
        assert torch.equal(mlp.run(x), want)
    mlp.setup(w, w, d)
    plain = mx.MLP()
    plain.setup(w, w, d)
    assert torch.equal(mlp.run(x), plain.run(x))


def test_a_second_setup_may_have_other_sizes():
    """Whatever the weights are and were: the intermediate of an earlier run does not stay."""
    x = {K: normal((5, K), K) for K in (128, 256)}
    mlp = mx.MLP()
    for compress in (None, "mxfp4", "fp8", None):
        for N, K in ((64, 128), (192, 256), (96, 256), (160, 128)):
            w, d = normal((N, K), N, 0.05), normal((K, N), N + 1, 0.05)
            mlp.setup(w, w, d, compress=compress)
            fresh = mx.MLP()
            fresh.setup(w, w, d, compress=compress)
            assert torch.equal(mlp.run(x[K]), fresh.run(x[K]))
