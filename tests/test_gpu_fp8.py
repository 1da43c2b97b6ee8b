"""Products in 8-bit floating point with a scale for each block of 128, their quantisers and the MLP over them, against their definitions in 64 bits."""
import copy

import numpy as np
import pytest
import torch

import ffn_util as u

pytestmark = pytest.mark.gpu

import mm_amx_amd as mx  # noqa: E402

E4 = torch.float8_e4m3fn


def bits(t):
    return t.detach().cpu().contiguous().view(torch.uint8).numpy()


def normal(shape, seed, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def weight(N, K, seed, pow2=False):
    """e4m3 weights [N, K] and scales as a checkpoint holds them."""
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn((N, K), generator=g) * 100).clamp(-448, 448).to(E4).cuda()
    s = torch.rand((u.blocks(N), u.blocks(K)), generator=g) * 1e-3 + 1e-4
    return w, (torch.exp2(torch.round(torch.log2(s))) if pow2 else s).cuda()


def in_wide(t, extra, fill):
    """The same values in rows `extra` elements longer than they are, and the whole buffer."""
    wide = torch.full((t.shape[0], t.shape[1] + extra), fill, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]], wide


# ---- quantisers --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (5, 129), (7, 7), (33, 1000), (130, 256), (2, 11008)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_rows_bits(M, K, dtype):
    x = normal((M, K), M * K, 3.0, dtype)
    q, s = mx.quantize_fp8(x)
    want_q, want_s = u.quantize_rows(u.f64(x))
    assert np.array_equal(u.f64(s), want_s)
    assert np.array_equal(bits(q), want_q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_special_values(dtype):
    x = torch.zeros((12, 256), dtype=dtype)
    x[1, 3] = 448.0                       # on the border: scale 1
    x[2, 3] = 450.0                       # past it: scale 2
    x[3, :128] = torch.arange(128) * 0.25 - 16
    x[4, 5], x[4, 6] = float("inf"), 1.0  # the block is NaN, the next one is not
    x[4, 200] = 2.0
    x[5, 0], x[5, 1] = float("nan"), 1.0
    x[6, 0] = 2.0 ** -133                 # subnormal
    x[7, 0] = 2.0 ** -126
    x[8, 0] = 3.0e38
    x[9, 0], x[9, 1:] = 448.0, 17.0       # 17 lies between 16 and 18: the even one
    x[10, 0], x[10, 1:] = -448.0, -19.0   # 19 between 18 and 20
    x[11, 0], x[11, 1:] = 448.0, 2.0 ** -10  # half of the smallest e4m3: to zero
    q, s = mx.quantize_fp8(x.cuda())
    want_q, want_s = u.quantize_rows(u.f64(x))
    assert np.array_equal(u.f64(s), want_s, equal_nan=True)
    nan = want_q & 127 == 127
    assert np.array_equal(bits(q) & 127 == 127, nan)
    assert np.array_equal(bits(q)[~nan], want_q[~nan])


def test_quantize_reads_rows_of_any_stride_and_pads_with_zeros():
    base = normal((9, 333), 5)
    for x in (base[:, 1:302], base[::2, 3:300], base[2:3, 5:6]):
        rows = mx.quantize_fp8(x)
        want_q, want_s = u.quantize_rows(u.f64(x))
        assert np.array_equal(bits(rows.q), want_q) and np.array_equal(u.f64(rows.scales), want_s)
        assert not bits(rows.padded)[:, x.shape[1]:].any()


@pytest.mark.parametrize("K,N", [(1, 1), (128, 128), (129, 33), (300, 257), (1000, 100), (17, 500)])
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_pack_bits(K, N, transpose):
    W = normal((N, K) if transpose else (K, N), K + N, 0.02)
    packed, s = mx.quantize_pack_fp8(W, transpose)
    assert packed.numel() == mx.packed_b_bytes(mx.F8, K, N)
    w = u.f64(W) if transpose else u.f64(W).T
    amax = np.array([[np.abs(w[n:n + 128, k:k + 128]).max() for k in range(0, K, 128)] for n in range(0, N, 128)])
    want_s = u.scale_of(amax)
    assert np.array_equal(u.f64(s), want_s)
    codes, pad = u.unpack_bytes(bits(packed), K, N)
    assert np.array_equal(codes & 127, u.encode(w / u.spread(want_s, N, K)) & 127)
    assert np.array_equal(u.decode(codes), u.decode(u.encode(w / u.spread(want_s, N, K))))
    assert not pad.any()


@pytest.mark.parametrize("K,N", [(128, 32), (200, 96), (1000, 160)])
def test_gate_up_pairs_hold_both_in_turn(K, N):
    g, gs = weight(N, K, 1)
    v, vs = weight(N, K, 2)
    packed, s = mx.pack_gate_up_fp8(g, v, (gs, vs))
    codes, _ = u.unpack_bytes(bits(packed), K, 2 * N)
    both = codes.reshape(N // 32, 2, 32, K)
    assert np.array_equal(both[:, 0].reshape(N, K), bits(g)) and np.array_equal(both[:, 1].reshape(N, K), bits(v))
    assert torch.equal(s, torch.cat([gs, vs]))
    gb, ub = normal((N, K), 3, 0.02), normal((N, K), 4, 0.5)
    packed, s = mx.pack_gate_up_fp8(gb, ub)
    one = [mx.pack_fp8(w) for w in (gb, ub)]
    both = u.unpack_bytes(bits(packed), K, 2 * N)[0].reshape(N // 32, 2, 32, K)
    for i, (p, sc) in enumerate(one):
        assert np.array_equal(both[:, i].reshape(N, K), u.unpack_bytes(bits(p), K, N)[0])
        assert torch.equal(s[i * u.blocks(N):(i + 1) * u.blocks(N)], sc)


# ---- products ----------------------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 128, 16), (1, 4096, 96), (2, 127, 33), (15, 129, 31), (16, 640, 160), (17, 1000, 200), (31, 2048, 129), (33, 300, 500), (48, 4100, 64),
         (64, 1152, 130), (65, 128, 257), (100, 515, 70), (127, 2304, 40), (129, 1000, 300), (200, 129, 513), (256, 1024, 256), (257, 384, 258),
         (300, 4096, 65), (391, 1000, 3001), (513, 700, 1030), (1000, 260, 90), (1030, 2050, 520), (2049, 130, 290)]


@pytest.mark.parametrize("M,K,N", SIZES)
def test_product(M, K, N):
    x = normal((M, K), 1)
    w, s = weight(N, K, 2)
    rows = mx.quantize_fp8(x)
    packed, scales = mx.pack_fp8(w, s)
    assert torch.equal(scales, s)
    want, bound = u.product(u.value_rows(bits(rows.q), u.f64(rows.scales)), u.f64(w) * u.spread(u.f64(s), N, K), 8)
    y = torch.full((M, N), 7.0, device="cuda")
    mx.gemm_fp8(rows, packed, scales, N, mx.Epilogue(y, mx.PP_NONE))
    u.close(y, want, bound, torch.float32, mx.last_kernel())
    # from bf16: the same rows, quantised on the way
    y2 = torch.empty_like(y)
    mx.gemm_fp8(x, packed, scales, N, mx.Epilogue(y2, mx.PP_NONE))
    u.close(y2, want, bound, torch.float32, mx.last_kernel())
    # bias, into bf16 rows with a gap that stays as it was
    b = normal((N,), 3, 0.3, torch.float32)
    y3, wide = in_wide(torch.empty((M, N), dtype=torch.bfloat16, device="cuda"), 5, 9.0)
    mx.gemm_fp8(rows, packed, scales, N, mx.Epilogue(y3, mx.PP_BIAS, bias=b))
    u.close(y3, want + u.f64(b), bound + u.U * np.abs(u.f64(b)) + u.U * np.abs(want), torch.bfloat16, mx.last_kernel())
    assert (wide[:, N:] == 9.0).all()


@pytest.mark.parametrize("M", [1, 16, 20, 40, 100, 130, 300])
def test_gelu_is_the_polynomial_of_the_other_products(M, po):
    K, N = 256, 96
    x, (w, s) = normal((M, K), 1), weight(N, K, 2)
    packed, scales = mx.pack_fp8(w, s * 0.05)
    plain, y = torch.empty((M, N), device="cuda"), torch.empty((M, N), device="cuda")
    b = normal((N,), 3, 0.3, torch.float32)
    mx.gemm_fp8(x, packed, scales, N, mx.Epilogue(plain, mx.PP_NONE))
    mx.gemm_fp8(x, packed, scales, N, mx.Epilogue(y, mx.PP_BIAS | mx.PP_GELU, bias=b))
    want = po.pp(plain.cpu().numpy(), po.PP_BIAS | po.PP_GELU, po.F32, bias=b.cpu().numpy())
    assert np.array_equal(y.cpu().numpy(), want)


@pytest.mark.parametrize("M,K,N", [(1, 128, 32), (3, 1000, 96), (16, 256, 160), (17, 700, 64), (40, 1152, 288), (64, 130, 32), (129, 512, 128), (257, 1000, 416), (600, 260, 96)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gate_up(M, K, N, dtype):
    x = normal((M, K), 1)
    (g, gs), (v, vs) = weight(N, K, 2), weight(N, K, 3)
    gs, vs = gs * 0.1, vs * 0.1
    packed, s = mx.pack_gate_up_fp8(g, v, (gs, vs))
    rows = mx.quantize_fp8(x)
    a = u.value_rows(bits(rows.q), u.f64(rows.scales))
    want, bound = u.gated(*u.product(a, u.f64(g) * u.spread(u.f64(gs), N, K), 8), *u.product(a, u.f64(v) * u.spread(u.f64(vs), N, K), 8))
    y, wide = in_wide(torch.empty((M, N), dtype=dtype, device="cuda"), 3, 9.0)
    mx.gemm_fp8(rows, packed, s, 2 * N, mx.Epilogue(y, mx.PP_SILU_GATE))
    u.close(y, want, bound, dtype, mx.last_kernel())
    assert (wide[:, N:] == 9.0).all()


@pytest.mark.parametrize("M,K,N,pair,tile", [(640, 300, 11000, False, "128x256"), (1200, 260, 5999, False, "128x256"), (640, 300, 11008, True, "128x256"), (1200, 260, 6016, True, "128x256"),
                                             (2300, 700, 3900, False, "256x192"), (2300, 700, 3904, True, "256x192")])
def test_large_tiles(M, K, N, pair, tile):
    """The two tiles that smaller products do not choose, their last rows and columns in part, over one band of eight rows of tiles and more.  N: packed columns."""
    x = normal((M, K), 1)
    rows = mx.quantize_fp8(x)
    a = u.value_rows(bits(rows.q), u.f64(rows.scales))
    if pair:
        (g, gs), (v, vs) = weight(N // 2, K, 2), weight(N // 2, K, 3)
        gs, vs = gs * 0.1, vs * 0.1
        packed, s = mx.pack_gate_up_fp8(g, v, (gs, vs))
        want, bound = u.gated(*u.product(a, u.f64(g) * u.spread(u.f64(gs), N // 2, K), 8), *u.product(a, u.f64(v) * u.spread(u.f64(vs), N // 2, K), 8))
    else:
        w, sw = weight(N, K, 2)
        packed, s = mx.pack_fp8(w, sw)
        want, bound = u.product(a, u.f64(w) * u.spread(u.f64(sw), N, K), 8)
    y, wide = in_wide(torch.empty((M, want.shape[1]), device="cuda"), 3, 9.0)
    mx.gemm_fp8(rows, packed, s, N, mx.Epilogue(y, mx.PP_SILU_GATE if pair else mx.PP_NONE))
    assert mx.last_kernel() == f"fp8_{tile}" + ("_pair" if pair else "")
    u.close(y, want, bound, torch.float32, mx.last_kernel())
    assert (wide[:, want.shape[1]:] == 9.0).all()


@pytest.mark.parametrize("M,K,N,pair,kernel", [
    (513, 1000, 4001, False, "64x128"), (700, 300, 2999, False, "64x128"), (200, 500, 11000, False, "64x128"), (513, 1000, 4032, True, "64x128"), (300, 260, 9024, True, "64x128"),
    (129, 129, 15936, True, "64x128"), (65, 3100, 705, False, "64x64_shared_k"), (33, 2950, 130, False, "64x64_shared_k"), (33, 3100, 704, True, "64x64_shared_k"),
    (70, 2950, 128, True, "64x64_shared_k"), (129, 1000, 300, False, "64x64"), (40, 1152, 576, True, "64x64"), (70, 130, 320, True, "64x64"),
    (20, 300, 9000, False, "rows_32"), (31, 515, 70, False, "rows_32"), (17, 300, 640, True, "rows_32_pair"), (16, 1000, 65, False, "rows_16"), (9, 1000, 192, True, "rows_16_pair")])
def test_every_kernel_that_products_choose(M, K, N, pair, kernel):
    """Sizes with rows, k and columns left over, an even and an odd number of blocks of k.  N: packed columns."""
    x = normal((M, K), 1)
    rows = mx.quantize_fp8(x)
    a = u.value_rows(bits(rows.q), u.f64(rows.scales))
    if pair:
        (g, gs), (v, vs) = weight(N // 2, K, 2), weight(N // 2, K, 3)
        gs, vs = gs * 0.1, vs * 0.1
        packed, s = mx.pack_gate_up_fp8(g, v, (gs, vs))
        want, bound = u.gated(*u.product(a, u.f64(g) * u.spread(u.f64(gs), N // 2, K), 8), *u.product(a, u.f64(v) * u.spread(u.f64(vs), N // 2, K), 8))
    else:
        w, sw = weight(N, K, 2)
        packed, s = mx.pack_fp8(w, sw)
        want, bound = u.product(a, u.f64(w) * u.spread(u.f64(sw), N, K), 8)
    for dtype in (torch.float32, torch.bfloat16):
        y, wide = in_wide(torch.empty((M, want.shape[1]), dtype=dtype, device="cuda"), 3, 9.0)
        mx.gemm_fp8(rows, packed, s, N, mx.Epilogue(y, mx.PP_SILU_GATE if pair else mx.PP_NONE))
        assert mx.last_kernel() == f"fp8_{kernel}"
        u.close(y, want, bound, dtype, kernel)
        assert (wide[:, want.shape[1]:] == 9.0).all()


@pytest.mark.parametrize("M", [1, 16, 33, 100, 300])
def test_rows_do_not_touch_each_other(M):
    """A row of infinities and NaN, and blocks of zeros, leave the other rows' bits as they are; the rows behind the last are not written."""
    K, N = 512, 160
    x, (w, s) = normal((M, K), 1), weight(N, K, 2)
    packed, scales = mx.pack_fp8(w, s)
    out = torch.full((M + 3, N), 5.0, device="cuda")
    mx.gemm_fp8(x, packed, scales, N, mx.Epilogue(out[:M], mx.PP_NONE))
    clean = out.clone()
    x[M // 2, 7], x[M // 2, 300] = float("inf"), float("nan")
    mx.gemm_fp8(x, packed, scales, N, mx.Epilogue(out[:M], mx.PP_NONE))
    assert torch.isnan(out[M // 2]).all()
    others = [m for m in range(M + 3) if m != M // 2]
    assert torch.equal(out[others], clean[others]) and (out[M:] == 5.0).all()
    x[M // 2] = 0
    mx.gemm_fp8(x, packed, scales, N, mx.Epilogue(out[:M], mx.PP_NONE))
    assert (out[M // 2] == 0).all()


@pytest.mark.parametrize("M", [1, 16, 20, 40, 100, 600])
def test_scales_whose_products_are_at_the_ends_of_32_bits(M):
    """Products of scales from 1.75 * 2^-126 to 1.5 * 2^127, bit for bit: values that are small multiples of 2^-9, so that a block's sum is exact and what is rounded is
    its one product with the scales (subnormal for the least of them)."""
    K, N = 128, 384
    g = torch.Generator().manual_seed(M)
    q, w = torch.randint(1, 8, (M, K), generator=g, dtype=torch.uint8), torch.randint(1, 8, (N, K), generator=g, dtype=torch.uint8)  # (codes of subnormals of e4m3)
    sA = torch.tensor([2.0 ** 100, 2.0 ** -100, 1.0])[torch.arange(M) % 3][None]
    sB = torch.tensor([[1.5 * 2.0 ** 27], [1.75 * 2.0 ** -26], [3.0]])
    packed, scales = mx.pack_fp8(w.view(E4).cuda(), sB.cuda())
    y = torch.empty((M, N), device="cuda")
    mx.gemm_fp8(mx.Fp8Rows.of(q.view(E4).cuda(), sA.cuda()), packed, scales, N, mx.Epilogue(y, mx.PP_NONE))
    sums = (q.double() @ w.double().t()) * 2.0 ** -18
    assert torch.equal(y.cpu(), (sums * (sA.double().t() * sB.double()[:, 0].repeat_interleave(128))).float())


def test_rows_from_elsewhere():
    """Values and scales that the quantiser did not make: any scales, rows of any stride and length."""
    g = torch.Generator().manual_seed(3)
    for M, K in ((5, 256), (40, 300), (1, 100), (200, 640)):
        N = 96
        base = (torch.randn((M, K + 16), generator=g) * 50).clamp(-448, 448).to(E4).cuda()
        s = (torch.rand((u.blocks(K), M), generator=g) + 0.5).cuda()
        w, ws = weight(N, K, 4)
        packed, scales = mx.pack_fp8(w, ws)
        y = torch.empty((M, N), device="cuda")
        for q in (base[:, :K], base[:, 1:K + 1]):
            rows = mx.Fp8Rows.of(q, s)
            mx.gemm_fp8(rows, packed, scales, N, mx.Epilogue(y, mx.PP_NONE))
            u.close(y, *u.product(u.value_rows(bits(q), u.f64(s)), u.f64(w) * u.spread(u.f64(ws), N, K), 8), torch.float32)


# ---- layers ------------------------------------------------------------------------------------------------------------
def test_linear_layer_takes_both_kinds_of_weights():
    M, K, N = 20, 300, 200
    x, wb = normal((M, K), 1), normal((N, K), 2, 0.02)
    lin = mx.LinearFp8()
    lin.set_weight(wb)
    y = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    lin.forward(x, y)
    sc = u.scale_of(np.array([[np.abs(u.f64(wb)[n:n + 128, k:k + 128]).max() for k in range(0, K, 128)] for n in range(0, N, 128)]))
    w = u.decode(u.encode(u.f64(wb) / u.spread(sc, N, K))) * u.spread(sc, N, K)
    a = u.value_rows(*u.quantize_rows(u.f64(x)))
    u.close(y, *u.product(a, w, 8), torch.bfloat16)
    other = copy.deepcopy(lin)
    y2 = torch.empty_like(y)
    other.forward(mx.quantize_fp8(x), y2)
    assert torch.equal(y, y2)


def test_scales_that_are_parameters():
    """torch.nn.Parameter requires a gradient unless told otherwise: what is packed is not part of a graph, and layers over it can be copied."""
    K, N = 256, 160
    x, (w, s), (d, ds) = normal((3, K), 1), weight(N, K, 2), weight(K, N, 3)
    p, dp = torch.nn.Parameter(s), torch.nn.Parameter(ds)
    assert p.requires_grad
    for packed, scales in (mx.pack_fp8(w, p), mx.pack_gate_up_fp8(w, w, (p, p))):
        assert not packed.requires_grad and not scales.requires_grad
    one, other = mx.LinearFp8(), mx.LinearFp8()
    one.set_weight(w, p)
    other.set_weight(w, s)
    y, y2 = torch.empty((3, N), device="cuda"), torch.empty((3, N), device="cuda")
    copy.deepcopy(one).forward(x, y)
    other.forward(x, y2)
    assert torch.equal(y, y2)
    mlp, same = mx.MLP(), mx.MLP()
    mlp.setup(w, w, d, scales=(p, p, dp))
    same.setup(w, w, d, scales=(s, s, ds))
    assert torch.equal(copy.deepcopy(mlp).run(x), same.run(x))


@pytest.mark.parametrize("M,K,N", [(1, 256, 96), (7, 300, 352), (16, 1024, 512), (30, 640, 256), (100, 512, 384), (200, 260, 160), (513, 384, 1056)])
def test_mlp(M, K, N):
    """Stage by stage: the intermediate that the gate/up product gives in fp32 is quantised to the same bits as by the quantiser.  Over both stages only
    values of h next to a border of e4m3 can fall on the other side.  The products' error is 1.5e-5 of their typical size (seven of eight
    cut off by 2^-14 of the largest product on average, as ffn_util.product has it, add up like independent errors), h = silu(g) u has that of both, 3e-5;
    so some 3e-5 / 2^-4 * 2 = 9.6e-4 of h fall on the other side, each by 2^-3 of itself at most: 3.9e-3 together in the 2-norm, beside bf16's 2^-8."""
    x = normal((M, K), 1)
    ws = [weight(*shape, 5 + i) for i, shape in enumerate(((N, K), (N, K), (K, N)))]
    ws = [(w, s * 0.2) for w, s in ws]
    mlp = mx.MLP()
    mlp.setup(*(w for w, _ in ws), scales=tuple(s for _, s in ws))
    y = mlp.run(x)
    full = [u.f64(w) * u.spread(u.f64(s), *w.shape) for w, s in ws]
    a = u.value_rows(*u.quantize_rows(u.f64(x)))
    h, _ = u.gated(a @ full[0].T, 0, a @ full[1].T, 0)
    want = u.value_rows(*u.quantize_rows(h)) @ full[2].T
    assert np.linalg.norm(u.f64(y) - want) <= (3.9e-3 + 2.0 ** -8) * np.linalg.norm(want)
    y32 = torch.empty((M, K), device="cuda")
    mlp.run(mx.quantize_fp8(x), y32)
    assert torch.equal(y32.to(torch.bfloat16), y)


@pytest.mark.parametrize("M,K,N", [(1, 256, 96), (16, 300, 352), (30, 640, 256), (200, 260, 160), (513, 384, 1056)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mlp_is_its_two_products_with_the_intermediate_quantised_from_32_bits(M, K, N, dtype):
    """Step by step through the public calls, bit for bit.  (Rounded to bf16 on the way, a value of the intermediate may come to lie on the border between two of e4m3: some in a
    hundred of them would go to the other one.)"""
    x = mx.quantize_fp8(normal((M, K), 1))
    ws = [weight(*shape, 5 + i) for i, shape in enumerate(((N, K), (N, K), (K, N)))]
    (g, gs), (v, vs), (d, ds) = [(w, s * 0.2) for w, s in ws]
    mlp = mx.MLP()
    mlp.setup(g, v, d, scales=(gs, vs, ds))
    y = mlp.run(x, torch.empty((M, K), dtype=dtype, device="cuda"))
    h = torch.empty((M, N), device="cuda")
    mx.gemm_fp8(x, *mx.pack_gate_up_fp8(g, v, (gs, vs)), 2 * N, mx.Epilogue(h, mx.PP_SILU_GATE))
    hq, want = mx.quantize_fp8(h), torch.empty_like(y)
    mx.gemm_fp8(hq, *mx.pack_fp8(d, ds), K, mx.Epilogue(want, mx.PP_NONE))
    assert torch.equal(y, want)
    value, bound = u.product(u.value_rows(bits(hq.q), u.f64(hq.scales)), u.f64(d) * u.spread(u.f64(ds), K, N), 8)
    u.close(y, value, bound, dtype)
    if M * N > 4000:
        assert not torch.equal(mx.quantize_fp8(h.to(torch.bfloat16)).q.view(torch.uint8), hq.q.view(torch.uint8))


def test_mlp_from_bf16_weights():
    M, K, N = 24, 256, 192
    x, w = normal((M, K), 1), [normal(s, 2 + i, 0.05) for i, s in enumerate(((N, K), (N, K), (K, N)))]
    mlp, bf = mx.MLP(), mx.MLP()
    mlp.setup(*w, compress="fp8")
    bf.setup(*w)
    # three quantisations to 4 significant bits (2^-4 at most, a third of that typically) against none
    d = (mlp.run(x).float() - bf.run(x).float()).norm() / bf.run(x).float().norm()
    assert d < 3 * 2.0 ** -4


def test_graph_and_streams():
    """Replays of a captured layer beside eager calls of it on another stream: the scratch of each is its own."""
    K, N = 512, 256
    mlp = mx.MLP()
    mlp.setup(normal((N, K), 1, 0.05), normal((N, K), 2, 0.05), normal((K, N), 3, 0.05), compress="fp8")
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
    w, s = weight(64, 128, 1)
    packed, scales = mx.pack_fp8(w, s)
    x = torch.empty((0, 128), dtype=torch.bfloat16, device="cuda")
    assert mx.quantize_fp8(x).shape == (0, 128)
    mx.gemm_fp8(x, packed, scales, 64, mx.Epilogue(torch.empty((0, 64), device="cuda"), mx.PP_NONE))
    mx.gemm_fp8(mx.quantize_fp8(x), packed, scales, 64, mx.Epilogue(torch.empty((0, 64), device="cuda"), mx.PP_NONE))


def test_packing_into_what_is_too_small_or_of_another_kind_is_refused():
    N, K = 96, 200
    (w, s), b = weight(N, K, 1), normal((N, K), 2)
    room = lambda n, rows: (torch.full((mx.packed_b_bytes(mx.F8, K, n) + 64,), 7, dtype=torch.uint8, device="cuda"), torch.zeros((rows, 2), device="cuda"))  # noqa: E731
    for pack, given, n, rows in ((lambda out: mx.pack_fp8(w, s, out=out), mx.pack_fp8(w, s), N, 1), (lambda out: mx.pack_fp8(b, out=out), mx.pack_fp8(b), N, 1),
                                 (lambda out: mx.pack_gate_up_fp8(w, w, (s, s), out=out), mx.pack_gate_up_fp8(w, w, (s, s)), 2 * N, 2),
                                 (lambda out: mx.pack_gate_up_fp8(b, b, out=out), mx.pack_gate_up_fp8(b, b), 2 * N, 2)):
        p, sc = room(n, rows)
        need = p.numel() - 64
        for bad in ((p[:need - 1], sc), (p[8:], sc), (p.view(torch.int8), sc), (p[:need].cpu(), sc), (p, sc[:, :1]), (p, sc.double()), (p, sc.t()[:, :1] if rows == 1 else sc.t()),
                    (p, torch.zeros((rows, 4), device="cuda")[:, ::2])):
            with pytest.raises(mx.MmxError):
                pack(bad)
        assert (p == 7).all()
        pack((p, sc))
        assert torch.equal(p[:need], given[0]) and (p[need:] == 7).all() and torch.equal(sc, given[1])


def test_refusals_on_the_gpu():
    w, s = weight(96, 256, 1)
    packed, scales = mx.pack_fp8(w, s)
    x = normal((4, 256), 1)
    y = torch.empty((4, 96), device="cuda")
    ok = lambda **k: mx.gemm_fp8(**{**dict(A=x, Bpacked=packed, b_scales=scales, N=96, ep=mx.Epilogue(y, mx.PP_NONE)), **k})  # noqa: E731
    ok()
    for bad in (dict(A=x.half()), dict(A=x[:, :128]), dict(A=x.t()), dict(A=w), dict(Bpacked=packed[:-1]), dict(Bpacked=packed.view(2, -1)),
                dict(b_scales=scales[:, :1]), dict(b_scales=scales.double()), dict(N=97), dict(N=0), dict(ep=mx.Epilogue(y[:, :95], mx.PP_NONE)),
                dict(ep=mx.Epilogue(y.half(), mx.PP_NONE)), dict(ep=mx.Epilogue(y, mx.PP_DEQUANT)), dict(ep=mx.Epilogue(y, mx.PP_QUANT)),
                dict(ep=mx.Epilogue(y, mx.PP_BIAS)), dict(ep=mx.Epilogue(y, mx.PP_BIAS, bias=torch.zeros(95, device="cuda"))),
                dict(ep=mx.Epilogue(y, mx.PP_SILU_GATE)), dict(ep=mx.Epilogue(y[:3], mx.PP_NONE)), dict(A=x.cpu())):
        with pytest.raises(mx.MmxError):
            ok(**bad)
    with pytest.raises(mx.MmxError):
        mx.quantize_fp8(x.half())
    with pytest.raises(mx.MmxError):
        mx.pack_fp8(w)  # e4m3 without scales
    with pytest.raises(mx.MmxError):
        mx.pack_fp8(w, s[:, :1])
    with pytest.raises(mx.MmxError):
        mx.pack_gate_up_fp8(w[:40], w[:40], (s, s))
    with pytest.raises(mx.MmxError):
        mx.Fp8Rows.of(w, s)
    with pytest.raises(mx.MmxError):
        mx.LinearFp8().forward(x, y)
