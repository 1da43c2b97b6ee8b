"""What the feed-forward block's entry points refuse, at the C ABI (before anything touches a device) and in the Python layer; and the 64-bit
definitions that the GPU tests use, against torch's own conversions."""
import ctypes as C

import numpy as np
import pytest
import torch

import ffn_util as u
import mm_amx_amd as mx
from mm_amx_amd import _lib as L

P = 1 << 20  # an address that is never read: every call below is refused on the host, or has nothing to do


@pytest.fixture(scope="module")
def lib():
    return L.lib()


def refused(rc, word):
    assert rc in (-1, -2), rc
    text = L.lib().mmx_last_error().decode()
    assert word in text, text


def test_quantisers(lib):
    rows = lambda **k: lib.mmx_quantize_rows_fp8(*{**dict(dt=1, x=P, ldx=512, M=4, K=256, q=P, ldq=256, s=P, lds=4, st=None), **k}.values())  # noqa: E731
    for bad, word in ((dict(dt=2), "dtype"), (dict(M=-1), "negative"), (dict(K=0), "positive"), (dict(x=None), "NULL"), (dict(x=P + 1), "aligned"), (dict(ldx=510), "apart"),
                      (dict(ldx=513), "aligned"), (dict(q=P + 8), "16-byte"), (dict(ldq=264), "16-byte"), (dict(ldq=240), "apart"), (dict(s=None), "NULL"),
                      (dict(s=P + 2), "aligned"), (dict(lds=3), "scales"), (dict(K=1 << 23), "up to"), (dict(dt=0), "apart"), (dict(M=1 << 22, lds=1 << 22), "up to")):
        refused(rows(**bad), word)
    assert rows(M=0, x=None, q=None) == 0
    pack = lambda **k: lib.mmx_quantize_pack_fp8(*{**dict(W=P, ldw=512, K=256, N=64, t=1, pair=0, packed=P, s=P, st=None), **k}.values())  # noqa: E731
    for bad, word in ((dict(W=None), "NULL"), (dict(ldw=510), "apart"), (dict(ldw=126, t=0), "apart"), (dict(pair=3), "pair"), (dict(pair=1, N=40), "32"),
                      (dict(packed=P + 8), "16-byte"), (dict(s=None), "NULL"), (dict(K=0), "positive")):
        refused(pack(**bad), word)
    both = lambda **k: lib.mmx_repack_gate_up_fp8(*{**dict(g=P, u=P, ldw=256, K=256, N=64, packed=P, st=None), **k}.values())  # noqa: E731
    for bad, word in ((dict(g=None), "NULL"), (dict(N=33), "32"), (dict(ldw=255), "row"), (dict(packed=P + 4), "16-byte")):
        refused(both(**bad), word)


def epilogue(steps=0, out=1, ld=128, C_=P, bias=None):
    return L._Epilogue(steps, out, C_, ld, bias, 1.0, None, 0.0, None)


def test_products(lib):
    def gemm(ep=None, **k):
        a = {**dict(dt=6, A=P, lda=256, s=P, lds=4, B=P, bs=P, M=4, K=256, N=64, ep=C.byref(ep or epilogue()), scratch=None, n=0, st=None), **k}
        return lib.mmx_gemm_fp8(*a.values())

    for bad, word in ((dict(dt=2), "dtype"), (dict(A=None), "NULL"), (dict(s=None), "NULL"), (dict(A=P + 8), "16-byte"), (dict(lda=128), "apart"), (dict(lda=1 << 24), "8 MiB"),
                      (dict(lds=3), "scales"), (dict(B=None), "NULL"), (dict(B=P + 8), "16-byte"), (dict(bs=None), "NULL"), (dict(K=0), "positive"), (dict(M=-1), "negative"),
                      (dict(dt=1, lda=512), "e4m3 activations only"), (dict(dt=0, s=None, lda=1024), "scratch"), (dict(dt=0, s=None, lda=1024, scratch=P + 16, n=1 << 20), "256-byte"),
                      (dict(dt=1, M=40, lds=40, s=None, lda=512), "scratch"),
                      (dict(ep=epilogue(out=2)), "dtype"), (dict(ep=epilogue(steps=1)), "DEQUANT"), (dict(ep=epilogue(steps=8)), "QUANT"), (dict(ep=epilogue(steps=2)), "bias"),
                      (dict(ep=epilogue(C_=None)), "NULL"), (dict(ep=epilogue(ld=126)), "row"), (dict(N=32, ep=epilogue(steps=16)), "64"),
                      (dict(ep=epilogue(steps=18, bias=P)), "SILU_GATE"), (dict(ep=epilogue(steps=64)), "unknown")):
        ep = bad.pop("ep", None)
        refused(gemm(ep, **bad), word)
    assert gemm(M=0, A=None) == 0
    assert lib.mmx_gemm_fp8_scratch_bytes(6, 4, 256, 64) == 0 and lib.mmx_gemm_fp8_scratch_bytes(1, 0, 256, 64) == 0
    assert lib.mmx_gemm_fp8_scratch_bytes(0, 4, 200, 64) >= 4 * 256 + 2 * 4 * 4
    assert lib.mmx_gemm_fp8_scratch_bytes(1, 400, 200, 64) >= 400 * 256 + 2 * 400 * 4

    need = lib.mmx_mlp_fp8_scratch_bytes(6, 4, 256, 64)
    mlp = lambda **k: lib.mmx_mlp_fp8(*{**dict(dt=6, x=P, ldx=256, s=P, lds=4, gu=P, gs=P, d=P, ds=P, yt=1, y=P, ldy=512, M=4, K=256, N=64, scratch=P, n=need, st=None), **k}.values())  # noqa: E731
    for bad, word in ((dict(N=40), "32"), (dict(gu=None), "NULL"), (dict(ds=None), "NULL"), (dict(yt=2), "dtype"), (dict(y=None), "NULL"), (dict(ldy=510), "row"), (dict(n=need - 1), "scratch"),
                      (dict(scratch=P + 128), "256-byte"), (dict(x=P + 1), "16-byte"), (dict(dt=0), "only")):
        refused(mlp(**bad), word)
    assert mlp(M=0) == 0


def test_experts(lib):
    route = lambda **k: lib.mmx_moe_route(*{**dict(x=P, ldx=256, r=P, ldr=256, T=4, H=128, E=8, k=2, flags=0, scale=1.0, bias=None, l=P, ids=P, w=P, st=None), **k}.values())  # noqa: E731
    for bad, word in ((dict(x=None), "NULL"), (dict(ldx=254), "apart"), (dict(r=None), "NULL"), (dict(E=0), "top_k"), (dict(E=1025), "1024"), (dict(k=0), "top_k"), (dict(k=9), "top_k"),
                      (dict(k=17, E=64), "top_k"), (dict(flags=4), "flags"), (dict(l=P + 4), "aligned"), (dict(ids=None), "NULL"), (dict(w=P + 1), "aligned"), (dict(bias=P + 2), "aligned"),
                      (dict(H=0), "positive"), (dict(T=-1), "negative")):
        refused(route(**bad), word)
    assert route(T=0) == 0
    need = lib.mmx_moe_experts_scratch_bytes(4, 128, 64, 2)
    assert need >= 4 * 2 * 2 * 64 * 2 and lib.mmx_moe_experts_scratch_bytes(0, 128, 64, 2) == 0
    ex = lambda **k: lib.mmx_moe_experts(*{**dict(dt=1, x=P, ldx=256, ids=P, w=P, T=4, H=128, I=64, E=8, k=2, gu=P, gs=None, d=P, ds=None, yt=1, y=P, ldy=256, scratch=P, n=need, st=None), **k}.values())  # noqa: E731
    for bad, word in ((dict(dt=2), "dtype"), (dict(I=40), "32"), (dict(I=0), "positive"), (dict(E=0), "experts"), (dict(k=17), "top_k"), (dict(yt=2), "dtype"), (dict(x=None), "NULL"),
                      (dict(ldy=254), "apart"), (dict(ids=None), "NULL"), (dict(n=need - 1), "scratch"), (dict(scratch=P + 128), "256-byte"), (dict(gu=P + 8), "16 bytes"), (dict(dt=6), "scales"), (dict(gs=P, ds=P), "scales"),
                      (dict(dt=6, gs=P, ds=P + 2), "aligned")):
        refused(ex(**bad), word)
    assert ex(T=0) == 0


def test_experts_that_one_launch_cannot_take(lib):
    """512 places of 2^14 workgroups of 512 threads are 2^32 of them."""
    T, H, I, E, k = 32, 1, 1 << 18, 512, 16
    refused(lib.mmx_moe_experts(1, P, 2, P, P, T, H, I, E, k, P, None, P, None, 1, P, 2, P, 1 << 62, None), "too many")


def test_block_norm(lib):
    base = dict(f=P, ldf=256, res=P, ldres=256, pw=None, gate=None, ldg=0, nw=None, r=P, ldr=256, z=P, ldz=256, zs=None, ldzs=0, rt=1, zt=1, post=0, pre=1, scale=1.0, eps=1e-6, off=0.0)

    def norm(M=4, H=128, **k):
        return lib.mmx_block_norm(C.byref(L._BlockNorm(*{**base, **k}.values())), M, H, None)

    for bad, word in ((dict(f=None), "NULL"), (dict(f=P + 1), "aligned"), (dict(ldf=254), "apart"), (dict(ldres=255), "aligned"), (dict(ldres=254), "apart"), (dict(rt=2), "residual"),
                      (dict(rt=0), "apart"), (dict(zt=0), "z of"), (dict(r=None, z=None), "neither"), (dict(pw=P), "off"), (dict(pre=0, nw=P), "off"), (dict(gate=P, ldg=128), "apart"),
                      (dict(gate=P + 1), "aligned"), (dict(nw=P + 1), "aligned"), (dict(ldz=254), "apart"), (dict(zt=6), "scales"), (dict(zt=6, zs=P, ldzs=3), "scales"),
                      (dict(zt=6, zs=P, ldzs=4, z=P + 8), "16-byte"), (dict(zt=6, zs=P, ldzs=4, ldz=112), "apart"), (dict(H=32769), "32768"), (dict(H=0), "positive"), (dict(M=-1), "negative")):
        refused(norm(**bad), word)
    assert lib.mmx_block_norm(None, 1, 1, None) == -1
    assert norm(M=0, f=None) == 0


def test_python_refuses_what_is_not_on_the_gpu():
    x, w = torch.zeros((4, 128), dtype=torch.bfloat16), torch.zeros((64, 128), dtype=torch.bfloat16)
    for call in (lambda: mx.quantize_fp8(x), lambda: mx.quantize_pack_fp8(w), lambda: mx.pack_fp8(w), lambda: mx.pack_gate_up_fp8(w, w), lambda: mx.moe_route(x, w, 2),
                 lambda: mx.block_norm(x), lambda: mx.LinearFp8().set_weight(w), lambda: mx.MLP().setup(w, w, w.t(), compress="fp8")):
        with pytest.raises(mx.MmxError, match="on the GPU|unit stride"):
            call()
    with pytest.raises(mx.MmxError):
        mx.MoE(2, scoring="other")
    with pytest.raises(mx.MmxError):
        mx.MLP().setup(w, w, w.t(), compress="int8")


def test_the_experts_setup_refuses_what_run_could_not_take():
    E, H, I = 4, 64, 32
    w = [torch.zeros(s, dtype=torch.bfloat16) for s in ((E, I, H), (E, I, H), (E, H, I))]
    router = torch.zeros((E, H), dtype=torch.bfloat16)
    for r, word in ((router.float(), "router must be"), ([[0.0] * H] * E, "router")):
        with pytest.raises(mx.MmxError, match=word):
            mx.MoE(2).setup(r, *w)


def test_the_experts_refuse_quantised_rows():
    moe = mx.MoE(2)
    moe.H, moe.gate_up = 128, torch.zeros(1, dtype=torch.uint8)
    with pytest.raises(mx.MmxError, match="quantised rows"):
        moe.run(mx.Fp8Rows.of(torch.zeros((3, 128), dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones((1, 3))))


def test_the_other_operators_refuse_e4m3(lib):
    for a in (torch.bfloat16, torch.int8, torch.uint8, torch.float8_e4m3fn):
        A, B = torch.zeros((64, 128), dtype=a), torch.zeros((128, 64)).to(torch.float8_e4m3fn)
        for const in (False, True):
            with pytest.raises(mx.MmxError, match="e4m3"):
                mx.Matmul(constB=const)(A, B, ppkernel=mx.BiasGeluStore(torch.zeros((64, 64))))
    ep = L._Epilogue(0, 1, P, 1024, None, 1.0, None, 0.0, None)
    for a, b in ((6, 6), (1, 6), (6, 1), (2, 6), (6, 2)):
        refused(lib.mmx_gemm(a, b, P, 1024, P, 64, 128, 64, 0, 64, C.byref(ep), None), "dtype")
    refused(lib.mmx_matvec(6, P, 1024, P, P, 64, 128, None), "dtype")
    ep.out_dtype = 6
    refused(lib.mmx_gemm(1, 1, P, 1024, P, 64, 128, 64, 0, 64, C.byref(ep), None), "dtype")


def test_rows_from_elsewhere_are_padded():
    q = torch.arange(-60, 60, dtype=torch.float32).view(3, 40).to(torch.float8_e4m3fn)
    s = torch.ones((1, 3))
    rows = mx.Fp8Rows.of(q, s)
    assert rows.padded.shape == (3, 128) and rows.shape == (3, 40)
    assert torch.equal(rows.q.view(torch.uint8), q.view(torch.uint8)) and not rows.padded.view(torch.uint8)[:, 40:].any()
    got_q, got_s = rows
    assert torch.equal(got_q.view(torch.uint8), q.view(torch.uint8)) and torch.equal(got_s, s)
    whole = torch.zeros((2, 256), dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert mx.Fp8Rows.of(whole, torch.ones((2, 2))).padded.data_ptr() == whole.data_ptr()
    turned = torch.zeros((256, 5), dtype=torch.uint8).view(torch.float8_e4m3fn).t()
    assert mx.Fp8Rows.of(turned, torch.ones((2, 5))).padded.stride() == (256, 1)
    for bad in ((q, torch.ones((3, 1))), (q, s.double()), (q.float(), s), (q[0], s)):
        with pytest.raises(mx.MmxError):
            mx.Fp8Rows.of(*bad)


def test_the_definitions_against_torch():
    codes = torch.arange(256, dtype=torch.uint8)
    v = codes.view(torch.float8_e4m3fn).float().double().numpy()
    assert np.array_equal(u.decode(np.arange(256)), v, equal_nan=True)
    x = torch.cat([torch.randn(20000, generator=torch.Generator().manual_seed(1)) * 100, torch.linspace(-20, 20, 4001) / 16, torch.tensor([0.0, 448.0, -448.0, 17.0, 19.0])]).clamp(-448, 448)
    assert np.array_equal(u.encode(x.double().numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert list(u.scale_of(np.array([0.0, 448.0, 449.0, 1.75, np.inf]))) [:4] == [2.0 ** -126, 1.0, 2.0, 2.0 ** -8]


def test_packed_weights_on_disk(tmp_path):
    from mm_amx_amd import packed_io
    K, N = 300, 160
    packed = torch.arange(L.packed_b_bytes(L.F8, K, N), dtype=torch.int64).to(torch.uint8)
    scales = torch.rand((2, 3))
    path = str(tmp_path / "w.safetensors")
    packed_io.save_packed(path, packed, "fp8", K, N, scales=scales)
    w = packed_io.load_packed(path, device="cpu")
    assert torch.equal(w["packed"], packed) and torch.equal(w["scales"], scales) and (w["dtype"], w["K"], w["N"]) == ("fp8", K, N)
    pair = torch.zeros(L.packed_b_bytes(L.F8, K, 320), dtype=torch.uint8)
    packed_io.save_packed(path, pair, "fp8", K, 320, scales=torch.rand((4, 3)), layout="gate_up")
    for bad in (dict(scales=None), dict(scales=scales[:1]), dict(scales=torch.rand(160)), dict(packed=packed[:-1])):
        with pytest.raises(mx.MmxError):
            packed_io.save_packed(path, **{**dict(packed=packed, dtype="fp8", K=K, N=N, scales=scales), **bad})
