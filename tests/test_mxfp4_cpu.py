"""What the entry points of microscaled 4-bit floating point refuse, at the C ABI (before anything touches a device) and in the Python layer; and the 64-bit
definitions that the GPU tests use."""
import ctypes as C

import numpy as np
import pytest
import torch

import mm_amx_amd as mx
import mxfp4_util as m4
from mm_amx_amd import _lib as L

P = 1 << 20  # an address that is never read: every call below is refused on the host, or has nothing to do


@pytest.fixture(scope="module")
def lib():
    return L.lib()


def refused(rc, word):
    assert rc in (-1, -2), rc
    text = L.lib().mmx_last_error().decode()
    assert word in text, text


def test_sizes(lib):
    from mm_amx_amd import mxfp4
    for rows, K in ((1, 1), (32, 256), (33, 257), (11008, 4096), (1 << 26, 1 << 22)):
        assert lib.mmx_mxfp4_bytes(rows, K) == mxfp4.packed_bytes(rows, K) == -(-rows // 32) * -(-K // 256) * 4352
    assert lib.mmx_mxfp4_bytes(0, 5) == lib.mmx_mxfp4_bytes(5, 0) == lib.mmx_mxfp4_bytes(-1, 5) == 0


def test_quantisers(lib):
    rows = lambda **k: lib.mmx_quantize_mxfp4(*{**dict(dt=1, x=P, ldx=512, M=4, K=256, pair=0, packed=P, st=None), **k}.values())  # noqa: E731
    for bad, word in ((dict(dt=2), "dtype"), (dict(dt=7), "dtype"), (dict(M=-1), "negative"), (dict(K=0), "positive"), (dict(x=None), "NULL"), (dict(x=P + 1), "aligned"), (dict(ldx=510), "apart"),
                      (dict(ldx=513), "aligned"), (dict(packed=P + 8), "16-byte"), (dict(packed=None), "NULL"), (dict(K=1 << 23), "up to"), (dict(dt=0), "apart"), (dict(pair=3), "pair"),
                      (dict(pair=-1), "pair"), (dict(pair=1), "32"), (dict(pair=2, M=40), "32"), (dict(M=(1 << 26) + 1), "up to")):
        refused(rows(**bad), word)
    assert rows(M=0, x=None, packed=None) == 0
    base = dict(q=P, ldq=128, s=P, lds=8, M=4, K=256, pair=0, packed=P, st=None)
    to = lambda **k: lib.mmx_repack_mxfp4(*{**base, **k}.values())  # noqa: E731
    back = lambda **k: lib.mmx_unpack_mxfp4(*[{**base, **k}[n] for n in ("packed", "M", "K", "q", "ldq", "s", "lds", "st")])  # noqa: E731
    for call in (to, back):
        for bad, word in ((dict(q=None), "NULL"), (dict(s=None), "NULL"), (dict(packed=None), "NULL"), (dict(packed=P + 4), "16-byte"), (dict(ldq=127), "apart"), (dict(lds=7), "apart"),
                          (dict(K=257), "apart"), (dict(M=-1), "negative"), (dict(K=0), "positive")):
            refused(call(**bad), word)
        assert call(M=0) == 0
    refused(to(pair=1), "32")
    de = lambda **k: lib.mmx_dequantize_mxfp4(*{**dict(packed=P, M=4, K=256, dt=1, y=P, ldy=512, st=None), **k}.values())  # noqa: E731
    for bad, word in ((dict(packed=None), "NULL"), (dict(dt=6), "dtype"), (dict(y=None), "NULL"), (dict(ldy=510), "apart"), (dict(dt=0), "apart"), (dict(packed=P + 2), "16-byte")):
        refused(de(**bad), word)
    assert de(M=0) == 0


def epilogue(steps=0, out=1, ld=128, C_=P, bias=None):
    return L._Epilogue(steps, out, C_, ld, bias, 1.0, None, 0.0, None)


def test_products(lib):
    def gemm(ep=None, **k):
        return lib.mmx_gemm_mxfp4(*{**dict(dt=7, A=P, lda=0, B=P, M=4, K=256, N=64, ep=C.byref(ep or epilogue()), scratch=None, n=0, st=None), **k}.values())

    for bad, word in ((dict(dt=2), "dtype"), (dict(dt=6), "dtype"), (dict(A=None), "NULL"), (dict(A=P + 8), "16-byte"), (dict(B=None), "NULL"), (dict(B=P + 8), "16-byte"), (dict(K=0), "positive"),
                      (dict(M=-1), "negative"), (dict(M=1 << 22), "up to"), (dict(dt=1, lda=510), "apart"), (dict(dt=0, lda=1024), "scratch"), (dict(dt=0, lda=1024, scratch=P + 16, n=1 << 20), "256-byte"),
                      (dict(dt=1, M=40, lda=512), "scratch"), (dict(ep=epilogue(out=2)), "dtype"), (dict(ep=epilogue(steps=1)), "DEQUANT"), (dict(ep=epilogue(steps=8)), "QUANT"),
                      (dict(ep=epilogue(steps=2)), "bias"), (dict(ep=epilogue(C_=None)), "NULL"), (dict(ep=epilogue(ld=126)), "row"), (dict(N=32, ep=epilogue(steps=16)), "64"),
                      (dict(ep=epilogue(steps=18, bias=P)), "SILU_GATE"), (dict(ep=epilogue(steps=64)), "unknown")):
        ep = bad.pop("ep", None)
        refused(gemm(ep, **bad), word)
    assert gemm(M=0, A=None) == 0
    assert lib.mmx_gemm_mxfp4_scratch_bytes(7, 4, 256, 64) == 0 and lib.mmx_gemm_mxfp4_scratch_bytes(1, 0, 256, 64) == 0
    assert lib.mmx_gemm_mxfp4_scratch_bytes(0, 4, 200, 64) >= 4352 and lib.mmx_gemm_mxfp4_scratch_bytes(1, 400, 200, 64) >= 13 * 4352

    need = lib.mmx_mlp_mxfp4_scratch_bytes(7, 4, 256, 64)
    mlp = lambda **k: lib.mmx_mlp_mxfp4(*{**dict(dt=7, x=P, ldx=0, gu=P, d=P, yt=1, y=P, ldy=512, M=4, K=256, N=64, scratch=P, n=need, st=None), **k}.values())  # noqa: E731
    for bad, word in ((dict(N=40), "32"), (dict(gu=None), "NULL"), (dict(d=P + 8), "16-byte"), (dict(yt=2), "dtype"), (dict(y=None), "NULL"), (dict(ldy=510), "row"), (dict(n=need - 1), "scratch"),
                      (dict(scratch=P + 128), "256-byte"), (dict(x=P + 1), "16-byte"), (dict(dt=6), "dtype"), (dict(N=1 << 23), "at most")):
        refused(mlp(**bad), word)
    assert mlp(M=0) == 0


def test_block_norm_into_packed_rows(lib):
    base = dict(f=P, ldf=256, res=None, ldres=0, pw=None, gate=None, ldg=0, nw=None, r=None, ldr=0, z=P, ldz=0, zs=None, ldzs=0, rt=1, zt=7, post=0, pre=1, scale=1.0, eps=1e-6, off=0.0)
    norm = lambda **k: lib.mmx_block_norm(C.byref(L._BlockNorm(*{**base, **k}.values())), 4, 128, None)  # noqa: E731
    refused(norm(z=P + 8), "16-byte")
    refused(norm(zt=5), "z of")
    refused(norm(f=None), "NULL")


def test_the_other_operators_refuse_packed_rows(lib):
    ep = L._Epilogue(0, 1, P, 1024, None, 1.0, None, 0.0, None)
    for a, b in ((7, 7), (1, 7), (7, 1)):
        refused(lib.mmx_gemm(a, b, P, 1024, P, 64, 128, 64, 0, 64, C.byref(ep), None), "dtype")
    rows = mx.Mxfp4Rows(torch.zeros(4352, dtype=torch.uint8), 3, 128)
    moe = mx.MoE(2)
    moe.H, moe.gate_up = 128, torch.zeros(1, dtype=torch.uint8)
    lin = mx.LinearFp8()
    lin._packed, lin.m_K, lin.m_N = torch.zeros(1, dtype=torch.uint8), 128, 32
    for call in (lambda: moe.run(rows), lambda: mx.quantize_fp8(rows), lambda: mx.quantize_mxfp4(rows), lambda: mx.block_norm(rows)):
        with pytest.raises(mx.MmxError):
            call()


def test_python_refuses_what_is_not_on_the_gpu():
    x, w = torch.zeros((4, 128), dtype=torch.bfloat16), torch.zeros((64, 128), dtype=torch.bfloat16)
    q, s = torch.zeros((64, 64), dtype=torch.uint8), torch.zeros((64, 4), dtype=torch.uint8)
    for call in (lambda: mx.quantize_mxfp4(x), lambda: mx.pack_mxfp4(w), lambda: mx.pack_mxfp4(q, s), lambda: mx.pack_gate_up_mxfp4(w, w), lambda: mx.Mxfp4Rows.of(q, s),
                 lambda: mx.block_norm(x, quantize="mxfp4"), lambda: mx.LinearMxfp4().set_weight(w), lambda: mx.MLP().setup(w, w, w.t(), compress="mxfp4"),
                 lambda: mx.MLP().setup(q, q, torch.zeros((128, 32), dtype=torch.uint8), scales=(s, s, torch.zeros((128, 2), dtype=torch.uint8))),
                 lambda: mx.dequantize_mxfp4(mx.Mxfp4Rows(torch.zeros(4352, dtype=torch.uint8), 3, 128))):
        with pytest.raises(mx.MmxError, match="on the GPU|unit stride"):
            call()
    with pytest.raises(mx.MmxError):
        mx.LinearMxfp4().forward(x, x)
    with pytest.raises(mx.MmxError):
        mx.dequantize_mxfp4(x)


def test_the_definitions():
    assert list(m4.encode(np.array([0.0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 6.9, -0.75, -6.0]))) == [0, 0, 1, 2, 2, 4, 4, 6, 6, 7, 7, 10, 15]
    assert list(m4.scale_of(np.array([0.0, 6.0, 6.99, 7.0, 13.9, 14.0, 1.75, np.inf, 2.0 ** -140, 3.0e38]))) == [1, 127, 127, 128, 128, 129, 126, 255, 1, 253]
    codes = np.arange(12, dtype=np.uint8).reshape(2, 6)
    assert np.array_equal(m4.single(m4.pairs(codes), 6), codes) and np.array_equal(m4.single(m4.pairs(codes[:, :5]), 5), codes[:, :5])


def test_any_true_value_of_quantize_means_e4m3(monkeypatch):
    """Only "mxfp4" asks for packed rows: the native call's own code for them comes from no caller."""
    seen = []

    class Native:
        @staticmethod
        def block_norm(*a):
            seen.append(a[10])  # (returns None: not taken, nothing done)

    monkeypatch.setattr(L, "_native", Native)
    monkeypatch.setattr(L, "_initialised", {0})
    monkeypatch.setattr(L, "_current_device", lambda: 0)
    monkeypatch.setattr(L, "_raw_stream", lambda device: 0)
    x = torch.zeros((4, 128), dtype=torch.bfloat16)
    for quantize, code in ((False, False), (0, False), (None, False), (True, True), ("fp8", True), (1, True), (2, True), (np.bool_(True), True), ("mxfp4", 2)):
        with pytest.raises(mx.MmxError, match="on the GPU"):
            mx.block_norm(x, quantize=quantize)
        assert seen[-1] == code and type(seen[-1]) is type(code), quantize


@pytest.mark.parametrize("compress", [None, "fp8", "mxfp4"])
def test_a_refused_setup_leaves_the_mlp_as_it_was(compress):
    mlp = mx.MLP()
    mlp.gate_up, mlp.down, mlp.m_N, mlp.m_K, mlp.mx4 = held = ("gate_up", "down", 96, 256, True)
    w = torch.zeros((64, 128), dtype=torch.bfloat16)
    with pytest.raises(mx.MmxError, match="on the GPU"):
        mlp.setup(w, w, torch.zeros((128, 64), dtype=torch.bfloat16), compress=compress)
    assert (mlp.gate_up, mlp.down, mlp.m_N, mlp.m_K, mlp.mx4) == held


def test_a_setup_lets_the_old_intermediate_go(monkeypatch):
    """run makes one of the new width: the old one, kept, was refused as too narrow."""
    mlp = mx.MLP()
    mlp.actUp = torch.zeros((4, 32))
    monkeypatch.setattr(L, "repack_gate_up", lambda gate, up: "gate_up")
    monkeypatch.setattr(L, "repack_b", lambda w, transpose: "down")
    w = torch.zeros((64, 128), dtype=torch.bfloat16)
    mlp.setup(w, w, torch.zeros((128, 64), dtype=torch.bfloat16))
    assert mlp.actUp is None and (mlp.gate_up, mlp.down, mlp.m_N, mlp.m_K, mlp.mx4) == ("gate_up", "down", 64, 128, False)
