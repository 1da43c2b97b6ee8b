"""Microscaled 4-bit floating point: e2m1 values with a scale, a power of two in 8 bits, for each row and 32 of k.  Rows of activations and
weights are quantised, or packed from what a checkpoint holds, multiplied, and read back.  As in ffn, arguments are checked here and every call
ends in the C ABI (include/mm_amx_amd.h says what each computes and how packed rows are laid out); nothing is computed by PyTorch.

A call's scratch is torch memory of its own, on the current stream.
"""
import ctypes as C

import torch

from . import _lib as L
from ._lib import MmxError
from .ffn import _gpu, _ptr, _result, _rows, _scratch

BLOCK = 32
CHUNK, CHUNK_BYTES = 256, 4352
_BYTES = tuple(t for t in (torch.uint8, getattr(torch, "float4_e2m1fn_x2", None)) if t is not None)
_SCALES = tuple(t for t in (torch.uint8, getattr(torch, "float8_e8m0fnu", None)) if t is not None)


def packed_bytes(rows, K):
    return -(-rows // 32) * -(-K // CHUNK) * CHUNK_BYTES


class Mxfp4Rows:
    """Quantised rows [M, K]: ``q`` uint8 [M, ceil(K / 2)], two values a byte with that of the lower k in the low half, and ``scales`` uint8
    [M, ceil(K / 32)], the value being e2m1 * 2^(scale - 127) (255: NaN).  Unpacks as ``q, scales = rows``; both are made on demand from ``packed``,
    which is what the products read."""

    def __init__(self, packed, M, K):
        self.packed, self.M, self.K = packed, M, K

    @classmethod
    def empty(cls, M, K, device):
        return cls(torch.empty(packed_bytes(M, K), dtype=torch.uint8, device=device), M, K)

    @classmethod
    def of(cls, q, scales, K=None):
        """From codes [M, ceil(K / 2)] and scales [M, ceil(K / 32)] made elsewhere, uint8 or torch's types of their size.  K: default 2 * q.shape[1]."""
        M, K = _codes(q, scales, "q", K)
        rows = cls.empty(M, K, q.device)
        if M:
            _repack(q, scales, M, K, 0, rows.packed)
        return rows

    @property
    def shape(self):
        return torch.Size((self.M, self.K))

    @property
    def device(self):
        return self.packed.device

    def __iter__(self):
        p = self._args("rows")
        q = torch.empty((self.M, (self.K + 1) // 2), dtype=torch.uint8, device=self.device)
        scales = torch.empty((self.M, -(-self.K // BLOCK)), dtype=torch.uint8, device=self.device)
        if self.M:
            L._check(L.lib().mmx_unpack_mxfp4(p, self.M, self.K, q.data_ptr(), q.shape[1], scales.data_ptr(), scales.shape[1], L._stream()))
        return iter((q, scales))

    @property
    def q(self):
        return tuple(self)[0]

    @property
    def scales(self):
        return tuple(self)[1]

    def _args(self, what):
        """Pointer, checked."""
        if not all(isinstance(n, int) for n in (self.M, self.K)) or self.M < 0 or self.K < 1:
            raise MmxError(f"{what}: [{self.M}, {self.K}] is no shape of quantised rows")
        return _packed(self.packed, what, self.M, self.K)


def _packed(p, what, rows, K):
    _gpu(p, what, (torch.uint8,), 1)
    need = packed_bytes(rows, K)
    if p.numel() < need or p.data_ptr() % 16:
        raise MmxError(f"{what} holds {p.numel()} bytes, packed [{rows}, {K}] takes {need}, 16-byte aligned")
    return p.data_ptr()


def _codes(q, scales, what, K=None):
    """(M, K) of codes and scales that belong together."""
    _gpu(q, what, _BYTES, 2), _gpu(scales, f"{what}'s scales", _SCALES, 2)
    K = 2 * q.shape[1] if K is None else K
    if not isinstance(K, int) or K < 1 or (K + 1) // 2 != q.shape[1]:
        raise MmxError(f"{what} [{q.shape[0]}, {q.shape[1]}] holds {2 * q.shape[1]} values a row, K = {K}")
    if tuple(scales.shape) != (q.shape[0], -(-K // BLOCK)):
        raise MmxError(f"{what}'s scales must be [{q.shape[0]}, {-(-K // BLOCK)}] (a row and a block of 32 each)")
    return q.shape[0], K


def _repack(q, scales, M, K, pair, packed):
    L._check(L.lib().mmx_repack_mxfp4(q.data_ptr(), _rows(q), scales.data_ptr(), _rows(scales), M, K, pair, packed.data_ptr(), L._stream()))


def quantize_mxfp4(x):
    """x [M, K] bf16 or fp32 -> Mxfp4Rows: a scale for each row and 32 of k, the least power of two with which the block's largest magnitude is
    less than 7, so that it rounds to 6 at most; ties to even."""
    if L._native is not None and L._initialised and len(getattr(x, "shape", ())) == 2:  # (regular calls; None: not one, nothing was done)
        made = L._made(L._native.quantize_mxfp4, x)
        if made is not None:
            return Mxfp4Rows(made, *x.shape)
    _gpu(x, "x", (torch.bfloat16, torch.float32), 2)
    M, K = x.shape
    if K == 0:
        raise MmxError("x has no columns")
    out = Mxfp4Rows.empty(M, K, x.device)
    if M:
        L._check(L.lib().mmx_quantize_mxfp4(L.dtype_code(x), x.data_ptr(), _rows(x), M, K, 0, out.packed.data_ptr(), L._stream()))
    return out


def dequantize_mxfp4(rows, dtype=torch.bfloat16):
    """Mxfp4Rows -> their values [M, K] in bf16 or fp32."""
    if not isinstance(rows, Mxfp4Rows):
        raise MmxError("rows must be Mxfp4Rows")
    if dtype not in (torch.bfloat16, torch.float32):
        raise MmxError("values come in torch.bfloat16 or torch.float32")
    if L._native is not None and L._initialised:
        made = L._made(L._native.dequantize_mxfp4, rows.packed, rows.M, rows.K, dtype == torch.float32)
        if made is not None:
            return made
    p = rows._args("rows")
    y = torch.empty((rows.M, rows.K), dtype=dtype, device=rows.device)
    if rows.M:
        L._check(L.lib().mmx_dequantize_mxfp4(p, rows.M, rows.K, L.dtype_code(y), y.data_ptr(), _rows(y), L._stream()))
    return y


def _weights(w, scales, what):
    """(N, K) of weights in torch's layout: bf16, or codes with scales."""
    if scales is None:
        N, K = _gpu(w, f"{what} without scales", (torch.bfloat16,), 2).shape
    else:
        N, K = _codes(w, scales, what)
    if N == 0 or K == 0:
        raise MmxError(f"{what} [{N}, {K}] is empty")
    return N, K


def _pack_into(w, scales, N, K, pair, packed):
    if scales is None:
        L._check(L.lib().mmx_quantize_mxfp4(L.BF16, w.data_ptr(), _rows(w), N, K, pair, packed.data_ptr(), L._stream()))
    else:
        _repack(w, scales, N, K, pair, packed)


def _memory(out, rows, K, device):
    if out is None:
        return (torch.zeros if rows % 32 else torch.empty)(packed_bytes(rows, K), dtype=torch.uint8, device=device)
    _packed(out, "out", rows, K)
    return out


def pack_mxfp4(w, scales=None, out=None):
    """Weights [N, K] in torch's layout, bf16 (quantised here) or codes uint8 [N, K / 2] with the scales [N, ceil(K / 32)] they came with -> packed
    weights (uint8); out: where to put them."""
    N, K = _weights(w, scales, "weights")
    packed = _memory(out, N, K, w.device)
    _pack_into(w, scales, N, K, 0, packed)
    return packed


def pack_gate_up_mxfp4(w_gate, w_up, scales=None, out=None):
    """Gate and up weights [N, K] as in pack_mxfp4 (scales: a pair) -> packed [2 N, K]."""
    given = (None, None) if scales is None else tuple(scales)
    if len(given) != 2:
        raise MmxError("scales must be a pair, gate's and up's")
    N, K = _weights(w_gate, given[0], "w_gate")
    if _weights(w_up, given[1], "w_up") != (N, K):
        raise MmxError("w_gate and w_up must have the same shape")
    if N % 32:
        raise MmxError(f"gate and up projections of {N} columns: a positive multiple of 32 is needed")
    packed = _memory(out, 2 * N, K, w_gate.device)
    for pair, w, s in ((1, w_gate, given[0]), (2, w_up, given[1])):
        _pack_into(w, s, N, K, pair, packed)
    return packed


def _activations(x, what):
    """(dtype code, M, K, pointer, row stride) of bf16 or fp32 rows or of Mxfp4Rows."""
    if isinstance(x, Mxfp4Rows):
        return L.F4, x.M, x.K, x._args(what), 0
    _gpu(x, what, (torch.bfloat16, torch.float32), 2)
    return L.dtype_code(x), x.shape[0], x.shape[1], x.data_ptr(), _rows(x)


def _native_activations(x):
    return (x.packed, x.M, x.K) if type(x) is Mxfp4Rows else (x, None, None)


def gemm_mxfp4(A, Bpacked, N, ep):
    """C = PP(A . B) in microscaled 4-bit floating point: A [M, K] is Mxfp4Rows, or bf16 / fp32 and quantised on the way; Bpacked from pack_mxfp4 or,
    with PP_SILU_GATE, pack_gate_up_mxfp4 (N then counts both halves).  ep: PP_BIAS, PP_GELU or both, or PP_SILU_GATE alone, into bf16 or fp32."""
    if not isinstance(ep, L.Epilogue):
        raise MmxError("ep must be an Epilogue")
    if L._native is not None and L._initialised:
        rc = L._made(L._native.gemm_mxfp4, *_native_activations(A), Bpacked, N, at_end=(ep.C, ep.steps, ep.bias, ep.deq, ep.deq_oc, ep.q, ep.q_oc))
        if rc is not None:
            return
    if not isinstance(N, int) or N <= 0:
        raise MmxError(f"N = {N} must be a positive int")
    dt, M, K, a, lda = _activations(A, "A")
    if K == 0:
        raise MmxError("A has no columns")
    pair = bool(ep.steps & L.PP_SILU_GATE)
    if pair and N % 64:
        raise MmxError("a gate/up pair has a multiple of 64 packed columns")
    b = _packed(Bpacked, "Bpacked", N, K)
    _result(ep.C, "C", M, N // 2 if pair else N)
    if ep.bias is not None and _gpu(ep.bias, "bias", (torch.float32,), 1).numel() != N:
        raise MmxError(f"bias holds {ep.bias.numel()} values, N = {N}")
    if M == 0:
        return
    d = ep.struct()
    need = L.lib().mmx_gemm_mxfp4_scratch_bytes(dt, M, K, N)
    scratch = _scratch(need, A.device)
    L._check(L.lib().mmx_gemm_mxfp4(dt, a, lda, b, M, K, N, C.byref(d), _ptr(scratch), need, L._stream()))


def mlp_mxfp4(x, gate_up, down, N, y=None):
    """y = (silu(x . gate) * (x . up)) . down: x [M, K] as in gemm_mxfp4; gate_up from pack_gate_up_mxfp4, down from pack_mxfp4 of the [K, N]
    down_proj weight.  y [M, K] bf16 or fp32 (default: a new bf16 tensor)."""
    if L._native is not None and L._initialised:
        made = L._made(L._native.mlp_mxfp4, *_native_activations(x), gate_up, down, N, y)
        if made is not None:
            return made
    if not isinstance(N, int) or N <= 0 or N % 32:
        raise MmxError("N must be a positive multiple of 32")
    dt, M, K, a, lda = _activations(x, "x")
    if K == 0:
        raise MmxError("x has no columns")
    gu, d = _packed(gate_up, "gate_up", 2 * N, K), _packed(down, "down", K, N)
    y = torch.empty((M, K), dtype=torch.bfloat16, device=x.device) if y is None else _result(y, "y", M, K)
    if M == 0:
        return y
    need = L.lib().mmx_mlp_mxfp4_scratch_bytes(dt, M, K, N)
    scratch = _scratch(need, x.device)
    L._check(L.lib().mmx_mlp_mxfp4(dt, a, lda, gu, d, L.dtype_code(y), y.data_ptr(), _rows(y), M, K, N, _ptr(scratch), need, L._stream()))
    return y
