"""The feed-forward block in 8-bit floating point: quantisation, products with a scale for each block of 128, the MLP over such
weights, a mixture-of-experts layer for a few tokens, and the norms around a block.  As in _lib, arguments are checked here and
every call ends in the C ABI (include/mm_amx_amd.h says what each computes); nothing is computed by PyTorch.

A call's scratch is torch memory of its own, on the current stream, so that calls on different streams and captured graphs
share none.
"""
import ctypes as C

import torch

from . import _lib as L
from ._lib import MmxError

BLOCK = 128
_E4M3 = torch.float8_e4m3fn


def _blocks(n):
    return -(-n // BLOCK)


def _gpu(t, what, dtypes, dim):
    """A tensor on the current GPU of one of these types and that many dimensions, unit stride in the last."""
    if not isinstance(t, torch.Tensor) or t.dim() != dim or t.dtype not in dtypes:
        raise MmxError(f"{what} must be a {dim}-D tensor of {' or '.join(str(d) for d in dtypes)}")
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        raise MmxError(f"{what} must have unit stride in its last dimension")
    L._dev(t, what)
    if t.get_device() != L._current_device():
        raise MmxError(f"{what} is on cuda:{t.get_device()}, the current device is cuda:{L._current_device()}")
    return t


def _rows(t):
    """The row stride of a 2-D tensor in bytes (that of a single row, which torch leaves arbitrary, is the row itself)."""
    return (t.shape[1] if t.shape[0] <= 1 else t.stride(0)) * t.element_size()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _scratch(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


class Fp8Rows:
    """Quantised activations [M, K]: ``q`` e4m3 [M, K] and ``scales`` fp32 [ceil(K / 128), M], the value of q[m, k] being
    q * scales[k // 128, m].  Unpacks as ``q, scales = rows``.  The rows are kept padded with zeros to whole blocks of 128."""

    def __init__(self, padded, scales, K):
        self.padded, self.scales, self.K = padded, scales, K

    @classmethod
    def empty(cls, M, K, device):
        # rows a multiple of 2 KiB apart meet in few channels of the L2: they get 128 bytes more between them
        n = _blocks(K) * BLOCK
        return cls(torch.empty((M, n + 128 if n % 2048 == 0 else n), dtype=_E4M3, device=device)[:, :n], torch.empty((_blocks(K), M), device=device), K)

    @classmethod
    def of(cls, q, scales):
        """From e4m3 values [M, K] and fp32 scales [ceil(K / 128), M] made elsewhere; values that are not rows of whole blocks, 16-byte
        aligned, are copied."""
        if not isinstance(q, torch.Tensor) or q.dtype != _E4M3 or q.dim() != 2:
            raise MmxError("q must be a 2-D tensor of torch.float8_e4m3fn")
        M, K = q.shape
        if not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or tuple(scales.shape) != (_blocks(K), M):
            raise MmxError(f"scales must be fp32 [{_blocks(K)}, {M}] (a block of 128 and a row each)")
        if q.device != scales.device:
            raise MmxError("q and its scales are on different devices")
        if K % BLOCK or (K and q.stride(1) != 1) or q.data_ptr() % 16 or (M > 1 and (q.stride(0) % 16 or q.stride(0) < K)):
            padded = torch.zeros((M, _blocks(K) * BLOCK), dtype=torch.uint8, device=q.device)
            padded[:, :K] = q.view(torch.uint8) if q.stride(1) == 1 or K == 1 else q.contiguous().view(torch.uint8)
            q = padded.view(_E4M3)
        if M and scales.shape[0] and (scales.stride(1) != 1 and M != 1 or scales.stride(0) < M):
            scales = scales.contiguous()
        return cls(q, scales, K)

    @property
    def q(self):
        return self.padded[:, :self.K]

    @property
    def shape(self):
        return torch.Size((self.padded.shape[0], self.K))

    @property
    def device(self):
        return self.padded.device

    def __iter__(self):
        return iter((self.q, self.scales))

    def _args(self, what):
        """(pointer, row stride, scales, their stride), checked."""
        M = self.padded.shape[0]
        q, s = _gpu(self.padded, what, (_E4M3,), 2), _gpu(self.scales, f"{what}'s scales", (torch.float32,), 2)
        if q.shape[1] != _blocks(self.K) * BLOCK or tuple(s.shape) != (_blocks(self.K), M):
            raise MmxError(f"{what} [{M}, {self.K}]: {tuple(q.shape)} values and {tuple(s.shape)} scales do not belong together")
        return q.data_ptr(), _rows(q), s.data_ptr(), M if s.shape[0] <= 1 else s.stride(0)


def quantize_fp8(x):
    """x [M, K] bf16 or fp32 -> Fp8Rows: a scale for each row and 128 of k, the least power of two with which the block's largest magnitude is
    at most 448."""
    if L._native is not None and L._initialised:  # (regular calls; None: not one, nothing was done)
        made = L._made(L._native.quantize_fp8, x)
        if made is not None:
            return Fp8Rows(made[0], made[1], x.shape[1])
    _gpu(x, "x", (torch.bfloat16, torch.float32), 2)
    M, K = x.shape
    if K == 0:
        raise MmxError("x has no columns")
    out = Fp8Rows.empty(M, K, x.device)
    if M:
        L._check(L.lib().mmx_quantize_rows_fp8(L.dtype_code(x), x.data_ptr(), _rows(x), M, K, out.padded.data_ptr(), _rows(out.padded), out.scales.data_ptr(),
                                               M, L._stream()))
    return out


def quantize_pack_fp8(W, transpose=False):
    """bf16 weights W [K, N] (or [N, K] with transpose) -> (packed e4m3 as a uint8 tensor, scales fp32 [ceil(N / 128), ceil(K / 128)])."""
    _gpu(W, "W", (torch.bfloat16,), 2)
    K, N = (W.shape[1], W.shape[0]) if transpose else W.shape
    packed = torch.empty(L._packed_bytes_host(L.F8, K, N), dtype=torch.uint8, device=W.device)
    scales = torch.empty((_blocks(N), _blocks(K)), device=W.device)
    L._check(L.lib().mmx_quantize_pack_fp8(W.data_ptr(), _rows(W), K, N, int(transpose), 0, packed.data_ptr(), scales.data_ptr(), L._stream()))
    return packed, scales


def _given_scales(scales, what, N, K):
    _gpu(scales, f"{what}'s scales", (torch.float32,), 2)
    if tuple(scales.shape) != (_blocks(N), _blocks(K)):
        raise MmxError(f"{what}'s scales must be [{_blocks(N)}, {_blocks(K)}] for [{N}, {K}] weights, a block of 128 x 128 each")
    return scales.detach().contiguous()  # (of a parameter: what is packed holds no graph)


def _packed_into(out, w, K, N, rows):
    """The caller's (packed, scales), checked, or new ones."""
    if out is None:
        return torch.empty(L._packed_bytes_host(L.F8, K, N), dtype=torch.uint8, device=w.device), torch.empty((rows, _blocks(K)), device=w.device)
    packed, scales = out
    _packed(packed, scales, "out", K, N, rows)
    return packed, scales


def pack_fp8(w, scales=None, out=None):
    """Weights w [N, K] in torch's layout, bf16 (quantised here) or e4m3 with the scales [ceil(N / 128), ceil(K / 128)] they came with
    -> (packed, scales); out: where to put both."""
    if scales is None:
        _gpu(w, "weights without scales", (torch.bfloat16,), 2)
    else:
        _gpu(w, "weights with scales", (_E4M3,), 2)
        scales = _given_scales(scales, "weights", *w.shape)
    N, K = w.shape
    packed, s = _packed_into(out, w, K, N, _blocks(N))
    if scales is None:
        L._check(L.lib().mmx_quantize_pack_fp8(w.data_ptr(), _rows(w), K, N, 1, 0, packed.data_ptr(), s.data_ptr(), L._stream()))
    else:
        L._check(L.lib().mmx_repack_b(L.F8, w.data_ptr(), _rows(w), K, N, 1, packed.data_ptr(), L._stream()))
        s.copy_(scales)
    return packed, s


def pack_gate_up_fp8(w_gate, w_up, scales=None, out=None):
    """Gate and up weights [N, K] as in pack_fp8 (scales: a pair) -> (packed [K, 2 N], scales of both, gate's rows first)."""
    for w in (w_gate, w_up):
        _gpu(w, "w_gate and w_up", (torch.bfloat16,) if scales is None else (_E4M3,), 2)
    if w_gate.shape != w_up.shape:
        raise MmxError("w_gate and w_up must have the same shape")
    N, K = w_gate.shape
    if N == 0 or N % 32:
        raise MmxError(f"gate and up projections of {N} columns: a positive multiple of 32 is needed")
    if scales is not None:
        scales = [_given_scales(s, n, N, K) for s, n in zip(scales, ("w_gate", "w_up"))]
    nb = _blocks(N)
    packed, s = _packed_into(out, w_gate, K, 2 * N, 2 * nb)
    if scales is None:
        for pair, w in ((1, w_gate), (2, w_up)):
            L._check(L.lib().mmx_quantize_pack_fp8(w.data_ptr(), _rows(w), K, N, 1, pair, packed.data_ptr(), s.data_ptr(), L._stream()))
    else:
        if _rows(w_gate) != _rows(w_up):
            w_gate, w_up = w_gate.contiguous(), w_up.contiguous()
        L._check(L.lib().mmx_repack_gate_up_fp8(w_gate.data_ptr(), w_up.data_ptr(), _rows(w_gate), K, N, packed.data_ptr(), L._stream()))
        s[:nb].copy_(scales[0])
        s[nb:].copy_(scales[1])
    return packed, s


def _activations(x, what):
    """(dtype code, M, K, pointer, row stride, scales, their stride) of bf16 or fp32 rows or of Fp8Rows."""
    if isinstance(x, Fp8Rows):
        q, ld, s, ld_s = x._args(what)
        return L.F8, x.shape[0], x.K, q, ld, s, ld_s
    _gpu(x, what, (torch.bfloat16, torch.float32), 2)
    return L.dtype_code(x), x.shape[0], x.shape[1], x.data_ptr(), _rows(x), None, 0


def _native_activations(x):
    return (x.padded, x.scales, x.K) if type(x) is Fp8Rows else (x, None, x.shape[1])


def _packed(p, s, what, K, N, rows):
    _gpu(p, what, (torch.uint8,), 1)
    _gpu(s, f"{what}'s scales", (torch.float32,), 2)
    need = L._packed_bytes_host(L.F8, K, N)
    if p.numel() < need or p.data_ptr() % 16:
        raise MmxError(f"{what} holds {p.numel()} bytes, a packed [{K}, {N}] matrix takes {need}, 16-byte aligned")
    if tuple(s.shape) != (rows, _blocks(K)) or not s.is_contiguous():
        raise MmxError(f"{what}'s scales must be contiguous [{rows}, {_blocks(K)}] for [{K}, {N}] weights")


def _result(y, what, M, N):
    _gpu(y, what, (torch.bfloat16, torch.float32), 2)
    if y.shape[0] != M or y.shape[1] != N:
        raise MmxError(f"{what} is {tuple(y.shape)}, the result is [{M}, {N}]")
    return y


def gemm_fp8(A, Bpacked, b_scales, N, ep):
    """C = PP(A . B) in e4m3 with a scale for each block of 128: A [M, K] is Fp8Rows, or bf16 / fp32 and quantised on the way;
    Bpacked and b_scales from quantize_pack_fp8, pack_fp8 or, with PP_SILU_GATE, pack_gate_up_fp8 (N then counts both halves).
    ep: PP_BIAS, PP_GELU or both, or PP_SILU_GATE alone, into bf16 or fp32.  The product of the scales that meet in a block is to be a normal number of fp32."""
    if not isinstance(ep, L.Epilogue):
        raise MmxError("ep must be an Epilogue")
    if L._native is not None and L._initialised and len(getattr(A, "shape", ())) == 2:
        rc = L._made(L._native.gemm_fp8, *_native_activations(A), Bpacked, b_scales, N, at_end=(ep.C, ep.steps, ep.bias, ep.deq, ep.deq_oc, ep.q, ep.q_oc))
        if rc is not None:
            return
    if not isinstance(N, int) or N <= 0:
        raise MmxError(f"N = {N} must be a positive int")
    dt, M, K, a, lda, s, ld_s = _activations(A, "A")
    pair = bool(ep.steps & L.PP_SILU_GATE)
    if pair and N % 64:
        raise MmxError("a gate/up pair has a multiple of 64 packed columns")
    _packed(Bpacked, b_scales, "Bpacked", K, N, 2 * _blocks(N // 2) if pair else _blocks(N))
    _result(ep.C, "C", M, N // 2 if pair else N)
    if ep.bias is not None:
        _gpu(ep.bias, "bias", (torch.float32,), 1)
        if ep.bias.numel() != N:
            raise MmxError(f"bias holds {ep.bias.numel()} values, N = {N}")
    if M == 0:
        return
    d = ep.struct()
    need = L.lib().mmx_gemm_fp8_scratch_bytes(dt, M, K, N)
    scratch = _scratch(need, A.device)
    L._check(L.lib().mmx_gemm_fp8(dt, a, lda, s, ld_s, Bpacked.data_ptr(), b_scales.data_ptr(), M, K, N, C.byref(d), _ptr(scratch), need, L._stream()))


def mlp_fp8(x, gate_up, down, N, y=None):
    """y = (silu(x . gate) * (x . up)) . down over e4m3 weights: x [M, K] as in gemm_fp8; gate_up, down: (packed, scales) pairs of pack_gate_up_fp8 and of
    pack_fp8 of the [K, N] down_proj weight.  y [M, K] bf16 or fp32 (default: a new bf16 tensor)."""
    if L._native is not None and L._initialised and len(getattr(x, "shape", ())) == 2:
        made = L._made(L._native.mlp_fp8, *_native_activations(x), *gate_up, *down, N, y)
        if made is not None:
            return made
    if not isinstance(N, int) or N <= 0 or N % 32:
        raise MmxError("N must be a positive multiple of 32")
    dt, M, K, a, lda, s, ld_s = _activations(x, "x")
    _packed(*gate_up, "w_gate_up", K, 2 * N, 2 * _blocks(N))
    _packed(*down, "w_down", N, K, _blocks(K))
    y = torch.empty((M, K), dtype=torch.bfloat16, device=x.device) if y is None else _result(y, "y", M, K)
    if M == 0:
        return y
    need = L.lib().mmx_mlp_fp8_scratch_bytes(dt, M, K, N)
    scratch = _scratch(need, x.device)
    L._check(L.lib().mmx_mlp_fp8(dt, a, lda, s, ld_s, gate_up[0].data_ptr(), gate_up[1].data_ptr(), down[0].data_ptr(), down[1].data_ptr(), L.dtype_code(y),
                                 y.data_ptr(), _rows(y), M, K, N, _ptr(scratch), need, L._stream()))
    return y


_SCORING = {"softmax": 0, "sigmoid": 1}  # MMX_MOE_SIGMOID
_RENORMALIZE = 2


def moe_route(x, router, top_k, scoring="softmax", renormalize=True, scale=1.0, bias=None):
    """-> (ids int32 [T, top_k], weights fp32 [T, top_k]) of x [T, H] bf16 over the experts of router [E, H] bf16: the top_k experts of the
    largest p + bias, p = softmax or sigmoid of the logits, and scale * p, divided by the sum of the chosen p if renormalize."""
    _gpu(x, "x", (torch.bfloat16,), 2), _gpu(router, "router", (torch.bfloat16,), 2)
    (T, H), E = x.shape, router.shape[0]
    if router.shape[1] != H:
        raise MmxError(f"x has {H} columns, router {router.shape[1]}")
    if scoring not in _SCORING:
        raise MmxError("scoring is 'softmax' or 'sigmoid'")
    if not isinstance(top_k, int) or not 1 <= top_k <= min(E, 16):
        raise MmxError(f"top_k = {top_k} of {E} experts (16 at most)")
    if bias is not None and _gpu(bias, "bias", (torch.float32,), 1).numel() != E:
        raise MmxError(f"bias holds {bias.numel()} values for {E} experts")
    ids = torch.empty((T, top_k), dtype=torch.int32, device=x.device)
    weights = torch.empty((T, top_k), device=x.device)
    if T:
        logits = torch.empty((T, E), dtype=torch.float64, device=x.device)
        L._check(L.lib().mmx_moe_route(x.data_ptr(), _rows(x), router.data_ptr(), _rows(router), T, H, E, top_k, _SCORING[scoring] | (_RENORMALIZE if renormalize else 0),
                                       scale, _ptr(bias), logits.data_ptr(), ids.data_ptr(), weights.data_ptr(), L._stream()))
    return ids, weights


def moe(x, router, top_k, gate_up, down, I, scoring="softmax", renormalize=True, scale=1.0, bias=None, y=None):
    """moe_route and moe_experts of its choices: a whole layer."""
    if L._native is not None and L._initialised and scoring in _SCORING:
        made = L._made(L._native.moe, x, router, bias, top_k, _SCORING[scoring] | (_RENORMALIZE if renormalize else 0), scale,
                       *(gate_up if type(gate_up) is tuple else (gate_up, None)), *(down if type(down) is tuple else (down, None)), I, y)
        if made is not None:
            return made
    ids, weights = moe_route(x, router, top_k, scoring, renormalize, scale, bias)
    return moe_experts(x, ids, weights, gate_up, down, router.shape[0], I, y=y)


def moe_experts(x, ids, weights, gate_up, down, E, I, y=None):
    """y[t] = sum over j of weights[t, j] * down_e(silu(gate_e . x[t]) * (up_e . x[t])), e = ids[t, j] (outside [0, E): no expert).
    x [T, H] bf16; gate_up and down: packed weights of all experts one behind the other as a uint8 tensor (bf16), or (packed, scales)
    pairs (e4m3).  y [T, H] bf16 or fp32 (default: a new bf16 tensor)."""
    _gpu(x, "x", (torch.bfloat16,), 2)
    T, H = x.shape
    _gpu(ids, "ids", (torch.int32,), 2), _gpu(weights, "weights", (torch.float32,), 2)
    if ids.shape[0] != T or ids.shape != weights.shape or not 1 <= ids.shape[1] <= 16 or not ids.is_contiguous() or not weights.is_contiguous():
        raise MmxError(f"ids and weights must be contiguous [{T}, top_k], top_k from 1 to 16")
    if not isinstance(I, int) or I <= 0 or I % 32:
        raise MmxError("I must be a positive multiple of 32")
    if not isinstance(E, int) or not 1 <= E <= 1024 or H == 0:
        raise MmxError("1 to 1024 experts over rows that are not empty")
    f8 = isinstance(gate_up, (tuple, list))
    if f8 != isinstance(down, (tuple, list)):
        raise MmxError("gate_up and down must both be e4m3 (packed, scales) or both packed bf16")
    parts = []
    for w, what, K, N, rows in ((gate_up, "gate_up", H, 2 * I, 2 * _blocks(I)), (down, "down", I, H, _blocks(H))):
        p, s = w if f8 else (w, None)
        _gpu(p, what, (torch.uint8,), 1)
        need = E * L._packed_bytes_host(L.F8 if f8 else L.BF16, K, N)
        if p.numel() < need or p.data_ptr() % 16:
            raise MmxError(f"{what} holds {p.numel()} bytes, {E} packed [{K}, {N}] matrices take {need}, 16-byte aligned")
        if f8 and (tuple(_gpu(s, f"{what}'s scales", (torch.float32,), 3).shape) != (E, rows, _blocks(K)) or not s.is_contiguous()):
            raise MmxError(f"{what}'s scales must be contiguous [{E}, {rows}, {_blocks(K)}]")
        parts += [p.data_ptr(), _ptr(s)]
    y = torch.empty((T, H), dtype=torch.bfloat16, device=x.device) if y is None else _result(y, "y", T, H)
    if T == 0:
        return y
    k = ids.shape[1]
    need = L.lib().mmx_moe_experts_scratch_bytes(T, H, I, k)
    scratch = _scratch(need, x.device)
    L._check(L.lib().mmx_moe_experts(L.F8 if f8 else L.BF16, x.data_ptr(), _rows(x), ids.data_ptr(), weights.data_ptr(), T, H, I, E, k, *parts,
                                     L.dtype_code(y), y.data_ptr(), _rows(y), scratch.data_ptr(), need, L._stream()))
    return y


def block_norm(f, residual=None, *, post=False, post_weight=None, gate=None, scale=1.0, pre=True, pre_weight=None, eps=1e-6, weight_offset=0.0,
               quantize=False, r=None, z=None):
    """The seam between two blocks in one pass over the rows of f [M, H] bf16:

        u = f, or with post  f / sqrt(mean(f^2) + eps) * (weight_offset + post_weight)
        r = residual + scale * gate * u
        z = r, or with pre   r / sqrt(mean(r^2) + eps) * (weight_offset + pre_weight)

    -> (r, z).  residual [M, H] bf16 or fp32, r like it (bf16 without one); gate bf16 [H], or [M, H] for a gate per row; weights bf16 [H] or None.
    z is bf16, or with quantize Fp8Rows.  r, z: where to put them (r may be residual itself; False: r is not wanted, and None in its place)."""
    if L._native is not None and L._initialised and z is None:
        made = L._made(L._native.block_norm, f, residual, post, post_weight, gate, scale, pre, pre_weight, eps, weight_offset, quantize, r)
        if made is not None:
            return (made[0], Fp8Rows(made[1], made[2], f.shape[1])) if quantize else made
    _gpu(f, "f", (torch.bfloat16,), 2)
    M, H = f.shape
    if H == 0:
        raise MmxError("f has no columns")
    if (post_weight is not None and not post) or (pre_weight is not None and not pre):
        raise MmxError("post_weight needs post, pre_weight needs pre")
    for t, what in ((post_weight, "post_weight"), (pre_weight, "pre_weight")):
        if t is not None and _gpu(t, what, (torch.bfloat16,), 1).numel() != H:
            raise MmxError(f"{what} holds {t.numel()} values, H = {H}")
    stream = torch.bfloat16
    if residual is not None:
        stream = _gpu(residual, "residual", (torch.bfloat16, torch.float32), 2).dtype
        if residual.shape != f.shape:
            raise MmxError(f"residual is {tuple(residual.shape)}, f {tuple(f.shape)}")
    ld_gate = 0
    if gate is not None:
        _gpu(gate, "gate", (torch.bfloat16,), 1 if isinstance(gate, torch.Tensor) and gate.dim() == 1 else 2)
        if gate.shape[-1] != H or (gate.dim() == 2 and gate.shape[0] not in (1, M)):
            raise MmxError(f"gate is {tuple(gate.shape)}, [{H}] or [{M}, {H}] are possible")
        ld_gate = 0 if gate.dim() == 1 or gate.shape[0] == 1 else gate.stride(0) * 2
    if r is None:
        r = torch.empty((M, H), dtype=stream, device=f.device)
    elif r is False:
        r = None
    elif _gpu(r, "r", (stream,), 2).shape != f.shape:
        raise MmxError(f"r is {tuple(r.shape)}, f {tuple(f.shape)}")
    if z is None:
        z = Fp8Rows.empty(M, H, f.device) if quantize else torch.empty((M, H), dtype=torch.bfloat16, device=f.device)
    elif isinstance(z, Fp8Rows) != bool(quantize) or z.shape != f.shape:
        raise MmxError(f"z must be {'Fp8Rows' if quantize else 'a bf16 tensor'} of {tuple(f.shape)}")
    zs, ld_zs = None, 0
    if quantize:
        zp, ldz, zs, ld_zs = z._args("z")
    else:
        zp, ldz = _gpu(z, "z", (torch.bfloat16,), 2).data_ptr(), _rows(z)
    if M:
        args = L._BlockNorm(f.data_ptr(), _rows(f), _ptr(residual), 0 if residual is None else _rows(residual), _ptr(post_weight), _ptr(gate), ld_gate, _ptr(pre_weight),
                            _ptr(r), 0 if r is None else _rows(r), zp, ldz, zs, ld_zs, L.F32 if stream == torch.float32 else L.BF16, L.F8 if quantize else L.BF16, int(post), int(pre),
                            scale, eps, weight_offset)
        L._check(L.lib().mmx_block_norm(C.byref(args), M, H, L._stream()))
    return r, z
