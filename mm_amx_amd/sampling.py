"""Drawing tokens from the logits that a head's product leaves: temperature, top_k, top_p and min_p, from random numbers that the caller gives.  As in
ffn, arguments are checked here and every call ends in the C ABI (include/mm_amx_amd.h defines what is drawn); nothing is computed by PyTorch.
"""
import ctypes as C

import torch

from . import _lib as L
from ._lib import MmxError
from .ffn import _gpu, _ptr, _rows, _scratch


def _asked(v, what, B, dtype, lo, hi):
    """(pointer, number) of a number for all rows or a tensor with one for each."""
    if isinstance(v, torch.Tensor):
        if _gpu(v, what, (dtype,), 1).numel() != B or not v.is_contiguous():
            raise MmxError(f"{what} must be a number or a contiguous {dtype} tensor [{B}]")
        return v.data_ptr(), 0
    if isinstance(v, bool) or not isinstance(v, int if dtype == torch.int32 else (int, float)) or not lo <= v <= hi:
        raise MmxError(f"{what} = {v} is out of range")
    if dtype == torch.int32:
        return None, v
    try:
        return None, float(v)
    except OverflowError:  # (a whole number that is below infinity, but no double)
        raise MmxError(f"{what} is out of range") from None


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """-> ids int32 [B]: a token for each row of logits [B, V] bf16 or fp32, given u fp32 [B] from [0, 1).

    Weights are e^((l - max l) / temperature); of their descending order (the lowest index of equal ones first) top_k (0: off) keeps the first k, top_p (1: off)
    of those the shortest run that holds top_p of their weight, min_p (0: off) of those what has min_p of the largest weight at least.  The token is the first in
    the order of the vocabulary up to which the weights that were kept come to more than u of their sum.  temperature 0 takes the largest; -inf and NaN are never
    drawn (a row of nothing else: -1).  Each of the four is a number, or a tensor [B] on the GPU with one for each row (int32 for top_k, else fp32).  out: where to
    put the ids."""
    if L._native is not None and L._initialised and out is None:
        made = L._made(L._native.sample, logits, u, temperature, top_k, top_p, min_p)
        if made is not None:
            return made
    B, V = _gpu(logits, "logits", (torch.bfloat16, torch.float32), 2).shape
    if V == 0:
        raise MmxError("logits have no columns")
    if _gpu(u, "u", (torch.float32,), 1).numel() != B or not u.is_contiguous():
        raise MmxError(f"u must be a contiguous tensor [{B}], a number for each row")
    (t_of, t), (k_of, k), (p_of, p), (m_of, m) = (_asked(temperature, "temperature", B, torch.float32, 0, float("inf")), _asked(top_k, "top_k", B, torch.int32, 0, 2 ** 31 - 1),
                                                  _asked(top_p, "top_p", B, torch.float32, 0, float("inf")), _asked(min_p, "min_p", B, torch.float32, 0, 1))
    if out is None:
        out = torch.empty(B, dtype=torch.int32, device=logits.device)
    elif _gpu(out, "out", (torch.int32,), 1).numel() != B or not out.is_contiguous():
        raise MmxError(f"out must be a contiguous tensor [{B}]")
    if B:
        need = L.lib().mmx_sample_scratch_bytes(B, V)
        scratch = _scratch(need, logits.device)
        args = L._Sample(logits.data_ptr(), _rows(logits), u.data_ptr(), t_of, k_of, p_of, m_of, t, p, m, out.data_ptr(), k, L.dtype_code(logits))
        L._check(L.lib().mmx_sample(C.byref(args), B, V, _ptr(scratch), need, L._stream()))
    return out
