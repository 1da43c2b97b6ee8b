"""What the drawing of tokens refuses, and the 64-bit definition that its GPU tests use, by hand."""
import ctypes as C

import numpy as np
import pytest
import torch

import mm_amx_amd as mx
import sample_util as su
from mm_amx_amd import _lib as L

P = 1 << 20  # an address that is never read


def test_refusals():
    lib = L.lib()
    need = lib.mmx_sample_scratch_bytes(4, 1000)
    base = dict(l=P, ld=4000, u=P, t_of=None, k_of=None, p_of=None, m_of=None, t=1.0, p=1.0, m=0.0, ids=P, k=0, dt=0)

    def call(B=4, V=1000, scratch=P, n=need, **k):
        return lib.mmx_sample(C.byref(L._Sample(*{**base, **k}.values())), B, V, scratch, n, None)

    for bad, word in ((dict(l=None), "NULL"), (dict(ld=3996), "apart"), (dict(l=P + 2), "aligned"), (dict(dt=1, l=P + 1), "aligned"), (dict(u=None), "NULL"), (dict(ids=None), "NULL"),
                      (dict(ids=P + 2), "aligned"), (dict(t_of=P + 1), "aligned"), (dict(k_of=P + 2), "aligned"), (dict(t=-1.0), "temperature"), (dict(t=float("nan")), "temperature"),
                      (dict(p=-0.5), "top_p"), (dict(m=1.5), "min_p"), (dict(k=-1), "top_k"), (dict(dt=2), "dtype"), (dict(V=0), "positive"), (dict(B=-1), "negative"),
                      (dict(B=65536), "up to"), (dict(V=(1 << 22) + 1), "up to"), (dict(n=need - 1), "scratch"), (dict(scratch=None), "scratch"), (dict(scratch=P + 128), "256-byte")):
        rc = call(**bad)
        assert rc in (-1, -2) and word in lib.mmx_last_error().decode(), (bad, rc, lib.mmx_last_error())
    assert lib.mmx_sample(None, 1, 1, None, 0, None) == -1
    assert call(B=0, l=None) == 0
    assert lib.mmx_sample_scratch_bytes(0, 5) == lib.mmx_sample_scratch_bytes(5, 0) == 0
    l, u = torch.zeros((2, 10)), torch.zeros(2)
    with pytest.raises(mx.MmxError, match="on the GPU"):
        mx.sample(l, u)


def test_the_definition():
    l = np.log([0.1, 0.4, 0.2, 0.3])
    draw = lambda u, **k: su.token(l, u, **k)  # noqa: E731
    assert [draw(u) for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.99, 1.0)] == [0, 0, 1, 1, 2, 2, 3, 3, 3]
    assert [draw(u, k=2) for u in (0.0, 0.5, 0.6, 0.99)] == [1, 1, 3, 3]
    assert list(su.kept(l, p=0.5)[0]) == [1, 3] and list(su.kept(l, p=0.39)[0]) == [1] and list(su.kept(l, p=0.0)[0]) == [1] and list(su.kept(l, p=0.71)[0]) == [1, 2, 3]
    assert list(su.kept(l, k=3, p=0.7)[0]) == [1, 3]  # (0.7 of the three's 0.9)
    assert list(su.kept(l, min_p=0.6)[0]) == [1, 3] and list(su.kept(l, min_p=1.0)[0]) == [1]
    assert draw(0.9, T=0.0) == 1 and su.token([1.0, 1.0], 0.9, T=0.0) == 0
    assert su.token([-np.inf, np.nan], 0.5) == -1 and su.token([0.0, np.inf, 1.0], 0.99) == 1
    assert list(su.kept(np.zeros(4), k=2)[0]) == [0, 1] and list(su.kept(np.zeros(4), p=0.6)[0]) == [0, 1, 2]


def test_whole_numbers_past_64_bits_are_refused():
    """What no double can hold is an argument out of range like any other."""
    from mm_amx_amd import sampling
    inf = float("inf")
    for v in (10 ** 400, -10 ** 400):
        with pytest.raises(mx.MmxError, match="out of range"):
            sampling._asked(v, "temperature", 4, torch.float32, 0, inf)
    assert sampling._asked(2 ** 70, "temperature", 4, torch.float32, 0, inf) == (None, 2.0 ** 70)
    assert sampling._asked(inf, "top_p", 4, torch.float32, 0, inf) == (None, inf)
    assert sampling._asked(40, "top_k", 4, torch.int32, 0, 2 ** 31 - 1) == (None, 40)
