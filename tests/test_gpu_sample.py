"""Drawing tokens from logits, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import sample_util as su

pytestmark = pytest.mark.gpu

import mm_amx_amd as mx  # noqa: E402


def logits(B, V, seed, std=2.0, dtype=torch.float32, peaks=12):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn((B, V), generator=g) * std
    l += 10 * (torch.rand((B, V), generator=g) < peaks / V) * torch.rand((B, V), generator=g)
    return l.to(dtype), torch.rand(B, generator=g)


def check(l, u, T=1.0, k=0, p=1.0, m=0.0):
    """Numbers, or a list with one for each row."""
    B = l.shape[0]
    rows = [[v] * B if not isinstance(v, list) else v for v in (T, k, p, m)]
    give = [torch.tensor(v, dtype=torch.int32 if i == 1 else torch.float32).cuda() if isinstance(v, list) else v for i, v in enumerate((T, k, p, m))]
    got = mx.sample(l.cuda(), u.cuda(), *give)
    assert got.dtype == torch.int32 and got.shape == (B,)
    exact = lambda v, of: float(np.float32(v)) if isinstance(of, list) else v  # noqa: E731 (tensors hold 32 bits)
    want = [su.token(l[b].double().numpy(), float(u[b]), exact(rows[0][b], T), rows[1][b], exact(rows[2][b], p), exact(rows[3][b], m)) for b in range(B)]
    assert got.tolist() == want
    return got


FILTERS = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (1.3, 0, 0.5, 0.0), (0.7, 20, 1.0, 0.0), (1.0, 0, 1.0, 0.05), (1.0, 2, 1.0, 0.0), (1.1, 700, 0.99, 0.001), (1.0, 3000, 1.0, 0.0),
           (1.0, 5000, 0.8, 0.0), (0.2, 0, 0.999, 0.0), (5.0, 0, 0.9, 0.3), (1.0, 1, 1.0, 0.0), (0.0, 40, 0.9, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 100, 0.7, 1.0), (0.05, 0, 0.9, 0.0), (30.0, 0, 0.9, 0.0)]


@pytest.mark.parametrize("V", [1, 2, 63, 1000, 1024, 1025, 8191, 32000, 50001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_filters(V, dtype):
    l, u = logits(7, V, V, dtype=dtype)
    for T, k, p, m in FILTERS:
        check(l, u, T, k, p, m)


@pytest.mark.parametrize("B,V", [(1, 131072), (33, 100003), (64, 20000), (300, 999), (600, 2500)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_each_row_asks_for_its_own(B, V, dtype):
    l, u = logits(B, V, B, dtype=dtype)
    rows = [FILTERS[b % len(FILTERS)] for b in range(B)]
    check(l, u, *([r[i] for r in rows] for i in range(4)))


def test_large_vocabularies_and_flat_rows():
    for V, std in ((1 << 20, 2.0), ((1 << 22) - 5, 0.1)):
        l, u = logits(2, V, 3, std=std)
        for f in ((1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 100, 0.9, 0.0), (1.0, 100000, 0.9, 0.0), (1.0, 0, 1.0, 0.2)):
            check(l, u, *f)


@pytest.mark.parametrize("V", [5, 1000, 3000, 70000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits_go_by_their_index(V, dtype):
    """All equal, and two values only: the run that stays ends among equal ones."""
    g = torch.Generator().manual_seed(V)
    u = torch.tensor([0.0, 0.3, 0.6, 0.999, 0.5, 0.9])
    same = torch.zeros((6, V), dtype=dtype)
    two = (torch.rand((6, V), generator=g) < 0.5).to(dtype)
    signs = torch.where(torch.rand((6, V), generator=g) < 0.5, 0.0, -0.0).to(dtype)  # (the two zeros are equal)
    for l in (same, two, signs):
        for f in ((1.0, 0, 1.0, 0.0), (1.0, 3, 1.0, 0.0), (1.0, V // 2 + 1, 1.0, 0.0), (1.0, 0, 0.37, 0.0), (1.0, V // 3 + 1, 0.41, 0.0), (1.0, 0, 0.77, 0.4), (0.0, 0, 1.0, 0.0)):
            check(l, u, *f)
    assert mx.sample(same.cuda(), u.cuda(), temperature=0.0).tolist() == [0] * 6


@pytest.mark.parametrize("V", [4, 1500, 40000])
@pytest.mark.parametrize("f", [(1.0, 0, 1.0, 0.0), (1.0, 50, 0.9, 0.0), (0.7, 0, 0.8, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.1), (1.0, 1, 1.0, 0.0)])
def test_masks_infinities_and_nan(V, f):
    l, u = logits(12, V, 1)
    inf = float("inf")
    l[0] = -inf                               # nothing is left
    l[1] = float("nan")
    l[2], l[2, V // 2] = -inf, -3.0           # one is
    l[3, ::2] = -inf
    l[4, 1::2] = float("nan")
    l[5, 1] = inf                             # beside it nothing has weight
    l[6, 0], l[6, V - 1] = inf, inf
    l[7] = torch.finfo(torch.float32).min     # masks of the lowest value: all equal
    l[8], l[8, 1] = torch.finfo(torch.float32).min, 2.0
    l[9] = inf
    l[10, 0], l[10, 1] = 3e38, -3e38
    l[11] = l[11] * 1e-30
    got = check(l, u, *f).tolist()
    assert got[0] == got[1] == -1 and got[2] == V // 2 and got[5] == 1 and got[6] in (0, V - 1) and got[8] == 1 and got[10] == 0


def test_the_ends_of_u():
    l, _ = logits(6, 3000, 2)
    l[:, 0] = l[:, 2999] = -float("inf")
    u = torch.tensor([0.0, 1.0, -1.0, float("nan"), 1.0 - 2.0 ** -24, 7.0])
    for f in ((1.0, 0, 1.0, 0.0), (1.0, 20, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.01)):
        got = mx.sample(l.cuda(), u.cuda(), *f).tolist()
        for b in range(6):
            at, w = su.kept(l[b].double().numpy(), *f)
            live = at[w > 0]
            assert got[b] == (live[0] if b in (0, 2, 3) else live[-1] if b in (1, 5) else su.token(l[b].double().numpy(), float(u[b]), *f)), (f, b)


def test_out_of_range_in_tensors_is_taken_as_the_nearest():
    l, u = logits(4, 2000, 3)
    nan, inf = float("nan"), float("inf")
    give = lambda v, t=torch.float32: torch.tensor(v, dtype=t).cuda()  # noqa: E731
    base = lambda **k: mx.sample(l.cuda(), u.cuda(), **k).tolist()  # noqa: E731
    assert base(temperature=give([-1.0, nan, 0.0, -inf])) == base(temperature=0.0)
    assert base(top_k=give([-5, 0, 2000, 2 ** 31 - 1], torch.int32)) == base()
    assert base(top_p=give([nan, 1.5, inf, 1.0])) == base() and base(top_p=give([-1.0, 0.0, -inf, 0.0])) == base(top_p=0.0)
    assert base(min_p=give([nan, -1.0, 0.0, -inf])) == base() and base(min_p=give([1.5, inf, 1.0, 2.0])) == base(min_p=1.0)
    assert base(temperature=inf, top_k=3) == [su.token(l[b].double().numpy(), float(u[b]), inf, 3) for b in range(4)]


@pytest.mark.parametrize("T", [float("inf"), 1e30])
@pytest.mark.parametrize("V", [2000, 40000])
def test_min_p_above_one_in_tensors_keeps_what_one_keeps(T, V):
    """Where the temperature makes every weight 1, a min_p of 1 drops none, and more than 1 is taken as 1."""
    l, u = logits(4, V, 5)
    m = [1.5, float("inf"), 1.0, 2.0]
    for k, p in ((0, 1.0), (40, 1.0), (40, 0.9), (0, 0.9)):
        got = check(l, u, T, k, p, m)
        assert torch.equal(got, mx.sample(l.cuda(), u.cuda(), T, k, p, 1.0))


@pytest.mark.parametrize("f", [(1.0, 0, 1.0, 0.0), (0.9, 30, 0.9, 0.0), (1.0, 0, 0.9, 0.0)])
def test_rows_of_any_stride_and_alignment(f):
    base, u = logits(20, 3333, 4, dtype=torch.bfloat16)
    wide = base.cuda()
    for sub in ((slice(None), slice(1, 3001)), (slice(0, None, 2), slice(3, 3300)), (slice(5, 6), slice(7, 3333))):
        l = wide[sub]
        want = [su.token(r.double().numpy(), float(x), *f) for r, x in zip(base[sub], u[:l.shape[0]])]
        assert mx.sample(l, u[:l.shape[0]].cuda(), *f).tolist() == want
    out = torch.full((22,), 77, dtype=torch.int32, device="cuda")
    assert mx.sample(wide, u.cuda(), *f, out=out[:20]).data_ptr() == out.data_ptr()
    assert out[:20].tolist() == mx.sample(wide, u.cuda(), *f).tolist() and out[20:].tolist() == [77, 77]


def test_frequencies_are_the_weights():
    """20000 draws from eight tokens: each one's count is within 6 standard deviations of what its share makes it."""
    l = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5, -3.0, 1.5, 0.0])
    n = 20000
    u = torch.rand(n, generator=torch.Generator().manual_seed(5)).cuda()
    ids = mx.sample(l.expand(n, 8).contiguous().cuda(), u, temperature=0.7, top_k=6)
    at, w = su.kept(l.double().numpy(), 0.7, 6)
    share = np.zeros(8)
    share[at] = w / w.sum()
    count = np.bincount(ids.cpu().numpy(), minlength=8)
    assert (np.abs(count - n * share) <= 6 * np.sqrt(n * share * (1 - share)) + 1e-9).all()


def test_graphs_and_streams():
    """Replays of captured draws with other logits and random numbers in place, beside eager ones on another stream."""
    l, u = logits(9, 30000, 6)
    l, u = l.cuda(), u.cuda()
    fs = ((1.0, 0, 1.0, 0.0), (0.9, 30, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05))
    side = torch.cuda.Stream()
    graphs = []
    for f in fs:
        with torch.cuda.stream(side):
            mx.sample(l, u, *f)
            side.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                ids = mx.sample(l, u, *f)
            graphs.append((gr, ids))
    for i in range(4):
        a, b = logits(9, 30000, 20 + i)
        torch.cuda.synchronize()
        l.copy_(a), u.copy_(b)
        want = [mx.sample(l, u, *f) for f in fs]
        torch.cuda.synchronize()
        for (gr, ids), f, w in zip(graphs, fs, want):
            with torch.cuda.stream(side):
                gr.replay()
            eager = mx.sample(l, u, *f)
            torch.cuda.synchronize()
            assert torch.equal(ids, w) and torch.equal(eager, w)


def test_block_head_and_token_together():
    """A norm into packed rows, an MLP, the norm in front of the head, the head and the draw, as a decode step runs them, against the same in 64 bits from its logits."""
    M, K, N, V = 5, 512, 768, 5000
    g = torch.Generator().manual_seed(7)
    t = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to(torch.bfloat16).cuda()  # noqa: E731
    f, r = t(M, K), t(M, K)
    mlp, head = mx.MLP(), mx.LinearMxfp4()
    mlp.setup(t(N, K, std=0.05), t(N, K, std=0.05), t(K, N, std=0.05), compress="mxfp4")
    head.set_weight(t(V, K, std=0.1))
    u = torch.rand(M, generator=g).cuda()

    def step():
        r1, z = mx.block_norm(f, r, quantize="mxfp4")
        y = mlp.run(z)
        _, z = mx.block_norm(y, r1, quantize="mxfp4", r=False)
        l = torch.empty((M, V), device="cuda")
        head.forward(z, l)
        return l, mx.sample(l, u, temperature=0.8, top_k=40, top_p=0.9)

    l, ids = step()
    assert ids.tolist() == [su.token(l[b].double().cpu().numpy(), float(u[b]), 0.8, 40, 0.9) for b in range(M)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            lg, ig = step()
    for _ in range(3):
        torch.cuda.synchronize()
        lg.zero_(), ig.zero_()
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(lg, l) and torch.equal(ig, ids)


def test_nothing_to_do_and_refusals():
    l, u = logits(4, 100, 8)
    l, u = l.cuda(), u.cuda()
    assert mx.sample(l[:0], u[:0]).shape == (0,)
    for bad in (dict(logits=l.half()), dict(logits=l[0]), dict(logits=l[:, :0]), dict(logits=l.t()), dict(logits=l.cpu()), dict(u=u[:3]), dict(u=u.double()), dict(u=u.cpu()), dict(temperature=-1.0),
                dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=2.0), dict(top_p=-0.1), dict(min_p=1.1), dict(min_p=float("nan")), dict(top_k=u), dict(temperature=u[:2]),
                dict(top_p=u.double()), dict(min_p=u.cpu()), dict(temperature="1"), dict(top_p=torch.stack((u, u), 1)[:, 0]), dict(out=torch.empty(3, dtype=torch.int32, device="cuda")),
                dict(out=torch.empty(4, device="cuda")), dict(u=torch.stack((u, u), 1)[:, 0])):
        with pytest.raises(mx.MmxError):
            mx.sample(**{**dict(logits=l, u=u), **bad})


def test_logits_of_more_than_4_gib():
    """Rows past 2^32 bytes, some of them against the definition."""
    B, V = 1100, 1 << 21
    l = torch.empty((B, V), dtype=torch.bfloat16, device="cuda")
    for b in range(0, B, 100):
        l[b:b + 100] = torch.randn((100, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(b)).to(torch.bfloat16)
    assert l.numel() * 2 > 2 ** 32
    u = torch.rand(B, generator=torch.Generator().manual_seed(1))
    for f in ((1.0, 0, 1.0, 0.0), (1.0, 50, 0.9, 0.0)):
        got = mx.sample(l, u.cuda(), *f).tolist()
        for b in (0, 700, 1098, 1099):
            assert got[b] == su.token(l[b].double().cpu().numpy(), float(u[b]), *f)


def test_large_logits_and_small_temperatures():
    """l / T far outside what a grid of bins holds, and logits whose differences are all that counts."""
    g = torch.Generator().manual_seed(3)
    u = torch.rand(6, generator=g)
    for scale, T in ((1e30, 1e30), (1e6, 1.0), (1e4, 1e4), (1.0, 1e-6), (1e-20, 1e-20), (3e37, 1.0)):
        for at in (0.0, 5.0, -7.0):  # (in units of the scale)
            l = (torch.randn((6, 3000), generator=g) * 2 + at) * scale
            for k, p, m in ((0, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.9, 0.0), (40, 0.9, 0.0), (0, 1.0, 0.05), (2000, 0.5, 0.0)):
                check(l, u, T, k, p, m)


@pytest.mark.parametrize("T", [5e-324, 1e-310, 6e-309, 1e-300, 1e-45, 1e30, float("inf")])
def test_temperatures_at_the_ends(T):
    l, u = logits(3, 5000, 11)
    l[0, 4321] = l[0, 4322] = 60.0
    l[1, :] = -1e-45
    l[1, 4000:4500] = 0.0
    for f in ((0, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.9, 0.0), (40, 0.9, 0.0), (0, 1.0, 0.5)):
        check(l, u, T, *f)


@pytest.mark.parametrize("V", [12000, 32000, 200001, 262144])
@pytest.mark.parametrize("std", [0.005, 0.2, 1.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_in_the_last_bin_than_a_list_holds(V, std, dtype):
    """Flat rows: the filters end among thousands of neighbours, in the row's highest bin and in others."""
    l, u = logits(3, V, V, std=std, dtype=dtype, peaks=0)
    l[2, 5000:60000] = l[2, 4999]  # (and among equal ones)
    for f in ((1.0, 0, 0.9, 0.0), (1.0, 50000, 1.0, 0.0), (2.0, 0, 0.5, 0.0), (0.5, 0, 0.999, 0.0), (1.0, V - 1, 1.0, 0.0), (1.0, 0, 0.0001, 0.0), (1.5, 0, 0.8, 0.6), (1.0, 20000, 0.7, 0.0)):
        check(l, u, *f)


def test_the_same_every_time():
    """Nothing depends on the order in which workgroups come: lists, sums and tokens of many replays."""
    l, u = logits(40, 50001, 9, dtype=torch.bfloat16)
    l, u = l.cuda(), u.cuda()
    for f in ((1.0, 0, 0.95, 0.0), (1.0, 300, 0.9, 0.01), (1.0, 0, 1.0, 0.0), (20.0, 0, 0.9, 0.0)):
        first = mx.sample(l, u, *f)
        for _ in range(20):
            assert torch.equal(mx.sample(l, u, *f), first)


def test_native_and_python_calls_agree(monkeypatch):
    from mm_amx_amd import _lib as L
    l, u = logits(9, 5000, 4)
    l, u = l.cuda(), u.cuda()
    rows = dict(temperature=torch.full((9,), 0.7, device="cuda"), top_k=torch.arange(9, dtype=torch.int32, device="cuda"), top_p=torch.full((9,), 0.9, device="cuda"),
                min_p=torch.full((9,), 0.01, device="cuda"))
    calls = lambda: [mx.sample(l, u), mx.sample(l, u, 0.7, 40, 0.9, 0.01), mx.sample(l, u, temperature=2, top_k=40), mx.sample(l, u, **rows)]  # noqa: E731
    native = calls()
    assert L._native is not None
    monkeypatch.setattr(L, "_native", None)
    assert all(torch.equal(a, b) for a, b in zip(native, calls()))


def test_whole_numbers_take_the_native_call(monkeypatch):
    """temperature=0, top_p=1 and their like are what programs write; the native call takes them as it takes floats."""
    from mm_amx_amd import _lib as L
    native, made = L._native, []
    assert native is not None

    class Spy:
        @staticmethod
        def sample(*a):
            made.append(native.sample(*a))
            return made[-1]

    l, u = logits(5, 3000, 10)
    l, u = l.cuda(), u.cuda()
    asked = (dict(temperature=0), dict(temperature=2, top_k=40), dict(top_p=1, min_p=0), dict(top_p=0), dict(min_p=1, temperature=1), dict(temperature=2 ** 31 - 1, top_k=3))
    want = [mx.sample(l, u, **{n: v if n == "top_k" else float(v) for n, v in a.items()}) for a in asked]
    monkeypatch.setattr(L, "_native", Spy)
    got = [mx.sample(l, u, **a) for a in asked]
    assert len(made) == len(asked) and all(m is not None for m in made)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for bad in (dict(temperature=-1), dict(top_p=-1), dict(min_p=2), dict(temperature=True)):
        with pytest.raises(mx.MmxError):
            mx.sample(l, u, **bad)


@pytest.mark.parametrize("V", [12000, 32000, 40000, 262144])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_k_ends_with_a_bin(V, dtype):
    """k as many as the bins above a border hold, one less and one more; and few of a flat row, where the parts that its bin is cut into hold one or two each."""
    g = torch.Generator().manual_seed(V)
    l = -1.0 - 2.0 * torch.rand((4, V), generator=g)
    for b in range(4):
        at = torch.randperm(V, generator=g)
        l[b, at[:3000]] = 0.001 + 0.06 * torch.rand(3000, generator=g)      # the row's first sixteenth
        l[b, at[3000:5000]] = -0.061 + 0.06 * torch.rand(2000, generator=g)  # and its second
    l, u = l.to(dtype), torch.rand(4, generator=g)
    for k in (2999, 3000, 3001, 4096, 4999, 5000, 5001):
        for m in (0.0, 0.9):
            check(l, u, 1.0, k, 1.0, m)
    for std in (0.005, 0.2, 2.0):
        l, u = logits(4, V, V + 1, std=std, dtype=dtype, peaks=0)
        for k in (2, 3, 5, 10, 20, 40, 50, 64, 100, 300, 1000):
            for T in (1.0, 30.0):
                check(l, u, T, k)


@pytest.mark.parametrize("V", [4096, 32000, 131072])
@pytest.mark.parametrize("T", [0.02, 0.1, 0.2])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_k_ends_far_below_the_largest(V, T, dtype):
    """Low temperatures: the run that top_k leaves reaches below e^-31.9 of the largest weight, past the histogram's grid."""
    l, u = logits(4, V, V, dtype=dtype)
    for k, p, m in ((50, 1.0, 0.0), (50, 0.9, 0.0), (2000, 1.0, 0.0), (2000, 0.95, 0.0), (50, 1.0, 1e-6)):
        check(l, u, T, k, p, m)


@pytest.mark.parametrize("V", [20, 3000, 40000])
def test_what_stays_can_be_drawn_however_small_its_weight(V):
    """Kept by top_k with weights from 1e-13 down to the smallest that 64 bits hold, in front of the others and behind them; what 64 bits hold as 0 is not drawn."""
    for d in (30.0, 36.0, 40.0, 100.0, 700.0, 740.0, 800.0):
        l = torch.full((4, V), -2000.0)
        l[:, 7], l[:, 2], l[:, V - 2] = 0.0, -d, -d - 1
        u = torch.tensor([0.0, 1.0, 0.5, 1.0 - 2.0 ** -24])
        for T, k in ((1.0, 3), (1.0, 10), (0.5, 3)):
            got = mx.sample(l.cuda(), u.cuda(), T, k).tolist()
            at, w = su.kept(l[0].double().numpy(), T, k)
            live = at[w > 0]
            assert got == [live[0], live[-1], 7, 7], (d, T, k)


def test_what_stays_beside_thousands_can_be_drawn_however_small_its_weight():
    """The same where more than a list holds lies above: a segment of such tokens alone is the first."""
    V = 262144
    l, u = torch.full((3, V), -40.0), torch.tensor([0.0, 1.0, 0.25])
    l[:, 100000:105000] = torch.rand((3, 5000), generator=torch.Generator().manual_seed(1))
    l[:, :50] = l[:, V - 50:] = -30.9
    check(l, u, 1.0, 5100)
    assert mx.sample(l.cuda(), u.cuda(), 1.0, 5100).tolist()[:2] == [0, V - 1]


@pytest.mark.parametrize("n", [2, 3, 4, 10, 20, 50, 96, 512, 3000, 4096, 5000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_p_that_equal_logits_hold_exactly(n, dtype):
    """n equal logits, alone and beside masked ones: where top_p is a whole number of them, it keeps as many and no more."""
    g = torch.Generator().manual_seed(n)
    u = torch.tensor([0.0, 1.0, 0.9, 0.5, 0.999])
    for at in (0.0, 0.37, -2.6, 1000.0):
        for V, mask in ((n, 0.0), (n + 1000, -float("inf")), (n + 1000, torch.finfo(torch.float32).min), (n + 40000, -float("inf")), (n + 3000, at - 50.0)):
            l = torch.full((5, V), mask)
            for b in range(5):
                l[b, torch.randperm(V, generator=g)[:n]] = at
            l = l.to(dtype)
            for p in (0.5, 0.25, 0.75, 0.9):
                for T in (1.0, 0.7):
                    check(l, u, T, 0, p)
        l = torch.full((5, n), at, dtype=dtype)
        check(l, u, 1.0, n, 0.5)
        check(l, u, 1.0, max(n - 1, 1), 0.5)


@pytest.mark.parametrize("n", [2, 4, 20, 512])
@pytest.mark.parametrize("V", [600, 5000, 40000])
def test_hardly_any_weight_adds_nothing_to_top_ps_share(n, V):
    """Beside n equal logits top_k keeps some of 1e-26 of their weight, which 64 bits add to n without a trace."""
    g = torch.Generator().manual_seed(n)
    u = torch.tensor([0.0, 1.0, 0.9, 0.5, 0.999])
    l = torch.full((5, V), -100.0)
    for b in range(5):
        at = torch.randperm(V, generator=g)
        l[b, at[:n + 40]] = -60.0 - torch.rand(n + 40, generator=g)
        l[b, at[:n]] = 0.0
    for k in (n, n + 1, n + 40):
        for p in (0.5, 0.25, 0.75):
            check(l, u, 1.0, k, p)


@pytest.mark.parametrize("B,V", [(600, 1500), (300, 31478), (200, 100003)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_u_of_1_takes_the_last_that_stays_in_every_row(B, V, dtype):
    """Whatever the sums of a row and of its segments were rounded to; the last tokens' weights lie below the sums' last bits."""
    l, _ = logits(B, V, B, std=0.8, dtype=dtype)
    l = l.cuda()
    u = torch.ones(B, device="cuda")
    u[::2] = 7.0
    assert mx.sample(l, u, 0.2).tolist() == [V - 1] * B
    assert mx.sample(l, u, 0.2, min_p=1e-300).tolist() == [V - 1] * B  # (every weight is more)
    for k in (3, 700, 6000):
        got = mx.sample(l, u, 0.2, top_k=k).tolist()
        for b in range(4):
            at, w = su.kept(l[b].double().cpu().numpy(), 0.2, k)
            assert got[b] == at[w > 0][-1]
