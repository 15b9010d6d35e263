"""GPU: sample_tokens against the rules in float64, at every path and at their borders.

The kernel's masses are multiples of 2^-39 of the largest weight (half of that off each) from weights good to 1e-14, the
plain form's are float64: prefix masses differ by at most V (2^-40 + 1e-14 w).  A test's numbers u and settings are such
that the plain form's decision keeps that distance from every border it meets; where a border is exact on both sides
(equal logits, powers of two) it is met on purpose."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tilequant_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def plain(z, u, t, k, p, m):
    """(token, distance of the nearest border in units of the whole mass) of one row of float64 logits."""
    n = len(z)
    if not t > 0:
        nan = np.isnan(z)
        return (int(np.argmax(nan)) if nan.any() else int(np.argmax(z))), 1.0
    z = np.where(np.isnan(z), -np.inf, z)
    if np.isposinf(z).any():
        z = np.where(np.isposinf(z), 0.0, -np.inf)
    if np.isneginf(z).all():
        return 0, 1.0
    order = np.argsort(-z, kind="stable")
    with np.errstate(invalid="ignore"):
        w = np.exp((z[order] - z[order[0]]) / np.float64(t))
    w = np.where(np.isneginf(z[order]), 0.0, w)         # also where t is infinite
    kept = k if 0 < k < n else n
    cum = np.cumsum(w)
    slack = 1.0
    if p < 1:
        before = cum - w
        target = p * cum[kept - 1]
        kept_p = int((before[:kept] < target).sum())
        slack = min(slack, np.abs(cum[:kept] - target).min() / cum[-1])
        kept = min(kept, max(kept_p, 1))
    kept = max(1, min(kept, int((w >= m).sum())))
    total = cum[kept - 1]
    at = min(int((cum[:kept] <= u * total).sum()), kept - 1)
    if kept > 1:
        slack = min(slack, np.abs(cum[:kept - 1] - u * total).min() / cum[-1])
    return int(order[at]), slack


def check(logits, u, t=1.0, k=0, p=1.0, m=0.0, exact=False):
    """One launch over all rows; rows whose plain decision is nearer to a border than the masses are exact are counted,
    not compared (at most 1 in 20)."""
    rows, vocab = logits.shape
    col = lambda x, dt: (torch.full((rows,), x) if not isinstance(x, torch.Tensor) else x).to(dt)   # noqa: E731
    u, tt, kk, pp, mm = col(u, torch.float32), col(t, torch.float32), col(k, torch.int32), col(p, torch.float32), col(m, torch.float32)
    got = sample_tokens(logits.to(DEV), u.to(DEV), temperature=tt.to(DEV), top_k=kk.to(DEV), top_p=pp.to(DEV),
                        min_p=mm.to(DEV)).cpu()
    z = logits.double().numpy()
    near = 0
    for b in range(rows):
        want, slack = plain(z[b], float(u[b]), float(tt[b]), int(kk[b]), float(pp[b]), float(mm[b]))
        if not exact and slack <= vocab * (2.0 ** -40 + 1e-14):
            near += 1
            continue
        assert got[b] == want, (b, int(got[b]), want, slack, float(u[b]), float(tt[b]), int(kk[b]), float(pp[b]), float(mm[b]))
    assert near <= rows / 20
    return got


def logits_like(rows, vocab, dtype, seed, peak=8.0, bulk=2.2):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn((rows, vocab), generator=g) * bulk
    few = max(1, min(60, vocab // 4))
    at = torch.randint(0, vocab, (rows, few), generator=g)
    z.scatter_(1, at, torch.randn((rows, few), generator=g) * 2.5 + peak)
    return z.to(dtype), torch.rand((rows,), generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 1000, 8191, 32001])
@pytest.mark.parametrize("setting", [dict(), dict(k=1), dict(k=5), dict(k=50, p=0.9), dict(p=0.9), dict(p=0.5, m=0.02),
                                     dict(m=0.1), dict(k=600, p=0.95), dict(t=0.6, k=200, p=0.8, m=0.01), dict(t=0.0),
                                     dict(t=1.5, k=700)])
def test_settings(setting, vocab, dtype):
    z, u = logits_like(24, vocab, dtype, seed=vocab)
    check(z, u, **setting)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_vocabulary_and_mixed_rows(dtype):
    rows, vocab = 40, 128256
    z, u = logits_like(rows, vocab, dtype, seed=9)
    z[::5] *= 0.3                                     # flat rows: thousands of tokens in the nucleus
    z[1::10] *= 3                                     # sharp ones
    g = torch.Generator().manual_seed(1)
    pick = lambda xs: torch.tensor(xs)[torch.randint(0, len(xs), (rows,), generator=g)]   # noqa: E731
    check(z, u, t=pick([0.0, 0.5, 1.0, 1.7]), k=pick([0, 0, 1, 40, 500, 513, 4000, 200000]), p=pick([1.0, 0.99, 0.9, 0.4, 0.0]),
          m=pick([0.0, 0.0, 0.001, 0.2, 1.5]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_rank_by_index(dtype):
    """Equal logits have exact masses on both sides: borders are met exactly, in index order, past the list's size too."""
    for vocab in (8, 640, 8192, 20000, 65536):
        z = torch.zeros((6, vocab), dtype=dtype)
        u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.625])
        got = check(z, u, exact=True)
        assert got[:4].tolist() == [0, vocab // 4, vocab // 2, 3 * vocab // 4]
        check(z, u, p=0.5, exact=True)
        check(z, u, k=vocab // 2, exact=True)
        check(z, u, k=vocab // 4 + 1, p=0.25, exact=True)
        check(z, u, m=1.0, exact=True)
    z = torch.zeros((4, 30000), dtype=dtype)          # two values: 10000 tokens at each of 1 and 0, the rest out
    z[:, ::3], z[:, 2::3] = 1, -float("inf")
    u = torch.tensor([0.1, 0.6, 0.8, 0.99])
    check(z, u)
    check(z, u, k=15000)
    check(z, u, p=0.9)


@pytest.mark.parametrize("vocab", [500, 30000])
def test_masked_infinite_and_nan_logits(vocab):
    inf, nan = float("inf"), float("nan")
    z = torch.randn((9, vocab), generator=torch.Generator().manual_seed(2))
    z[0] = -inf                                       # nothing left: argmax's answer
    z[1, :-1] = -inf                                  # one left, the last
    z[2] = nan
    z[3, ::2] = nan
    z[4, 17] = z[4, 33] = z[4, 400] = inf             # equally likely, the others not at all
    z[5] = inf
    z[6] = -3.0e38
    z[7, :] = -0.0
    z[7, 250:] = 0.0
    z[8, 3], z[8, 4] = 3.0e38, -3.0e38
    u = torch.tensor([0.9, 0.3, 0.9, 0.4, 0.5, 0.7, 0.5, 0.5, 0.99])
    for s in (dict(), dict(k=3), dict(p=0.9), dict(m=0.5), dict(k=600), dict(p=0.3, k=100), dict(t=0.0)):
        for dt in (torch.float32, torch.bfloat16):
            got = check(z.to(dt), u, exact=True, **s)
            if s.get("t", 1.0) > 0:
                assert got[0] == 0 and got[1] == vocab - 1 and got[4] in (17, 33, 400)
    assert check(z, u, t=0.0)[2] == 0 and check(z, u, t=0.0)[3] == 0


@pytest.mark.parametrize("vocab", [3001, 40000])
def test_odd_settings(vocab):
    z, u = logits_like(7, vocab, torch.float32, seed=3)
    z[:, 5::7] = -float("inf")
    for s in (dict(t=float("inf")), dict(t=1e-30), dict(t=float("nan")), dict(t=-1.0), dict(p=0.0), dict(p=-1.0), dict(p=2.0),
              dict(m=1.0), dict(m=2.0), dict(k=-5), dict(k=2 ** 31 - 1), dict(k=3001), dict(k=3000), dict(t=1e30),
              dict(k=0, p=1e-9), dict(m=1e-30), dict(m=1e-40)):
        check(z, u, **s)
    check(z, torch.tensor([0.0, 1.0, 1.5, 0.0, 1.0, 1.0, 0.0]), exact=True, p=0.9)     # numbers outside [0, 1)
    check(z, torch.tensor([0.0, 1.0, 1.5, 0.0, 1.0, 1.0, 0.0]), exact=True, k=20)


@pytest.mark.parametrize("setting", [dict(), dict(temperature=0.0), dict(temperature=float("nan")), dict(top_k=1), dict(top_k=40),
                                     dict(top_k=512), dict(top_k=513), dict(top_k=10 ** 12), dict(top_k=-3), dict(min_p=0.05),
                                     dict(top_p=0.8), dict(top_p=0.8, min_p=0.01), dict(top_k=300, top_p=0.9, min_p=0.02),
                                     dict(temperature=0.0, top_k=40, top_p=0.5)])
@pytest.mark.parametrize("vocab", [400, 40000])
def test_numbers_for_all_rows_equal_vectors(vocab, setting):
    z, u = logits_like(9, vocab, torch.bfloat16, seed=vocab + 1)
    z[3], z[4, ::2], z[5, 7] = -float("inf"), float("nan"), float("inf")
    z, u = z.to(DEV), u.to(DEV)
    types = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    vectors = {n: torch.full((9,), min(v, 2 ** 31 - 1) if n == "top_k" else v, dtype=types[n], device=DEV)
               for n, v in setting.items()}
    assert torch.equal(sample_tokens(z, u, **setting), sample_tokens(z, u, **vectors))


@pytest.mark.parametrize("vocab", [50, 30000])
def test_numbers_far_outside_give_the_ends(vocab):
    """Below 0: the first kept token, 1 and above: the last, however large."""
    z, _ = logits_like(8, vocab, torch.float32, seed=3)
    z = z[:1].expand(8, -1).contiguous()
    u = torch.tensor([0.0, -1.0, -float("inf"), float("nan"), 1.0, 1e9, 3e38, float("inf")])
    for setting in (dict(top_k=20), dict(top_p=0.7), dict()):
        got = sample_tokens(z.to(DEV), u.to(DEV), **setting).tolist()
        assert got[:4] == got[:1] * 4 and got[4:] == got[4:5] * 4 and got[0] == int(z[0].argmax())


def test_strides_and_alignment():
    """Views with odd row strides and odd first elements, and an output that the caller holds."""
    base = torch.randn((6, 1111), generator=torch.Generator().manual_seed(4)) * 3
    u = torch.rand((6,), generator=torch.Generator().manual_seed(5)).to(DEV)
    for dt in (torch.bfloat16, torch.float32):
        whole = base.to(dt).to(DEV)
        for lo, hi in ((0, 1111), (1, 1111), (3, 1000), (5, 6), (7, 900)):
            for s in (dict(top_k=9), dict(top_p=0.8)):
                want = sample_tokens(whole[:, lo:hi].contiguous(), u, **s)
                out = torch.full((6,), -1, dtype=torch.int64, device=DEV)
                assert sample_tokens(whole[:, lo:hi], u, out=out, **s) is out and torch.equal(out, want)


def test_draws_follow_the_distribution():
    """20000 numbers spread evenly over [0, 1) on one row: every token's count is its probability to one draw."""
    rows, vocab = 20000, 100
    z = (torch.randn((1, vocab), generator=torch.Generator().manual_seed(6)) * 2).to(torch.bfloat16)
    u = (torch.arange(rows) + 0.5) / rows
    got = sample_tokens(z.expand(rows, vocab).contiguous().to(DEV), u.to(DEV), temperature=0.8, top_p=0.97).cpu()
    w = torch.exp(z[0].double() / 0.8)
    w, order = torch.sort(w, descending=True, stable=True)
    kept = int((w.cumsum(0) - w < 0.97 * w.sum()).sum())
    p = torch.zeros(vocab, dtype=torch.float64)
    p[order[:kept]] = w[:kept] / w[:kept].sum()
    assert ((torch.bincount(got, minlength=vocab) - p * rows).abs() <= 1 + 1e-6 * rows).all()


def test_captured_and_replayed():
    z, _ = logits_like(5, 9000, torch.bfloat16, seed=7)
    z, u = z.to(DEV), torch.zeros(5, device=DEV)
    t, k = torch.ones(5, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV)
    sample_tokens(z, u, temperature=t, top_k=k, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_tokens(z, u, temperature=t, top_k=k, top_p=0.9)
    for i in range(6):
        u.copy_(torch.rand((5,), generator=torch.Generator().manual_seed(i)))
        t.fill_(0.5 + 0.2 * i)
        k.fill_([0, 1, 20, 700, 0, 3][i])
        graph.replay()
        assert torch.equal(got, sample_tokens(z, u, temperature=t, top_k=k, top_p=0.9))


def test_two_streams_at_once():
    z, u = logits_like(64, 20000, torch.bfloat16, seed=8)
    z, u = z.to(DEV), u.to(DEV)
    want = [sample_tokens(z, u, top_p=0.9), sample_tokens(z, u, top_k=30)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for s, kw in zip(streams, (dict(top_p=0.9), dict(top_k=30))):
            with torch.cuda.stream(s):
                got.append(sample_tokens(z, u, **kw))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_greedy_rows_equal_the_decoders_step():
    """Temperature 0 is torch.argmax, NaN first, as the decoder's greedy step takes it."""
    z, u = logits_like(16, 4001, torch.bfloat16, seed=10)
    z[3, 700] = z[3, 90] = float("nan")
    z[4] = 1.0
    z = z.to(DEV)
    assert torch.equal(sample_tokens(z, u.to(DEV), temperature=0.0), z.argmax(dim=-1))


def test_refusals_on_the_device():
    z, u = torch.zeros((3, 50), device=DEV), torch.zeros(3, device=DEV)
    for bad in (lambda: sample_tokens(z[0], u), lambda: sample_tokens(z.double(), u), lambda: sample_tokens(z.t(), u),
                lambda: sample_tokens(z, u[:2]), lambda: sample_tokens(z, u.double()),
                lambda: sample_tokens(z, u, top_k=torch.zeros(3, device=DEV)),
                lambda: sample_tokens(z, u, top_p=torch.zeros(2, device=DEV)),
                lambda: sample_tokens(z, u, out=torch.zeros(3, device=DEV)),
                lambda: sample_tokens(z[:1].expand(3, 50), u),
                lambda: sample_tokens(torch.zeros((1, 500001), device=DEV), u[:1])):
        with pytest.raises(ValueError):
            bad()
    assert sample_tokens(z[:0], u[:0]).shape == (0,)
