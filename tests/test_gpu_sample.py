"""The next ids (thvm_b200.sampling, sm100_sample) against the definition in 64
bits: the kept set id by id, ties, settings at their ends, masked rows, the
probabilities of the draw."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _kept(row, T, k, p, m):
    """(the kept ids in order, their d) of one f64 row."""
    ids = np.nonzero(row > -np.inf)[0]
    order = ids[np.lexsort((ids, -row[ids]))]
    d = (row[order] - row[order[0]]) / T
    if k is not None and k > 0:
        order, d = order[:k], d[:k]
    w = np.exp(d)
    n = len(order)
    if p is not None and p < 1:
        before = np.cumsum(w) - w
        n = max(1, int((before < p * w.sum()).sum()))
    if m is not None:
        n = min(n, max(1, int((w >= m).sum())))
    return order[:n], d[:n]


def _sampler():
    from thvm_b200.sampling import Sampler
    return Sampler("cuda")


def _set(v, n, dtype):
    import torch
    return None if v is None else torch.full((n,), v, dtype=dtype).cuda()


def _run(logits, noise, T=1.0, k=None, p=None, m=None):
    import torch
    B = len(logits)
    return _sampler()(logits, noise, temperature=_set(T, B, torch.float32), top_k=_set(k, B, torch.int32),
                      top_p=_set(p, B, torch.float32), min_p=_set(m, B, torch.float32))


def _levels(V, rng, levels):
    """Logits on few distinct values (many ties), a bf16-exact grid."""
    return rng.integers(0, levels, V).astype(np.float32) * 0.25 - 4


ROWS = {
    "spread": lambda V, rng: (3 * rng.standard_normal(V)).astype(np.float32),
    "ties": lambda V, rng: _levels(V, rng, 40),
    "two values": lambda V, rng: _levels(V, rng, 2),
    "all equal": lambda V, rng: np.full(V, -1.5, np.float32),
    "steep": lambda V, rng: (80 * rng.standard_normal(V)).astype(np.float32),
    "masked": lambda V, rng: np.where(rng.random(V) < 0.9, -np.inf, rng.standard_normal(V)).astype(np.float32),
    "lowest": lambda V, rng: np.where(rng.random(V) < 0.9, np.finfo(np.float32).min, rng.standard_normal(V)).astype(np.float32),
    "around zero": lambda V, rng: (1e-3 * rng.standard_normal(V)).astype(np.float32) * (rng.random(V) < 0.7),
}

FILTERS = [dict(k=1), dict(k=7), dict(k=50), dict(k=1000), dict(p=0.3), dict(p=0.9), dict(p=0.999), dict(m=0.05),
           dict(k=40, p=0.8), dict(k=300, p=0.95, m=0.01), dict(T=0.3, p=0.7), dict(T=2.5, k=20, m=0.3), dict(p=0.0),
           dict(k=0, p=1.0, m=0.0), dict(m=2.0)]


@pytest.mark.parametrize("V", [1, 5, 33, 1000, 50257, 131072])
@pytest.mark.parametrize("kind", list(ROWS))
def test_kept_set(kind, V):
    """Each row of a call is the same logits with one id's random number nearly
    zero: that id is chosen exactly where it is kept.  Ids around the cut, the
    first, the last and some others; an id within 1e-5 of a weight cut (f32 sums
    of the forerunners) is not asked for."""
    import torch
    rng = np.random.default_rng(V + len(kind))
    row = ROWS[kind](V, rng)
    if not (row > -np.inf).any():
        row[V // 2] = 0.5
    x = torch.from_numpy(row).cuda()
    for f in FILTERS:
        a = dict(T=1.0, k=None, p=None, m=None) | f
        kept, _ = _kept(row.astype(np.float64), np.float64(np.float32(a["T"])), a["k"],
                        None if a["p"] is None else np.float64(np.float32(a["p"])),
                        None if a["m"] is None else np.float64(np.float32(a["m"])))
        order, d = _kept(row.astype(np.float64), np.float64(np.float32(a["T"])), None, None, None)
        n = len(kept)
        asked = sorted({i for i in [0, 1, 2, n - 3, n - 2, n - 1, n, n + 1, n + 2, n + 40, 2 * n, len(order) // 2,
                                    len(order) - 1] if 0 <= i < len(order)})
        w = np.exp(d)
        if a["p"] is not None and a["p"] < 1:
            tot = w[:a["k"]].sum() if a["k"] else w.sum()
            before = np.cumsum(w) - w
            asked = [i for i in asked if i == 0 or abs(before[i] / tot - np.float32(a["p"])) > 1e-5]
        if a["m"] is not None:
            asked = [i for i in asked if i == 0 or abs(w[i] / max(a["m"], 1e-30) - 1) > 1e-5]
        ids = order[asked]
        # an id far below the largest needs a random number whose logarithm reaches that far: only those are asked
        ok = d[asked] > -85
        ids, asked = ids[ok], np.array(asked)[ok]
        noise = torch.ones(len(ids), V, device="cuda")
        noise[torch.arange(len(ids)), torch.from_numpy(ids.copy()).cuda()] = 1e-38
        tok, logp = _run(x.expand(len(ids), V).contiguous(), noise, **a)
        got = tok.cpu().numpy()
        want = np.where(asked < n, ids, order[0])
        # where the asked id is left out, ids of equal score at the top decide for the lowest
        assert (got == want).all(), (kind, V, f, n, list(zip(asked, ids, got, want)))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 17), (7, 1001), (32, 50257), (64, 102400), (5, 131072), (2, 300001)])
def test_draws_match_the_definition(B, V, bf16):
    """Ids and log-probabilities of whole batches, each row with its own settings, rows strided.

    A logarithm of a sum of n weights in f32 is good to a few 2^-24 of itself and of the sum's terms: 1e-5
    absolute covers both.  Where the two best scores are within 1e-5 either may win."""
    import torch
    rng = np.random.default_rng(B * V + bf16)
    x = (2.5 * rng.standard_normal((B, V + 3))).astype(np.float32)
    x[rng.random(x.shape) < 0.2] = -np.inf
    x[:, 0] = 1.0
    noise = rng.exponential(size=(B, V + 5)).astype(np.float32)
    T = rng.uniform(0.4, 1.5, B).astype(np.float32)
    T[B // 2::5] = 0
    k = rng.choice([0, 1, 20, 64, 500, 5000, V], B).astype(np.int32)
    p = rng.choice([1.0, 0.95, 0.9, 0.5], B).astype(np.float32)
    m = rng.choice([0.0, 0.0, 0.02], B).astype(np.float32)
    xt = torch.from_numpy(x).cuda()
    xt = (xt.bfloat16() if bf16 else xt)[:, :V]
    d = lambda a: torch.from_numpy(a).cuda()
    tok, logp = _sampler()(xt, d(noise)[:, :V], temperature=d(T), top_k=d(k), top_p=d(p), min_p=d(m))
    tok, logp, x = tok.cpu().numpy(), logp.cpu().numpy(), xt.double().cpu().numpy()
    for b in range(B):
        if T[b] == 0:
            assert tok[b] == int(np.argmax(x[b])) and logp[b] == 0
            continue
        ids, dd = _kept(x[b], np.float64(T[b]), int(k[b]), np.float64(p[b]), np.float64(m[b]))
        score = dd - np.log(noise[b, ids].astype(np.float64))
        at = np.nonzero(ids == tok[b])[0]
        assert len(at) == 1, (b, tok[b])
        assert score[at[0]] >= score.max() - 1e-5
        assert abs(logp[b] - (dd[at[0]] - np.log(np.exp(dd).sum()))) <= 1e-5 * (1 + abs(dd[at[0]]))


def test_rows_with_nothing_nan_and_infinities():
    import torch
    inf, nan, big = math.inf, math.nan, float(np.finfo(np.float32).max)
    rows = [[-inf] * 6, [nan] * 6, [nan, 1, 2, -inf, 2, 0], [inf, 1, inf, 0, 0, 0], [-big] * 6, [big, -big, 0, 0, 0, 0],
            [-inf, -inf, -3, -inf, -inf, -inf]]
    x = torch.tensor(rows).cuda()
    ones = torch.ones_like(x)
    for T in (0.0, 1.0, 1e-3):
        for f in (dict(), dict(k=2), dict(p=0.5), dict(m=0.1), dict(k=3, p=0.9, m=0.2)):
            tok, logp = _run(x, ones, T=T, **f)
            assert tok.tolist() == [-1, -1, 2, 0, 0, 0, 2], (T, f, tok.tolist())
            assert logp[:2].tolist() == [-inf, -inf] and bool(torch.isfinite(logp[2:]).all())
    # random numbers of zero, infinity and NaN: zero wins, the others never
    noise = torch.tensor([[1.0, 0, 1, 0, 1, 1]]).cuda()
    x = torch.zeros(1, 6).cuda()
    assert _run(x, noise)[0].tolist() == [1]
    assert _run(x, torch.tensor([[inf, nan, inf, 5, nan, inf]]).cuda())[0].tolist() == [3]
    assert _run(x, torch.full((1, 6), nan).cuda())[0].tolist() == [0]
    # negative zero and zero are equal logits
    x = torch.tensor([[-0.0, 0.0, -0.0, 0.0]]).cuda()
    assert _run(x, torch.tensor([[1, 1e-30, 1, 1]]).cuda(), k=1)[0].tolist() == [0]
    assert _run(x, torch.tensor([[1, 1, 1e-30, 1e-20]]).cuda(), k=3)[0].tolist() == [2]


def test_many_rows_on_every_cluster_size_repeat_to_the_bit():
    """The same rows in batches of every launch shape, and again: ids and log-probabilities do not move."""
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(9)
    V = 40001
    x = 2 * torch.randn(200, V, device="cuda", generator=g)
    x = (x * 8).round() / 8   # many equal logits
    noise = torch.empty(200, V, device="cuda").exponential_(generator=g)
    f = dict(T=0.9, p=0.95)
    tok, logp = _run(x, noise, **f)
    for _ in range(3):
        again = _run(x, noise, **f)
        assert torch.equal(again[0], tok) and torch.equal(again[1], logp)
    for n in (1, 20, 100):
        t, lp = _run(x[:n], noise[:n], **f)
        assert torch.equal(t, tok[:n]) and float((lp - logp[:n]).abs().max()) <= 1e-5


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,V", [(34, 33333), (35, 33333), (70, 8200), (72, 33333), (100, 2049), (101, 50257), (148, 9001),
                                 (149, 33333)])
def test_draws_around_the_changes_of_launch_shape(B, V, bf16):
    """Ids and log-probabilities where another number of CTAs takes a row, and where a part is hardly worth one.

    The tolerances are those of whole batches above: the sums are over as many weights or fewer."""
    import torch
    rng = np.random.default_rng(B + V + bf16)
    x = (2.5 * rng.standard_normal((B, V))).astype(np.float32)
    x[rng.random(x.shape) < 0.2] = -np.inf
    x[:, V - 1] = 1.0
    noise = rng.exponential(size=(B, V)).astype(np.float32)
    T = rng.uniform(0.4, 1.5, B).astype(np.float32)
    k = rng.choice([0, 1, 20, 64, 500, 2000, V], B).astype(np.int32)
    p = rng.choice([1.0, 0.95, 0.9, 0.5], B).astype(np.float32)
    m = rng.choice([0.0, 0.0, 0.02], B).astype(np.float32)
    xt = torch.from_numpy(x).cuda()
    xt = xt.bfloat16() if bf16 else xt
    d = lambda a: torch.from_numpy(a).cuda()
    tok, logp = _sampler()(xt, d(noise), temperature=d(T), top_k=d(k), top_p=d(p), min_p=d(m))
    tok, logp, x = tok.cpu().numpy(), logp.cpu().numpy(), xt.double().cpu().numpy()
    for b in range(B):
        ids, dd = _kept(x[b], np.float64(T[b]), int(k[b]), np.float64(p[b]), np.float64(m[b]))
        score = dd - np.log(noise[b, ids].astype(np.float64))
        at = np.nonzero(ids == tok[b])[0]
        assert len(at) == 1, (b, tok[b])
        assert score[at[0]] >= score.max() - 1e-5
        assert abs(logp[b] - (dd[at[0]] - np.log(np.exp(dd).sum()))) <= 1e-5 * (1 + abs(dd[at[0]]))


@pytest.mark.parametrize("kind", list(ROWS))
def test_kept_set_in_pairs_of_ctas(kind):
    """A hundred copies of a row, one id's random number nearly zero in each: that id is chosen exactly where top-k keeps it."""
    import torch
    V, B = 30011, 100
    rng = np.random.default_rng(5)
    row = ROWS[kind](V, rng)
    if not (row > -np.inf).any():
        row[V // 2] = 0.5
    order, d = _kept(row.astype(np.float64), 1.0, None, None, None)
    # an id far below the largest needs a random number whose logarithm reaches that far: only those are asked
    order = order[d > -85]
    x = torch.from_numpy(row).cuda().expand(B, V).contiguous()
    for k in (1, 20, 700, 4000):
        asked = [min(max(0, min(k, len(order)) - B // 2 + i), len(order) - 1) for i in range(B)]
        noise = torch.ones(B, V, device="cuda")
        noise[torch.arange(B), torch.from_numpy(order[asked].copy()).cuda()] = 1e-38
        got = _run(x, noise, k=k)[0].cpu().numpy()
        assert (got == np.where(np.array(asked) < k, order[asked], order[0])).all(), (kind, k)


def test_probabilities_of_the_draw():
    """20000 draws over 12 ids with top-p: frequencies within 5 standard deviations of the kept ids' probabilities,
    none of the others."""
    import torch
    rng = np.random.default_rng(12)
    row = rng.standard_normal(12).astype(np.float32) * 1.5
    ids, d = _kept(row.astype(np.float64), 0.8, None, 0.85, None)
    prob = np.zeros(12)
    prob[ids] = np.exp(d) / np.exp(d).sum()
    n = 20000
    g = torch.Generator("cuda")
    g.manual_seed(1)
    noise = torch.empty(n, 12, device="cuda").exponential_(generator=g)
    tok, logp = _run(torch.from_numpy(row).cuda().expand(n, 12).contiguous(), noise, T=0.8, p=0.85)
    tok = tok.cpu().numpy()
    f = np.bincount(tok, minlength=12) / n
    assert (np.abs(f - prob) <= 5 * np.sqrt(prob * (1 - prob) / n)).all()
    np.testing.assert_allclose(logp.cpu().numpy(), np.log(prob[tok]), atol=1e-5)


def test_no_settings_same_as_neutral_ones_and_side_stream():
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(3)
    x = torch.randn(9, 4099, device="cuda", generator=g)
    noise = torch.empty(9, 4099, device="cuda").exponential_(generator=g)
    s = _sampler()
    a = s(x, noise)
    b = _run(x, noise, T=1.0, k=0, p=1.0, m=0.0)
    want = (x - noise.log()).argmax(-1)
    assert a[0].tolist() == b[0].tolist() == want.tolist() and torch.equal(a[1], b[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    tok = torch.zeros(9, dtype=torch.int32, device="cuda")
    with torch.cuda.stream(side):
        s(x, noise, tok=tok)
    side.synchronize()
    assert tok.tolist() == want.tolist()
    graph = torch.cuda.CUDAGraph()
    logp = torch.empty(9, device="cuda")
    with torch.cuda.graph(graph):
        s(x, noise, tok=tok, logp=logp)
    x.copy_(torch.randn(9, 4099, device="cuda", generator=g))
    graph.replay()
    assert tok.tolist() == (x - noise.log()).argmax(-1).tolist()


def test_refusals():
    import torch
    from thvm_b200 import _lib as L
    s = _sampler()
    x, n = torch.zeros(2, 8).cuda(), torch.ones(2, 8).cuda()
    with pytest.raises(ValueError):
        s(x.half(), n)
    with pytest.raises(ValueError):
        s(x, n[:, :7])
    with pytest.raises(ValueError):
        s(x[:1].expand(2, 8), n)
    with pytest.raises(ValueError):
        s(x.t().contiguous().t(), n)
    with pytest.raises(ValueError):
        s(x, n, temperature=torch.ones(3).cuda())
    with pytest.raises(ValueError):
        s(x, n, top_k=torch.ones(2).cuda())
    with pytest.raises(L.Sm100Error):
        s(x[:, :0], n[:, :0])
    tok, logp = s(x[:0], n[:0])
    assert tok.numel() == 0 and logp.numel() == 0


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [6, 1000, 40001])
def test_no_top_p_leaves_the_first_id(V, bf16):
    """top_p of 0, below it or NaN: the first id alone, whatever the other filters leave and however many ids tie with it;
    NaN in temperature or min_p does the same."""
    import torch
    nan = math.nan
    rng = np.random.default_rng(V)
    g = torch.Generator("cuda")
    g.manual_seed(V)
    x = torch.zeros(3, V)
    x[0, rng.permutation(V)[:max(1, V // 5)]] = 2.0   # many equal largest logits above equal ones
    x[1] = torch.from_numpy(_levels(V, rng, 40))
    x[2] = torch.from_numpy(rng.standard_normal(V).astype(np.float32))
    x = (x.bfloat16() if bf16 else x).cuda()
    want = [int(np.flatnonzero(r == r.max())[0]) for r in x.float().cpu().numpy()]
    for _ in range(4):
        noise = torch.empty(3, V, device="cuda").exponential_(generator=g)
        for f in (dict(p=0.0), dict(p=-1.0), dict(p=nan), dict(k=300, p=0.0), dict(k=300, p=-0.5), dict(k=300, p=nan),
                  dict(k=2, p=0.0), dict(k=700, p=0.0, m=0.01), dict(p=nan, m=0.5), dict(p=1e-45), dict(k=300, p=1e-45),
                  dict(m=nan), dict(k=300, m=nan), dict(T=nan), dict(T=nan, p=0.9)):
            tok, logp = _run(x, noise, **f)
            assert tok.tolist() == want and logp.tolist() == [0.0] * 3, (f, tok.tolist(), want)


def test_infinity_ties_with_the_largest_float():
    """+inf counts as the largest float: of the two the lower id comes first, within a thread's ids and between threads."""
    import torch
    big = float(np.finfo(np.float32).max)
    for V, a, b in ((6, 0, 5), (6, 2, 3), (5000, 1, 4000), (5000, 6, 2048 + 6), (60000, 3, 59999)):
        x = torch.zeros(2, V)
        x[0, a], x[0, b] = big, math.inf
        x[1, a], x[1, b] = math.inf, big
        noise = torch.ones(2, V).cuda()
        for f in (dict(T=0.0), dict(T=1.0), dict(k=1), dict(p=0.1), dict(k=2, p=0.4)):
            tok, logp = _run(x.cuda(), noise, **f)
            assert tok.tolist() == [a, a], (V, a, b, f, tok.tolist())


@pytest.mark.parametrize("V", [61, 3000, 40001])
@pytest.mark.parametrize("base", [1e4, -3e3, 700.0])
def test_min_p_at_low_temperatures_beside_large_logits(V, base):
    """Logits whose spacing in f32 is near the temperature: what min-p keeps is every id whose weight reaches it.

    l - l_max is exact here (neighbours of one size), so w is good to |d| 2^-23 and 2^-22; an id within 1e-5 of the bound is not
    asked for.  As above, the id with a random number of nearly nothing is chosen exactly where it is kept."""
    import torch
    rng = np.random.default_rng(V)
    step = float(np.spacing(np.float32(abs(base))))
    row = (np.float32(base) - np.float32(step) * rng.integers(0, 40, V).astype(np.float32)).astype(np.float32)
    for spread in (0.05, 0.31, 0.9, 1.7):
        T = np.float32(step / spread)
        order, d = _kept(row.astype(np.float64), np.float64(T), None, None, None)
        w = np.exp(d)
        before = np.cumsum(w) - w
        for m in (1e-6, 0.02, 0.3, 0.7):
            for extra in (dict(), dict(k=V - 1), dict(p=0.99), dict(p=0.9999)):
                p = np.float64(np.float32(extra.get("p", 1.0)))
                kept = (w >= np.float64(np.float32(m))) & (before < p * w.sum()) & (np.arange(V) < extra.get("k", V))
                sure = (np.abs(w / np.float64(np.float32(m)) - 1) > 1e-5) & (np.abs(before / w.sum() - p) > 1e-5)
                n = int(kept.sum())   # a beginning of the order
                ends = np.append(np.flatnonzero(np.diff(d) < 0), V - 1)   # the last id of each level
                asked = [i for i in sorted({0, 1, n // 2, n - 2, n - 1, n, n + 1, *ends.tolist()})
                         if 0 <= i < V and sure[i] and i < 4 * n + 50][:24]
                ids = order[asked]
                noise = torch.ones(len(ids), V, device="cuda")
                noise[torch.arange(len(ids)), torch.from_numpy(ids.copy()).cuda()] = 1e-38
                x = torch.from_numpy(row).cuda().expand(len(ids), V).contiguous()
                tok, _ = _run(x, noise, T=float(T), m=m, **extra)
                want = np.where(np.array(asked) < n, ids, order[0])
                assert (tok.cpu().numpy() == want).all(), (V, base, spread, m, extra, n, asked)
