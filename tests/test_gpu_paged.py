"""The paged key / value cache (thvm_b200.paged): append with per-head norms
and rotation, reading back, and attention, against the formulas in 64 bits.

Tolerances, from the roundings that the operators state:
  bf16 values     one rounding to 8 significant bits (2^-8 of the value, half a
                  unit) of an f32 result whose own error is a few 2^-24 of the
                  largest term (2^-18 of the head's largest value)
  4-bit values    half a step s, plus the rounding of s (15 s 2^-8) and of the
                  minimum (2^-8 of it) to bf16, plus the bf16 value read back
  attention       each weight enters the second product rounded to at least 8
                  bits: 2^-8 of sum p |v|; logits in f32 (2^-12 of it is ample);
                  one rounding of the output
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GROUP = 64


def _table(lengths, page, rng, max_pages=None, spare=3):
    """A shuffled page table for sequences of these lengths; returns (table, n_pages)."""
    import torch
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    ids = rng.permutation(total)
    t = np.full((len(lengths), max_pages or max(max(need), 1)), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = ids[at:at + n]
        at += n
    return torch.from_numpy(t).cuda(), total


def _cache(lengths, kv, hd, page, bits, rng, **kw):
    import torch
    from thvm_b200.paged import PagedCache
    table, total = _table(lengths, page, rng, **kw)
    c = PagedCache.empty(len(lengths), table.shape[1], total, kv, hd, page, bits)
    c.table.copy_(table)
    # rows that no call has written hold whatever was there: NaN patterns, which must never reach a result
    c.pool.copy_(torch.full_like(c.pool, 0xFF))
    return c


def _unpack(c):
    """The pool by its documented layout: values f64 [n_pages, kv, 2, page, hd], (scale, minimum) f64 in 4 bits."""
    import torch
    n, kv, _ = c.pool.shape
    page, hd = c.page, c.head_dim
    x = c.pool.view(n, kv, 2, -1)
    if c.bits == 16:
        return x.contiguous().view(torch.bfloat16).double().view(n, kv, 2, page, hd), None
    codes = x[..., :page * hd // 2].reshape(n, kv, 2, page, hd // 2)
    marks = x[..., page * hd // 2:].contiguous().view(torch.bfloat16).double().view(n, kv, 2, page, hd // GROUP, 2)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    s, m = (marks[..., i].repeat_interleave(GROUP, -1) for i in (0, 1))
    return m + code * s, marks


def _rows(c, pos, seq):
    """Values (and scales) of token pos[t] of sequence seq[t], [T, kv, 2, hd]."""
    v, marks = _unpack(c)
    at = c.table[seq.long(), (pos // c.page).long()].long()
    r = (pos % c.page).long()
    return v[at, :, :, r], None if marks is None else marks[at, :, :, r]


def _tables(n, rot):
    import torch
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
    return a.cos().float().cuda(), a.sin().float().cuda()


def _want(qkv, pos, H, kv, hd, g_q, g_k, cos, sin, pairs, eps):
    """q, k, v in f64 by the formulas."""
    import torch
    x = qkv.double().view(len(qkv), -1, hd)
    out = [x[:, :H], x[:, H:H + kv], x[:, H + kv:]]
    for i, g in ((0, g_q), (1, g_k)):
        if g is not None:
            out[i] = out[i] / torch.sqrt((out[i] ** 2).mean(-1, keepdim=True) + eps) * g.double()
        if cos is not None:
            half = cos.shape[1]
            j = torch.arange(half, device=x.device)
            a, b = (2 * j, 2 * j + 1) if pairs else (j, j + half)
            cc, ss = (t.double()[pos.long()][:, None] for t in (cos, sin))
            y = out[i].clone()
            y[..., a], y[..., b] = out[i][..., a] * cc - out[i][..., b] * ss, out[i][..., b] * cc + out[i][..., a] * ss
            out[i] = y
    return out


def _near(got, want, rel=2.0 ** -8):
    err = (got.double() - want).abs()
    tol = rel * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True)
    assert bool((err <= tol).all()), float((err - tol).max())


APPEND = [
    # heads, kv, hd, page, rows per sequence, starts, norm, rot, pairs, f32
    (1, 1, 64, 16, [1], [0], False, 0, False, True),
    (12, 12, 64, 16, [1], [15], True, 64, False, False),
    (4, 1, 64, 32, [5, 1, 33], [0, 31, 16], True, 32, True, True),
    (7, 7, 64, 16, [3, 18], [14, 1], False, 16, False, False),
    (8, 2, 128, 64, [1] * 9, [0, 63, 64, 65, 127, 128, 1, 2, 500], True, 128, False, True),
    (28, 4, 128, 32, [37, 64], [3, 0], True, 64, True, False),
    (5, 5, 128, 16, [129], [7], False, 128, True, True),
    (16, 2, 256, 16, [21, 2], [11, 30], True, 256, False, False),
    (3, 1, 256, 64, [70], [60], True, 48, False, True),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}p{c[3]}r{c[7]}")
def test_append_matches_the_formulas(case, bits):
    import torch
    H, kv, hd, page, new, start, norm, rot, pairs, f32 = case
    rng = np.random.default_rng(hd + sum(new) + bits)
    c = _cache([a + n for a, n in zip(start, new)], kv, hd, page, bits, rng)
    before = c.pool.clone()
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(start, new)]).int().cuda()
    seq = torch.arange(len(new)).repeat_interleave(torch.tensor(new)).int().cuda()
    T, width = len(pos), (H + 2 * kv) * hd
    order = torch.from_numpy(rng.permutation(T)).cuda()   # rows come in any order
    pos, seq = pos[order].contiguous(), seq[order].contiguous()
    x = torch.from_numpy(rng.standard_normal((T, width + 16)).astype(np.float32) * 2).cuda()
    x = (x if f32 else x.bfloat16())[:, 8:8 + width]      # strided rows
    g = [torch.from_numpy(rng.uniform(0.5, 1.5, hd).astype(np.float32)).cuda() for _ in range(2)] if norm else [None] * 2
    cos, sin = _tables(700, rot) if rot else (None, None)
    q = c.append(x, pos, seq, H, *g, cos, sin, pairs, eps=1e-5)
    wq, wk, wv = _want(x, pos, H, kv, hd, *g, cos, sin, pairs, 1e-5)
    _near(q, wq)
    got, marks = _rows(c, pos, seq)
    want = torch.stack((wk, wv), 2)
    if bits == 16:
        _near(got, want)
    else:
        y = want.unflatten(-1, (-1, GROUP))
        lo, hi = y.amin(-1), y.amax(-1)
        step = ((hi - lo) / 15).repeat_interleave(GROUP, -1)
        lo = lo.abs().repeat_interleave(GROUP, -1)
        assert bool(((got - want).abs() <= (0.5 + 15 * 2.0 ** -8) * step + 2.0 ** -8 * lo + 1e-5).all())
    k, v = c.read(pos, seq)
    assert torch.equal(k, got[:, :, 0].float().bfloat16()) and torch.equal(v, got[:, :, 1].float().bfloat16())
    # nothing but the rows' own bytes changed
    n, token = c.pool.shape[0], 2 * hd if bits == 16 else hd // 2
    touched = torch.zeros(n, page, dtype=torch.bool, device="cuda")
    touched[c.table[seq.long(), (pos // page).long()].long(), (pos % page).long()] = True
    a, b = (t.view(n, kv, 2, -1)[..., :page * token].view(n, kv, 2, page, token) for t in (before, c.pool))
    assert bool((a == b).all(-1).all(2).all(1)[~touched].all())
    assert c.status() == 0


def _sum_squares_in_order(x):
    """sum x^2 over the last dimension in f32, each step rounded: 256 dimensions first add their halves, 128 add up runs of 4
    neighbours, and then what there is adds its halves until one is left."""
    s = x * x
    if s.shape[-1] == 256:
        s = s[..., :128] + s[..., 128:]
    if s.shape[-1] == 128:
        r = s.unflatten(-1, (32, 4))
        s = ((r[..., 0] + r[..., 1]) + r[..., 2]) + r[..., 3]
    while s.shape[-1] > 1:
        half = s.shape[-1] // 2
        s = s[..., :half] + s[..., half:]
    return s


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("hd,H,kv,rot,pairs", [(64, 6, 3, 64, False), (64, 4, 2, 32, True), (128, 6, 3, 128, False),
                                               (128, 8, 2, 64, True), (256, 4, 2, 256, True), (256, 2, 1, 128, False)])
def test_append_is_the_stated_order_to_the_bit(hd, H, kv, rot, pairs, f32, bits):
    """Queries, codes, scales and minima equal, bit for bit, f32 arithmetic in the stated order with every step rounded on its
    own: a key near a tie takes the same code in any call shape."""
    import torch
    rng = np.random.default_rng(hd + H + f32)
    n, eps = 700, 1e-6
    c = _cache([n], kv, hd, 64, bits, rng)
    x = torch.from_numpy((2 * rng.standard_normal((n, (H + 2 * kv) * hd))).astype(np.float32)).cuda()
    x = x if f32 else x.bfloat16()
    g_q, g_k = (torch.from_numpy(rng.uniform(0.5, 1.5, hd).astype(np.float32)).cuda() for _ in range(2))
    cos, sin = _tables(n, rot)
    pos, seq = torch.arange(n, dtype=torch.int32).cuda(), torch.zeros(n, dtype=torch.int32).cuda()
    q = c.append(x, pos, seq, H, cos=cos, sin=sin, pairs=pairs, g_q=g_q, g_k=g_k, eps=eps)

    y = x.float().view(n, -1, hd)
    out = []
    for h, g in ((y[:, :H], g_q), (y[:, H:H + kv], g_k)):
        h = h * torch.rsqrt(_sum_squares_in_order(h) * (1.0 / hd) + eps) * g
        j = torch.arange(rot // 2, device="cuda")
        a, b = (2 * j, 2 * j + 1) if pairs else (j, j + rot // 2)
        u, w, cc, ss = h[..., a], h[..., b], cos[:, None], sin[:, None]
        r = h.clone()
        r[..., a], r[..., b] = u * cc - w * ss, w * cc + u * ss
        out.append(r)
    assert torch.equal(q.view(n, H, hd).view(torch.int16), out[0].bfloat16().view(torch.int16))
    kvs = torch.stack((out[1], y[:, H + kv:]), 2)   # [n, kv, 2, hd]
    page = c.table[0, (pos // 64).long()].long()
    pool = c.pool[page].view(n, kv, 2, -1)
    row = (pos % 64).long()
    if bits == 16:
        got = pool.view(n, kv, 2, 64, hd * 2)[torch.arange(n), :, :, row]
        assert torch.equal(got.contiguous().view(torch.int16), kvs.bfloat16().view(torch.int16))
        return
    codes = pool[..., :64 * hd // 2].reshape(n, kv, 2, 64, hd // 2)[torch.arange(n), :, :, row]
    marks = pool[..., 64 * hd // 2:].reshape(n, kv, 2, 64, hd // GROUP * 4)[torch.arange(n), :, :, row]
    grp = kvs.unflatten(-1, (-1, GROUP))
    mn, mx = grp.amin(-1), grp.amax(-1)
    third = torch.tensor(1.0, device="cuda") / 15
    scale, least = ((mx - mn) * third).bfloat16(), mn.bfloat16()
    assert torch.equal(marks.contiguous().view(torch.int16), torch.stack((scale, least), -1).flatten(-2).view(torch.int16))
    code = torch.round((grp - least.float()[..., None]) / scale.float()[..., None]).clamp(0, 15).to(torch.uint8).flatten(-2)
    assert torch.equal(codes, code[..., 0::2] | code[..., 1::2] << 4)


def test_append_skips_rows_outside_the_cache_and_keeps_nan_visible():
    import torch
    from thvm_b200 import _lib as L
    rng = np.random.default_rng(3)
    c = _cache([40, 20], 2, 64, 16, 4, rng, max_pages=4)
    before = c.pool.clone()
    pos = torch.tensor([5, 64, -1, 3, 48, 9], dtype=torch.int32).cuda()   # 64: past the table; 48: an empty slot
    seq = torch.tensor([0, 0, 0, 2, 0, -1], dtype=torch.int32).cuda()
    x = torch.randn(6, 6 * 64).cuda()
    x[0, 2 * 64 + 7] = float("nan")    # key head 0
    x[0, 4 * 64 + 9] = float("inf")    # value head 0
    q = c.append(x, pos, seq, 2)
    assert c.status() == L.DECODE_ERR_ARG
    assert c.status() == 0             # read once
    assert bool((q[1:] == 0).all()) and bool((q[0] != 0).any())
    k, v = c.read(pos[:1].contiguous(), seq[:1].contiguous())
    assert bool(torch.isnan(k[0, 0]).all()) and bool(torch.isnan(v[0, 0]).all())
    assert bool(torch.isfinite(k[0, 1]).all()) and bool(torch.isfinite(v[0, 1]).all())
    page = int(c.table[0, 0])
    same = (c.pool == before).all(-1).all(-1)
    assert bool(same[torch.arange(len(same)) != page].all())
    k, v = c.read(pos, seq)
    assert bool((k[1:] == 0).all()) and bool((v[1:] == 0).all())
    assert c.status() == L.DECODE_ERR_ARG
    # past the rotation tables
    cos, sin = _tables(5, 64)
    q = c.append(x[:1], pos[:1].contiguous(), seq[:1].contiguous(), 2, cos=cos, sin=sin)
    assert c.status() == L.DECODE_ERR_ARG and bool((q == 0).all())
    assert c.append(x[:0], pos[:0], seq[:0], 2).shape == (0, 2, 64)


def test_append_constant_groups_and_offsets():
    """A constant group reads as its (bf16) value; a far offset costs its bf16 rounding and no more."""
    import torch
    rng = np.random.default_rng(4)
    c = _cache([3], 1, 64, 16, 4, rng)
    x = torch.zeros(3, 3 * 64).cuda()
    x[0, 64:128] = 1.7
    x[1, 64:128] = 100 + torch.rand(64).cuda()
    x[2, 128:192] = 1e-30 * torch.randn(64).cuda()
    pos, seq = torch.arange(3).int().cuda(), torch.zeros(3).int().cuda()
    c.append(x, pos, seq, 1)
    k, v = c.read(pos, seq)
    assert bool((k[0] == torch.tensor(1.7).bfloat16().cuda()).all())
    assert float((k[1].float() - x[1, 64:128]).abs().max()) <= 0.5 + 0.5 / 15 + 0.25   # m and the value read, in bf16
    want = x[2, 128:192]
    assert float((v[2, 0].float() - want).abs().max()) <= (0.6 / 15 + 2.0 ** -7) * float(want.max() - want.min())
    assert c.status() == 0


ATTEND = [
    # heads, kv, hd, page, lengths, rows per sequence
    (1, 1, 64, 16, [1], [1]),
    (12, 12, 64, 16, [37], [1]),
    (25, 25, 64, 16, [1, 15, 16, 17, 300], [1] * 5),
    (8, 1, 64, 32, [64, 0, 63, 65, 1000], [1] * 5),
    (32, 8, 128, 64, [2500, 1, 129, 0, 64], [1] * 5),
    (28, 4, 128, 32, [5000], [1]),
    (16, 16, 128, 16, [130, 255], [1, 1]),
    (64, 8, 128, 64, [100, 7, 513], [4, 4, 2]),
    (6, 2, 128, 16, [40, 3, 200], [5, 7, 0]),      # more rows than tokens: the first see none
    (8, 8, 128, 16, [90, 33], [33, 33]),
    (40, 1, 64, 16, [77, 500], [1, 3]),            # 40 query heads on one key head
    (16, 2, 256, 16, [300, 17], [1, 1]),
    (5, 1, 256, 64, [200, 64], [9, 2]),
    (4, 4, 64, 32, [3] * 70, [1] * 70),
]


def _fill(c, lens, rng, spread=1.0):
    """Random keys and values through append, with a few strong key channels."""
    import torch
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    seq = torch.arange(len(lens)).repeat_interleave(torch.tensor(lens)).int().cuda()
    x = torch.from_numpy(rng.standard_normal((len(pos), 3 * c.kv_heads * c.head_dim)).astype(np.float32)).cuda() * spread
    x[:, c.kv_heads * c.head_dim::37] *= 3
    if len(pos):
        c.append(x, pos, seq, c.kv_heads)


def _attend_want(c, q, lens, rows, scale):
    """(out, sum p |v|) in f64 from the values that the cache holds."""
    import torch
    values, _ = _unpack(c)
    H, G = q.shape[1], q.shape[1] // c.kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    at = 0
    for s, (n, r) in enumerate(zip(lens, rows)):
        if n:
            pages = c.table[s, :-(-n // c.page)].long()
            x = values[pages].permute(0, 3, 2, 1, 4).reshape(-1, 2, c.kv_heads, c.head_dim)[:n]
            for i in range(r):
                m = n - r + i + 1
                if m <= 0:
                    continue
                qi = q[at + i].double().view(c.kv_heads, G, -1)
                p = torch.softmax(torch.einsum("kgd,nkd->kgn", qi, x[:m, 0]) * scale, -1)
                out[at + i] = torch.einsum("kgn,nkd->kgd", p, x[:m, 1]).reshape(H, -1)
                size[at + i] = torch.einsum("kgn,nkd->kgd", p, x[:m, 1].abs()).reshape(H, -1)
        at += r
    return out, size


def _check_attention(got, want, size):
    err = (got.double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * size + 1e-30
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}p{c[3]}n{len(c[4])}x{max(c[5])}")
def test_attention_matches_the_formula(case, bits):
    import torch
    H, kv, hd, page, lens, rows = case
    rng = np.random.default_rng(H + hd + sum(lens) + bits)
    c = _cache(lens, kv, hd, page, bits, rng)
    _fill(c, lens, rng)
    T = sum(rows)
    wide = torch.from_numpy(rng.standard_normal((T, H * hd + 24)).astype(np.float32)).cuda().bfloat16()
    q = wide[:, 8:8 + H * hd].unflatten(1, (H, hd))       # strided rows
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    ragged = rows != [1] * len(lens)
    q_off = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32).cuda()
    want, size = _attend_want(c, q, lens, rows, hd ** -0.5)
    for _ in range(2):   # the scratch is left ready for the next call
        got = c.attend(q, kv_len, q_off=q_off if ragged else None, max_rows=max(rows))
        _check_attention(got, want, size)
    if not ragged:       # the same rows by offsets, and with room for more rows than there are
        _check_attention(c.attend(q, kv_len, q_off=q_off, max_rows=3), want, size)
    assert c.status() == 0


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_of_strong_logits_and_small_values(bits):
    """Logits in the hundreds (a softmax that is one key), tiny and huge values."""
    import torch
    rng = np.random.default_rng(11)
    lens = [700, 65]
    for spread in (12.0, 1e-6, 1e4):
        c = _cache(lens, 2, 128, 32, bits, rng)
        _fill(c, lens, rng, spread)
        q = torch.from_numpy(rng.standard_normal((2, 8, 128)).astype(np.float32)).cuda().bfloat16()
        kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
        scale = 0.5 if spread > 1 else 1.0
        if spread == 1e4:
            q *= 1e-3
        want, size = _attend_want(c, q, lens, [1, 1], scale)
        got = c.attend(q, kv_len, scale=scale)
        err = (got.double() - want).abs()
        # logits of size z come with an f32 error of up to 2^-20 z, each weight with that much more
        z = float(12.0 * 128 * 0.5 * 9 if spread == 12.0 else 64)
        assert bool((err <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12 + 2.0 ** -20 * z) * size).all())
        assert c.status() == 0


def test_attention_leaves_out_pages_outside_the_pool():
    """A bad page id: its tokens are left out of the softmax, the status says so; a length past the table is cut."""
    import torch
    from thvm_b200 import _lib as L
    rng = np.random.default_rng(5)
    for bits in (4, 16):
        c = _cache([200, 48], 2, 64, 16, bits, rng)
        _fill(c, [200, 48], rng)
        q = torch.from_numpy(rng.standard_normal((2, 4, 64)).astype(np.float32)).cuda().bfloat16()
        kv_len = torch.tensor([200, 48], dtype=torch.int32).cuda()
        full, _ = _attend_want(c, q, [200, 48], [1, 1], 0.125)
        assert c.status() == 0
        c.table[0, 2:4] = torch.tensor([-1, 10 ** 6], dtype=torch.int32).cuda()
        got = c.attend(q, kv_len)
        assert c.status() == L.DECODE_ERR_ARG
        keep = torch.tensor([i for i in range(200) if not 32 <= i < 64]).cuda()
        values, _ = _unpack(c)
        pages = c.table[0, :13].long().clamp(0, c.pool.shape[0] - 1)
        x = values[pages].permute(0, 3, 2, 1, 4).reshape(-1, 2, 2, 64)[keep]
        p = torch.softmax(torch.einsum("kgd,nkd->kgn", q[0].double().view(2, 2, 64), x[:, 0]) * 0.125, -1)
        o = torch.einsum("kgn,nkd->kgd", p, x[:, 1]).reshape(4, 64)
        size = torch.einsum("kgn,nkd->kgd", p, x[:, 1].abs()).reshape(4, 64)
        _check_attention(got[0], o, size)
        _check_attention(got[1:], full[1:], torch.full_like(full[1:], 8.0))
        # every page of a row gone: zeros
        c.table[1, :3] = -1
        got = c.attend(q, kv_len)
        assert bool((got[1] == 0).all()) and c.status() == L.DECODE_ERR_ARG
        c.attend(q, torch.tensor([10 ** 6, 0], dtype=torch.int32).cuda())
        assert c.status() == L.DECODE_ERR_ARG


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("hd,H,kv", [(64, 4, 2), (128, 8, 1), (256, 4, 2)])
def test_later_tokens_that_are_not_finite_stay_out_of_earlier_rows(bits, hd, H, kv):
    """Five new rows a sequence; the keys and values of the last two tokens hold NaN and infinities: the rows before
    them are as without, the rows that see them are not finite."""
    import torch
    rng = np.random.default_rng(hd + bits)
    lens, rows = [70, 16, 5], [5, 5, 5]
    c = _cache(lens, kv, hd, 16, bits, rng)
    _fill(c, lens, rng)
    T = sum(rows)
    q = torch.from_numpy(rng.standard_normal((T, H, hd)).astype(np.float32)).cuda().bfloat16()
    want, size = _attend_want(c, q, lens, rows, hd ** -0.5)
    bad = torch.from_numpy(rng.standard_normal((6, 3 * kv * hd)).astype(np.float32)).cuda()
    bad[0::2] = float("nan")
    bad[1::2, ::3] = float("inf")
    pos = torch.tensor([x for n in lens for x in (n - 2, n - 1)], dtype=torch.int32).cuda()
    c.append(bad, pos, torch.tensor([0, 0, 1, 1, 2, 2], dtype=torch.int32).cuda(), kv)
    got = c.attend(q, torch.tensor(lens, dtype=torch.int32).cuda(),
                   q_off=torch.tensor([0, 5, 10, 15], dtype=torch.int32).cuda(), max_rows=5)
    early = torch.tensor([5 * s + r for s in range(3) for r in range(3)]).cuda()
    _check_attention(got[early], want[early], size[early])
    late = torch.tensor([5 * s + r for s in range(3) for r in (3, 4)]).cuda()
    assert bool(torch.isnan(got[late]).any(-1).all())


def test_attention_repeats_to_the_bit():
    """Units cut between CTAs are joined in one order, whichever CTA comes last."""
    import torch
    rng = np.random.default_rng(13)
    for bits, lens in ((4, [9000, 3]), (16, [3000, 700, 1])):
        c = _cache(lens, 2, 128, 64, bits, rng)
        _fill(c, lens, rng)
        q = torch.from_numpy(rng.standard_normal((len(lens), 8, 128)).astype(np.float32)).cuda().bfloat16()
        kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
        first = c.attend(q, kv_len)
        for _ in range(30):
            assert torch.equal(c.attend(q, kv_len), first)


def test_attention_offsets_past_two_gigabytes():
    """A pool of 5 GB whose used pages lie at its far end."""
    import torch
    from thvm_b200.paged import PagedCache
    rng = np.random.default_rng(6)
    kv, hd, page = 8, 128, 64
    n_pages = 5 * (1 << 30) // (kv * 4 * page * hd)
    c = PagedCache.empty(1, 4, n_pages, kv, hd, page, 16)
    c.table.copy_(torch.tensor([[n_pages - 1, n_pages // 2, n_pages - 2, 1]], dtype=torch.int32))
    pos, seq = torch.arange(200).int().cuda(), torch.zeros(200).int().cuda()
    x = torch.from_numpy(rng.standard_normal((200, 3 * kv * hd)).astype(np.float32)).cuda()
    c.append(x, pos, seq, kv)
    k, v = c.read(pos, seq)
    assert torch.equal(k, x[:, kv * hd:2 * kv * hd].bfloat16().view(200, kv, hd))
    assert torch.equal(v, x[:, 2 * kv * hd:].bfloat16().view(200, kv, hd))
    q = torch.from_numpy(rng.standard_normal((1, 16, hd)).astype(np.float32)).cuda().bfloat16()
    got = c.attend(q, torch.tensor([200], dtype=torch.int32).cuda())
    p = torch.softmax(torch.einsum("kgd,nkd->kgn", q[0].double().view(kv, 2, hd), k.double()) * hd ** -0.5, -1)
    _check_attention(got[0], torch.einsum("kgn,nkd->kgd", p, v.double()).reshape(16, hd),
                     torch.einsum("kgn,nkd->kgd", p, v.double().abs()).reshape(16, hd))
    assert c.status() == 0


def test_paged_calls_on_another_stream_and_in_a_graph():
    """append and attend captured into one graph on a side stream: replays follow the device positions."""
    import torch
    rng = np.random.default_rng(8)
    H, kv, hd, page = 8, 2, 128, 16
    c = _cache([100, 100], kv, hd, page, 4, rng)
    _fill(c, [60, 33], rng)
    kv_len = torch.tensor([61, 34], dtype=torch.int32).cuda()
    pos, seq = kv_len - 1, torch.arange(2).int().cuda()
    x = torch.from_numpy(rng.standard_normal((2, (H + 2 * kv) * hd)).astype(np.float32)).cuda()
    q, o = (torch.empty(2, H, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.append(x, pos, seq, H, out=q)
        c.attend(q, kv_len, out=o)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(x, pos, seq, H, out=q)
        c.attend(q, kv_len, out=o)
    for step in range(20):
        x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
        g.replay()
        want, size = _attend_want(c, q, [61 + step, 34 + step], [1, 1], hd ** -0.5)
        _check_attention(o, want, size)
        pos += 1
        kv_len += 1
    assert c.status() == 0


def test_refusals():
    import torch
    from thvm_b200 import _lib as L
    from thvm_b200.paged import PagedCache
    c = PagedCache.empty(2, 2, 4, 2, 64, 16, 16)
    i = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()
    x = torch.zeros(1, 6 * 64).cuda()
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        PagedCache.empty(2, 2, 4, 2, 96, 16, 16)
    with pytest.raises(ValueError):
        PagedCache(c.pool, c.table.long(), 16, 64, 16)
    with pytest.raises(ValueError):
        c.append(x[:, :64], i(0), i(0), 2)
    with pytest.raises(ValueError):
        c.append(x.half(), i(0), i(0), 2)
    with pytest.raises(ValueError):
        c.append(x, i(0, 1), i(0), 2)
    with pytest.raises(ValueError):
        c.append(x, i(0), i(0), 2, cos=torch.zeros(4, 32).cuda())
    with pytest.raises(ValueError):
        c.append(x.expand(3, -1), i(0, 1, 2), i(0, 0, 0), 2)
    with pytest.raises(L.Sm100Error):   # rot 24
        c.append(x, i(0), i(0), 2, cos=torch.zeros(4, 12).cuda(), sin=torch.zeros(4, 12).cuda())
    with pytest.raises(L.Sm100Error):   # rows that do not start on 16 bytes
        c.append(torch.zeros(2, 6 * 64 + 1).cuda()[:, 1:], i(0, 1), i(0, 0), 2)
    with pytest.raises(ValueError):
        c.attend(q.float(), i(1, 1))
    with pytest.raises(ValueError):
        c.attend(q, i(1))
    with pytest.raises(ValueError):
        c.attend(torch.zeros(2, 3, 64, dtype=torch.bfloat16, device="cuda"), i(1, 1))   # 3 heads on 2
    with pytest.raises(L.Sm100Error):
        c.attend(q[:1], i(1, 1))        # one row for two sequences, no offsets
    with pytest.raises(L.Sm100Error):
        c.attend(q, i(1, 1), scale=-0.5)
    assert c.attend(q[:0], i(0, 0), q_off=i(0, 0, 0)).shape == (0, 4, 64)
    small = L.Sm100PagedAttnArgs(q.data_ptr(), c.table.data_ptr(), None, q.data_ptr(), q.data_ptr(), 0, 0, 2, 4, 1, 1.0)
    assert L.lib().sm100_paged_attention(c._desc, ctypes.byref(small), None) == L.ERR_ARG
    assert b"scratch" in L.lib().sm100_last_error()
    assert c.status() == 0


def test_long_sums_of_codes_do_not_lean():
    """65536 tokens a sequence whose values cancel in pairs, equal weights (q = 0): the output is zero.

    A value is m + c s with s = 205 / 1024, m = -7.5 s rounded to bf16, codes c and 15 - c in turn: a pair's sum is
    2 m + 15 s, the rounding of m that is left.  The formula's output is m + 7.5 s, below 2^-9 of |v|'s mean.  Weights are
    1 and their products with s exact, so what is left is the f32 sums' rounding: of terms whose running sum stays
    within a tile's, 2^-17 of the mean |v| is ample; sums of 16384 offset codes that are rounded towards zero
    lean by 2^-13 of it.  Sequences share 16 pages, so that each warp's sums are long and the pool small."""
    import torch
    from thvm_b200.paged import PagedCache
    rng = np.random.default_rng(21)
    n_seq, kv, hd, page, n = 64, 8, 128, 64, 65536
    c = PagedCache.empty(n_seq, n // page, 16, kv, hd, page, 4)
    c.table.copy_(torch.from_numpy(rng.permuted(np.tile(np.arange(16, dtype=np.int32), (n_seq, n // page // 16)), axis=1)))
    x = c.pool.view(16, kv, 2, -1)
    code = torch.from_numpy(rng.integers(0, 16, (16, kv, 2, page // 2, hd)).astype(np.uint8)).cuda()
    code = torch.stack((code, 15 - code), 4).flatten(3, 4)   # tokens 2 i and 2 i + 1
    x[..., :page * hd // 2] = (code[..., 0::2] | code[..., 1::2] << 4).flatten(3)
    s = torch.tensor(205 / 1024).bfloat16()
    m = (-7.5 * s.float()).bfloat16()
    x[..., page * hd // 2:] = torch.stack((s, m)).cuda().view(torch.uint8).repeat(page * hd // GROUP)
    for H in (8, 64):   # both forms of the products: up to 4 query columns, and 8
        q = torch.zeros(n_seq, H, hd, dtype=torch.bfloat16, device="cuda")
        got = c.attend(q, torch.full((n_seq,), n, dtype=torch.int32).cuda()).double()
        want = float(m) + 7.5 * float(s)
        assert float((got - want).abs().max()) <= 2.0 ** -8 * abs(want) + 2.0 ** -17 * 4 * float(s)
    assert c.status() == 0


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("H", [1, 4, 8])
def test_weights_keep_sixteen_bits(bits, H):
    """Values +-a whose weighted sum nearly cancels, so that the output's own rounding is small and the weights' shows.

    A weight enters as two bf16 parts: off by at most 2^-8 of 2^-8 of it; its logit's f32 error (below 16) and 2^x add
    2^-18, the sums of 32 tokens 2^-19: 2^-15 of sum p |v| holds all.  Weights of 8 bits are off by 2^-9 of the root of
    sum p^2, some 2^-11."""
    import torch
    rng = np.random.default_rng(31 + bits + H)
    n, hd = 32, 64
    c = _cache([n], 1, hd, 16, bits, rng)
    x = torch.from_numpy(rng.standard_normal((n, 3 * hd)).astype(np.float32)).cuda()
    q = torch.from_numpy(rng.standard_normal((1, H, hd)).astype(np.float32)).cuda().bfloat16()
    q[:] = q[:, :1]
    pos, seq = torch.arange(n).int().cuda(), torch.zeros(n).int().cuda()
    c.append(x, pos, seq, 1)
    k = _unpack(c)[0][c.table[0, pos.long() // 16].long(), 0, 0, pos.long() % 16]
    p = torch.softmax(k @ q[0, 0].double() * hd ** -0.5, 0).cpu().numpy()
    sign, left = np.zeros(n), 0.0
    for i in np.argsort(-p):      # the largest first, each against what is left
        sign[i] = -1.0 if left > 0 else 1.0
        left += sign[i] * p[i]
    a = 7.5 * 0.25                # codes 0 and 15, scale 1 / 4
    along = torch.from_numpy(rng.choice([-1.0, 1.0], hd)).float()
    along[:2] = torch.tensor([1.0, -1.0])
    x[:, 2 * hd:] = (a * torch.from_numpy(sign).float()[:, None] * along).cuda()
    c.append(x, pos, seq, 1)
    want, size = _attend_want(c, q, [n], [1], hd ** -0.5)
    assert float(want.abs().max()) <= 0.02 * a   # they do cancel
    err = (c.attend(q, torch.tensor([n], dtype=torch.int32).cuda()).double() - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() + 2.0 ** -15 * size).all()), float((err / size).max())


@pytest.mark.parametrize("warm", [True, False])
def test_graph_stays_right_after_wider_eager_calls(warm):
    """A decode step in 4 bits (4 query columns a unit), eagerly first or not, is captured; then a part of a prompt and verify
    rows run eagerly, others take memory and fill it, and the graph is replayed between eager calls: the graph's results,
    theirs and the others' memory hold."""
    import torch
    rng = np.random.default_rng(41)
    H, kv, hd, page, n = 8, 2, 128, 64, 6000    # units cut between CTAs: parts and counters are used
    c = _cache([n], kv, hd, page, 4, rng)
    _fill(c, [n], rng)
    q = torch.from_numpy(rng.standard_normal((33, H, hd)).astype(np.float32)).cuda().bfloat16()
    kv_len = torch.tensor([n], dtype=torch.int32).cuda()
    o = torch.empty(1, H, hd, dtype=torch.bfloat16, device="cuda")
    if warm:
        c.attend(q[:1], kv_len, out=o)
    at = c.scratch.ptr
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.attend(q[:1], kv_len, out=o)
        c.attend(q[:1], kv_len, out=o)
    for rows in (33, 4):    # before the first replay
        want, size = _attend_want(c, q[:rows], [n], [rows], hd ** -0.5)
        got = c.attend(q[:rows], kv_len, q_off=torch.tensor([0, rows], dtype=torch.int32).cuda(), max_rows=rows)
        _check_attention(got, want, size)
    assert c.scratch.ptr == at or not warm
    others = [torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda") for _ in range(16)]
    want, size = _attend_want(c, q[:1], [n], [1], hd ** -0.5)
    for _ in range(3):
        o.zero_()
        g.replay()
        _check_attention(o, want, size)
        _check_attention(c.attend(q[:1], kv_len), want, size)
    assert all(bool((t == 7).all()) for t in others)
    assert c.status() == 0


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("hd,H,kv", [(64, 4, 2), (128, 16, 2), (256, 2, 2)])
def test_nan_scores_reach_their_rows(bits, hd, H, kv):
    """A key with a NaN, alone in its warp, tile or CTA or not: every row and head that sees it is NaN, the other key head's
    are the formula's.  A NaN in a query makes its head NaN, and no other."""
    import torch
    rng = np.random.default_rng(hd + bits)
    G = H // kv
    for n, at in ((1, 0), (17, 16), (33, 32), (65, 64), (129, 128), (200, 0), (6000, 0), (6000, 3011), (6000, 5999)):
        c = _cache([n], kv, hd, 16, bits, rng)
        _fill(c, [n], rng)
        q = torch.from_numpy(rng.standard_normal((1, H, hd)).astype(np.float32)).cuda().bfloat16()
        kv_len = torch.tensor([n], dtype=torch.int32).cuda()
        want, size = _attend_want(c, q, [n], [1], hd ** -0.5)
        broken = q.clone()
        broken[0, 1, 5] = float("nan")
        got = c.attend(broken, kv_len)
        assert bool(torch.isnan(got[0, 1]).all()), n
        rest = [h for h in range(H) if h != 1]
        _check_attention(got[:, rest], want[:, rest], size[:, rest])
        k, v = c.read(torch.tensor([at], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda())
        x = torch.cat((torch.zeros(kv * hd).cuda(), k.flatten().float(), v.flatten().float()))[None]
        x[0, kv * hd + 3] = float("nan")   # key head 0
        c.append(x, torch.tensor([at], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda(), kv)
        got = c.attend(q, kv_len)
        assert bool(torch.isnan(got[0, :G]).all()), (n, at)
        want, size = _attend_want(c, q, [n], [1], hd ** -0.5)   # (4 bits: the values were put in once more)
        _check_attention(got[:, G:], want[:, G:], size[:, G:])
        assert c.status() == 0


@pytest.mark.parametrize("bits", [16, 4])
def test_nan_scores_of_later_tokens_stay_out(bits):
    """Verify rows: the rows before a NaN key are the formula's, the others NaN, also where the key is a tile's first."""
    import torch
    rng = np.random.default_rng(bits)
    for n in (66, 130, 260):
        c = _cache([n], 1, 128, 64, bits, rng)
        _fill(c, [n], rng)
        q = torch.from_numpy(rng.standard_normal((4, 4, 128)).astype(np.float32)).cuda().bfloat16()
        want, size = _attend_want(c, q, [n], [4], 128 ** -0.5)
        x = torch.zeros(1, 3 * 128).cuda()
        x[0, 128] = float("nan")
        c.append(x, torch.tensor([n - 2], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda(), 1)
        got = c.attend(q, torch.tensor([n], dtype=torch.int32).cuda(), q_off=torch.tensor([0, 4], dtype=torch.int32).cuda(),
                       max_rows=4)
        _check_attention(got[:2], want[:2], size[:2])
        assert bool(torch.isnan(got[2:]).all())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("scale", [0.0, 1e-42, 1e-30])
def test_scale_zero_is_the_mean(bits, scale):
    """With a scale of nothing a row is the mean of the values that it sees, for lengths that end inside a tile, later tokens
    of other rows, idle sequences and units cut between CTAs."""
    import torch
    rng = np.random.default_rng(bits)
    for lens, rows in (([1, 17, 33, 0, 130, 64], [1] * 6), ([40, 3, 100], [5, 7, 4]), ([5001], [1]), ([90], [33])):
        c = _cache(lens, 2, 64, 16, bits, rng)
        _fill(c, lens, rng)
        q = torch.from_numpy(rng.standard_normal((sum(rows), 4, 64)).astype(np.float32)).cuda().bfloat16()
        q_off = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32).cuda()
        want, size = _attend_want(c, q, lens, rows, scale)
        got = c.attend(q, torch.tensor(lens, dtype=torch.int32).cuda(), q_off=q_off, max_rows=max(rows), scale=scale)
        assert bool(torch.isfinite(got).all())
        _check_attention(got, want, size)
        assert c.status() == 0


def test_status_of_one_cache_is_not_taken_by_another():
    import torch
    from thvm_b200 import _lib as L
    from thvm_b200.paged import PagedCache
    a, b = (PagedCache.empty(1, 2, 2, 1, 64) for _ in range(2))
    one = torch.zeros(1, dtype=torch.int32).cuda()
    assert a.status() == b.status() == 0
    a.read(one, one)                         # an empty slot of the table
    assert b.status() == L.DECODE_ERR_ARG    # the GPU's word: b hears of it too,
    assert a.status() == L.DECODE_ERR_ARG    # and a still does
    assert a.status() == b.status() == 0
    c = PagedCache.empty(1, 2, 2, 1, 64)
    b.read(one, one)
    assert a.status() == b.status() == c.status() == L.DECODE_ERR_ARG and c.status() == 0


@pytest.mark.parametrize("bits", [16, 4])
def test_rows_and_lengths_outside_set_the_status(bits):
    """Offsets that fall or leave q, and lengths below 0: that sequence has no rows (no keys), the others are right, rows of no
    sequence stay as they are, and the status says so."""
    import torch
    from thvm_b200 import _lib as L
    rng = np.random.default_rng(51)
    i = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()
    c = _cache([40, 20], 2, 64, 16, bits, rng)
    _fill(c, [40, 20], rng)
    q = torch.from_numpy(rng.standard_normal((4, 4, 64)).astype(np.float32)).cuda().bfloat16()
    want, size = _attend_want(c, q, [40, 20], [2, 2], 0.125)
    out = torch.empty_like(q)

    def run(kv_len, q_off):
        out.fill_(7.0)
        c.attend(q, kv_len, q_off=q_off, max_rows=2, out=out)
        return c.status()

    assert run(i(40, 20), i(0, 2, 4)) == 0
    _check_attention(out, want, size)
    for q_off in (i(0, 2, 99), i(0, 2, 1), i(0, 2, -1), i(0, 2, 5)):
        assert run(i(40, 20), q_off) == L.DECODE_ERR_ARG
        _check_attention(out[:2], want[:2], size[:2])
        assert bool((out[2:] == 7).all())
    assert run(i(40, 20), i(-2, 0, 2)) == L.DECODE_ERR_ARG and bool((out[2:] == 7).all())
    assert run(i(40, 20), i(9, 9, 9)) == L.DECODE_ERR_ARG and bool((out == 7).all())    # nothing to do, and past q
    assert run(i(40, 20), i(1, 1, 1)) == 0 and bool((out == 7).all())
    assert run(i(40, -3), i(0, 2, 4)) == L.DECODE_ERR_ARG
    _check_attention(out[:2], want[:2], size[:2])
    assert bool((out[2:] == 0).all())
    assert run(i(40, -3), i(0, 0, 0)) == L.DECODE_ERR_ARG
