"""The decoder over a paged cache (thvm_b200.paged_decoder) against a plain f64
evaluation of the same model with its stated roundings (bf16 matmul operands,
the cache's values).

Tolerance: the two differ where an f32 sum lands on the other side of a bf16
rounding boundary (one part in 2^8 of an operand's element, in few elements) and
in 4 bits where a key or value falls on the other side of a step's middle; a
logit is a sum over hundreds of such terms, so 2^-5 of the largest logit is
ample for either, and an error in a position, a page or a head is far above it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Plain:
    """One sequence, token by token."""

    def __init__(self, cfg, w):
        import torch
        self.cfg = cfg
        self.w = {k: torch.from_numpy(v).bfloat16().double() if v.ndim == 2 else torch.from_numpy(v).double()
                  for k, v in w.items()}
        self.kv = [([], []) for _ in range(cfg.n_layers)]
        self.pos = 0

    @staticmethod
    def _bf(x):
        return x.float().bfloat16().double()

    def _norm(self, x, g):
        return x / (x.pow(2).mean(-1, keepdim=True) + self.cfg.eps).sqrt() * g

    def _held(self, x):
        if self.cfg.bits == 16:
            return self._bf(x)
        import torch
        y = x.unflatten(-1, (-1, 64))
        lo = y.amin(-1, keepdim=True)
        s, lo = self._bf((y.amax(-1, keepdim=True) - lo) / 15), self._bf(lo)
        return (lo + s * torch.round((y - lo) / s).clamp(0, 15)).flatten(-2)

    def logits(self, tok):
        import torch
        c, w = self.cfg, self.w
        half = c.head_dim // 2
        a = self.pos * c.rope_base ** (-torch.arange(half, dtype=torch.float64) * 2 / c.head_dim)
        cos, sin = a.cos().float().double(), a.sin().float().double()
        rot = lambda x: torch.cat((x[:, :half] * cos - x[:, half:] * sin, x[:, half:] * cos + x[:, :half] * sin), -1)
        h = w["emb"][tok].clone()
        for i in range(c.n_layers):
            p = f"h.{i}."
            qkv = (w[p + "qkv"] @ self._bf(self._norm(h, w[p + "norm1"]))).view(-1, c.head_dim)
            q, k, v = qkv.split([c.heads, c.kv_heads, c.kv_heads])
            q, k = rot(self._norm(q, w[p + "g_q"])), rot(self._norm(k, w[p + "g_k"]))
            self.kv[i][0].append(self._held(k))
            self.kv[i][1].append(self._held(v))
            K, V = (torch.stack(t, 1) for t in self.kv[i])            # [kv, n, hd]
            q = self._bf(q).view(c.kv_heads, -1, c.head_dim)
            o = torch.softmax(q @ K.transpose(1, 2) * c.head_dim ** -0.5, -1) @ V
            h = h + w[p + "o"] @ self._bf(o.reshape(-1))
            gu = w[p + "gu"] @ self._bf(self._norm(h, w[p + "norm2"]))
            g, u = gu.split(c.hidden)
            h = h + w[p + "down"] @ self._bf(g * torch.sigmoid(g) * u)
        self.pos += 1
        return w["lm_head"] @ self._bf(self._norm(h, w["norm"]))


@pytest.mark.parametrize("bits,hd,heads,kv", [(4, 64, 8, 2), (16, 64, 6, 6), (4, 128, 4, 1), (16, 128, 8, 4)])
def test_decoder_matches_the_plain_model(bits, hd, heads, kv):
    import torch
    from thvm_b200.paged_decoder import PagedConfig, PagedDecoder, paged_weights
    cfg = PagedConfig(n_layers=2, dim=256, heads=heads, kv_heads=kv, head_dim=hd, hidden=384, vocab=500, max_ctx=128,
                      bits=bits)
    w = paged_weights(cfg, seed=3)
    dec = PagedDecoder(cfg, w, n_seq=4, n_pages=24)
    seen = []
    draw = dec._draw
    dec._draw = lambda logits, slots: (seen.append((list(slots), logits.double().cpu().clone())), draw(logits, slots))[1]
    rng = np.random.default_rng(1)
    plain, fed = {}, {}

    def check():
        slots, logits = seen.pop()
        for s, row in zip(slots, logits):
            for t in fed[s]:
                want = plain[s].logits(t)
            fed[s] = []
            assert float((row - want).abs().max()) <= 2.0 ** -5 * float(want.abs().max())

    def admit(n, **kw):
        prompt = rng.integers(0, cfg.vocab, n)
        s = dec.admit(prompt, **kw)
        plain[s], fed[s] = Plain(cfg, w), [int(v) for v in prompt]
        check()
        return s

    def step():
        before = dict(dec.next_id)
        ids = dec.step()
        for s in ids:
            fed[s].append(before[s])
        check()

    a = admit(45, temperature=0.7, top_k=20)         # two parts
    b = admit(3, temperature=0.0)
    for _ in range(4):
        step()
    c = admit(16, top_p=0.9)                         # ends on a page
    for _ in range(3):
        step()
    dec.release(a)
    d = admit(33, temperature=1.2, min_p=0.05)       # the pages and the slot of a
    assert d == a
    for _ in range(20):
        step()
    assert dec.status() == 0
    for s in (b, c, d):
        dec.release(s)
    assert sorted(dec.free_pages) == list(range(24)) and dec.step() == {}


def test_greedy_stream_does_not_depend_on_the_batch():
    """Greedy ids of a request alone and beside others: the same, row for row."""
    from thvm_b200.paged_decoder import PagedConfig, PagedDecoder, paged_weights
    cfg = PagedConfig(dim=256, hidden=256, vocab=300, max_ctx=64, bits=16)
    w = paged_weights(cfg, seed=5)
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, cfg.vocab, n) for n in (5, 40, 17)]

    def alone(p):
        dec = PagedDecoder(cfg, w, n_seq=1, n_pages=8)
        s = dec.admit(p, temperature=0.0)
        return [dec.next_id[s]] + [dec.step()[s] for _ in range(10)]

    dec = PagedDecoder(cfg, w, n_seq=3, n_pages=16)
    slots = [dec.admit(p, temperature=0.0) for p in prompts]
    out = [[dec.next_id[s]] for s in slots]
    for _ in range(10):
        ids = dec.step()
        for o, s in zip(out, slots):
            o.append(ids[s])
    assert out == [alone(p) for p in prompts]


def test_refusals():
    from thvm_b200.paged_decoder import PagedConfig, PagedDecoder, paged_weights
    cfg = PagedConfig(n_layers=1, dim=256, hidden=256, vocab=300, max_ctx=64)
    w = paged_weights(cfg)
    with pytest.raises(ValueError):
        PagedDecoder(cfg, w, n_seq=33, n_pages=4)
    dec = PagedDecoder(cfg, w, n_seq=2, n_pages=2)
    with pytest.raises(ValueError):
        dec.admit([])
    with pytest.raises(ValueError):
        dec.admit(range(64))
    with pytest.raises(RuntimeError):
        dec.admit(range(40))        # three pages of two
    s = dec.admit(range(32), temperature=0.0)
    with pytest.raises(RuntimeError):
        dec.step()                  # a third page
    dec.release(s)
    dec.admit([1, 2])
    dec.admit([3])
    with pytest.raises(RuntimeError):
        dec.admit([4])
    assert len(dec.step()) == 2 and dec.status() == 0


def test_a_request_that_fails_or_fills_its_cache_leaves_the_others():
    """A request that raises while it is admitted gives its slot and pages back; one that fills its cache is named, and the
    others go on once it is released."""
    from thvm_b200.paged_decoder import PagedConfig, PagedDecoder, paged_weights
    cfg = PagedConfig(n_layers=1, dim=256, hidden=256, vocab=300, max_ctx=64)
    w = paged_weights(cfg)
    dec = PagedDecoder(cfg, w, n_seq=2, n_pages=8)
    a = dec.admit([5, 6, 7], temperature=0.0)
    state = (sorted(dec.free_pages), list(dec.free_slots), dict(dec.length), dict(dec.next_id))
    for _ in range(3):   # more often than there are slots
        with pytest.raises((TypeError, ValueError)):
            dec.admit(range(20), top_k="many")
        assert (sorted(dec.free_pages), list(dec.free_slots), dict(dec.length), dict(dec.next_id)) == state
    b = dec.admit(range(63), temperature=0.0)
    assert set(dec.step()) == {a, b}
    before = (dict(dec.length), dict(dec.next_id))
    with pytest.raises(RuntimeError, match=rf"\[{b}\]"):
        dec.step()
    assert (dict(dec.length), dict(dec.next_id)) == before
    dec.release(b)

    alone = PagedDecoder(cfg, w, n_seq=1, n_pages=8)
    s = alone.admit([5, 6, 7], temperature=0.0)
    want = [alone.step()[s] for _ in range(5)]
    assert [before[1][a]] + [dec.step()[a] for _ in range(4)] == want
    assert dec.status() == 0
