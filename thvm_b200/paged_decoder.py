"""A decoder served over a paged cache: grouped-query attention with per-head
norms and position rotation, a gated feed-forward, ids by sampling; requests of
any length join and leave between passes, each holding the pages that its
tokens need.

A pass takes up to 32 rows (the skinny GEMM's batch): one new token of each
running request, or a part of a prompt.  Per layer

    x = bf16(rmsnorm(h)); qkv = x W_qkv^T
    q = norm, rotate and append (PagedCache.append); a = PagedCache.attend(q)
    h += a W_o^T;  x = bf16(rmsnorm(h)); h += bf16(silu(gate x) * up x) W_d^T

then logits = bf16(rmsnorm(h)) W_lm^T and the next ids by Sampler.

    dec = PagedDecoder(cfg, weights, n_seq=8, n_pages=256)
    s = dec.admit(prompt_ids, temperature=0.8, top_p=0.95)
    while ...: ids = dec.step()          # {s: next id}
    dec.release(s)

PyTorch provides memory, copies and the random numbers; the kernels of a pass
and of the draw are the library's.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import numpy as np

from . import _lib as L
from .paged import PagedCache, Scratch
from .sampling import Sampler

MAX_ROWS = 32


@dataclass(frozen=True)
class PagedConfig:
    n_layers: int = 2
    dim: int = 512
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    hidden: int = 1024
    vocab: int = 1000
    max_ctx: int = 1024
    page: int = 16
    bits: int = 4
    rope_base: float = 10000.0
    eps: float = 1e-6

    @property
    def qkv(self) -> int:
        return (self.heads + 2 * self.kv_heads) * self.head_dim


def paged_weights(cfg: PagedConfig, seed: int = 0, std: float = 0.05) -> dict[str, np.ndarray]:
    """Seeded synthetic weights: matrices N(0, std), norms around 1 (f32; the
    model keeps matrices and the embedding in bf16)."""
    rng = np.random.default_rng(seed)
    mat = lambda *s: rng.standard_normal(s, dtype=np.float32) * np.float32(std)
    vec = lambda n: rng.uniform(0.8, 1.2, n).astype(np.float32)
    w = {"emb": mat(cfg.vocab, cfg.dim) * np.float32(20)}
    for i in range(cfg.n_layers):
        p = f"h.{i}."
        w[p + "norm1"], w[p + "norm2"] = vec(cfg.dim), vec(cfg.dim)
        w[p + "g_q"], w[p + "g_k"] = vec(cfg.head_dim), vec(cfg.head_dim)
        w[p + "qkv"], w[p + "o"] = mat(cfg.qkv, cfg.dim), mat(cfg.dim, cfg.heads * cfg.head_dim)
        w[p + "gu"], w[p + "down"] = mat(2 * cfg.hidden, cfg.dim), mat(cfg.dim, cfg.hidden)
    w["norm"], w["lm_head"] = vec(cfg.dim), mat(cfg.vocab, cfg.dim)
    return w


class PagedDecoder:
    def __init__(self, cfg: PagedConfig, weights: dict[str, np.ndarray], n_seq: int, n_pages: int, seed: int = 0):
        import torch
        if not 1 <= n_seq <= MAX_ROWS:
            raise ValueError(f"n_seq {n_seq} (1 .. {MAX_ROWS}: a pass holds a row of every request)")
        self.torch, self.cfg, self.lib, self.n_seq = torch, cfg, L.lib(), n_seq
        dev = self.dev = torch.device("cuda", torch.cuda.current_device())
        put = lambda k, v: torch.from_numpy(v).to(dev, torch.bfloat16 if v.ndim == 2 else torch.float32)
        self.w = {k: put(k, v) for k, v in weights.items()}
        freq = cfg.rope_base ** (-torch.arange(cfg.head_dim // 2, dtype=torch.float64) * 2 / cfg.head_dim)
        angle = torch.arange(cfg.max_ctx, dtype=torch.float64)[:, None] * freq
        self.cos, self.sin = angle.cos().float().to(dev), angle.sin().float().to(dev)
        max_pages = -(-cfg.max_ctx // cfg.page)
        scratch = Scratch()   # the layers run one after the other
        self.cache = [PagedCache.empty(n_seq, max_pages, n_pages, cfg.kv_heads, cfg.head_dim, cfg.page, cfg.bits, dev, scratch)
                      for _ in range(cfg.n_layers)]
        self.table = self.cache[0].table
        for c in self.cache[1:]:   # a page has the same number in every layer
            c.table = self.table
            c.desc.table = self.table.data_ptr()
        self.sampler = Sampler(dev)
        self.noise_from = torch.Generator(device=dev)
        self.noise_from.manual_seed(seed)
        z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=dev)
        R, bf = MAX_ROWS, torch.bfloat16
        self.h, self.x, self.qkv = z(R, cfg.dim), z(R, cfg.dim, dt=bf), z(R, cfg.qkv)
        self.gu, self.act, self.logits = z(R, 2 * cfg.hidden), z(R, cfg.hidden, dt=bf), z(R, cfg.vocab)
        self.ws = z(int(self.lib.sm100_skinny_ws_bytes(R)) // 4)
        self.counters = z(max(cfg.qkv, 2 * cfg.hidden, cfg.vocab, cfg.dim) // 128 + 1, dt=torch.int32)
        self.free_pages = list(range(n_pages - 1, -1, -1))
        self.free_slots = list(range(n_seq - 1, -1, -1))
        self.pages: dict[int, list[int]] = {}      # slot -> its pages
        self.length: dict[int, int] = {}           # slot -> tokens in the cache
        self.next_id: dict[int, int] = {}          # slot -> the id to append next
        self.settings: dict[int, tuple] = {}       # slot -> (temperature, top_k, top_p, min_p)

    # -- one launcher per kernel ------------------------------------------------
    def _stream(self):
        return ctypes.c_void_p(self.torch.cuda.current_stream().cuda_stream)

    def _norm(self, x, g, y, T):
        L.check(self.lib.sm100_ds_rmsnorm(x.data_ptr(), g.data_ptr(), y.data_ptr(), T, self.cfg.dim, self.cfg.eps,
                                          self._stream()), "ds_rmsnorm")

    def _linear(self, x, w, y, T, residual=None):
        a = L.Sm100SkinnyArgs()
        a.x, a.w, a.y, a.ws, a.counters = (t.data_ptr() for t in (x, w, y, self.ws, self.counters))
        a.residual = residual.data_ptr() if residual is not None else None
        a.M, (a.N, a.K), a.flags = T, w.shape, L.SK_RESIDUAL if residual is not None else 0
        L.check(self.lib.sm100_skinny_bf16(ctypes.byref(a), self._stream()), "skinny")

    # -- a pass ---------------------------------------------------------------
    def _pass(self, rows: list[tuple[int, list[int]]]):
        """rows: (slot, ids) whose tokens follow the slot's cached ones, in
        rising slots, at most 32 ids in all.  Appends them; the logits of every
        row, f32 [T, vocab] (a view of the model's own buffer)."""
        torch, c = self.torch, self.cfg
        ids = [t for _, ts in rows for t in ts]
        T = len(ids)
        pos = [self.length[s] + i for s, ts in rows for i in range(len(ts))]
        seq = [s for s, ts in rows for _ in ts]
        for s, ts in rows:
            self.length[s] += len(ts)
            while len(self.pages[s]) * c.page < self.length[s]:
                if not self.free_pages:
                    raise RuntimeError("no free page")
                self.pages[s].append(self.free_pages.pop())
                self.table[s, len(self.pages[s]) - 1] = self.pages[s][-1]
        count = dict((s, len(ts)) for s, ts in rows)
        off = np.concatenate([[0], np.cumsum([count.get(s, 0) for s in range(self.n_seq)])])
        lens = [self.length.get(s, 0) for s in range(self.n_seq)]
        host = np.concatenate([ids, pos, seq, off, lens]).astype(np.int32)
        tok, pos, seq, off, lens = torch.from_numpy(host).to(self.dev).split([T, T, T, self.n_seq + 1, self.n_seq])
        st, w = self._stream, self.w
        L.check(self.lib.sm100_ds_embed(w["emb"].data_ptr(), tok.data_ptr(), self.h.data_ptr(), T, c.vocab, c.dim, st()),
                "ds_embed")
        for i in range(c.n_layers):
            p = f"h.{i}."
            self._norm(self.h, w[p + "norm1"], self.x, T)
            self._linear(self.x, w[p + "qkv"], self.qkv, T)
            q = self.cache[i].append(self.qkv[:T], pos, seq, c.heads, w[p + "g_q"], w[p + "g_k"], self.cos, self.sin, eps=c.eps)
            o = self.cache[i].attend(q, lens, q_off=off, max_rows=max(count.values()))
            self._linear(o, w[p + "o"], self.h, T, residual=self.h)
            self._norm(self.h, w[p + "norm2"], self.x, T)
            self._linear(self.x, w[p + "gu"], self.gu, T)
            L.check(self.lib.sm100_ds_silu_mul(self.gu.data_ptr(), self.act.data_ptr(), T, c.hidden, st()), "ds_silu_mul")
            self._linear(self.act, w[p + "down"], self.h, T, residual=self.h)
        self._norm(self.h, w["norm"], self.x, T)
        self._linear(self.x, w["lm_head"], self.logits, T)
        return self.logits[:T]

    def _draw(self, logits, slots):
        """The next id of each row (of slots' settings)."""
        torch = self.torch
        noise = torch.empty(logits.shape, device=self.dev).exponential_(generator=self.noise_from)
        t, k, p, m = zip(*(self.settings[s] for s in slots))
        f = lambda v, dt=torch.float32: torch.tensor(v, dtype=dt, device=self.dev)
        tok, _ = self.sampler(logits, noise, temperature=f(t), top_k=f(k, torch.int32), top_p=f(p), min_p=f(m))
        return [int(v) for v in tok.cpu()]

    # -- requests -----------------------------------------------------------------
    def admit(self, prompt, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0) -> int:
        """Runs a prompt (in parts of 32) and draws the request's first id; its slot."""
        prompt = [int(v) for v in prompt]
        if not prompt or len(prompt) >= self.cfg.max_ctx:
            raise ValueError(f"prompt of {len(prompt)} ids (cache of {self.cfg.max_ctx})")
        if not self.free_slots:
            raise RuntimeError("no free slot")
        if -(-len(prompt) // self.cfg.page) > len(self.free_pages):
            raise RuntimeError("no free page")
        s = self.free_slots.pop()
        self.pages[s], self.length[s], self.settings[s] = [], 0, (temperature, top_k, top_p, min_p)
        try:
            for at in range(0, len(prompt), MAX_ROWS):
                part = prompt[at:at + MAX_ROWS]
                logits = self._pass([(s, part)])
            self.next_id[s] = self._draw(logits[len(part) - 1:], [s])[0]
        except BaseException:   # the request was not admitted: its slot and pages are free again
            self.release(s)
            raise
        return s

    def step(self) -> dict[int, int]:
        """Appends every request's last id and draws the next: {slot: id}."""
        slots = sorted(self.next_id)
        full = [s for s in slots if self.length[s] + 1 > self.cfg.max_ctx]
        if full:   # nothing has changed: the others go on once these are released
            raise RuntimeError(f"requests {full} fill their cache: release them")
        need = sum(self.length[s] % self.cfg.page == 0 for s in slots)
        if need > len(self.free_pages):
            raise RuntimeError("no free page")
        if not slots:
            return {}
        logits = self._pass([(s, [self.next_id[s]]) for s in slots])
        self.next_id = dict(zip(slots, self._draw(logits, slots)))
        return dict(self.next_id)

    def release(self, s: int):
        """Ends a request: its pages and its slot are free."""
        self.free_pages += reversed(self.pages.pop(s))
        self.next_id.pop(s, None)
        del self.length[s], self.settings[s]
        self.free_slots.append(s)
        self.table[s] = -1

    def status(self) -> int:
        """Error bits of the pass's kernels on this GPU, other users' of them
        included (0: none); waits for the GPU."""
        return self.cache[0].status() | int(self.lib.sm100_skinny_status()) << 16
