"""A paged key / value cache and the operators over it (include/thvm_sm100.h):
append with the per-head norms and the position rotation of a decoder's
queries and keys, attention of the new rows over the cached tokens, and the
cached rows as values.

    cache = PagedCache.empty(n_seq=8, max_pages=64, n_pages=256, kv_heads=8, head_dim=128, bits=4)
    cache.table[s, i] = page of tokens i * page .. of sequence s
    q = cache.append(qkv, pos, seq, heads=32, g_q=g_q, g_k=g_k, cos=cos, sin=sin)
    o = cache.attend(q, kv_len)

PyTorch holds the memory; every call launches on torch's current stream of the
cache's GPU and returns without waiting.  Calls on one PagedCache share its scratch, so they
belong on one stream; a cache given the `scratch` of another shares that too
(the layers of a decoder need one between them).
"""
from __future__ import annotations

import ctypes
import weakref

from . import _lib as L

_addressof = ctypes.addressof
_caches: dict[int, weakref.WeakSet] = {}   # by GPU: who is to hear of its status word


class Scratch:
    """The attention's workspace.  A cache's first attention takes what its widest
    call needs, so no later one moves it.  No memory is given back, since a
    captured graph may hold its address: neither what a cache of wider heads
    outgrows, nor what a first attention under capture takes, which is zeroed by
    the graph's replays alone and so stays with the graph."""

    def __init__(self):
        self.held, self.ptr, self.nbytes = [], 0, 0

    def take(self, nbytes: int, device) -> tuple[int, int]:
        """(address, bytes) of a workspace of nbytes or more."""
        import torch
        if self.held and self.held[-1].device != device:
            raise ValueError(f"a scratch on {self.held[-1].device} for a cache on {device}")
        if nbytes > self.nbytes:
            self.held.append(torch.zeros(nbytes, dtype=torch.uint8, device=device))   # counters start at zero
            if torch.cuda.is_current_stream_capturing():
                return self.held[-1].data_ptr(), nbytes
            self.ptr, self.nbytes = self.held[-1].data_ptr(), nbytes
        return self.ptr, self.nbytes


class PagedCache:
    def __init__(self, pool, table, page: int, head_dim: int, bits: int, scratch: Scratch | None = None):
        """pool: uint8 [n_pages, kv_heads, block] (sm100_paged_block_bytes);
        table: int32 [n_seq, max_pages], both on the GPU and dense."""
        import torch
        self.torch, self.lib = torch, L.lib()
        block = int(self.lib.sm100_paged_block_bytes(page, head_dim, bits))
        if not block:
            raise ValueError(f"page {page} (16, 32, 64), head_dim {head_dim} (64, 128, 256), bits {bits} (4, 16)")
        if pool.dtype != torch.uint8 or pool.dim() != 3 or pool.shape[2] != block or not pool.is_contiguous() or \
                not pool.is_cuda:
            raise ValueError(f"pool must be uint8 [n_pages, kv_heads, {block}] on a GPU, got {pool.dtype} "
                             f"{tuple(pool.shape)} on {pool.device}")
        if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous() or table.device != pool.device:
            raise ValueError("table must be int32 [n_seq, max_pages] beside the pool")
        self.pool, self.table = pool, table
        self.page, self.head_dim, self.bits, self.kv_heads = page, head_dim, bits, pool.shape[1]
        self.scratch = scratch or Scratch()
        self.desc = L.Sm100PagedCache(pool.data_ptr(), table.data_ptr(), pool.shape[0], page, pool.shape[1], head_dim,
                                      bits, table.shape[0], table.shape[1])
        self._desc = ctypes.addressof(self.desc)
        self._raw_stream = torch._C._cuda_getCurrentRawStream
        self._device, self._index, self._n_seq = pool.device, pool.device.index, table.shape[0]
        # what every call looks up
        self._empty, self._bf16, self._f32, self._i32 = torch.empty, torch.bfloat16, torch.float32, torch.int32
        self._rows = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16}
        self._append, self._read, self._attention = (
            self.lib.sm100_paged_append, self.lib.sm100_paged_read, self.lib.sm100_paged_attention)
        self._on = L.OnDevice(self._index)
        self._bits = 0   # of the status word, taken by another cache's status()
        _caches.setdefault(self._index, weakref.WeakSet()).add(self)
        self._need: dict[tuple[int, int], int] = {}
        # 8 query columns a unit are the widest layout
        self._widest = int(self.lib.sm100_paged_attention_ws_bytes(self._desc, self.kv_heads, 8))

    @classmethod
    def empty(cls, n_seq: int, max_pages: int, n_pages: int, kv_heads: int, head_dim: int, page: int = 32,
              bits: int = 16, device="cuda", scratch: Scratch | None = None) -> "PagedCache":
        """A pool of zeros and a table of empty slots (-1)."""
        import torch
        block = int(L.lib().sm100_paged_block_bytes(page, head_dim, bits))
        pool = torch.zeros(n_pages, kv_heads, block, dtype=torch.uint8, device=device)
        table = torch.full((n_seq, max_pages), -1, dtype=torch.int32, device=device)
        return cls(pool, table, page, head_dim, bits, scratch)

    def _refuse(self, what: str, wanted: str, t):
        raise ValueError(f"{what} must be {wanted} beside the pool, got {t.dtype} {tuple(t.shape)}"
                         f"{'' if t.is_contiguous() else ' (strided)'} on {t.device}")

    def _dense(self, what: str, t, dtype, n: int):
        """The address of n dense values of dtype on the pool's GPU."""
        if t.dtype is not dtype or t.get_device() != self._index or t.numel() != n or not t.is_contiguous():
            self._refuse(what, f"{n} dense {dtype} values", t)
        return t.data_ptr()

    def append(self, qkv, pos, seq, heads: int, g_q=None, g_k=None, cos=None, sin=None, pairs: bool = False,
               eps: float = 1e-6, out=None):
        """Rows of a fused projection ([T, (heads + 2 kv_heads) * head_dim], f32
        or bf16, rows may be strided) at pos[t] of sequence seq[t]: norms and
        rotation of queries and keys, keys and values into the cache; returns
        the queries, bf16 [T, heads, head_dim] (sm100_paged_append)."""
        hd, dense, i32, f32 = self.head_dim, self._dense, self._i32, self._f32
        T, width = qkv.shape
        step, one = qkv.stride()
        dtype = self._rows.get(qkv.dtype)
        if dtype is None or width != (heads + 2 * self.kv_heads) * hd or qkv.get_device() != self._index or one != 1 or \
                (T > 1 and step < width):
            self._refuse("qkv", f"f32 or bf16 [T, {(heads + 2 * self.kv_heads) * hd}] with dense rows", qkv)
        if out is None:
            out = self._empty((T, heads, hd), dtype=self._bf16, device=self._device)
            out_ptr = out.data_ptr()
        else:
            if tuple(out.shape) != (T, heads, hd):
                self._refuse("out", f"{(T, heads, hd)}", out)
            out_ptr = dense("out", out, self._bf16, T * heads * hd)
        rot = n_pos = 0
        cos_ptr = sin_ptr = None
        if cos is not None or sin is not None:
            if cos is None or sin is None or cos.dim() != 2 or cos.shape != sin.shape:
                raise ValueError("cos and sin come together, f32 [n_pos, rot / 2]")
            n_pos, half = cos.shape
            rot = 2 * half
            cos_ptr, sin_ptr = dense("cos", cos, f32, n_pos * half), dense("sin", sin, f32, n_pos * half)
        a = L.Sm100PagedAppendArgs(
            qkv.data_ptr(), None if g_q is None else dense("g_q", g_q, f32, hd),
            None if g_k is None else dense("g_k", g_k, f32, hd), cos_ptr, sin_ptr, dense("pos", pos, i32, T),
            dense("seq", seq, i32, T), out_ptr, step if T > 1 else 0, T, heads, dtype, rot, n_pos, pairs, eps)
        rc = self._on(self._append, self._desc, _addressof(a), self._raw_stream(self._index))
        if rc:
            L.check(rc, "paged_append")
        return out

    def read(self, pos, seq):
        """(keys, values), bf16 [T, kv_heads, head_dim], of token pos[t] of
        sequence seq[t] (sm100_paged_read)."""
        T = pos.numel()
        both = self._empty((2, T, self.kv_heads, self.head_dim), dtype=self._bf16, device=self._device)
        k, v = both.unbind(0)
        rc = self._on(self._read, self._desc, self._dense("pos", pos, self._i32, T), self._dense("seq", seq, self._i32, T),
                      k.data_ptr(), v.data_ptr(), T, self._raw_stream(self._index))
        if rc:
            L.check(rc, "paged_read")
        return k, v

    def attend(self, q, kv_len, q_off=None, max_rows: int = 1, scale: float | None = None, out=None):
        """softmax(q k^T scale) v of the new rows q (bf16 [T, heads, head_dim]),
        bf16 [T, heads, head_dim].  kv_len [n_seq] counts the cached tokens, the
        new ones among them; sequence s has the rows q_off[s] .. q_off[s + 1] - 1
        (at most max_rows), without q_off row s alone; rows that no sequence has
        are not written (sm100_paged_attention)."""
        hd, dense, i32 = self.head_dim, self._dense, self._i32
        T, heads, d = q.shape
        step, head, one = q.stride()
        if q.dtype is not self._bf16 or d != hd or q.get_device() != self._index or one != 1 or \
                (heads > 1 and head != hd) or (T > 1 and step < heads * hd):
            self._refuse("q", f"bf16 [T, heads, {hd}] with dense rows", q)
        if out is None:
            out = self._empty((T, heads, hd), dtype=self._bf16, device=self._device)
            out_ptr = out.data_ptr()
        else:
            if out.shape != q.shape:
                self._refuse("out", f"{tuple(q.shape)}", out)
            out_ptr = dense("out", out, self._bf16, T * heads * hd)
        need = self._need.get((heads, max_rows))
        if need is None:
            need = int(self.lib.sm100_paged_attention_ws_bytes(self._desc, heads, max_rows))
            if not need:
                raise ValueError(f"heads {heads} (a multiple of {self.kv_heads}), max_rows {max_rows}")
            self._need[heads, max_rows] = need
        ws, ws_bytes = self.scratch.ptr, self.scratch.nbytes
        if ws_bytes < self._widest:
            ws, ws_bytes = self._on(self.scratch.take, self._widest, self._device)
        a = L.Sm100PagedAttnArgs(q.data_ptr(), dense("kv_len", kv_len, i32, self._n_seq),
                                 None if q_off is None else dense("q_off", q_off, i32, self._n_seq + 1), out_ptr,
                                 ws, ws_bytes, step if T > 1 else 0, T, heads, max_rows,
                                 hd ** -0.5 if scale is None else scale)
        rc = self._on(self._attention, self._desc, _addressof(a), self._raw_stream(self._index))
        if rc:
            L.check(rc, "paged_attention")
        return out

    def status(self) -> int:
        """Error bits of the paged calls on this GPU since this cache last asked
        (0: none); waits for the GPU.  The library has one word a GPU, which
        reading clears: every cache hears of every bit, its own calls' or not."""
        bits = int(self._on(self.lib.sm100_paged_status))
        for c in list(_caches[self._index]):
            c._bits |= bits
        bits, self._bits = self._bits, 0
        return bits
