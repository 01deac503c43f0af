"""A paged key / value cache and the operators over it (include/thvm_sm100.h):
append with the per-head norms and the position rotation of a decoder's
queries and keys, attention of the new rows over the cached tokens, and the
cached rows as values.

    cache = PagedCache.empty(n_seq=8, max_pages=64, n_pages=256, kv_heads=8, head_dim=128, bits=4)
    cache.table[s, i] = page of tokens i * page .. of sequence s
    q = cache.append(qkv, pos, seq, heads=32, g_q=g_q, g_k=g_k, cos=cos, sin=sin)
    o = cache.attend(q, kv_len)

PyTorch holds the memory; every call launches on torch's current stream and
returns without waiting.  Calls on one PagedCache share its scratch, so they
belong on one stream; a cache given the `scratch` of another shares that too
(the layers of a decoder need one between them).
"""
from __future__ import annotations

import ctypes

from . import _lib as L


class Scratch:
    """The attention's workspace: grows to what its calls need."""

    def __init__(self):
        self.buf, self.ptr, self.nbytes = None, 0, 0

    def take(self, nbytes: int, device):
        if nbytes > self.nbytes:
            import torch
            self.buf = torch.zeros(nbytes, dtype=torch.uint8, device=device)   # counters start at zero
            self.ptr, self.nbytes = self.buf.data_ptr(), nbytes
        return self


class PagedCache:
    def __init__(self, pool, table, page: int, head_dim: int, bits: int, scratch: Scratch | None = None):
        """pool: uint8 [n_pages, kv_heads, block] (sm100_paged_block_bytes);
        table: int32 [n_seq, max_pages], both on the GPU and dense."""
        import torch
        self.torch, self.lib = torch, L.lib()
        block = int(self.lib.sm100_paged_block_bytes(page, head_dim, bits))
        if not block:
            raise ValueError(f"page {page} (16, 32, 64), head_dim {head_dim} (64, 128, 256), bits {bits} (4, 16)")
        if pool.dtype != torch.uint8 or pool.dim() != 3 or pool.shape[2] != block or not pool.is_contiguous():
            raise ValueError(f"pool must be uint8 [n_pages, kv_heads, {block}], got {pool.dtype} {tuple(pool.shape)}")
        if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous() or table.device != pool.device:
            raise ValueError("table must be int32 [n_seq, max_pages] beside the pool")
        self.pool, self.table = pool, table
        self.page, self.head_dim, self.bits, self.kv_heads = page, head_dim, bits, pool.shape[1]
        self.scratch = scratch or Scratch()
        self.desc = L.Sm100PagedCache(pool.data_ptr(), table.data_ptr(), pool.shape[0], page, pool.shape[1], head_dim,
                                      bits, table.shape[0], table.shape[1])
        self._desc = ctypes.addressof(self.desc)
        self._raw_stream = torch._C._cuda_getCurrentRawStream
        self._index = pool.device.index
        self._need: dict[tuple[int, int], int] = {}

    @classmethod
    def empty(cls, n_seq: int, max_pages: int, n_pages: int, kv_heads: int, head_dim: int, page: int = 32,
              bits: int = 16, device="cuda", scratch: Scratch | None = None) -> "PagedCache":
        """A pool of zeros and a table of empty slots (-1)."""
        import torch
        block = int(L.lib().sm100_paged_block_bytes(page, head_dim, bits))
        pool = torch.zeros(n_pages, kv_heads, block, dtype=torch.uint8, device=device)
        table = torch.full((n_seq, max_pages), -1, dtype=torch.int32, device=device)
        return cls(pool, table, page, head_dim, bits, scratch)

    def _int32(self, what: str, t, n: int):
        if t.dtype != self.torch.int32 or t.device != self.pool.device or not t.is_contiguous() or t.numel() != n:
            raise ValueError(f"{what} must be {n} dense int32 values beside the pool, got {t.dtype} {tuple(t.shape)}")
        return t.data_ptr()

    def _float(self, what: str, t, shape: tuple):
        if t.dtype != self.torch.float32 or t.device != self.pool.device or not t.is_contiguous() or tuple(t.shape) != shape:
            raise ValueError(f"{what} must be f32 {shape} beside the pool, got {t.dtype} {tuple(t.shape)}")
        return t.data_ptr()

    def append(self, qkv, pos, seq, heads: int, g_q=None, g_k=None, cos=None, sin=None, pairs: bool = False,
               eps: float = 1e-6, out=None):
        """Rows of a fused projection ([T, (heads + 2 kv_heads) * head_dim], f32
        or bf16, rows may be strided) at pos[t] of sequence seq[t]: norms and
        rotation of queries and keys, keys and values into the cache; returns
        the queries, bf16 [T, heads, head_dim] (sm100_paged_append)."""
        torch, hd = self.torch, self.head_dim
        T, width = qkv.shape
        if qkv.dtype not in (torch.float32, torch.bfloat16) or width != (heads + 2 * self.kv_heads) * hd or \
                qkv.device != self.pool.device or qkv.stride(1) != 1 or (T > 1 and qkv.stride(0) < width):
            raise ValueError(f"qkv must be f32 or bf16 [T, {(heads + 2 * self.kv_heads) * hd}] beside the pool with "
                             f"dense rows, got {qkv.dtype} {tuple(qkv.shape)}")
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin come together")
        if out is None:
            out = torch.empty(T, heads, hd, dtype=torch.bfloat16, device=qkv.device)
        elif out.dtype != torch.bfloat16 or tuple(out.shape) != (T, heads, hd) or not out.is_contiguous() or \
                out.device != self.pool.device:
            raise ValueError(f"out must be dense bf16 {(T, heads, hd)}")
        a = L.Sm100PagedAppendArgs(
            qkv.data_ptr(), None if g_q is None else self._float("g_q", g_q, (hd,)),
            None if g_k is None else self._float("g_k", g_k, (hd,)),
            None if cos is None else self._float("cos", cos, (cos.shape[0], cos.shape[1])),
            None if sin is None else self._float("sin", sin, tuple(cos.shape)), self._int32("pos", pos, T),
            self._int32("seq", seq, T), out.data_ptr(), qkv.stride(0) if T > 1 else 0, T, heads,
            L.DT_F32 if qkv.dtype == torch.float32 else L.DT_BF16, 0 if cos is None else 2 * cos.shape[1],
            0 if cos is None else cos.shape[0], pairs, eps)
        L.check(self.lib.sm100_paged_append(self._desc, ctypes.addressof(a), self._raw_stream(self._index)),
                "paged_append")
        return out

    def read(self, pos, seq):
        """(keys, values), bf16 [T, kv_heads, head_dim], of token pos[t] of
        sequence seq[t] (sm100_paged_read)."""
        torch = self.torch
        T = pos.numel()
        k = torch.empty(T, self.kv_heads, self.head_dim, dtype=torch.bfloat16, device=self.pool.device)
        v = torch.empty_like(k)
        L.check(self.lib.sm100_paged_read(self._desc, self._int32("pos", pos, T), self._int32("seq", seq, T),
                                          k.data_ptr(), v.data_ptr(), T, self._raw_stream(self._index)), "paged_read")
        return k, v

    def attend(self, q, kv_len, q_off=None, max_rows: int = 1, scale: float | None = None, out=None):
        """softmax(q k^T scale) v of the new rows q (bf16 [T, heads, head_dim]),
        bf16 [T, heads, head_dim].  kv_len [n_seq] counts the cached tokens, the
        new ones among them; sequence s has the rows q_off[s] .. q_off[s + 1] - 1
        (at most max_rows), without q_off row s alone (sm100_paged_attention)."""
        torch, hd = self.torch, self.head_dim
        T, heads, d = q.shape
        if q.dtype != torch.bfloat16 or d != hd or q.device != self.pool.device or q.stride(2) != 1 or \
                (heads > 1 and q.stride(1) != hd) or (T > 1 and q.stride(0) < heads * hd):
            raise ValueError(f"q must be bf16 [T, heads, {hd}] beside the pool with dense rows, got {q.dtype} {tuple(q.shape)}")
        if out is None:
            out = torch.empty(T, heads, hd, dtype=torch.bfloat16, device=q.device)
        elif out.dtype != torch.bfloat16 or out.shape != q.shape or not out.is_contiguous() or \
                out.device != self.pool.device:
            raise ValueError(f"out must be dense bf16 {tuple(q.shape)}")
        n_seq = self.table.shape[0]
        need = self._need.get((heads, max_rows))
        if need is None:
            need = int(self.lib.sm100_paged_attention_ws_bytes(self._desc, heads, max_rows))
            if not need:
                raise ValueError(f"heads {heads} (a multiple of {self.kv_heads}), max_rows {max_rows}")
            self._need[heads, max_rows] = need
        ws = self.scratch.take(need, self.pool.device)
        a = L.Sm100PagedAttnArgs(q.data_ptr(), self._int32("kv_len", kv_len, n_seq),
                                 None if q_off is None else self._int32("q_off", q_off, n_seq + 1), out.data_ptr(),
                                 ws.ptr, ws.nbytes, q.stride(0) if T > 1 else 0, T, heads, max_rows,
                                 hd ** -0.5 if scale is None else scale)
        L.check(self.lib.sm100_paged_attention(self._desc, ctypes.addressof(a), self._raw_stream(self._index)),
                "paged_attention")
        return out

    def status(self) -> int:
        """Sticky error bits of the paged calls (0: none); waits for the GPU."""
        return int(self.lib.sm100_paged_status())
