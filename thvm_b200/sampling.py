"""The next ids from logits: temperature, top-k, top-p and min-p, drawn with
given random numbers (sm100_sample in include/thvm_sm100.h).

    sampler = Sampler("cuda")
    noise.exponential_()
    tok, logp = sampler(logits, noise, temperature=t, top_k=k, top_p=p, min_p=m)
"""
from __future__ import annotations

import ctypes

from . import _lib as L

_addressof = ctypes.addressof


class Sampler:
    def __init__(self, device="cuda"):
        import torch
        self.torch, self.lib = torch, L.lib()
        self.device = torch.device(device)
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        # what every call looks up
        self._index, self._raw_stream, self._sample = self.device.index, torch._C._cuda_getCurrentRawStream, self.lib.sm100_sample
        self._on = L.OnDevice(self._index)
        self._empty, self._f32, self._i32 = torch.empty, torch.float32, torch.int32
        self._rows = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16}

    def _setting(self, what: str, t, dtype, B: int):
        if t.dtype is not dtype or t.get_device() != self._index or t.numel() != B or not t.is_contiguous():
            raise ValueError(f"{what} must be {B} dense {dtype} values on {self.device}, got {t.dtype} {tuple(t.shape)}")
        return t.data_ptr()

    def __call__(self, logits, noise, temperature=None, top_k=None, top_p=None, min_p=None, tok=None, logp=None):
        """(tok int32 [B], logp f32 [B]) of logits [B, V] (f32 or bf16) and
        noise [B, V] (f32, from the unit exponential distribution); rows may be
        strided.  temperature, top_p, min_p f32 [B] and top_k int32 [B], or None;
        tok and logp to write into, or None for new ones."""
        setting, f32, i32 = self._setting, self._f32, self._i32
        B, V = logits.shape
        step, one = logits.stride()
        noise_step, noise_one = noise.stride()
        dtype = self._rows.get(logits.dtype)
        if dtype is None or logits.get_device() != self._index or (V > 1 and one != 1) or (B > 1 and step < V):
            raise ValueError(f"logits must be f32 or bf16 [B, V] on {self.device} with dense rows, got {logits.dtype}")
        if noise.dtype is not f32 or noise.shape != logits.shape or noise.get_device() != self._index or \
                (V > 1 and noise_one != 1) or (B > 1 and noise_step < V):
            raise ValueError(f"noise must be f32 {(B, V)} on {self.device} with dense rows")
        tok_ptr = logp_ptr = None
        if tok is None:
            tok = self._empty(B, dtype=i32, device=self.device)
            tok_ptr = tok.data_ptr()
        if logp is None:
            logp = self._empty(B, dtype=f32, device=self.device)
            logp_ptr = logp.data_ptr()
        a = L.Sm100SampleArgs(
            logits.data_ptr(), noise.data_ptr(),
            None if temperature is None else setting("temperature", temperature, f32, B),
            None if top_k is None else setting("top_k", top_k, i32, B),
            None if top_p is None else setting("top_p", top_p, f32, B),
            None if min_p is None else setting("min_p", min_p, f32, B),
            tok_ptr or setting("tok", tok, i32, B), logp_ptr or setting("logp", logp, f32, B),
            step if B > 1 else 0, noise_step if B > 1 else 0, B, V, dtype)
        rc = self._on(self._sample, _addressof(a), self._raw_stream(self._index))
        if rc:
            L.check(rc, "sample")
        return tok, logp
