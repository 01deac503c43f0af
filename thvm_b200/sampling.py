"""The next ids from logits: temperature, top-k, top-p and min-p, drawn with
given random numbers (sm100_sample in include/thvm_sm100.h).

    sampler = Sampler("cuda")
    noise.exponential_()
    tok, logp = sampler(logits, noise, temperature=t, top_k=k, top_p=p, min_p=m)
"""
from __future__ import annotations

import ctypes

from . import _lib as L


class Sampler:
    def __init__(self, device="cuda"):
        import torch
        self.torch, self.lib = torch, L.lib()
        self.device = torch.device(device)
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._raw_stream = torch._C._cuda_getCurrentRawStream

    def _setting(self, what: str, t, dtype, B: int):
        if t is None:
            return None
        if t.dtype != dtype or t.numel() != B or not t.is_contiguous() or t.device != self.device:
            raise ValueError(f"{what} must be {B} dense {dtype} values on {self.device}, got {t.dtype} {tuple(t.shape)}")
        return t.data_ptr()

    def __call__(self, logits, noise, temperature=None, top_k=None, top_p=None, min_p=None, tok=None, logp=None):
        """(tok int32 [B], logp f32 [B]) of logits [B, V] (f32 or bf16) and
        noise [B, V] (f32, from the unit exponential distribution); rows may be
        strided.  temperature, top_p, min_p f32 [B] and top_k int32 [B], or None;
        tok and logp to write into, or None for new ones."""
        torch = self.torch
        B, V = logits.shape
        if logits.dtype not in (torch.float32, torch.bfloat16) or logits.device != self.device or \
                (V > 1 and logits.stride(1) != 1) or (B > 1 and logits.stride(0) < V):
            raise ValueError(f"logits must be f32 or bf16 [B, V] on {self.device} with dense rows, got {logits.dtype}")
        if noise.dtype != torch.float32 or noise.shape != logits.shape or noise.device != self.device or \
                (V > 1 and noise.stride(1) != 1) or (B > 1 and noise.stride(0) < V):
            raise ValueError(f"noise must be f32 {(B, V)} on {self.device} with dense rows")
        if tok is None:
            tok = torch.empty(B, dtype=torch.int32, device=self.device)
        if logp is None:
            logp = torch.empty(B, dtype=torch.float32, device=self.device)
        a = L.Sm100SampleArgs(logits.data_ptr(), noise.data_ptr(),
                              self._setting("temperature", temperature, torch.float32, B),
                              self._setting("top_k", top_k, torch.int32, B),
                              self._setting("top_p", top_p, torch.float32, B),
                              self._setting("min_p", min_p, torch.float32, B),
                              self._setting("tok", tok, torch.int32, B), self._setting("logp", logp, torch.float32, B),
                              logits.stride(0) if B > 1 else 0, noise.stride(0) if B > 1 else 0, B, V,
                              L.DT_F32 if logits.dtype == torch.float32 else L.DT_BF16)
        L.check(self.lib.sm100_sample(ctypes.addressof(a), self._raw_stream(self.device.index)), "sample")
        return tok, logp
