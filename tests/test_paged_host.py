"""Argument checks of the paged cache and the sampler, on the CPU: calls outside
their contracts come back with a status and a message before anything touches
a device."""
import ctypes
import math

from thvm_b200 import _lib as L

P = 1 << 20   # an aligned stand-in address; never dereferenced


def _cache(**kw):
    a = dict(pool=P, table=P, n_pages=4, page=16, kv_heads=2, head_dim=64, bits=16, n_seq=2, max_pages=2) | kw
    return L.Sm100PagedCache(*(a[n] for n, _ in L.Sm100PagedCache._fields_))


def _append(c, **kw):
    a = dict(qkv=P, g_q=P, g_k=P, cos_t=P, sin_t=P, pos=P, seq=P, q_out=P, ld=0, T=1, heads=4, dtype=L.DT_F32, rot=64,
             n_pos=8, pairs=0, eps=1e-6) | kw
    a = L.Sm100PagedAppendArgs(*(a[n] for n, _ in L.Sm100PagedAppendArgs._fields_))
    return L.lib().sm100_paged_append(ctypes.byref(c), ctypes.byref(a), None)


def _attend(c, **kw):
    a = dict(q=P, kv_len=P, q_off=P, out=P, ws=P, ws_bytes=1 << 40, ld_q=0, T=2, heads=4, max_rows=1, scale=1.0) | kw
    a = L.Sm100PagedAttnArgs(*(a[n] for n, _ in L.Sm100PagedAttnArgs._fields_))
    return L.lib().sm100_paged_attention(ctypes.byref(c), ctypes.byref(a), None)


def _sample(**kw):
    a = dict(logits=P, noise=P, temperature=None, top_k=None, top_p=None, min_p=None, tok=P, logp=None, ld=0,
             ld_noise=0, B=1, V=8, dtype=L.DT_F32) | kw
    a = L.Sm100SampleArgs(*(a[n] for n, _ in L.Sm100SampleArgs._fields_))
    return L.lib().sm100_sample(ctypes.byref(a), None)


def test_struct_layouts():
    assert ctypes.sizeof(L.Sm100PagedCache) == 48
    assert ctypes.sizeof(L.Sm100PagedAppendArgs) == 104 and L.Sm100PagedAppendArgs.ld.offset == 64
    assert ctypes.sizeof(L.Sm100PagedAttnArgs) == 72 and L.Sm100PagedAttnArgs.T.offset == 56
    assert ctypes.sizeof(L.Sm100SampleArgs) == 96 and L.Sm100SampleArgs.B.offset == 80


def test_block_bytes():
    f = L.lib().sm100_paged_block_bytes
    assert f(16, 64, 16) == 2 * 16 * 64 * 2
    assert f(32, 128, 4) == 2 * 32 * (64 + 8)
    assert f(64, 256, 4) == 2 * 64 * (128 + 16)
    for bad in ((8, 64, 16), (48, 64, 16), (16, 96, 4), (16, 64, 8), (0, 0, 0), (-16, 64, 4)):
        assert f(*bad) == 0


def test_cache_refusals():
    for bad in (dict(pool=None), dict(table=None), dict(pool=P + 8), dict(n_pages=0), dict(kv_heads=0), dict(n_seq=0),
                dict(max_pages=0), dict(max_pages=1 << 28)):
        c = _cache(**bad)
        assert _append(c) == _attend(c) == L.ERR_ARG, bad
        assert L.lib().sm100_paged_read(ctypes.byref(c), P, P, P, P, 1, None) == L.ERR_ARG
        assert L.lib().sm100_paged_attention_ws_bytes(ctypes.byref(c), 4, 1) == 0
    for bad in (dict(page=8), dict(head_dim=96), dict(bits=8)):
        c = _cache(**bad)
        assert _append(c) == _attend(c) == L.ERR_UNSUPPORTED, bad
        assert b"head_dim" in L.lib().sm100_last_error()


def test_append_refusals():
    c = _cache()
    for bad in (dict(qkv=None), dict(pos=None), dict(seq=None), dict(q_out=None), dict(T=-1), dict(heads=0),
                dict(heads=3), dict(qkv=P + 4), dict(q_out=P + 2), dict(g_q=P + 4), dict(cos_t=None), dict(sin_t=None),
                dict(sin_t=P + 4), dict(rot=0), dict(rot=24), dict(rot=80), dict(n_pos=0), dict(ld=511), dict(ld=514),
                dict(dtype=L.DT_BF16, ld=516)):
        assert _append(c, **bad) == L.ERR_ARG, bad
    assert _append(c, dtype=L.DT_I32) == L.ERR_UNSUPPORTED
    assert _append(c, T=0) == L.OK
    assert L.lib().sm100_paged_read(ctypes.byref(c), P, P, P, P + 2, 1, None) == L.ERR_ARG
    assert L.lib().sm100_paged_read(ctypes.byref(c), P, P, P, P, 0, None) == L.OK


def test_attention_refusals():
    c = _cache()
    for bad in (dict(q=None), dict(kv_len=None), dict(out=None), dict(ws=None), dict(T=-1), dict(heads=3),
                dict(max_rows=0), dict(q_off=None, T=1), dict(q_off=None, max_rows=2), dict(q=P + 8), dict(out=P + 8),
                dict(ws=P + 8), dict(ld_q=100), dict(ld_q=260), dict(ws_bytes=0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf"))):
        assert _attend(c, **bad) == L.ERR_ARG, bad
    assert _attend(c, T=0) == L.OK
    assert L.lib().sm100_paged_attention_ws_bytes(ctypes.byref(c), 4, 1) > 0


def test_sample_refusals():
    for bad in (dict(logits=None), dict(noise=None), dict(tok=None), dict(B=-1), dict(V=0), dict(ld=7), dict(ld_noise=7),
                dict(ld=-1)):
        assert _sample(**bad) == L.ERR_ARG, bad
    assert _sample(dtype=L.DT_I32) == L.ERR_UNSUPPORTED
    assert _sample(B=0) == L.OK


def test_scratch_keeps_what_a_graph_may_hold(monkeypatch):
    import pytest
    import torch
    from thvm_b200.paged import Scratch
    cpu, capturing = torch.device("cpu"), []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: bool(capturing))
    s = Scratch()
    small = s.take(64, cpu)[0]
    assert s.take(32, cpu) == s.take(64, cpu) == (small, 64)     # large enough: it stays where it is
    large = s.take(128, cpu)[0]
    assert large != small and s.take(1, cpu) == (large, 128)
    assert [b.data_ptr() for b in s.held] == [small, large]      # the earlier memory is no one else's
    with pytest.raises(ValueError):
        s.take(16, torch.device("cuda", 0))
    capturing.append(True)
    assert s.take(128, cpu) == (large, 128)
    graph = s.take(129, cpu)                                     # zeroed by replays: the graph's alone
    assert graph[1] == 129 and graph[0] not in (small, large) and s.held[-1].data_ptr() == graph[0]
    capturing.clear()
    assert s.take(128, cpu) == (large, 128)
    assert s.take(129, cpu)[0] not in (small, large, graph[0])


def test_widest_workspace_is_that_of_eight_columns():
    f = L.lib().sm100_paged_attention_ws_bytes
    for bits in (4, 16):
        for hd in (64, 128, 256):
            c = _cache(bits=bits, head_dim=hd)
            most = f(ctypes.byref(c), 2, 8)
            assert all(f(ctypes.byref(c), 2 * g, r) <= most for g in (1, 2, 5, 64) for r in (1, 2, 7, 4096))


def test_attention_refuses_a_scale_whose_logarithm_base_overflows():
    assert _attend(_cache(), scale=3e38) == L.ERR_ARG


class FakePool:
    """A pool or another tensor on cuda:1, as far as the calls look at one."""
    is_cuda = True

    def __init__(self, dtype, *shape):
        import torch
        self.dtype, self.shape, self.device = dtype, shape, torch.device("cuda", 1)
        self.numel = lambda: math.prod(shape)
        self.dim, self.is_contiguous, self.get_device, self.data_ptr = lambda: len(shape), lambda: True, lambda: 1, lambda: P
        steps = [1]
        for n in shape[:0:-1]:
            steps.insert(0, steps[0] * n)
        self.stride = lambda: tuple(steps)


def test_calls_make_their_gpu_current(monkeypatch):
    """A cache and a sampler on cuda:1 while cuda:0 is current: each call of the library runs with cuda:1 current, on its
    stream, and cuda:0 is current again afterwards."""
    import torch
    from thvm_b200 import paged, sampling
    current = [0]

    class Guard:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 + index)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(paged.Scratch, "take", lambda self, n, device: (P, n))
    seen = []

    def call(name):
        return lambda *a: seen.append((name, current[0], a[-1] if a else None)) or 0

    real, i32, f32, u8, bf16 = L.lib(), torch.int32, torch.float32, torch.uint8, torch.bfloat16
    block = int(real.sm100_paged_block_bytes(16, 64, 16))

    class Fake:
        sm100_paged_block_bytes, sm100_paged_attention_ws_bytes = real.sm100_paged_block_bytes, real.sm100_paged_attention_ws_bytes
        sm100_paged_append, sm100_paged_read, sm100_paged_attention = call("append"), call("read"), call("attend")
        sm100_paged_status, sm100_sample = call("status"), call("sample")

    monkeypatch.setattr(L, "lib", lambda: Fake)
    monkeypatch.setattr(torch, "empty", lambda shape, dtype, device: FakePool(dtype, *(shape if isinstance(shape, tuple) else (shape,))))
    FakePool.unbind = lambda self, d: (FakePool(self.dtype, *self.shape[1:]),) * 2
    for here in (0, 1):
        current[0] = here
        c = paged.PagedCache(FakePool(u8, 4, 2, block), FakePool(i32, 2, 2), 16, 64, 16)
        c.append(FakePool(f32, 2, 8 * 64), FakePool(i32, 2), FakePool(i32, 2), 4)
        c.read(FakePool(i32, 2), FakePool(i32, 2))
        c.attend(FakePool(bf16, 2, 4, 64), FakePool(i32, 2))
        c.status()
        s = sampling.Sampler(torch.device("cuda", 1))
        s(FakePool(f32, 2, 8), FakePool(f32, 2, 8))
        assert current[0] == here
        assert seen == [("append", 1, 1001), ("read", 1, 1001), ("attend", 1, 1001), ("status", 1, None), ("sample", 1, 1001)]
        seen.clear()


def test_a_cache_is_on_a_gpu():
    import pytest
    from thvm_b200.paged import PagedCache
    with pytest.raises(ValueError):
        PagedCache.empty(2, 2, 4, 2, 64, device="cpu")


def test_append_refuses_more_heads_than_it_can_count():
    big = (1 << 31) - 2
    assert _append(_cache(), heads=big) == L.ERR_ARG
    assert _append(_cache(kv_heads=1 << 30), heads=1 << 30) == L.ERR_ARG
    assert _append(_cache(kv_heads=1 << 30), heads=1 << 30, T=5) == L.ERR_ARG
    assert _append(_cache(), heads=1 << 20, T=1 << 20) == L.ERR_ARG
