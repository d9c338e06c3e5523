"""The powers of two of an 8-bit key-value cache are memory of torch's allocator: it is told of each stream that a call uses them on, so that a handle may go while calls are queued."""
import ctypes

import pytest


class _Scales:
    def __init__(self):
        self.on = []

    def record_stream(self, stream):
        self.on.append(stream)


def test_each_stream_is_told_once(monkeypatch):
    """(no device: what a call asks for the current stream)"""
    import torch
    from bam_amd import kv
    cache = kv.KVCache.__new__(kv.KVCache)
    cache.h, cache._owned, cache._index, cache.device, cache.scales, cache._scales_on = ctypes.c_void_p(), [], 0, torch.device("cuda", 0), _Scales(), set()
    now = [0]
    monkeypatch.setattr(kv, "_current", lambda: 0)
    monkeypatch.setattr(kv, "_stream", lambda: ctypes.c_void_p(now[0]))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    for now[0] in (0, 16, 16, 0, 32, 16):
        assert (cache._queue().value or 0) == now[0]
    assert cache.scales.on == [0, 16, 32]
    cache.scales = None                              # 16 bits
    for now[0] in (0, 48):
        cache._queue()


@pytest.mark.gpu
def test_a_handle_that_goes_while_calls_are_queued():
    import torch
    import bam_amd
    from test_gpu_kv import _i32, _starts
    from test_gpu_parity import Rig
    with Rig(bam_amd, 1 << 22) as r:
        array = r.array((1 << 22) // 8, 4096, 1024)
        kv = bam_amd.KVCache(array, 1, 128, n_blocks=512, stored=torch.float8_e4m3fn)
        size, at = kv.scales.numel(), kv.scales.data_ptr()
        n = 32 * 512
        k = torch.randn(n, 1, 128, device="cuda").to(torch.bfloat16)
        args = [_i32([n]), torch.arange(512, dtype=torch.int32, device="cuda").view(1, -1), _starts([n])]
        torch.cuda.synchronize()
        side, done = torch.cuda.Stream(), torch.cuda.Event()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            kv.append(k, k, *args)
            done.record()
        kv.close()
        del kv
        others = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(8)]
        pending = not done.query()
        assert pending and at not in [x.data_ptr() for x in others]
        side.synchronize()
        assert not r.c.aborted()
