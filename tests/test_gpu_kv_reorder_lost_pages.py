"""Copies of a reordering whose pages could not be had, of the page that they come from and of the one that they go to.  The target swallows every command: waits are bounded, and the launches end."""
import pytest

from test_gpu_kv import _i32, _starts
from test_gpu_parity import Rig, bam  # noqa: F401  (bam is the module fixture)

pytestmark = pytest.mark.gpu


def _cache(bam, r, stored, dtype):
    """64 pages for 64 blocks of one head; float8_e4m3fn by its name: a block holds 32 tokens, else 16"""
    import torch
    dt = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    return bam.KVCache(r.array(1 << 17, 4096, 64), 1, 128, dt, n_blocks=64, stored=torch.float8_e4m3fn if stored == "e4m3" else None)


def _fill(kv, blocks):
    """whole blocks of new rows, one after the other: nothing of them is read from the store"""
    import torch
    t = kv.block_tokens
    for b in blocks:
        k = torch.randn(t, 1, 128, generator=torch.Generator().manual_seed(b)).to(kv.dtype).cuda()
        kv.append(k, k, _i32([t]), _i32([b]).view(1, 1), starts=_starts([t]))
    torch.cuda.synchronize()


@pytest.mark.parametrize("stored", ["16", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_the_source(bam, stored, dtype):
    """NaN in the place of what was not there, in a page that is resident and held finite rows: only the copy can have put it there"""
    import torch
    with Rig(bam, 1 << 20, backing=True, n_queues=1, depth=1024, drop_every=1, limit=100_000) as r:
        kv = _cache(bam, r, stored, dtype)
        t, rest = kv.block_tokens, 9
        _fill(kv, [5])
        assert not r.c.aborted()
        lens, table, _ = kv.reorder(_i32([0, 0]), _i32([rest]), _i32([3]).view(1, 1), _i32([4, 5]))
        torch.cuda.synchronize()
        assert r.c.aborted() and lens.tolist() == [rest, rest] and table.tolist() == [[3], [5]]
        k, v = kv.read(t, _i32([t]), table[1:], starts=_starts([t]))
        for x in (k, v):
            assert bool(torch.isnan(x[:rest]).all()), x[:rest]
        kv.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_the_powers_of_two_of_pages_that_copies_do_not_reach(bam, dtype):
    """thousands of copies by way of sixteen slots, of a page that is lost on the way: most waits for a slot are given up, and a page that was not had keeps the powers of two that go with what it holds"""
    import torch
    n = 4000
    with Rig(bam, 2 * (n + 1) * 4096, backing=True, n_queues=1, depth=1024, drop_every=1, limit=100_000) as r:
        kv = bam.KVCache(r.array((n + 1) * 1024, 4096, 16), 1, 128, {"bf16": torch.bfloat16, "f16": torch.float16}[dtype], n_blocks=n + 1, stored=torch.float8_e4m3fn)
        _fill(kv, [n])
        assert not r.c.aborted()
        kv.scales[:n] = 77
        source = kv.scales[n, 0, :, :9].clone()
        lens, table, _ = kv.reorder(_i32([0] * (n + 1)), _i32([9]), _i32([n]).view(1, 1), torch.arange(-1, n, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert r.c.aborted() and bool((lens == 9).all()) and table[:, 0].tolist() == [n] + list(range(n))
        got = kv.scales[:n, 0]
        kept, copied = (got == 77).all(-1), (got[..., :9] == source).all(-1) & (got[..., 9:] == 77).all(-1)
        assert bool((kept | copied).all()) and bool(kept.any()), (int(kept.sum()), int(copied.sum()))
        kv.close()
