"""The key-value cache at its edges: tables shorter than what they are asked for, starts that say more rows than there are, calls that share a small cache, reads that
fail, weights far below the largest.  Tolerances as in test_gpu_kv."""
import numpy as np
import pytest

from test_gpu_kv import Cache, _i32, _near, _starts, _table
from test_gpu_parity import bam  # noqa: F401  (the module fixture)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- tables shorter than the lengths

@pytest.mark.parametrize("dtype,dim,page", [("bf16", 256, 4096), ("bf16", 128, 4096), ("f16", 64, 4096), ("f16", 16, 512), ("bf16", 80, 4096)])
@pytest.mark.parametrize("width", [1, 3, 5, 6])
@pytest.mark.parametrize("new", [1, 3, 40, 70])
@pytest.mark.parametrize("window,sinks", [(0, 0), (290, 2), (50, 64)])
def test_tokens_past_the_table_are_not_seen(bam, dtype, dim, page, width, new, window, sinks):
    """blocks of 8, 16 and 32 tokens, tables that end inside a step of 32 and a tile of 64 tokens, and what other sequences have in the page cache far from what this one has"""
    import torch
    lens = [300, 200]
    with Cache(bam, 80, 1, dim, dtype, page) as c:
        table = _table(lens, c.t, 80)
        k, v = torch.randn(500, 1, dim).to(c.dtype), torch.randn(500, 1, dim).to(c.dtype)
        v[300:] += 100
        c.fill(lens, table, k=k, v=v)
        table = table[:, :width].contiguous()
        news = [new, min(new, 4)]
        q = torch.randn(sum(news), 2, dim, generator=torch.Generator().manual_seed(new)).to(c.dtype)
        want, tol, lse = c.want(q, lens, news, table, window, sinks)
        got, got_lse = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), max_new=new, window=window, sinks=sinks, return_lse=True)
        _near(got, want, tol)
        none = torch.isinf(lse)
        assert bool((got_lse.cpu()[none] == -np.inf).all())
        _near(got_lse.cpu()[~none], lse[~none], 2.0 ** -16 * (1 + lse[~none].abs()))
        assert not c.rig.c.aborted()
