"""The key-value cache in 8 bits at its edges: as test_gpu_kv_edges, whose checks hold for what the cache has; several calls that share a small page cache, pages that never come, a cache past 4 GiB, and
calls while another device is the current one."""
import threading

import pytest

import test_gpu_kv_edges as edges
from test_gpu_kv import UNIT, _i32, _near, _starts, _table
from test_gpu_kv8 import Cache8, _kept, _same
from test_gpu_parity import Rig, bam  # noqa: F401  (bam is the module fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture
def eight(monkeypatch):
    monkeypatch.setattr(edges, "Cache", Cache8)


@pytest.mark.parametrize("dtype,dim,page", [("bf16", 256, 4096), ("bf16", 128, 4096), ("f16", 64, 4096), ("f16", 16, 512), ("bf16", 80, 4096), ("bf16", 256, 16384)])
@pytest.mark.parametrize("width", [1, 3, 5, 6])
@pytest.mark.parametrize("new", [1, 3, 40, 70])
@pytest.mark.parametrize("window,sinks", [(0, 0), (290, 2), (50, 64)])
def test_tokens_past_the_table_are_not_seen(bam, eight, dtype, dim, page, width, new, window, sinks):
    edges.test_tokens_past_the_table_are_not_seen(bam, dtype, dim, page, width, new, window, sinks)


@pytest.mark.parametrize("max_new", [1, 3, 20, 40, 70])
def test_rows_beyond_max_new_are_left(bam, eight, max_new):
    edges.test_rows_beyond_max_new_are_left(bam, max_new)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n_seqs", [1, 200])
def test_a_split_that_is_done_again_counts_once(bam, dim, n_seqs):
    """an infinity among values that some rows see and others do not leaves a split to be done row by row: its pages are counted by whoever does it.  An access is a wave's visit of a page: four steps of
    32 tokens are a wave's each, and a block of 64 tokens has two of them"""
    import torch
    with Cache8(bam, 32, 2, dim, "bf16") as c:
        lens = [100]
        table = _table(lens, c.t, 32)
        v = torch.randn(100, 2, dim).to(c.dtype)
        v[98] = float("inf")
        c.fill(lens, table, v=v)
        q = torch.randn(3 * n_seqs, 4, dim).to(c.dtype).cuda()
        c.kv.array.stats()
        c.kv.attend(q, _i32(lens * n_seqs), table.cuda().expand(n_seqs, -1), starts=_starts([3] * n_seqs), max_new=3)
        st = c.kv.array.stats()
        visits = sum(len({t // c.t for t in range(first, min(100, first + 32))}) for first in range(0, 100, 32))
        assert st["access_cnt"] == st["hit_cnt"] == n_seqs * 2 * 2 * visits, st


@pytest.mark.parametrize("new", [1, 5, 70])
def test_attention_twice_is_the_same(bam, new):
    """bit for bit, split over the length and joined; lengths much shorter than the table"""
    import torch
    with Cache8(bam, 512, 1, 64, "bf16") as c:
        lens = [9000, 3000, 40]
        table = _table(lens, c.t, 512, width=500)
        c.fill(lens, table)
        news = [new, new, min(new, 40)]
        q = torch.randn(sum(news), 4, 64).to(torch.bfloat16)
        first = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news))
        for _ in range(4):
            assert torch.equal(c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news)), first)
        last = [new - 1, 2 * new - 1, sum(news) - 1]
        want, tol, _ = c.want(q[last], lens, [1, 1, 1], table)
        _near(first[last], want, tol)


@pytest.mark.parametrize("dim,page,cache_pages", [(128, 4096, 16), (256, 4096, 32), (64, 16384, 16), (16, 512, 33)])
@pytest.mark.parametrize("news", [[1, 1], [3, 5], [40, 70]])
def test_four_calls_at_a_time(bam, dim, page, cache_pages, news):
    """layers in one array behind a page cache of a few pages, each on a stream of its own, with appends, reads and reorderings among the attentions"""
    import torch
    from bam_amd.host import make_array
    calls, t, heads, n_blocks = 4, 1 << ((page // dim).bit_length() - 1), 2, 20
    lens = [9 * t + 3, 6 * t + 1]
    pages = 2 * heads * n_blocks
    with Rig(bam, calls * pages * page, backing=True, n_queues=16, depth=256, stage_bytes=max(4096, min(page, 8192))) as r:
        pc, rg, array = make_array(r.c, calls * pages * page // 8, page, cache_pages)
        layers = []
        for j in range(calls):
            c = Cache8.__new__(Cache8)          # what the layer should hold, without a store of its own
            c.dtype, c.name, c.heads, c.dim, c.n_blocks, c.u, c.t = torch.bfloat16, "bf16", heads, dim, n_blocks, UNIT["bf16"], t
            c.k = torch.zeros(n_blocks, heads, t, dim, dtype=torch.float64)
            c.v = torch.zeros_like(c.k)
            c.kv = bam.KVCache(array, heads, dim, first_page=j * pages, n_blocks=n_blocks, stored=torch.float8_e4m3fn)
            c.table = _table(lens, t, n_blocks, seed=j)
            free = [b for b in range(n_blocks) if b not in c.table.flatten().tolist()]
            c.kk, c.vv = c.fill(lens, c.table, seed=j)
            c.q = torch.randn(sum(news), 2 * heads, dim, generator=torch.Generator().manual_seed(j)).to(c.dtype)
            c.args = [x.cuda() for x in (c.kk, c.vv, c.q, c.table)] + [_i32(lens), _starts(lens), _starts(news), _i32([0, 0, 1]), _i32(free[:3])]
            c.want_out, c.tol, _ = c.want(c.q, lens, news, c.table)
            layers.append(c)
        torch.cuda.synchronize()
        got, start = [[] for _ in layers], threading.Barrier(calls)

        def work(j):
            torch.cuda.set_device(0)
            c = layers[j]
            k, v, q, table, dl, all_starts, starts, parents, spare = c.args
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(60)
                for rep in range(3):
                    out = c.kv.attend(q, dl, table, starts=starts, max_new=max(news))
                    back = None
                    if j % 3 == rep:
                        new_lens, new_table, _ = c.kv.reorder(parents, dl, table, spare)
                        back = c.kv.read(2 * lens[0] + lens[1], new_lens, new_table, starts=_starts([lens[0], lens[0], lens[1]]))
                    else:
                        c.kv.append(k, v, dl, table, starts=all_starts)
                    torch.cuda.current_stream().synchronize()
                    got[j].append((out, back))

        threads = [threading.Thread(target=work, args=(j,)) for j in range(calls)]
        for x in threads:
            x.start()
        for x in threads:
            x.join()
        assert not r.c.aborted()
        for j, c in enumerate(layers):
            assert len(got[j]) == 3, j
            for out, back in got[j]:
                _near(out, c.want_out, c.tol, j)
                for got_rows, rows in zip(back or (), (c.kk, c.vv)):
                    _same(got_rows, _kept(torch.cat([rows[:lens[0]], rows]), "bf16"))
            c.kv.close()
        for x in (array, rg, pc):
            x.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_rows_of_lost_pages_read_as_nan(bam, dtype):
    """the target swallows every command: the waits are bounded, rows whose keys and values never came are NaN, out of reads and attention, and those that were there are as they were"""
    import torch
    with Rig(bam, 1 << 20, backing=True, n_queues=1, depth=1024, drop_every=1, limit=100_000) as r:
        kv = bam.KVCache(r.array(1 << 17, 4096, 64), 1, 128, {"bf16": torch.bfloat16, "f16": torch.float16}[dtype], n_blocks=64, stored=torch.float8_e4m3fn)
        table = torch.tensor([[3, 7]], dtype=torch.int32, device="cuda")
        k = torch.randn(32, 1, 128).to(kv.dtype).cuda()
        v = k.flip(2).contiguous()
        kv.append(k, v, _i32([32]), table, starts=_starts([32]))          # a block of new rows: nothing is read
        torch.cuda.synchronize()
        assert not r.c.aborted()
        got_k, got_v = kv.read(45, _i32([45]), table, starts=_starts([45]))
        out = kv.attend(k[:1], _i32([45]), table)
        torch.cuda.synchronize()
        assert r.c.aborted() and r.t.stats()["dropped"] >= 1
        _same(got_k[:32], _kept(k.cpu(), dtype))
        _same(got_v[:32], _kept(v.cpu(), dtype))
        assert bool(torch.isnan(got_k[32:]).all()) and bool(torch.isnan(got_v[32:]).all()) and bool(torch.isnan(out).all())
        kv.close()


def test_a_cache_past_4_gib(bam):
    """slots and rows whose offsets pass 32 bits: rows of some sequences against torch's own conversion, attention over them in 64 bits on the device, and a copied last block at the far end"""
    import torch
    heads, dim, per = 8, 128, 32
    n_seqs, length = 37, 65536                       # 5 GB of pages
    n_blocks = n_seqs * length // per + 2
    with Rig(bam, 1 << 40, n_queues=16, depth=256) as r:
        kv = bam.make_kv_cache(r.c, n_blocks, heads, dim, stored=torch.float8_e4m3fn)
        assert kv.block_tokens == per and 2 * n_blocks * heads * 4096 > 1 << 32
        gen = torch.Generator(device="cuda").manual_seed(3)
        order = torch.randperm(n_blocks, generator=torch.Generator().manual_seed(1)).to(torch.int32)
        table, spare = order[:-2].view(n_seqs, -1).cuda(), order[-2:].cuda()
        lens = _i32([length - 7 * b for b in range(n_seqs)])
        n = int(lens.sum())
        starts = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), lens.cumsum(0).to(torch.int32)])
        k = torch.randn(n, heads, dim, generator=gen, dtype=torch.bfloat16, device="cuda")
        kv.append(k, k, lens, table, starts=starts)
        q = torch.randn(n_seqs, 16, dim, generator=gen, dtype=torch.bfloat16, device="cuda")
        out = kv.attend(q, lens, table)
        for b in (0, 17, n_seqs - 1):
            rows = k[int(starts[b]):int(starts[b + 1])]
            by = torch.exp2(torch.ceil(torch.log2(rows.double().abs().amax(-1, keepdim=True) / 448)))
            held = (rows.double() / by).float().to(torch.float8_e4m3fn).double() * by
            m = rows.shape[0]
            got_k, got_v = kv.read(m, lens[b:b + 1], table[b:b + 1], starts=_i32([0, m]))
            assert torch.equal(got_k.double(), held) and torch.equal(got_v.double(), held)
            for h in (0, 9, 15):
                w = torch.softmax(held[:, h // 2] @ q[b, h].double() * dim ** -0.5, 0)
                want = w @ held[:, h // 2]
                # the bound of test_gpu_kv for bfloat16, scores of up to a few times 1e-5 off
                _near(out[b, h], want.cpu(), (1.01 * 2.0 ** -8 * want.abs() + (1.01 * 2.0 ** -8 + 2.0 ** -14) * (w @ held[:, h // 2].abs())).cpu(), (b, h))
        b = n_seqs - 1
        new_lens, new_table, _ = kv.reorder(_i32([b, b]), lens, table, spare)
        ends = kv.read(18, new_lens, new_table, starts=_i32([0, 9, 18]))
        assert torch.equal(ends[0][:9], got_k[-9:]) and torch.equal(ends[0][9:], got_k[-9:]) and torch.equal(ends[1][9:], got_v[-9:])
        kv.close()
        assert not r.c.aborted()


def test_another_device_is_the_current_one(bam, monkeypatch):
    """kernels would go to the other device, whose they are not"""
    import torch
    from bam_amd import kv as binding
    with Cache8(bam, 4, 1, 64, "bf16") as c:
        x, lens, table = torch.ones(1, 1, 64, dtype=c.dtype, device="cuda"), _i32([1]), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
        calls = (lambda: c.kv.append(x, x, lens, table), lambda: c.kv.read(1, lens, table), lambda: c.kv.attend(x, lens, table), lambda: c.kv.reorder(_i32([0]), lens, table, _i32([3])))
        for call in calls:
            call()
        monkeypatch.setattr(binding, "_current", lambda: 1)
        for call in calls:
            with pytest.raises(bam.BamError, match="current device"):
                call()
