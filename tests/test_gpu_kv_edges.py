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


# ---------------------------------------------------------------- starts that say more rows than there are

@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("starts,rows", [([0, 9, 40], 23), ([0, 30, 77], 12), ([-5, 20, 2 ** 31 - 1], 60), ([2 ** 31 - 1, -2 ** 31, 50], 50), ([0, 70, 40], 40)])
def test_no_more_rows_than_there_are(bam, dtype, dim, starts, rows):
    """what lies behind the given rows is neither read nor written; the rows that are there have the places that starts gives them, in all three calls"""
    import ctypes
    import torch
    heads, lens, behind = 2, [150, 160], 80
    with Cache(bam, 64, heads, dim, dtype) as c:
        table = _table([200, 200], c.t, 64)
        c.fill([200, 200], table)
        dl, dt, ds = _i32(lens), table.cuda(), _i32(starts)
        # (sequence, position) of each row that has one
        places = {}
        for i in range(rows):
            b = 1 if starts[1] <= i else 0
            if max(starts[b], 0) <= i < starts[b + 1] and lens[b] - (starts[b + 1] - i) >= 0:
                places[i] = (b, lens[b] - (starts[b + 1] - i))
        k = torch.randn(rows + behind, heads, dim).to(c.dtype)
        k[rows:] = float("nan")
        v = k.flip(2).contiguous()
        c.kv.append(k.cuda()[:rows], v.cuda()[:rows], dl, dt, starts=ds)
        for i, (b, p) in places.items():
            c.k[int(table[b, p // c.t]), :, p % c.t] = k[i]
            c.v[int(table[b, p // c.t]), :, p % c.t] = v[i]
        all_k, all_v = c.kv.read(400, _i32([200, 200]), dt, starts=_i32([0, 200, 400]))
        at = [(int(table[b, p // c.t]), p % c.t) for b in range(2) for p in range(200)]
        assert torch.equal(all_k.cpu(), torch.stack([c.k[b, :, x] for b, x in at])) and torch.equal(all_v.cpu(), torch.stack([c.v[b, :, x] for b, x in at]))
        # rows out, with numbers behind the two outputs that have to stay
        from bam_amd import kv as binding
        out = torch.full((2, rows + behind, heads, dim), 7.0, dtype=c.dtype, device="cuda")
        what = binding._READ.pack(rows, 2, ds.data_ptr(), dl.data_ptr(), dt.data_ptr(), dt.stride(0), dt.shape[1])
        assert c.kv.L.bam_kv_read(c.kv.h, what, ctypes.c_void_p(out[0].data_ptr()), ctypes.c_void_p(out[1].data_ptr()), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        assert bool((out[:, rows:] == 7).all())
        for i in range(rows):
            x = out[:, i].cpu()
            assert torch.equal(x[0], k[i]) and torch.equal(x[1], v[i]) if i in places else not bool(x.any()), i
        # attention: rows of no sequence stay as they are
        q = torch.randn(rows, 2 * heads, dim).to(c.dtype)
        got = torch.full((rows + behind, 2 * heads, dim), 7.0, dtype=c.dtype, device="cuda")
        c.kv.attend(q.cuda(), dl, dt, starts=ds, out=got[:rows])
        assert bool((got[rows:] == 7).all())
        for i in range(rows):
            b = 1 if starts[1] <= i else 0
            if i in places:
                b, p = places[i]
                want, tol, _ = c.want(q[i:i + 1], [p + 1, p + 1], [1 - b, b], table)
                _near(got[i:i + 1], want, tol, i)
            else:
                assert bool((got[i] == (0 if max(starts[b], 0) <= i < starts[b + 1] else 7)).all()), i
        assert not c.rig.c.aborted()


# ---------------------------------------------------------------- several calls over one small page cache

CALLS = 6


@pytest.mark.parametrize("dim,page,cache_pages", [(128, 4096, 32), (256, 4096, 64), (64, 16384, 16), (64, 4096, 40), (16, 512, 33)])
@pytest.mark.parametrize("news", [[1, 1], [3, 5], [40, 70]])
def test_six_calls_at_a_time(bam, dim, page, cache_pages, news):
    """layers whose blocks lie in one array behind a page cache of a few pages, each on a stream of its own: no wave keeps a page while it waits for a slot, so none waits for what the
    others have; appends and reads among the attentions"""
    import threading
    import torch
    from bam_amd.host import make_array
    from test_gpu_parity import Rig
    t, heads = 1 << ((page // (2 * dim)).bit_length() - 1), 2
    lens = [9 * t + 3, 6 * t + 1]
    n_blocks = 17
    pages = 2 * heads * n_blocks
    with Rig(bam, CALLS * pages * page, backing=True, n_queues=16, depth=256, stage_bytes=max(4096, min(page, 8192))) as r:
        pc, rg, array = make_array(r.c, CALLS * pages * page // 8, page, cache_pages)
        layers = []
        for j in range(CALLS):
            c = Cache.__new__(Cache)          # what the layer should hold, without a store of its own
            c.dtype, c.heads, c.dim, c.n_blocks, c.u, c.t = torch.bfloat16, heads, dim, n_blocks, 2.0 ** -8, t
            c.k = torch.zeros(n_blocks, heads, t, dim, dtype=c.dtype)
            c.v = torch.zeros_like(c.k)
            c.kv = bam.KVCache(array, heads, dim, first_page=j * pages, n_blocks=n_blocks)
            c.table = _table(lens, t, n_blocks, seed=j)
            k, v = c.fill(lens, c.table, seed=j)
            c.q = torch.randn(sum(news), 2 * heads, dim, generator=torch.Generator().manual_seed(j)).to(c.dtype)
            c.args = [x.cuda() for x in (k, v, c.q, c.table)] + [_i32(lens), _starts(lens), _starts(news)]
            c.want_out, c.tol, _ = c.want(c.q, lens, news, c.table)
            layers.append(c)
        torch.cuda.synchronize()
        got, start = [[] for _ in layers], threading.Barrier(CALLS)

        def work(j):
            torch.cuda.set_device(0)
            c = layers[j]
            k, v, q, table, dl, all_starts, starts = c.args
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(60)
                for rep in range(3):
                    out = c.kv.attend(q, dl, table, starts=starts, max_new=max(news))
                    back = c.kv.read(sum(lens), dl, table, starts=all_starts) if j % 3 == rep else None
                    if j % 3 != rep:
                        c.kv.append(k, v, dl, table, starts=all_starts)
                    torch.cuda.current_stream().synchronize()
                    got[j].append((out, back))

        threads = [threading.Thread(target=work, args=(j,)) for j in range(CALLS)]
        for x in threads:
            x.start()
        for x in threads:
            x.join()
        assert not r.c.aborted()
        for j, c in enumerate(layers):
            assert len(got[j]) == 3, j
            for out, back in got[j]:
                _near(out, c.want_out, c.tol, j)
                assert back is None or (torch.equal(back[0], c.args[0]) and torch.equal(back[1], c.args[1])), j
            c.kv.close()
        for x in (array, rg, pc):
            x.close()


# ---------------------------------------------------------------- pages that could not be had

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_rows_of_lost_pages_read_as_nan(bam, dtype):
    """the target swallows every command: the waits are bounded, rows whose keys and values never came are NaN, and those that were there are as they were.  (One wave
    waits, for two pages, in a queue that is never full.)"""
    import torch
    from test_gpu_parity import Rig
    with Rig(bam, 1 << 20, backing=True, n_queues=1, depth=1024, drop_every=1, limit=100_000) as r:
        kv = bam.KVCache(r.array(1 << 17, 4096, 64), 1, 128, {"bf16": torch.bfloat16, "f16": torch.float16}[dtype], n_blocks=64)
        table = torch.tensor([[3, 7]], dtype=torch.int32, device="cuda")
        k = torch.randn(16, 1, 128).to(kv.dtype).cuda()
        v = k.flip(2).contiguous()
        kv.append(k, v, _i32([16]), table, starts=_starts([16]))          # a block of new rows: nothing is read
        torch.cuda.synchronize()
        assert not r.c.aborted()
        got_k, got_v = kv.read(25, _i32([25]), table, starts=_starts([25]))
        torch.cuda.synchronize()
        assert r.c.aborted() and r.t.stats()["dropped"] >= 1
        assert torch.equal(got_k[:16], k) and torch.equal(got_v[:16], v)
        assert bool(torch.isnan(got_k[16:]).all()) and bool(torch.isnan(got_v[16:]).all())
        kv.close()


# ---------------------------------------------------------------- weights far below the largest

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("low", [12.5, 23.4, 25.0])
@pytest.mark.parametrize("new,n", [(1, 1 << 19), (5, 1 << 19), (40, 1 << 17), (100, 1 << 17)])
def test_one_peak_over_a_long_flat_tail(bam, dtype, low, new, n):
    """one token above all others, of 2^-low of its weight each, which hold up to ninety times its share of the sum or a hundredth of it: their part is not lost in the weights'
    rounding, wherever the peak is.  Bounds: weights and output are rounded to the type once (u each), scores are off by e as in test_gpu_kv, what rounds to nothing is below 2^-36 of the
    largest, and sums in 32 bits are off by 2^-24 for each addition: one workgroup for all adds a weight at a time in tiles, n / 4 to a lane (sums of eight by four waves for few rows), and
    16 weighted values at a time (32 by four waves)."""
    import torch
    dim, u = 64, {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    per = 16384 // (2 * dim)
    adds, mixes = (n // 4, n // 16) if new * 2 > 32 else (n // 128 + 16, n // 128)
    with Cache(bam, n // per, 1, dim, dtype, 16384) as c:
        c.k = c.v = None
        table = torch.arange(n // per, dtype=torch.int32).view(1, -1)
        q = torch.zeros(new, 2, dim, dtype=c.dtype)
        q[:, :, 0] = 8
        for peak in (0, 70001, n - new):
            k, v = torch.zeros(n, 1, dim, dtype=c.dtype, device="cuda"), torch.full((n, 1, dim), -1.0, dtype=c.dtype, device="cuda")
            k[peak, 0, 0] = low * np.log(2)          # times 8 and a scale of an eighth
            v[peak] = 1
            c.kv.append(k, v, _i32([n]), table.cuda(), starts=_starts([n]))
            x = float(k[peak, 0, 0])
            tail = (torch.arange(n - new, n, dtype=torch.float64) * np.exp(-x))[:, None, None]          # of the peak's weight
            want = (1 - tail) / (1 + tail)
            e = 2 * dim * 2.0 ** -24 * x
            tol = (1.01 * u + 2.0 ** -24 * adds) * want.abs() + 1.01 * u + 2.0 ** -24 * mixes + 2.0 ** -19 + e
            sums = x + torch.log1p(tail[:, :, 0]).expand(new, 2)
            for max_len in (n, 1):                   # split over the length, and by one workgroup
                got, lse = c.kv.attend(q.cuda(), _i32([n]), table.cuda(), starts=_starts([new]), max_new=new, max_len=max_len, return_lse=True)
                _near(got, want.expand(new, 2, dim), tol.expand(new, 2, dim), (peak, max_len))
                _near(lse, sums, 2.0 ** -24 * adds + 2.0 ** -19 + e + 2.0 ** -22 * sums.abs(), (peak, max_len))
        assert not c.rig.c.aborted()


# ---------------------------------------------------------------- counters

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n_seqs", [1, 200])
def test_a_split_that_is_done_again_counts_once(bam, dim, n_seqs):
    """an infinity among values that some rows see and others do not leaves a split to be done row by row: its pages are counted by whoever does it"""
    import torch
    with Cache(bam, 32, 2, dim, "bf16") as c:
        lens = [100]
        table = _table(lens, c.t, 32)
        v = torch.randn(100, 2, dim).to(c.dtype)
        v[98] = float("inf")
        c.fill(lens, table, v=v)
        q = torch.randn(3 * n_seqs, 4, dim).to(c.dtype).cuda()
        c.kv.array.stats()
        c.kv.attend(q, _i32(lens * n_seqs), table.cuda().expand(n_seqs, -1), starts=_starts([3] * n_seqs), max_new=3)
        st = c.kv.array.stats()
        assert st["access_cnt"] == st["hit_cnt"] == n_seqs * 2 * 2 * -(-100 // c.t), st


# ---------------------------------------------------------------- more new rows than were announced

@pytest.mark.parametrize("max_new", [1, 3, 20, 40, 70])
def test_rows_beyond_max_new_are_left(bam, max_new):
    """few rows, tiles of two and of four waves: of each sequence the first max_new rows are as without it, the others as the output was"""
    import torch
    lens, news = [150, 90, 130], [75, 2, 74]
    with Cache(bam, 32, 1, 128, "bf16") as c:
        table = _table(lens, c.t, 32)
        c.fill(lens, table)
        q = torch.randn(sum(news), 2, 128).to(c.dtype)
        want, tol, _ = c.want(q, lens, news, table)
        out = torch.full(q.shape, 7.0, dtype=c.dtype, device="cuda")
        c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), max_new=max_new, out=out)
        at = 0
        for n in news:
            m = min(n, max_new)
            _near(out[at:at + m], want[at:at + m], tol[at:at + m], at)
            assert bool((out[at + m:at + n] == 7).all()), at
            at += n


# ---------------------------------------------------------------- gradients

def test_tensors_that_require_gradients_are_refused(bam):
    """outputs carry no graph: what would be lost without a word is refused, unless gradients are not being recorded"""
    import torch
    with Cache(bam, 4, 1, 64, "bf16") as c:
        lens, table = _i32([1]), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
        x, w, angles = (torch.ones(*s, dtype=t, device="cuda") for s, t in (((1, 1, 64), c.dtype), ((64,), c.dtype), ((4, 32), torch.float32)))
        good = {"k": x, "v": x, "q": x, "q_norm": w, "k_norm": w, "cos": angles, "sin": angles}
        for name, t in good.items():
            args = dict(good, **{name: t.clone().requires_grad_()})
            k, v = args.pop("k"), args.pop("v")
            with pytest.raises(bam.BamError, match="gradients"):
                c.kv.append(k, v, lens, table, **args)
            with torch.no_grad():
                c.kv.append(k, v, lens, table, **args)
        with pytest.raises(bam.BamError, match="gradients"):
            c.kv.attend(x.clone().requires_grad_(), lens, table)
        with torch.inference_mode():
            assert not c.kv.attend(x.clone().requires_grad_(), lens, table).requires_grad


# ---------------------------------------------------------------- refusals

@pytest.mark.parametrize("wrong", [{"head_dim": 120}, {"head_dim": 48, "page_size": 512}, {"n_blocks": 0}, {"dtype": "float32"}, {"max_range": 0}])
def test_a_refused_cache_leaves_nothing_open(bam, wrong):
    """its page cache, range and array are closed when the error comes out, not when the error is let go of, which may be after the controller is gone"""
    import gc
    import torch
    from test_gpu_parity import Rig
    args = {"n_blocks": 4, "n_heads": 1, "head_dim": 64, "page_size": 4096, **wrong}
    if "dtype" in args:
        args["dtype"] = getattr(torch, args["dtype"])

    def open_ones():
        return {id(x): x for x in gc.get_objects() if type(x) in (bam.PageCache, bam.Range, bam.Array) and x.h}

    with Rig(bam, 1 << 20) as r:
        before = open_ones()
        with pytest.raises(bam.BamError) as kept:
            bam.make_kv_cache(r.c, **args)
        assert not open_ones().keys() - before.keys()
    assert "KVCache" in str(kept.value) or "bam_" in str(kept.value)


# ---------------------------------------------------------------- heads between the widths that kernels are built for

@pytest.mark.parametrize("dtype,dim,page", [("bf16", 144, 4096), ("f16", 176, 8192), ("bf16", 192, 16384), ("f16", 240, 4096), ("bf16", 112, 4096), ("f16", 48, 1024), ("bf16", 256, 4096)])
@pytest.mark.parametrize("group,news", [(1, [1, 1, 1]), (5, [4, 1, 3]), (2, [25, 3, 17]), (3, [30, 41, 2])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (37, 5)])
def test_other_head_sizes(bam, dtype, dim, page, group, news, window, sinks):
    """one row and few, tiles of two waves (33 to 64 rows of a head of keys) and of four; rows with norms and rotations into them and out"""
    import torch
    from test_gpu_kv import _rotated
    lens, heads = [200, 133, 90], 2
    gen = torch.Generator().manual_seed(dim)
    with Cache(bam, 160, heads, dim, dtype, page) as c:
        table = _table(lens, c.t, 160)
        c.fill(lens, table)
        n = sum(news)
        rows = c.rows_of(lens, news)
        x = torch.randn(3, n, heads * group, dim, generator=gen).to(c.dtype)
        w = (1 + 0.2 * torch.randn(2, dim, generator=gen)).to(c.dtype)
        rot = dim if group % 2 else dim // 32 * 16
        angle = torch.rand(200, rot // 2, generator=gen) * 6.28
        cos, sin, style = angle.cos(), angle.sin(), "half" if group > 1 else "pairs"
        dev = [c_.cuda() for c_ in (x[0, :, :heads], x[1, :, :heads], x[2])]
        q = c.kv.append(dev[0], dev[1], _i32(lens), table.cuda(), starts=_starts(news), q=dev[2], q_norm=w[0].cuda(), k_norm=w[1].cuda(), cos=cos.cuda(), sin=sin.cuda(), rotary=style)
        got_k, got_v = (y.cpu() for y in c.kv.read(n, _i32(lens), table.cuda(), starts=_starts(news)))
        assert torch.equal(got_v, x[1, :, :heads])
        for i, (b, p) in enumerate(rows):
            for h in range(heads):
                for got, row, weight in ((q[i, h], x[2, i, h], w[0]), (got_k[i, h], x[0, i, h], w[1])):
                    y, size = _rotated(row, weight, p, cos, sin, style, 1e-6)
                    _near(got, y, 1.01 * c.u * y.abs() + 2.0 ** -18 * size + 2.0 ** -25, (i, h))
        c.note(got_k, got_v, rows, table)
        want, tol, lse = c.want(q.cpu(), lens, news, table, window, sinks)
        got, got_lse = c.kv.attend(q, _i32(lens), table.cuda(), starts=_starts(news), max_new=max(news), window=window, sinks=sinks, return_lse=True)
        _near(got, want, tol)
        _near(got_lse, lse, 2.0 ** -16 * (1 + lse.abs()))
        assert not c.rig.c.aborted()


def test_arguments_out_of_range_are_refused(bam):
    """numbers that do not fit the fields of a call, and a store offset inside a page, which was taken for the page's beginning"""
    import torch
    from test_gpu_parity import Rig
    with Cache(bam, 4, 1, 64, "bf16") as c:
        x, lens, table = torch.ones(1, 1, 64, dtype=c.dtype, device="cuda"), _i32([1]), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
        for kw in ({"window": 1 << 31}, {"window": (1 << 32) + 5}, {"sinks": 1 << 40}, {"max_len": 1 << 31}, {"scale": 1e39}, {"scale": "x"}):
            with pytest.raises(bam.BamError):
                c.kv.attend(x, lens, table, **kw)
        for kw in ({"eps": 1e39, "k_norm": x[0, 0]}, {"eps": -1e-6, "k_norm": x[0, 0]}, {"eps": float("nan"), "q": x, "q_norm": x[0, 0]}, {"eps": None}):
            with pytest.raises(bam.BamError):
                c.kv.append(x, x, lens, table, **kw)
        with pytest.raises(bam.BamError):
            c.kv.read(-1, lens, table, starts=_starts([1]))
    with Rig(bam, 1 << 20) as r:
        for offset in (1, 4095, -4096):
            with pytest.raises(bam.BamError):
                bam.make_kv_cache(r.c, 4, 1, 64, disk_offset_bytes=offset)
        bam.make_kv_cache(r.c, 4, 1, 64, disk_offset_bytes=8192).close()
