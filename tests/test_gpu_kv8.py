"""The key-value cache in 8 bits: rows in and out, and attention over it, against the definition in 64 bits on the CPU.

What is kept of a row is worked out here in 64 bits without the eight-bit type: k the least whole number for which the row's largest is at most 448 * 2^k, numbers as
multiples of an eighth of their own power of two (of 2^-9 below 2^-6).  Values go in as they are, and keys are normed and turned in 64 bits, so what comes out has to be that, number for number
(test_keys_are_rounded_once); beside the number itself it is off by half a step (2^-4 of the number, or 2^-10 * 2^k), for which test_rows_in_and_out leaves 2^-17 of the terms that were added up besides.  Attention goes over what the cache holds, by the bounds of test_gpu_kv.
"""
import numpy as np
import pytest

from test_gpu_kv import UNIT, Cache, _i32, _near, _rotated, _starts, _table, _type
from test_gpu_parity import Rig, bam  # noqa: F401  (bam is the module fixture)

pytestmark = pytest.mark.gpu

POWERS = {"bf16": (-110, 120), "f16": (-24, 8)}
MOST = {"bf16": 1.875 * 2.0 ** 127, "f16": 1.875 * 2.0 ** 15}


def _powers(x, dtype):
    """k of each row, in 64 bits"""
    import torch
    low, high = POWERS[dtype]
    top = torch.where(torch.isfinite(x), x.double().abs(), torch.zeros(())).clamp(max=MOST[dtype]).amax(-1)
    part, e = torch.frexp(top)                       # top = part * 2^e, a half <= part < 1
    k = e - 9 + (part > 0.875)
    return torch.where(top > 0, k, torch.full_like(k, low)).clamp(low, high)


def _kept(x, dtype):
    """what rows stand for, in 64 bits"""
    import torch
    k = _powers(x, dtype)[..., None]
    y = torch.ldexp(x.double().clamp(-MOST[dtype], MOST[dtype]), -k)
    unit = torch.ldexp(torch.ones((), dtype=torch.float64), torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4)
    y = torch.ldexp(torch.round(y / unit) * unit, k)
    return torch.where(torch.isfinite(x), y, torch.full_like(y, float("nan")))


class Cache8(Cache):
    """as Cache, in 8 bits: what it should hold is rounded"""

    def __init__(self, bam, n_blocks, heads, dim, dtype, page=4096, cache_pages=None, backing=False, scales=None):
        import torch
        self.dtype, self.name, self.heads, self.dim, self.n_blocks = _type(dtype), dtype, heads, dim, n_blocks
        self.u = UNIT[dtype]
        self.rig = Rig(bam, 2 * n_blocks * heads * page, backing=backing, n_queues=8, depth=128)
        self.kv = bam.make_kv_cache(self.rig.c, n_blocks, heads, dim, page_size=page, cache_pages=cache_pages, dtype=self.dtype, stored=torch.float8_e4m3fn, scales=scales)
        self.t = self.kv.block_tokens
        assert self.t == 1 << ((page // dim).bit_length() - 1) and self.kv.stored is torch.float8_e4m3fn
        self.k = torch.zeros(n_blocks, heads, self.t, dim, dtype=torch.float64)
        self.v = torch.zeros_like(self.k)

    def note(self, k, v, rows, table):
        super().note(_kept(k, self.name), _kept(v, self.name), rows, table)


def _same(got, want):
    """bit for bit but for a zero's sign and a NaN's bits"""
    import torch
    got, want = got.cpu(), want.to(got.dtype)
    bad = ~((got == want) | (torch.isnan(got) & torch.isnan(want)))
    assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


# ---------------------------------------------------------------- rows

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,page", [(64, 4096), (128, 4096), (256, 4096), (16, 512), (80, 4096), (208, 8192)])
def test_every_number_of_the_type(bam, dtype, dim, page):
    """all 65536 bit patterns, sorted by magnitude and at random, in rows beside others: each comes out as it has to, infinities as NaN"""
    import torch
    every = torch.arange(65536).to(torch.int32).to(torch.int16).view(_type(dtype))
    order = torch.argsort(every.abs().float(), stable=True)
    mixed = torch.randperm(65536, generator=torch.Generator().manual_seed(1))
    n = 2 * 65536 // dim
    x = torch.cat([every[order], every[mixed]])[:n * dim].view(n, 1, dim)
    with Cache8(bam, 2 + n // (1 << ((page // dim).bit_length() - 1)), 1, dim, dtype, page) as c:
        table = _table([n], c.t, c.n_blocks)
        c.kv.append(x.flip(0).cuda(), x.cuda(), _i32([n]), table.cuda(), starts=_starts([n]))
        k, v = c.kv.read(n, _i32([n]), table.cuda(), starts=_starts([n]))
        _same(v, _kept(x, dtype))
        _same(k, _kept(x.flip(0), dtype))
        # and the powers of two, in the order of the pages
        for p in (0, 1, n // 2, n - 1):
            got = c.kv.scales[int(table[0, p // c.t]), 0, :, p % c.t].cpu().int() - 127
            assert got.tolist() == [int(_powers(x[n - 1 - p, 0], dtype)), int(_powers(x[p, 0], dtype))], p


@pytest.mark.parametrize("dtype,dim,heads,q_heads,page,rot,style,norm,lens,news", [
    ("bf16", 128, 2, 8, 4096, 128, "half", True, [1, 33, 16, 100], [1, 1, 1, 1]),
    ("f16", 64, 3, 3, 4096, 32, "pairs", False, [5, 64, 31], [5, 40, 1]),
    ("bf16", 80, 1, 5, 4096, 80, "half", True, [17, 200], [17, 77]),
    ("f16", 256, 2, 2, 4096, 256, "pairs", True, [9, 8, 40], [9, 0, 33]),
    ("bf16", 16, 1, 1, 512, 16, "half", False, [50], [23]),
    ("f16", 96, 2, 4, 16384, 48, "half", True, [300, 130], [129, 130]),
    ("bf16", 128, 2, 0, 8192, 0, "half", True, [70], [70]),
])
@pytest.mark.parametrize("aligned", [True, False])
def test_rows_in_and_out(bam, dtype, dim, heads, q_heads, page, rot, style, norm, lens, news, aligned):
    import torch
    gen = torch.Generator().manual_seed(11)
    n, dt, eps = sum(news), _type(dtype), 1e-5
    with Cache8(bam, 64, heads, dim, dtype, page) as c:
        table = _table(lens, c.t, 64)
        before = [a - b for a, b in zip(lens, news)]
        if sum(before):
            c.fill(before, table)
        qkv = (torch.randn(n, q_heads + 2 * heads, dim, generator=gen) * torch.exp(torch.randn(n, 1, 1, generator=gen) * 2)).to(dt)
        dev = qkv.cuda() if aligned else torch.cat([qkv, qkv[..., :3]], -1).cuda()[..., :dim]
        q, k, v = dev[:, :q_heads], dev[:, q_heads:q_heads + heads], dev[:, q_heads + heads:]
        w = (1 + 0.2 * torch.randn(2, dim, generator=gen)).to(dt)
        angle = torch.rand(max(lens), rot // 2, generator=gen) * 6.28
        cos, sin = (angle.cos(), angle.sin()) if rot else (None, None)
        got = c.kv.append(k, v, _i32(lens), table.cuda(), starts=_starts(news), q=q if q_heads else None, q_norm=w[0].cuda() if norm and q_heads else None,
                          k_norm=w[1].cuda() if norm else None, eps=eps, cos=cos.cuda() if rot else None, sin=sin.cuda() if rot else None, rotary=style)
        got_k, got_v = c.kv.read(n, _i32(lens), table.cuda(), starts=_starts(news))
        _same(got_v, _kept(qkv[:, q_heads + heads:], dtype))
        for i, (b, p) in enumerate(c.rows_of(lens, news)):
            for h in range(q_heads + heads):
                is_q = h < q_heads
                y, size = _rotated(qkv[i, h], (w[0] if is_q else w[1]) if norm else None, p, cos, sin, style, eps)
                if is_q:
                    _near(got[i, h], y, 1.01 * c.u * y.abs() + 2.0 ** -18 * size + 2.0 ** -25, (i, h))
                else:
                    k_top = float(_powers(y * (1 + 2.0 ** -17), dtype))
                    _near(got_k[i, h - q_heads], y, 1.01 * 2.0 ** -4 * y.abs() + 2.0 ** (k_top - 10) + 2.0 ** -17 * size + 2.0 ** -25, (i, h))
        # what was there before is as it was
        if sum(before):
            old_k, old_v = c.kv.read(sum(before), _i32(before), table.cuda(), starts=_starts(before))
            rows = c.rows_of(before, before)
            _same(old_k, torch.stack([c.k[int(table[b, p // c.t]), :, p % c.t] for b, p in rows]))
            _same(old_v, torch.stack([c.v[int(table[b, p // c.t]), :, p % c.t] for b, p in rows]))
        assert not c.rig.c.aborted()


@pytest.mark.parametrize("dtype,dim,page,rot,style,norm", [("bf16", 128, 4096, 128, "half", True), ("bf16", 64, 4096, 32, "pairs", True), ("f16", 256, 4096, 256, "half", True), ("f16", 80, 4096, 64, "half", False),
                                                           ("bf16", 96, 8192, 0, "half", True), ("f16", 16, 512, 16, "pairs", True)])
def test_keys_are_rounded_once(bam, dtype, dim, page, rot, style, norm):
    """what is kept of a key is what the definition in 64 bits rounds to, number for number: of rows of all sizes, and rows that are tiny beside eps.  (Borders of two codes that 64 bits miss by their
    own error of some 2^-50 are not met.)"""
    import torch
    gen = torch.Generator().manual_seed(dim)
    n, dt, eps = 700, _type(dtype), 2.0 ** -17
    with Cache8(bam, 2 + n // (1 << ((page // dim).bit_length() - 1)), 1, dim, dtype, page) as c:
        table = _table([n], c.t, c.n_blocks)
        k = (torch.randn(n, 1, dim, generator=gen) * torch.exp2(torch.randint(-9, 9, (n, 1, 1), generator=gen).float())).to(dt)
        w = (1 + 0.2 * torch.randn(dim, generator=gen)).to(dt) if norm else None
        angle = torch.rand(n, rot // 2, generator=gen) * 6.28
        cos, sin = (angle.cos(), angle.sin()) if rot else (None, None)
        c.kv.append(k.cuda(), k.cuda(), _i32([n]), table.cuda(), starts=_starts([n]), k_norm=None if w is None else w.cuda(), eps=eps, cos=cos.cuda() if rot else None, sin=sin.cuda() if rot else None, rotary=style)
        got, _ = c.kv.read(n, _i32([n]), table.cuda(), starts=_starts([n]))
        want = torch.stack([_rotated(k[i, 0], w, i, cos, sin, style, eps)[0] for i in range(n)])
        _same(got[:, 0], _kept(want, dtype))


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype,dim,heads,group,page,lens,news,window,sinks", [
    ("bf16", 128, 2, 4, 4096, [1, 2, 31, 32, 33, 300], [1] * 6, 0, 0),
    ("f16", 64, 1, 1, 4096, [1, 129, 511], [1] * 3, 0, 0),
    ("bf16", 256, 1, 8, 4096, [77, 8], [1] * 2, 0, 0),
    ("f16", 96, 2, 3, 4096, [200, 65], [1] * 2, 40, 3),
    ("bf16", 80, 1, 16, 8192, [257, 100], [1] * 2, 64, 0),
    ("f16", 16, 1, 2, 512, [1000], [1], 100, 70),
    ("bf16", 32, 2, 20, 16384, [700], [1], 0, 0),
    ("bf16", 64, 1, 40, 4096, [130], [1], 0, 0),
    ("f16", 128, 1, 2, 4096, [150, 3, 40], [3, 3, 3], 0, 0),
    ("bf16", 128, 2, 1, 4096, [130, 260], [4, 4], 33, 2),
    ("f16", 64, 2, 4, 4096, [77], [77], 0, 0),
    ("bf16", 128, 1, 5, 4096, [70, 90, 5, 64], [70, 21, 5, 0], 0, 0),
    ("f16", 128, 2, 2, 8192, [200, 129], [200, 65], 48, 4),
    ("bf16", 80, 1, 3, 4096, [150], [131], 0, 0),
    ("f16", 256, 1, 2, 16384, [90], [90], 0, 0),
    ("bf16", 256, 2, 4, 4096, [200, 60], [100, 20], 0, 0),
    ("f16", 208, 1, 2, 4096, [150], [140], 40, 3),
    ("bf16", 144, 1, 2, 4096, [150], [20], 0, 0),
    ("bf16", 96, 2, 1, 4096, [333], [333], 100, 17),
])
def test_attention(bam, dtype, dim, heads, group, page, lens, news, window, sinks):
    import torch
    gen = torch.Generator().manual_seed(5)
    with Cache8(bam, 256, heads, dim, dtype, page) as c:
        table = _table(lens, c.t, 256)
        n_all = sum(lens)
        # rows of different sizes: each has a power of two of its own
        by = torch.exp2(torch.randint(-3, 2, (2, n_all, heads, 1), generator=gen).float())
        k, v = (torch.randn(2, n_all, heads, dim, generator=gen) * by).to(c.dtype)
        c.fill(lens, table, k=k, v=v)
        n = sum(news)
        q = (torch.randn(n, heads * group, dim, generator=gen) * 1.5).to(c.dtype)
        want, tol, lse = c.want(q, lens, news, table, window, sinks)
        one = all(m == 1 for m in news)
        for starts in ([None, _starts(news)] if one else [_starts(news)]):
            got, got_lse = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=starts, max_new=max(news), window=window, sinks=sinks, return_lse=True)
            _near(got, want, tol)
            _near(got_lse, lse, 2.0 ** -16 * (1 + lse.abs()))
        for max_len in (1, 64, 1 << 20):
            _near(c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), max_new=max(news), max_len=max_len, window=window, sinks=sinks), want, tol, max_len)
        _near(c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), window=window, sinks=sinks, scale=-0.3), *c.want(q, lens, news, table, window, sinks, -0.3)[:2])
        assert not c.rig.c.aborted()


@pytest.mark.parametrize("dtype,group,news", [("bf16", 4, [1, 1, 1, 1, 1]), ("f16", 2, [3, 1, 4, 2, 5]), ("bf16", 3, [50, 40, 30, 1, 60])])
def test_rows_that_see_nothing(bam, dtype, group, news):
    import torch
    with Cache8(bam, 64, 1, 128, dtype) as c:
        lens = [0, 2, 90, 33, 64]
        table = _table([64, 64, 96, 64, 64], c.t, 64, width=3)
        c.fill([64, 64, 96, 64, 64], table)
        table[2, 1] = -1
        table[3, 0] = 64
        table[3, 1] = 1 << 30
        n = sum(news)
        q = torch.randn(n, group, 128).to(c.dtype)
        want, tol, lse = c.want(q, lens, news, table)
        got, got_lse = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), return_lse=True)
        _near(got, want, tol)
        empty = torch.isinf(lse)
        assert bool(empty.any()) and bool((got.cpu()[empty] == 0).all()) and bool((got_lse.cpu()[empty] == -np.inf).all())
        long = [200, 2, 96, 33, 300]
        _near(c.kv.attend(q.cuda(), _i32(long), table.cuda(), starts=_starts(news)), *c.want(q, long, news, table)[:2])
        assert not c.rig.c.aborted()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), "scale"])
@pytest.mark.parametrize("window,sinks,new", [(0, 0, 1), (0, 0, 6), (0, 0, 90), (40, 2, 1), (40, 2, 5), (40, 2, 90)])
def test_what_is_not_seen_may_be_anything(bam, dtype, odd, window, sinks, new):
    """what is not finite at tokens to come, behind the window and past the end, and past the end powers of two that no row has: rows that do not see them are as without, those that do show them"""
    import torch
    lens = [100]
    with Cache8(bam, 16, 1, 64, dtype) as c:
        table = _table([128], c.t, 16)
        k = torch.randn(128, 1, 64).to(c.dtype)
        v = torch.randn(128, 1, 64).to(c.dtype)
        c.fill([128], table, k=k, v=v)
        q = torch.randn(new, 2, 64).to(c.dtype)
        want, tol, _ = c.want(q, lens, [new], table, window, sinks)
        for what in ("k", "v"):
            for at in (99, 97, 110, 20, 5) if odd != "scale" else (110, 127):
                bad_k, bad_v = k.clone(), v.clone()
                if odd != "scale":
                    (bad_k if what == "k" else bad_v)[at] = odd
                c.fill([128], table, k=bad_k, v=bad_v)
                if odd == "scale":
                    c.kv.scales[int(table[0, at // c.t]), 0, 0 if what == "k" else 1, at % c.t] = 255
                got = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts([new]), window=window, sinks=sinks).cpu()
                for i, (_, p) in enumerate(c.rows_of(lens, [new])):
                    if not (at <= p and (not window or p - at < window or at < sinks)):
                        _near(got[i], want[i], tol[i], (what, at, i))
                    elif odd != "scale":
                        assert bool(torch.isnan(got[i]).all()), (what, at, i)


@pytest.mark.parametrize("dim,page,heads,cache_pages,new", [(128, 4096, 2, 32, 1), (128, 4096, 2, 40, 40), (64, 4096, 1, 16, 3), (256, 4096, 1, 32, 1), (256, 4096, 1, 32, 70), (32, 512, 1, 64, 9), (128, 8192, 1, 33, 70)])
def test_a_cache_smaller_than_what_is_kept(bam, dim, page, heads, cache_pages, new):
    """what does not fit goes to the store and comes back: rows, attention over all of them, and the store's own content; a cache that is opened again over the pages, with the scales"""
    import torch
    t = 1 << ((page // dim).bit_length() - 1)
    n_blocks = 40
    lens = [12 * t + 3, 20 * t, 5]
    with Cache8(bam, n_blocks, heads, dim, "bf16", page, cache_pages=cache_pages, backing=True) as c:
        table = _table(lens, c.t, n_blocks)
        k, v = c.fill(lens, table)
        for _ in range(2):
            got_k, got_v = c.kv.read(sum(lens), _i32(lens), table.cuda(), starts=_starts(lens))
            _same(got_k, _kept(k, "bf16"))
            _same(got_v, _kept(v, "bf16"))
        news = [new, new, min(new, 5)]
        q = torch.randn(sum(news), 2 * heads, dim).to(torch.bfloat16)
        want, tol, _ = c.want(q, lens, news, table)
        for _ in range(3):
            _near(c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), max_new=new), want, tol)
        st = c.kv.array.stats()
        assert st["read_io_cnt"] > 0 and st["hit_cnt"] + st["miss_cnt"] == st["access_cnt"], st
        # one more token each, in blocks that are on the store
        k1, v1 = torch.randn(3, heads, dim).to(torch.bfloat16), torch.randn(3, heads, dim).to(torch.bfloat16)
        c.kv.append(k1.cuda(), v1.cuda(), _i32(lens), table.cuda())
        c.note(k1, v1, c.rows_of(lens, [1, 1, 1]), table)
        torch.cuda.synchronize()
        c.kv._owned[2].flush()
        torch.cuda.synchronize()
        codes = c.rig.backing(2 * n_blocks * heads * page // 8).view(np.uint8).reshape(n_blocks, heads, 2, page)
        scales = c.kv.scales.cpu().int().numpy() - 127
        for b, n in enumerate(lens):
            for p in (0, n // 2, n - 1):
                block, x = int(table[b, p // t]), p % t
                place = (x & ~12) | (x & 4) << 1 | (x & 8) >> 1
                for h in range(heads):
                    keys = codes[block, h, 0, :t * dim].reshape(dim // 16, t, 16)[:, place].reshape(-1)
                    values = codes[block, h, 1, :t * dim].reshape(t // 8, dim // 2, 8, 2)[x // 8, :, x % 8].reshape(-1)
                    for got, kept, kind in ((keys, c.k, 0), (values, c.v, 1)):
                        y = torch.from_numpy(got.copy()).view(torch.float8_e4m3fn).double() * 2.0 ** int(scales[block, h, kind, x])
                        assert torch.equal(y, kept[block, h, x])
        # another handle over the same pages
        again = bam.KVCache(c.kv.array, heads, dim, torch.bfloat16, n_blocks=n_blocks, stored=torch.float8_e4m3fn, scales=c.kv.scales)
        q = torch.randn(3, 2 * heads, dim).to(torch.bfloat16)
        _near(again.attend(q.cuda(), _i32(lens), table.cuda()), *c.want(q, lens, [1, 1, 1], table)[:2])
        again.close()
        assert not c.rig.c.aborted()


def test_streams_and_graphs(bam):
    """on another stream than the tensors' own, and replayed several times with other work between, as eagerly"""
    import torch
    lens, news, hq = [150, 90, 33], [1, 1, 1], 8
    with Cache8(bam, 64, 2, 128, "bf16") as c:
        table = _table([200, 200, 200], c.t, 64).cuda()
        dl = _i32(lens)
        c.fill(lens, table.cpu())
        k = torch.randn(3, 2, 128).to(torch.bfloat16).cuda()
        v, q = k.flip(2).contiguous(), torch.randn(3, hq, 128).to(torch.bfloat16).cuda()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            c.kv.append(k, v, dl, table)
            eager = c.kv.attend(q, dl, table)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        q_in, out = q.clone(), torch.empty_like(q)
        with torch.cuda.graph(graph):
            dl.add_(1)
            c.kv.append(k, v, dl, table)
            c.kv.attend(q_in, dl, table, out=out)
        dl.copy_(_i32([n - 1 for n in lens]))
        for step in range(4):
            graph.replay()
            torch.cuda.synchronize()
            now = [n + step for n in lens]
            c.note(k.cpu(), v.cpu(), c.rows_of(now, news), table.cpu())
            again = c.kv.attend(q, _i32(now), table)
            assert torch.equal(out, again), step
            if step == 0:
                assert torch.equal(out, eager)
            _near(out, *c.want(q.cpu(), now, news, table.cpu())[:2])


@pytest.mark.parametrize("new", [1, 40])
def test_with_reads_without_a_reference_switched_off(bam, monkeypatch, new):
    import torch
    monkeypatch.setenv("BAM_FAST_READS", "0")
    lens = [100, 45]
    with Cache8(bam, 32, 2, 64, "bf16") as c:
        table = _table(lens, c.t, 32)
        c.fill(lens, table)
        q = torch.randn(2 * new, 4, 64).to(torch.bfloat16)
        want, tol, _ = c.want(q, lens, [new, new], table, 50, 2)
        _near(c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts([new, new]), window=50, sinks=2), want, tol)
        assert not c.rig.c.aborted()


def test_refusals(bam):
    import torch
    e4 = torch.float8_e4m3fn
    with Rig(bam, 1 << 20) as r:
        a = r.array((1 << 20) // 8, 4096, 64)
        good = torch.zeros(16, 1, 2, 32, dtype=torch.uint8, device="cuda")
        for kw in ({"stored": torch.float8_e5m2}, {"stored": torch.float16}, {"stored": None, "scales": good}, {"head_dim": 120}, {"head_dim": 0}, {"head_dim": 272}, {"n_heads": 0}, {"n_blocks": 0},
                   {"n_blocks": -1}, {"scales": good[:15]}, {"scales": good.int()}, {"scales": good.cpu()}, {"scales": good.transpose(0, 3)}, {"n_blocks": 129, "scales": None}, {"dtype": torch.float32}):
            with pytest.raises(bam.BamError):
                bam.KVCache(a, **{"n_heads": 1, "head_dim": 128, "n_blocks": 16, "stored": e4, "scales": good if "stored" not in kw else None, **kw})
        with pytest.raises(bam.BamError):
            bam.KVCache(r.array(1 << 12, 512, 64), 1, 64, n_blocks=1, stored=e4)                # eight rows to a page
        kv = bam.KVCache(a, 1, 128, n_blocks=16, stored=e4, scales=good)
        assert kv.scales is good and kv.block_tokens == 32
        kv.close()
        kv = bam.KVCache(a, 1, 128, n_blocks=16, stored=torch.bfloat16)
        assert kv.scales is None and kv.block_tokens == 16
        kv.close()


@pytest.mark.parametrize("dtype,dim,page", [("bf16", 144, 4096), ("f16", 176, 8192), ("bf16", 192, 16384), ("f16", 240, 4096), ("bf16", 112, 4096), ("f16", 48, 1024), ("bf16", 256, 4096), ("f16", 80, 4096), ("bf16", 96, 8192), ("f16", 64, 1024)])
@pytest.mark.parametrize("group,news", [(1, [1, 1, 1]), (5, [4, 1, 3]), (2, [25, 3, 17]), (3, [30, 41, 2])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (37, 5)])
def test_other_head_sizes(bam, dtype, dim, page, group, news, window, sinks):
    """one row and few, tiles of two waves (33 to 64 rows of a head of keys) and of four, blocks of 16 tokens and more"""
    import torch
    lens, heads = [200, 133, 90], 2
    gen = torch.Generator().manual_seed(dim)
    with Cache8(bam, 100, heads, dim, dtype, page) as c:
        table = _table(lens, c.t, 100)
        c.fill(lens, table)
        q = torch.randn(sum(news), heads * group, dim, generator=gen).to(c.dtype)
        want, tol, lse = c.want(q, lens, news, table, window, sinks)
        got, got_lse = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), max_new=max(news), window=window, sinks=sinks, return_lse=True)
        _near(got, want, tol)
        _near(got_lse, lse, 2.0 ** -16 * (1 + lse.abs()))
        assert not c.rig.c.aborted()
