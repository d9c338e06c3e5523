"""The key-value cache in the pages of an array: rows in and out, and attention over it, against the definition in 64 bits on the CPU.

Tolerances, for outputs rounded to a type of unit roundoff u (2^-8 of bfloat16 with its 8 bits, 2^-11 of float16 with 11), are bounds worked out for each element:
rows: u |y| for the rounding, and 2^-18 of the terms that were added up for 32-bit arithmetic of a few hundred steps;
attention: u |y| for the rounding, and of sum_t w_t |v_t| a share of u (weights are rounded to the type once), 2^-18 (32-bit sums) and twice the error of a
score in 32 bits, D 2^-24 sum |q k| scale; in float16, weights below 2^-14 of the largest are rounded to multiples of 2^-24.
"""
import numpy as np
import pytest

from test_gpu_parity import Rig, SEED, bam  # noqa: F401  (bam is the module fixture)

pytestmark = pytest.mark.gpu

UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _type(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


class Cache:
    """A key-value cache on a store of its own and, beside it, what it should hold: [block][head][token][dim] in the cache's type on the CPU."""

    def __init__(self, bam, n_blocks, heads, dim, dtype, page=4096, cache_pages=None, backing=False, fail_every=0):
        import torch
        self.dtype, self.heads, self.dim, self.n_blocks = _type(dtype), heads, dim, n_blocks
        self.u = UNIT[dtype]
        self.rig = Rig(bam, 2 * n_blocks * heads * page, backing=backing, n_queues=8, depth=128)
        self.kv = bam.make_kv_cache(self.rig.c, n_blocks, heads, dim, page_size=page, cache_pages=cache_pages, dtype=self.dtype)
        self.t = self.kv.block_tokens
        assert self.t == 1 << ((page // (2 * dim)).bit_length() - 1)
        self.k = torch.zeros(n_blocks, heads, self.t, dim, dtype=self.dtype)
        self.v = torch.zeros_like(self.k)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.kv.close()
        self.rig.close()

    def rows_of(self, lens, news):
        """(sequence, position) of every packed row"""
        return [(b, n - m + j) for b, (n, m) in enumerate(zip(lens, news)) for j in range(m)]

    def note(self, k, v, rows, table):
        for i, (b, p) in enumerate(rows):
            if p < 0 or p // self.t >= table.shape[1]:
                continue
            block = int(table[b, p // self.t])
            if 0 <= block < self.n_blocks:
                self.k[block, :, p % self.t] = k[i]
                self.v[block, :, p % self.t] = v[i]

    def fill(self, lens, table, seed=1, k=None, v=None):
        """all tokens of all sequences go in as new rows"""
        import torch
        gen = torch.Generator().manual_seed(seed)
        n = sum(lens)
        k = torch.randn(n, self.heads, self.dim, generator=gen).to(self.dtype) if k is None else k
        v = (torch.randn(n, self.heads, self.dim, generator=gen) + 0.5).to(self.dtype) if v is None else v
        self.kv.append(k.cuda(), v.cuda(), _i32(lens), table.cuda(), starts=_starts(lens))
        self.note(k, v, self.rows_of(lens, lens), table)
        return k, v

    def want(self, q, lens, news, table, window=0, sinks=0, scale=None):
        """outputs, bounds of their errors, and logarithms of sums, in 64 bits"""
        import torch
        hq = q.shape[1]
        group = hq // self.heads
        scale = self.dim ** -0.5 if scale is None else scale
        out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
        lse = torch.full(q.shape[:2], -np.inf, dtype=torch.float64)
        k64, v64, q64 = self.k.double(), self.v.double(), q.double()
        for i, (b, p) in enumerate(self.rows_of(lens, news)):
            seen = [t for t in range(max(0, p + 1)) if not window or p - t < window or t < sinks]
            seen = [t for t in seen if t // self.t < table.shape[1] and 0 <= int(table[b, t // self.t]) < self.n_blocks]
            if not seen:
                continue
            t = torch.tensor(seen)
            block = table[b].long()[t // self.t]
            for h in range(hq):
                k, v = k64[block, h // group, t % self.t], v64[block, h // group, t % self.t]
                x = k @ q64[i, h] * scale
                lse[i, h] = torch.logsumexp(x, 0)
                w = torch.exp(x - lse[i, h])
                out[i, h] = w @ v
                e = self.dim * 2.0 ** -24 * float((k.abs() @ q64[i, h].abs()).max()) * abs(scale)
                mass = w @ v.abs()
                tol[i, h] = 1.01 * self.u * out[i, h].abs() + (1.01 * self.u + 2.0 ** -18 + 2 * e) * mass + 1e-12
                if self.dtype == torch.float16:
                    tol[i, h] += 2.0 ** -24 * v.abs().sum(0) / float(torch.exp(x - x.max()).sum()) + 2.0 ** -25
        return out, tol, lse


def _i32(x):
    import torch
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def _starts(news):
    return _i32(np.concatenate([[0], np.cumsum(news)]))


def _table(lens, t, n_blocks, seed=3, width=None):
    import torch
    need = [-(-max(n, 0) // t) for n in lens]
    assert sum(need) <= n_blocks
    order = torch.randperm(n_blocks, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    out = torch.full((len(lens), max(max(need), 1) if width is None else width), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        out[b, :k] = order[at:at + k]
        at += k
    return out


def _near(got, want, tol, what=""):
    import torch
    got = got.double().cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - want).abs().max()), float((got - want).abs().sub(tol).max()), torch.nonzero(bad)[:4].tolist())


# ---------------------------------------------------------------- rows

def _rotated(x, weight, pos, cos, sin, style, eps):
    """one row in 64 bits, and the size of what was added up for each number"""
    import torch
    x = x.double().clone()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean() + eps) * weight.double()
    size = x.abs()
    if cos is not None:
        c, s, half = cos[pos].double(), sin[pos].double(), cos.shape[1]
        i = torch.arange(half)
        a, b = (i, i + half) if style == "half" else (2 * i, 2 * i + 1)
        y = x.clone()
        y[a], y[b] = x[a] * c - x[b] * s, x[b] * c + x[a] * s
        size = size.clone()
        size[a] = size[b] = x[a].abs() + x[b].abs()
        return y, size
    return x, size


@pytest.mark.parametrize("dtype,dim,heads,q_heads,page,rot,style,norm,lens,news", [
    ("bf16", 128, 2, 8, 4096, 128, "half", True, [1, 33, 16, 100], [1, 1, 1, 1]),
    ("f16", 64, 3, 3, 4096, 32, "pairs", False, [5, 64, 31], [5, 40, 1]),
    ("bf16", 80, 1, 5, 4096, 80, "half", True, [17, 200], [17, 77]),
    ("f16", 256, 2, 2, 4096, 256, "pairs", True, [9, 8, 40], [9, 0, 33]),
    ("bf16", 16, 1, 1, 512, 16, "half", False, [50], [23]),
    ("f16", 96, 2, 4, 16384, 48, "half", True, [300, 130], [129, 130]),
    ("bf16", 128, 2, 0, 8192, 0, "half", True, [70], [70]),
])
def test_rows_in_and_out(bam, dtype, dim, heads, q_heads, page, rot, style, norm, lens, news):
    import torch
    gen = torch.Generator().manual_seed(11)
    n, dt, eps = sum(news), _type(dtype), 1e-5
    with Cache(bam, 64, heads, dim, dtype, page) as c:
        table = _table(lens, c.t, 64)
        before = [a - b for a, b in zip(lens, news)]
        if sum(before):
            c.fill(before, table)
        qkv = (torch.randn(n, q_heads + 2 * heads, dim, generator=gen) * 2).to(dt)
        dev = qkv.cuda()
        q, k, v = dev[:, :q_heads], dev[:, q_heads:q_heads + heads], dev[:, q_heads + heads:]
        w = (1 + 0.2 * torch.randn(2, dim, generator=gen)).to(dt)
        angle = torch.rand(max(lens), rot // 2, generator=gen) * 6.28
        cos, sin = (angle.cos(), angle.sin()) if rot else (None, None)
        got = c.kv.append(k, v, _i32(lens), table.cuda(), starts=_starts(news), q=q if q_heads else None, q_norm=w[0].cuda() if norm and q_heads else None,
                          k_norm=w[1].cuda() if norm else None, eps=eps, cos=cos.cuda() if rot else None, sin=sin.cuda() if rot else None, rotary=style)
        got_k, got_v = c.kv.read(n, _i32(lens), table.cuda(), starts=_starts(news))
        assert torch.equal(got_v.cpu().view(torch.int16), qkv[:, q_heads + heads:].contiguous().view(torch.int16))
        for i, (b, p) in enumerate(c.rows_of(lens, news)):
            for h in range(q_heads + heads):
                is_q = h < q_heads
                y, size = _rotated(qkv[i, h], (w[0] if is_q else w[1]) if norm else None, p, cos, sin, style, eps)
                g = got[i, h] if is_q else got_k[i, h - q_heads]
                _near(g, y, 1.01 * c.u * y.abs() + 2.0 ** -18 * size + 2.0 ** -25, (i, h))
        # what was there before is as it was
        if sum(before):
            old_k, old_v = c.kv.read(sum(before), _i32(before), table.cuda(), starts=_starts(before))
            rows = c.rows_of(before, before)
            want_k = torch.stack([c.k[int(table[b, p // c.t]), :, p % c.t] for b, p in rows])
            want_v = torch.stack([c.v[int(table[b, p // c.t]), :, p % c.t] for b, p in rows])
            assert torch.equal(old_k.cpu(), want_k) and torch.equal(old_v.cpu(), want_v)
        assert not c.rig.c.aborted()


def test_rows_without_a_place_are_dropped(bam):
    """positions before the first, past the table, blocks the cache does not have: nothing is written, and they read as zeros; a position past the tables of
    angles gives NaN"""
    import torch
    with Cache(bam, 8, 1, 64, "bf16") as c:
        assert c.t == 32
        table = torch.tensor([[0, 1], [2, -1], [3, 8], [4, 5]], dtype=torch.int32)
        c.fill([64, 32, 32, 64], table)
        lens, news = [70, 40, 64, 2], [10, 16, 40, 4]
        n = sum(news)
        k = torch.randn(n, 1, 64).to(torch.bfloat16)
        v = torch.randn(n, 1, 64).to(torch.bfloat16)
        c.kv.append(k.cuda(), v.cuda(), _i32(lens), table.cuda(), starts=_starts(news))
        rows = c.rows_of(lens, news)
        c.note(k, v, rows, table)
        has = torch.tensor([p >= 0 and p // c.t < 2 and 0 <= int(table[b, p // c.t]) < 8 for b, p in rows])
        assert 0 < int(has.sum()) < n
        got_k, got_v = c.kv.read(n, _i32(lens), table.cuda(), starts=_starts(news))
        assert torch.equal(got_k.cpu(), torch.where(has[:, None, None], k, torch.zeros_like(k)))
        assert torch.equal(got_v.cpu(), torch.where(has[:, None, None], v, torch.zeros_like(v)))
        # everything else as it was
        full = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32)
        all_k, all_v = c.kv.read(192, _i32([64, 64, 64]), full.cuda(), starts=_starts([64, 64, 64]))
        want = torch.stack([c.k[int(full[b, p // 32]), :, p % 32] for b in range(3) for p in range(64)])
        assert torch.equal(all_k.cpu(), want)
        angles = torch.ones(60, 16).cuda()
        q = torch.ones(10, 2, 64, dtype=torch.bfloat16).cuda()
        got = c.kv.append(k[:10].cuda(), v[:10].cuda(), _i32([64]), table[:1].contiguous().cuda(), starts=_starts([10]), q=q, cos=angles, sin=angles)
        nan = torch.isnan(got[:, :, :32]).all(-1).all(-1).cpu()
        assert nan.tolist() == [False] * 6 + [True] * 4 and not bool(torch.isnan(got[:, :, 32:]).any())
        assert not c.rig.c.aborted()


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype,dim,heads,group,page,lens,news,window,sinks", [
    ("bf16", 128, 2, 4, 4096, [1, 2, 31, 32, 33, 300], [1] * 6, 0, 0),
    ("f16", 64, 1, 1, 4096, [1, 129, 511], [1] * 3, 0, 0),
    ("bf16", 256, 1, 8, 4096, [77, 8], [1] * 2, 0, 0),
    ("f16", 96, 2, 3, 4096, [200, 65], [1] * 2, 40, 3),
    ("bf16", 80, 1, 16, 8192, [257, 100], [1] * 2, 64, 0),
    ("f16", 16, 1, 2, 512, [1000], [1], 100, 70),
    ("bf16", 32, 2, 20, 16384, [700], [1], 0, 0),                        # more heads than a tile of sixteen rows
    ("bf16", 64, 1, 40, 4096, [130], [1], 0, 0),
    ("f16", 128, 1, 2, 4096, [150, 3, 40], [3, 3, 3], 0, 0),             # drafted tokens
    ("bf16", 128, 2, 1, 4096, [130, 260], [4, 4], 33, 2),
    ("f16", 64, 2, 4, 4096, [77], [77], 0, 0),                           # prompts
    ("bf16", 128, 1, 5, 4096, [70, 90, 5, 64], [70, 21, 5, 0], 0, 0),
    ("f16", 128, 2, 2, 8192, [200, 129], [200, 65], 48, 4),
    ("bf16", 80, 1, 3, 4096, [150], [131], 0, 0),
    ("f16", 256, 1, 2, 16384, [90], [90], 0, 0),
    ("bf16", 96, 2, 1, 4096, [333], [333], 100, 17),
])
def test_attention(bam, dtype, dim, heads, group, page, lens, news, window, sinks):
    import torch
    gen = torch.Generator().manual_seed(5)
    with Cache(bam, 256, heads, dim, dtype, page) as c:
        table = _table(lens, c.t, 256)
        c.fill(lens, table)
        n = sum(news)
        q = (torch.randn(n, heads * group, dim, generator=gen) * 1.5).to(c.dtype)
        want, tol, lse = c.want(q, lens, news, table, window, sinks)
        one = all(m == 1 for m in news)
        for starts in ([None, _starts(news)] if one else [_starts(news)]):
            got, got_lse = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=starts, max_new=max(news), window=window, sinks=sinks, return_lse=True)
            _near(got, want, tol)
            _near(got_lse, lse, 2.0 ** -16 * (1 + lse.abs()))
        # announced lengths decide how work is shared out, and nothing else
        for max_len in (1, 64, 1 << 20):
            _near(c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), max_new=max(news), max_len=max_len, window=window, sinks=sinks), want, tol, max_len)
        _near(c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), window=window, sinks=sinks, scale=-0.3), *c.want(q, lens, news, table, window, sinks, -0.3)[:2])
        assert not c.rig.c.aborted()


@pytest.mark.parametrize("new", [1, 5, 70])
def test_attention_twice_is_the_same(bam, new):
    """bit for bit, split over the length and joined"""
    import torch
    with Cache(bam, 512, 1, 64, "bf16") as c:
        lens = [9000]
        table = _table(lens, c.t, 512)
        c.fill(lens, table)
        q = torch.randn(new, 4, 64).to(torch.bfloat16)
        first = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts([new]))
        for _ in range(4):
            assert torch.equal(c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts([new])), first)
        want, tol, _ = c.want(q[-1:], lens, [1], table)
        _near(first[-1:], want, tol)


@pytest.mark.parametrize("dtype,group,news", [("bf16", 4, [1, 1, 1, 1, 1]), ("f16", 2, [3, 1, 4, 2, 5]), ("bf16", 3, [50, 40, 30, 1, 60])])
def test_rows_that_see_nothing(bam, dtype, group, news):
    """no tokens, fewer tokens than rows, blocks that are not there"""
    import torch
    with Cache(bam, 64, 1, 64, dtype) as c:
        lens = [0, 2, 90, 33, 64]
        table = _table([64, 64, 96, 64, 64], c.t, 64, width=3)
        c.fill([64, 64, 96, 64, 64], table)
        table[2, 1] = -1
        table[3, 0] = 64
        table[3, 1] = 1 << 30
        n = sum(news)
        q = torch.randn(n, group, 64).to(c.dtype)
        want, tol, lse = c.want(q, lens, news, table)
        got, got_lse = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts(news), return_lse=True)
        _near(got, want, tol)
        empty = torch.isinf(lse)
        assert bool(empty.any()) and bool((got.cpu()[empty] == 0).all()) and bool((got_lse.cpu()[empty] == -np.inf).all())
        _near(got_lse.cpu()[~empty], lse[~empty], 2.0 ** -16 * (1 + lse[~empty].abs()))
        # lengths past the table: what lies past it is not visible
        long = [200, 2, 96, 33, 300]
        _near(c.kv.attend(q.cuda(), _i32(long), table.cuda(), starts=_starts(news)), *c.want(q, long, news, table)[:2])
        assert not c.rig.c.aborted()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("window,sinks,new", [(0, 0, 1), (0, 0, 6), (0, 0, 90), (40, 2, 1), (40, 2, 5), (40, 2, 90)])
def test_what_is_not_seen_may_be_anything(bam, dtype, odd, window, sinks, new):
    """infinities and NaN in keys and values of tokens to come, behind the window and past the end: rows that do not see them are as without, those that do show them"""
    import torch
    lens = [100]
    with Cache(bam, 16, 1, 64, dtype) as c:
        table = _table([128], c.t, 16)
        k = torch.randn(128, 1, 64).to(c.dtype)
        v = torch.randn(128, 1, 64).to(c.dtype)
        c.fill([128], table, k=k, v=v)
        q = torch.randn(new, 2, 64).to(c.dtype)
        want, tol, _ = c.want(q, lens, [new], table, window, sinks)
        for what in ("k", "v"):
            for at in (99, 97, 110, 20, 5):
                bad_k, bad_v = k.clone(), v.clone()
                (bad_k if what == "k" else bad_v)[at] = odd
                c.fill([128], table, k=bad_k, v=bad_v)
                got = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts([new]), window=window, sinks=sinks).cpu()
                for i, (_, p) in enumerate(c.rows_of(lens, [new])):
                    if not (at <= p and (not window or p - at < window or at < sinks)):
                        _near(got[i], want[i], tol[i], (what, at, i))
                    elif what == "v":
                        assert not bool(torch.isfinite(got[i]).any()), (what, at, i)
                    elif odd != odd:
                        assert bool(torch.isnan(got[i]).all()), (what, at, i)


def test_scores_far_apart(bam):
    """one token far above the others, all equal, and scores near the end of the type's range"""
    import torch
    lens, new = [200], 3
    with Cache(bam, 32, 1, 64, "bf16") as c:
        table = _table(lens, c.t, 32)
        k = torch.randn(200, 1, 64).to(torch.bfloat16)
        v = torch.randn(200, 1, 64).to(torch.bfloat16)
        for kind in ("peak", "equal", "huge"):
            kk = k.clone()
            if kind == "peak":
                kk[57] = 30
            elif kind == "equal":
                kk[:] = kk[0]
            else:
                kk = (kk.float() * 1e17).to(torch.bfloat16)
            c.fill(lens, table, k=kk, v=v)
            q = torch.randn(new, 2, 64).to(torch.bfloat16)
            want, tol, _ = c.want(q, lens, [new], table)
            got = c.kv.attend(q.cuda(), _i32(lens), table.cuda(), starts=_starts([new]))
            if kind == "huge":
                # a score's last bits are larger than one: only that the winner takes all
                assert bool(torch.isfinite(got).all())
            else:
                _near(got, want, tol, kind)


@pytest.mark.parametrize("shape", ["fused", "offset", "transposed"])
def test_strides_and_alignment(bam, shape):
    import torch
    lens, news, hq = [130, 77], [1, 1], 4
    with Cache(bam, 32, 2, 80, "bf16") as c:
        table = _table(lens, c.t, 32)
        c.fill(lens, table)
        base = torch.randn(2, hq, 80).to(torch.bfloat16)
        if shape == "fused":
            q = torch.zeros(2, hq + 4, 80, dtype=torch.bfloat16, device="cuda")[:, 2:2 + hq]
        elif shape == "offset":
            q = torch.zeros(2, hq, 83, dtype=torch.bfloat16, device="cuda")[:, :, 3:]
        else:
            q = torch.zeros(hq, 2, 80, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
        q.copy_(base)
        wide = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
        wide[:, 5:5 + table.shape[1]] = table.cuda()
        want, tol, _ = c.want(base, lens, news, table)
        _near(c.kv.attend(q, _i32(lens), wide[:, 5:5 + table.shape[1]]), want, tol)
        # and as new rows: keys and values with such strides
        k, v = q[:, :2], q[:, 2:]
        c.kv.append(k, v, _i32(lens), wide[:, 5:5 + table.shape[1]])
        got_k, got_v = c.kv.read(2, _i32(lens), table.cuda())
        assert torch.equal(got_k.cpu(), base[:, :2]) and torch.equal(got_v.cpu(), base[:, 2:])
        # one row of blocks for every sequence
        shared = table[:1].cuda().expand(2, -1)
        c.k, c.v = c.k.clone(), c.v.clone()
        c.note(base[:, :2], base[:, 2:], c.rows_of(lens, news), table)
        _near(c.kv.attend(q, _i32([77, 77]), shared), *c.want(base, [77, 77], news, table[:1].expand(2, -1))[:2])


@pytest.mark.parametrize("dim,page,heads,cache_pages,new", [(128, 4096, 2, 32, 1), (128, 4096, 2, 40, 40), (64, 4096, 1, 16, 3), (256, 4096, 1, 64, 1), (32, 512, 1, 64, 9), (128, 8192, 1, 33, 70)])
def test_a_cache_smaller_than_what_is_kept(bam, dim, page, heads, cache_pages, new):
    """what does not fit goes to the store and comes back: rows, attention over all of them, and the store's own content after a flush"""
    import torch
    t = 1 << ((page // (2 * dim)).bit_length() - 1)
    n_blocks = 40
    lens = [12 * t + 3, 20 * t, 5]
    with Cache(bam, n_blocks, heads, dim, "bf16", page, cache_pages=cache_pages, backing=True) as c:
        table = _table(lens, c.t, n_blocks)
        k, v = c.fill(lens, table)
        for _ in range(2):
            got_k, got_v = c.kv.read(sum(lens), _i32(lens), table.cuda(), starts=_starts(lens))
            assert torch.equal(got_k.cpu(), k) and torch.equal(got_v.cpu(), v)
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
        q = torch.randn(3, 2 * heads, dim).to(torch.bfloat16)
        want, tol, _ = c.want(q, lens, [1, 1, 1], table)
        _near(c.kv.attend(q.cuda(), _i32(lens), table.cuda()), want, tol)
        # the pages as they lie on the store
        torch.cuda.synchronize()
        c.kv._owned[2].flush()
        torch.cuda.synchronize()
        words = c.rig.backing(2 * n_blocks * heads * page // 8).view(np.int16).reshape(n_blocks, heads, 2, page // 2)
        for b, n in enumerate(lens):
            for p in (0, n // 2, n - 1):
                block, x = int(table[b, p // t]), p % t
                place = x if t == 8 else (x & ~12) | (x & 4) << 1 | (x & 8) >> 1
                for h in range(heads):
                    keys = words[block, h, 0, :t * dim].reshape(dim // 8, t, 8)[:, place].reshape(-1)
                    values = words[block, h, 1, :t * dim].reshape(t // 8, dim, 8)[p % t // 8, :, p % 8]
                    assert np.array_equal(keys, c.k[block, h, p % t].view(torch.int16).numpy())
                    assert np.array_equal(values, c.v[block, h, p % t].view(torch.int16).numpy())
        assert not c.rig.c.aborted()


@pytest.mark.parametrize("dim,page", [(128, 4096), (64, 4096), (32, 4096), (64, 16384), (256, 4096)])
@pytest.mark.parametrize("odd", [0, 5])
def test_new_blocks_that_do_not_fit(bam, dim, page, odd):
    """many blocks at once into a cache that holds a few of their pages: whoever writes a page, its rows are all there when it has gone to the store and come back"""
    import torch
    t = 1 << ((page // (2 * dim)).bit_length() - 1)
    lens = [20 * t + odd, 15 * t - odd, 9 * t + odd]
    with Cache(bam, 64, 2, dim, "f16", page, cache_pages=64 if t == 8 else 32, backing=True) as c:
        table = _table(lens, c.t, 64)
        for seed in (1, 2, 3):
            k, v = c.fill(lens, table, seed=seed)
            got_k, got_v = c.kv.read(sum(lens), _i32(lens), table.cuda(), starts=_starts(lens))
            assert torch.equal(got_k.cpu(), k) and torch.equal(got_v.cpu(), v), seed
        assert not c.rig.c.aborted()


def test_new_blocks_are_not_read(bam):
    """a block whose tokens are all new needs nothing from the store; what is not written of its pages is zero"""
    import torch
    with Cache(bam, 16, 2, 128, "bf16", backing=True) as c:
        table = _table([40], c.t, 16)
        c.kv.array.stats()
        c.fill([40], table)
        assert c.kv.array.stats()["read_io_cnt"] == 0
        k, v = c.kv.read(48, _i32([48]), table.cuda(), starts=_starts([48]))
        assert bool((k[40:] == 0).all()) and bool((v[40:] == 0).all())
        # a block that begins with a token of an earlier call is read
        one = torch.randn(1, 2, 128).to(torch.bfloat16).cuda()
        fresh = torch.tensor([[i for i in range(16) if i not in table[0].tolist()][:3]], dtype=torch.int32)
        c.kv.append(one, one, _i32([18]), fresh.cuda())
        assert c.kv.array.stats()["read_io_cnt"] == 4
        c.kv.append(one, one, _i32([33]), fresh.cuda())
        assert c.kv.array.stats()["read_io_cnt"] == 0


def test_streams_and_graphs(bam):
    """on another stream than the tensors' own, and replayed several times with other work between, as eagerly"""
    import torch
    lens, news, hq = [150, 90, 33], [1, 1, 1], 8
    with Cache(bam, 64, 2, 128, "bf16") as c:
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


def test_accesses_are_counted(bam):
    import torch
    lens = [100]
    with Cache(bam, 16, 2, 128, "bf16") as c:
        table = _table(lens, c.t, 16)
        c.fill(lens, table)
        c.kv.array.stats()
        c.kv.attend(torch.randn(1, 4, 128).to(torch.bfloat16).cuda(), _i32(lens), table.cuda())
        st = c.kv.array.stats()
        assert st["access_cnt"] == st["hit_cnt"] == 2 * 2 * 7, st


def test_refusals(bam):
    import torch
    bf, i32 = torch.bfloat16, torch.int32
    with Rig(bam, 1 << 20) as r:
        a = r.array((1 << 20) // 8, 4096, 64)
        for kw in ({"head_dim": 120}, {"head_dim": 272}, {"head_dim": 0}, {"n_heads": 0}, {"n_blocks": 129}, {"n_blocks": 0}, {"dtype": torch.float32}, {"first_page": 1, "n_blocks": 128}, {"n_blocks": None}):
            with pytest.raises(bam.BamError):
                bam.KVCache(a, **{"n_heads": 1, "head_dim": 128, "n_blocks": 128, **kw})
        with pytest.raises(bam.BamError):
            bam.KVCache(r.array(1 << 12, 512, 64), 1, 64, n_blocks=1)                # four rows to a page
        with pytest.raises(bam.BamError):
            bam.KVCache(r.array(1 << 14, 4096, 15), 1, 64, n_blocks=1)
        kv = bam.KVCache(a, 2, 128, n_blocks=32, first_page=3)
        q, k = torch.zeros(2, 4, 128, dtype=bf, device="cuda"), torch.zeros(2, 2, 128, dtype=bf, device="cuda")
        lens, table = _i32([1, 1]), torch.zeros(2, 1, dtype=i32, device="cuda")
        out, angles = torch.empty_like(q), torch.zeros(4, 64, device="cuda")
        good = kv.attend(q, lens, table)
        assert good.shape == q.shape
        for args, kw in (((q[:, :3], lens, table), {}), ((q.half(), lens, table), {}), ((q[:, :, :64], lens, table), {}), ((q.transpose(1, 2), lens, table), {}), ((q.cpu(), lens, table), {}),
                         ((q, lens.long(), table), {}), ((q, lens[:1], table), {}), ((q, lens, table.long()), {}), ((q, lens, table[:1]), {}), ((q, lens, table[:, :0]), {}),
                         ((q, lens, table), {"starts": _i32([0, 1])}), ((q[:1], lens, table), {}), ((q, lens, table), {"window": -1}), ((q, lens, table), {"sinks": -1}),
                         ((q, lens, table), {"max_len": 0}), ((q, lens, table), {"starts": _i32([0, 1, 2]), "max_new": 0}), ((q, lens, table), {"scale": float("nan")}),
                         ((q, lens, table), {"scale": float("inf")}), ((q, lens, table), {"out": out[:1]}), ((q, lens, table), {"out": torch.empty(4, 2, 128, dtype=bf, device="cuda").transpose(0, 1)})):
            with pytest.raises(bam.BamError):
                kv.attend(*args, **kw)
        for args, kw in (((k[:, :1], k, lens, table), {}), ((k, k[:1], lens, table), {}), ((k, k, lens, table), {"q": q[:1]}), ((k, k, lens, table), {"q_norm": k[0, 0]}),
                         ((k, k, lens, table), {"k_norm": k[0, 0, :64]}), ((k, k, lens, table), {"k_norm": k[0, 0].float()}), ((k, k, lens, table), {"cos": angles}),
                         ((k, k, lens, table), {"cos": angles[:, :12].contiguous(), "sin": angles[:, :12].contiguous()}), ((k, k, lens, table), {"cos": angles.half(), "sin": angles.half()}),
                         ((k, k, lens, table), {"cos": torch.zeros(4, 72, device="cuda"), "sin": torch.zeros(4, 72, device="cuda")}),
                         ((k, k, lens, table), {"cos": angles, "sin": angles, "rotary": "other"}), ((k, k, lens, table), {"out": out})):
            with pytest.raises(bam.BamError):
                kv.append(*args, **kw)
        # nothing to do
        none = torch.zeros(0, dtype=i32, device="cuda")
        assert kv.attend(q[:0], none, table[:0]).shape == (0, 4, 128)
        assert kv.append(k[:0], k[:0], none, table[:0]) is None
        assert kv.read(0, none, table[:0])[0].shape == (0, 2, 128)
        kv.close()
        torch.cuda.synchronize()
        assert not r.c.aborted()
