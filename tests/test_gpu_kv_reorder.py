"""Reordering of the key-value cache's sequences behind a choice of beams, in 16 bits and in 8, against the same steps on the CPU: numbers are moved, so everything is compared exactly."""
import random

import pytest

from test_gpu_kv import Cache, _i32, _near, _starts, _table
from test_gpu_kv8 import Cache8, _kept
from test_gpu_parity import bam  # noqa: F401  (the module fixture)

pytestmark = pytest.mark.gpu


def _expected(parents, lens, table, spare, t, n_blocks):
    """(lens, table, spare, copies (from block, to block, tokens)) of the new sequences"""
    width = len(table[0])

    def last(o):
        i, rest = lens[o] // t, lens[o] % t
        return table[o][i] if lens[o] > 0 and rest and i < width and 0 <= table[o][i] < n_blocks else None
    there = [0 <= p < len(lens) for p in parents]
    freed = [last(o) for o in range(len(lens)) if o not in parents and last(o) is not None]
    new_lens, new_table, new_spare, copies = [], [], list(spare), []
    for i, p in enumerate(parents):
        if not there[i]:
            new_lens.append(0)
            new_table.append([-1] * width)
            continue
        new_lens.append(lens[p])
        row = [b if k * t < lens[p] else -1 for k, b in enumerate(table[p])]
        if p in parents[:i] and last(p) is not None:
            row[lens[p] // t] = spare[i]
            if 0 <= spare[i] < n_blocks:
                copies.append((last(p), spare[i], lens[p] % t))
            new_spare[i] = freed.pop(0) if freed else -1
        new_table.append(row)
    return new_lens, new_table, new_spare, copies


def _call(c, parents, lens, table, spare):
    import torch
    width = len(table[0])
    got = c.kv.reorder(_i32(parents), _i32(lens), torch.tensor(table, dtype=torch.int32, device="cuda").view(-1, width), _i32(spare))
    want = _expected(parents, lens, table, spare, c.t, c.n_blocks)
    for a, b in zip(got, want):
        assert a.dtype is torch.int32 and a.cpu().tolist() == b
    for source, target, rest in want[3]:
        c.k[target, :, :rest] = c.k[source, :, :rest]
        c.v[target, :, :rest] = c.v[source, :, :rest]
    return got


def _compare(c, lens, table, what=""):
    """all tokens of all sequences"""
    import torch
    rows = [(b, p) for b, n in enumerate(lens) for p in range(n)]
    k, v = c.kv.read(len(rows), _i32(lens), table, starts=_starts(lens))
    t = table.cpu().long()
    for got, held in ((k, c.k), (v, c.v)):
        want = torch.stack([held[t[b, p // c.t], :, p % c.t] for b, p in rows])
        assert torch.equal(got.cpu().double(), want.double()), what


KINDS = {"16": Cache, "8": Cache8}


@pytest.mark.parametrize("kind", ["16", "8"])
@pytest.mark.parametrize("dtype,dim,heads,page,cache_pages", [
    ("bf16", 128, 2, 4096, None), ("f16", 64, 3, 4096, None), ("bf16", 80, 1, 8192, None), ("f16", 256, 2, 16384, None), ("bf16", 64, 1, 32768, None), ("f16", 16, 1, 512, None), ("bf16", 112, 2, 4096, None),
    ("bf16", 128, 2, 4096, 64), ("f16", 64, 2, 32768, 64), ("bf16", 256, 1, 8192, 64),
])
def test_beams_go_on(bam, kind, dtype, dim, heads, page, cache_pages):
    """several steps of a search: choices at random, a token more for each beam, attention; also with most pages on the store"""
    import torch
    rng = random.Random(5)
    with KINDS[kind](bam, 60, heads, dim, dtype, page, cache_pages=cache_pages, backing=cache_pages is not None) as c:
        t = c.t
        per = [2 * t + 3, t - 1, 3 * t, 5]
        # a prompt each; then three beams of each
        table = _table(per, t, 60, width=5)
        c.fill(per, table)
        used = {b for row in table.tolist() for b in row if b >= 0}
        free = [b for b in range(60) if b not in used]
        take = lambda: free.pop()  # noqa: E731
        parents = [r for r in range(4) for _ in range(3)]
        spare = [take() for _ in parents]
        lens, table, spare = _call(c, parents, per, table.tolist(), spare)
        for step in range(8):
            now = lens.cpu().tolist()
            _compare(c, now, table, step)
            # a token more, in a block of the beam's own where it begins one
            now = [n + 1 for n in now]
            rows = table.cpu()
            for b, n in enumerate(now):
                if (n - 1) % t == 0:
                    rows[b, (n - 1) // t] = take()
            table = rows.cuda()
            k = torch.randn(12, heads, dim, generator=torch.Generator().manual_seed(step)).to(c.dtype)
            c.kv.append(k.cuda(), k.flip(2).cuda(), _i32(now), table)
            c.note(k, k.flip(2), [(b, n - 1) for b, n in enumerate(now)], rows)
            q = torch.randn(12, 2 * heads, dim, generator=torch.Generator().manual_seed(step)).to(c.dtype)
            _near(c.kv.attend(q.cuda(), _i32(now), table), *c.want(q, now, [1] * 12, rows)[:2], step)
            # in every request some beams go on, one of them at least twice
            parents = []
            for r in range(4):
                a, b = rng.sample(range(3), 2)
                parents += rng.choice([[a, a, b], [b, a, a], [a, a, a], [a, b, a], [0, 1, 2]])
                parents[-3:] = [3 * r + x for x in parents[-3:]]
            lens, table, spare = _call(c, parents, now, rows.tolist(), spare.cpu().tolist())
            spare = torch.tensor([take() if x < 0 and len(free) > 14 else x for x in spare.cpu().tolist()], dtype=torch.int32, device="cuda")
            if len(free) <= 14:
                break
        assert step >= 2
        assert not c.rig.c.aborted()


@pytest.mark.parametrize("kind", ["16", "8"])
def test_what_is_not_there(bam, kind):
    """parents, spare blocks and last blocks that are not there, lengths of nothing, of whole blocks and past the table, fewer and more sequences than before"""
    import torch
    with KINDS[kind](bam, 24, 1, 128, "bf16") as c:
        t = c.t
        lens = [t + 1, 0, 2 * t, 5, 3 * t + 7, t + 4, 9, -3]
        table = [[0, 1], [2, 3], [4, 5], [6, 7], [8, 9], [10, 24], [-1, 11], [12, 13]]
        c.fill([2 * t] * 8, torch.tensor(table, dtype=torch.int32))
        spare = list(range(14, 24))
        for parents in ([0, 0, 0], [1, 1], [2, 2, 3, 3], [4, 4, 5, 5, 6, 6, 7, 7], [8, -1, 1 << 30, -(1 << 31), 0], [3], [0, 3, 0, 3, 0, 3, 0, 3, 0, 3]):
            got = _call(c, parents, lens, table, spare[:len(parents)])
            held = [(x, min(n, 2 * t)) for x, n in enumerate(got[0].cpu().tolist())]
            rows = [x for x, n in held if n > 0 and parents[x] in (0, 2, 3)]
            if rows:
                _compare(c, [held[x][1] for x in rows], got[1][rows])
        for none in (-1, 24, 1 << 30, -(1 << 31)):
            _call(c, [0, 0, 3, 3], lens, table, [none] * 4)
        empty = torch.zeros(0, dtype=torch.int32, device="cuda")
        new = c.kv.reorder(empty, _i32(lens), torch.tensor(table, dtype=torch.int32, device="cuda"), empty)
        assert [tuple(x.shape) for x in new] == [(0,), (0, 2), (0,)]
        assert not c.rig.c.aborted()


@pytest.mark.parametrize("n_old,n_new", [(1, 300), (70, 9000), (9000, 9000), (4097, 130)])
def test_many_sequences(bam, n_old, n_new):
    """more than are looked at at a time"""
    rng = random.Random(n_old)
    with Cache(bam, 2 * 9000 + 300, 1, 16, "f16", 512) as c:
        import torch
        t = c.t
        assert t == 16
        lens = [rng.randint(1, 15) for _ in range(n_old)]
        table = [[b] for b in range(n_old)]
        n = sum(lens)
        k = torch.randn(n, 1, 16).to(c.dtype)
        c.kv.append(k.cuda(), k.flip(2).cuda(), _i32(lens), torch.tensor(table, dtype=torch.int32, device="cuda"), starts=_starts(lens))
        c.note(k, k.flip(2), c.rows_of(lens, lens), torch.tensor(table))
        parents = [rng.randrange(n_old) for _ in range(n_new)]
        new_lens, new_table, _ = _call(c, parents, lens, table, [9000 + i for i in range(n_new)])
        _compare(c, new_lens.cpu().tolist(), new_table)


def test_graphs(bam):
    """select, reorder, append and attend in one graph, replayed with other work between, as eagerly"""
    import torch
    beams, heads, dim, vocab = 4, 2, 64, 500
    outs = []
    for captured in (False, True):
        with Cache8(bam, 200, heads, dim, "bf16") as c:
            gen = torch.Generator(device="cuda").manual_seed(7)
            prompt = 3 * c.t + 9
            blocks = torch.randperm(200, generator=torch.Generator().manual_seed(1)).to(torch.int32)
            table0 = torch.full((1, 12), -1, dtype=torch.int32)
            table0[0, :4] = blocks[:4]
            c.fill([prompt], table0)
            w = torch.randn(heads * 2 * dim, vocab, generator=gen, device="cuda").to(torch.bfloat16)
            emb = torch.randn(vocab, heads, dim, generator=gen, device="cuda").to(torch.bfloat16)
            lens, table, spare = c.kv.reorder(_i32([0] * beams), _i32([prompt]), table0.cuda(), blocks[4:8].cuda())
            scores = torch.tensor([[0.0] + [-1e30] * (beams - 1)], device="cuda")
            q = torch.randn(beams, 2 * heads, dim, generator=gen, device="cuda").to(torch.bfloat16)

            def step():
                out = c.kv.attend(q, lens, table)
                sums, chosen, tokens = bam.beam_select(out.view(beams, -1) @ w, scores)
                new = c.kv.reorder(chosen[0], lens, table, spare)
                for a, b in zip((lens, table, spare, scores), (*new, sums)):
                    a.copy_(b)
                k = emb[tokens[0].long()]
                lens.add_(1)
                c.kv.append(k, k, lens, table)
                return tokens

            seen = []
            if captured:
                # (what a first call sets up is set up before the capture; what it changes is put back)
                kept = [x.clone() for x in (lens, table, spare, scores)]
                step()
                for a, b in zip((lens, table, spare, scores), kept):
                    a.copy_(b)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    tokens = step()
                for _ in range(6):
                    graph.replay()
                    torch.cuda.synchronize()
                    seen.append(tokens.clone())
                    bam.beam_select(torch.randn(8, 300, device="cuda"), torch.zeros(2, 4, device="cuda"))
            else:
                for _ in range(6):
                    seen.append(step().clone())
            k, v = c.kv.read(int(lens.sum()), lens, table, starts=torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), lens.cumsum(0).to(torch.int32)]))
            outs.append([torch.stack(seen).cpu(), lens.cpu(), scores.cpu(), k.cpu(), v.cpu()])
            assert not c.rig.c.aborted()
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_pages_that_could_not_be_had(bam):
    """the target swallows every command: the launch ends, and the tokens of the copy are NaN"""
    import torch
    from test_gpu_parity import Rig
    with Rig(bam, 1 << 20, backing=True, n_queues=1, depth=1024, drop_every=1, limit=100_000) as r:
        kv = bam.KVCache(r.array(1 << 17, 4096, 64), 1, 128, torch.bfloat16, n_blocks=64)
        table = torch.tensor([[3]], dtype=torch.int32, device="cuda")
        lens, new, spare = kv.reorder(_i32([0, 0]), _i32([9]), table, _i32([4, 5]))
        torch.cuda.synchronize()
        assert r.c.aborted()
        k, v = kv.read(9, _i32([9]), new[1:], starts=_starts([9]))
        assert bool(torch.isnan(k).all()) and bool(torch.isnan(v).all())
        kv.close()


def test_refusals(bam):
    import torch
    with Cache(bam, 8, 1, 64, "bf16") as c:
        parents, lens, table, spare = _i32([0, 1]), _i32([5, 6]), torch.zeros(2, 3, dtype=torch.int32, device="cuda"), _i32([4, 5])
        c.kv.reorder(parents, lens, table, spare)
        for args in ((parents.long(), lens, table, spare), (parents, lens.long(), table, spare), (parents, lens, table.long(), spare), (parents, lens, table, spare.long()), (parents.cpu(), lens, table, spare),
                     (parents, lens, table, spare.cpu()), (parents, lens, table, spare[:1]), (parents, lens[:1], table, spare), (parents, lens, table[:1], spare), (parents, lens, table[:, :0], spare),
                     (parents[None], lens, table, spare), (_i32([0, 0, 1, 1])[::2], lens, table, spare), (parents, lens, table, _i32([4, 4, 5, 5])[::2]), (parents, lens[:0], table[:0], spare),
                     (parents, lens, table.T.contiguous().T, spare)):
            with pytest.raises(bam.BamError):
                c.kv.reorder(*args)
