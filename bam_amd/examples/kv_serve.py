"""Serving from a key-value cache that lies behind the page cache: prompts go in, then tokens one at a time, by way of the calls of bam_amd.KVCache.

    python -m bam_amd.examples.kv_serve [--batch N] [--prompt N] [--steps N] [--layers N] [--resident SHARE] [--eight] [--beams N] [--check]

A stack of attention layers (norms of queries and keys, rotary positions, grouped heads, every other layer with a sliding window and four first tokens) with random
weights, and nothing but attention in it.  Each layer's keys and values are a range of one array; the page cache holds a share of all pages, the
others are written to the store when their slots are needed and fetched again by the waves that want them.  --eight keeps keys and values in 8 bits.  --check compares every layer's
last output with plain torch over all tokens.

--beams N searches for each request's continuation of the largest probability, N beams to a request, over a vocabulary of random embeddings: selection (bam_amd.beam_select), reordering of every layer's
sequences behind it (KVCache.reorder), the next tokens.  All layers share lengths, tables and spare blocks; the first to be reordered says which those are.
"""
import argparse
import time

import torch

import bam_amd

HEADS, KV_HEADS, DIM, PAGE, WINDOW, SINKS, VOCAB = 16, 4, 64, 4096, 96, 4, 1000
EPS = 1e-6


class Layer:
    def __init__(self, array, first_page, n_blocks, hidden, gen, window, dtype, stored):
        self.kv = bam_amd.KVCache(array, KV_HEADS, DIM, dtype, first_page=first_page, n_blocks=n_blocks, stored=stored)
        self.window, self.sinks = window, SINKS if window else 0
        self.w_in = (torch.randn(hidden, (HEADS + 2 * KV_HEADS) * DIM, generator=gen) / hidden ** 0.5).to(dtype).cuda()
        self.w_out = (torch.randn(HEADS * DIM, hidden, generator=gen) / (HEADS * DIM) ** 0.5).to(dtype).cuda()
        self.q_norm, self.k_norm = ((1 + 0.1 * torch.randn(DIM, generator=gen)).to(dtype).cuda() for _ in range(2))

    def step(self, x, lens, table, starts, cos, sin, max_new):
        qkv = (x @ self.w_in).view(x.shape[0], -1, DIM)
        q = self.kv.append(qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:], lens, table, starts=starts, q=qkv[:, :HEADS],
                           q_norm=self.q_norm, k_norm=self.k_norm, eps=EPS, cos=cos, sin=sin)
        out = self.kv.attend(q, lens, table, starts=starts, max_new=max_new, window=self.window, sinks=self.sinks)
        return qkv, x + out.view(x.shape[0], -1) @ self.w_out


def plain(qkv, layer, cos, sin, held):
    """the layer's attention over all tokens of one sequence, the last token's output, in 32 bits; held: its length and row of blocks, for keys and values as the cache has them (8 bits are
    not what went in)"""
    def normed(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x[..., :DIM // 2], x[..., DIM // 2:]
        c, s = cos[:x.shape[0], None], sin[:x.shape[0], None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    n = qkv.shape[0]
    q, k, v = normed(qkv[:, :HEADS], layer.q_norm)[-1], normed(qkv[:, HEADS:HEADS + KV_HEADS], layer.k_norm), qkv[:, HEADS + KV_HEADS:].float()
    if layer.kv.stored is torch.float8_e4m3fn:
        k, v = (x.float() for x in layer.kv.read(n, *held, starts=torch.tensor([0, n], dtype=torch.int32, device="cuda")))
    k, v = (x.repeat_interleave(HEADS // KV_HEADS, 1) for x in (k, v))
    t = torch.arange(n, device="cuda")
    seen = (n - 1 - t < layer.window) | (t < layer.sinks) if layer.window else t >= 0
    score = (k * q).sum(-1) * DIM ** -0.5
    weight = torch.softmax(score.masked_fill(~seen[:, None], float("-inf")), 0)
    return (weight[..., None] * v).sum(0)


def search(a, layers, x, lens, table, blocks, hidden, gen, dtype, cos, sin, seen):
    """the best `beams` continuations of each request by `steps` tokens: their tokens and sums of log-probabilities, and what was chosen among; nothing waits for the device"""
    n, beams, t = a.batch * a.beams, a.beams, layers[0].kv.block_tokens
    embedding = torch.randn(VOCAB, hidden, generator=gen).to(dtype).cuda()
    head = (4 * torch.randn(hidden, VOCAB, generator=gen) / hidden ** 0.5).to(dtype).cuda()
    free, used = blocks.cuda(), torch.zeros((), dtype=torch.int64, device="cuda")

    def blocks_for(wanted, others):
        """a free block for each that wants one"""
        got = torch.where(wanted, free[(used + wanted.cumsum(0) - 1).clamp(0, free.numel() - 1)], others)
        used.add_(wanted.sum())
        return got

    every = torch.ones(n, dtype=torch.bool, device="cuda")
    # a sequence for each beam of each request's prompt; they are alike, so only the first one counts
    parents = torch.arange(a.batch, dtype=torch.int32, device="cuda").repeat_interleave(beams)
    lens, table, spare = reorder(layers, parents, lens, table, blocks_for(every, parents))
    scores = torch.full((a.batch, beams), float("-inf"), device="cuda")
    scores[:, 0] = 0
    x = x.repeat_interleave(beams, 0)
    rows = [[[torch.cat(s)] for s in kind for _ in range(beams)] for kind in seen] if seen else None
    history, logs, worst = torch.zeros(n, 0, dtype=torch.int32, device="cuda"), [], 0.0
    for _ in range(a.steps):
        logits, before = (x / x.float().std(-1, keepdim=True).to(dtype)) @ head, scores
        scores, chosen, tokens = bam_amd.beam_select(logits, scores)
        parents, tokens = chosen.flatten(), tokens.flatten()
        logs.append((logits, before, parents, tokens))
        # (a spare block that was used comes back as another, but for the first ones)
        lens, table, spare = reorder(layers, parents, lens, table, blocks_for(spare < 0, spare))
        history = torch.cat([history[parents.long()], tokens[:, None]], 1)
        at = (lens // t).long()[:, None]
        table.scatter_(1, at, blocks_for(lens % t == 0, table.gather(1, at)[:, 0])[:, None])
        lens = lens + 1
        x = embedding[tokens.long()]
        for i, layer in enumerate(layers):
            went_in = x
            qkv, x = layer.step(x, lens, table, None, cos, sin, 1)
            if rows:
                rows[i] = [rows[i][p] + [qkv[b:b + 1]] for b, p in enumerate(parents.tolist())]
                want = torch.stack([plain(torch.cat(r), layer, cos, sin, (lens[b:b + 1], table[b:b + 1])) for b, r in enumerate(rows[i])])
                want = went_in.float() + want.view(n, -1) @ layer.w_out.float()
                worst = max(worst, float((x.float() - want).abs().max() / want.abs().max()))
    return {"tokens": history.view(a.batch, beams, -1), "sums": scores, "logs": logs, "worst_of_beams": worst}


def reorder(layers, parents, lens, table, spare):
    """every layer's copies go to the same blocks"""
    for layer in layers:
        new = layer.kv.reorder(parents, lens, table, spare)
    return new


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--prompt", type=int, default=700)
    p.add_argument("--steps", type=int, default=40)
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--resident", type=float, default=0.5)
    p.add_argument("--eight", action="store_true")
    p.add_argument("--beams", type=int, default=0)
    p.add_argument("--check", action="store_true")
    a = p.parse_args(argv)
    dtype, hidden = torch.bfloat16, 256
    stored = torch.float8_e4m3fn if a.eight else None
    gen = torch.Generator().manual_seed(1)
    tokens = PAGE // ((1 if a.eight else 2) * DIM)               # of a block
    prompts = [max(1, a.prompt - 37 * b % max(1, a.prompt)) for b in range(a.batch)]
    per_seq = -(-(a.prompt + a.steps) // tokens)
    # of beams: the prompts' blocks, those that each begins, and one for its first copy and one for the next
    n_blocks = per_seq * a.batch if not a.beams else (per_seq + a.beams * (a.steps // tokens + 4)) * a.batch
    pages = 2 * KV_HEADS * n_blocks * a.layers
    target = bam_amd.Target("/dev/libnvm-kv-serve", pages * PAGE, 512, backing=True, n_io_threads=4)
    ctrl = bam_amd.Controller("/dev/libnvm-kv-serve", 1, 0, queue_depth=256, n_queues=16)
    cache, rng, array = bam_amd.host.make_array(ctrl, pages * PAGE // 8, PAGE, max(64, int(pages * a.resident)))
    layers = [Layer(array, 2 * KV_HEADS * n_blocks * i, n_blocks, hidden, gen, WINDOW if i % 2 else 0, dtype, stored) for i in range(a.layers)]
    assert layers[0].kv.block_tokens == tokens
    blocks = torch.randperm(n_blocks, generator=gen).to(torch.int32)
    table = blocks[:per_seq * a.batch].view(a.batch, per_seq).cuda()
    angle = torch.arange(a.prompt + a.steps, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, DIM, 2, dtype=torch.float64) / DIM)
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    seen = [[[] for _ in range(a.batch)] for _ in layers]       # for --check: what went into each layer, and its last output
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    worst = 0.0

    def run(x, starts, news):
        at = [0]
        for m in news:
            at.append(at[-1] + m)
        for i, layer in enumerate(layers):
            before = x
            qkv, x = layer.step(x, lens, table, starts, cos, sin, max(news))
            if a.check:
                for b in range(a.batch):
                    seen[i][b].append(qkv[at[b]:at[b + 1]])
                nonlocal worst
                want = torch.stack([plain(torch.cat(seen[i][b]), layer, cos, sin, (lens[b:b + 1], table[b:b + 1])) for b in range(a.batch)])
                last = [k - 1 for k in at[1:]]
                want = before[last].float() + want.view(a.batch, -1) @ layer.w_out.float()
                worst = max(worst, float((x[last].float() - want).abs().max() / want.abs().max()))
        return x

    starts = torch.tensor([0] + list(torch.tensor(prompts).cumsum(0)), dtype=torch.int32, device="cuda")
    x = torch.randn(sum(prompts), hidden, generator=gen).to(dtype).cuda()
    array.stats()
    x = run(x, starts, prompts)[(starts[1:] - 1).long()]
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    if a.beams:
        found = search(a, layers, x, lens, table, blocks[per_seq * a.batch:], hidden, gen, dtype, cos, sin, seen if a.check else None)
        worst = max(worst, found["worst_of_beams"])
    for _ in range(0 if a.beams else a.steps):
        lens += 1
        x = run(x / x.float().std(-1, keepdim=True).to(dtype), None, [1] * a.batch)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - t0
    stats, aborted = array.stats(), ctrl.aborted()
    for layer in layers:
        layer.kv.close()
    for o in (array, rng, cache, ctrl, target):
        o.close()
    result = {"tokens_per_s": a.batch * max(1, a.beams) * a.steps / seconds, "pages": pages, "page_reads": stats["read_io_cnt"], "hits": stats["hit_cnt"], "misses": stats["miss_cnt"],
              "aborted": aborted, "worst": worst if a.check else None}
    print(", ".join(f"{k} {v}" for k, v in result.items()))
    if a.beams:
        result.update(found)
    return result


if __name__ == "__main__":
    main()
